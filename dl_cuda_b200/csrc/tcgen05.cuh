// Tensor-core primitives of sm_100a used by the attention kernels: tensor-map (TMA) loads of
// [token, column] tiles in the 128-byte swizzle, the shared-memory and instruction descriptors of
// tcgen05.mma (kind::f16, bf16 operands, fp32 accumulators in TMEM), and TMEM loads and stores in
// the 32x32b shape, where a thread reads or writes its own lane (one row of the accumulator).
//
// A tile is stored as blocks of 64 columns: block c holds rows of 128 bytes (64 bf16), 8 rows to a
// swizzle atom of 1024 bytes.  The same bytes serve as a K-major operand (the product runs over the
// columns) and as an MN-major one (it runs over the rows); only the descriptor differs.
#pragma once

#include <cuda.h>

#include "tma.cuh"

namespace dlb {

constexpr int kBlockCols = 64;  // bf16 columns of a block: 128 bytes

// ---------------------------------------------------------------- host side
// Map of a [batch, head, token, column] bf16 tensor with the given strides (elements); a box is
// `rows` tokens by 64 columns of one head.  Columns and tokens outside the tensor read as zero.
// Returns 0 or a CUDA driver error.
int make_heads_map(CUtensorMap *map, const void *ptr, int dim, int tokens, int heads, int batch, long long token_stride,
                   long long head_stride, long long batch_stride, int rows);

// -------------------------------------------------------------- device side
__device__ __forceinline__ void tma_load_rows(void *smem, const CUtensorMap *map, uint64_t *bar, int col, int token,
                                              int head, int batch) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(smem)), "l"(map), "r"(smem_u32(bar)), "r"(col), "r"(token), "r"(head), "r"(batch)
      : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// Whole warp: reserves `cols` TMEM columns (a power of two >= 32); the base address lands in *slot.
__device__ __forceinline__ void tmem_alloc(uint32_t *slot, int cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base, int cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Makes generic-proxy writes to shared memory visible to the tensor cores and the copy engine.
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Arrives on `bar` when every MMA this thread has issued so far is complete.
__device__ __forceinline__ void tc_commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

constexpr uint64_t kDescSwizzle128 = (2ull << 61) | (1ull << 46);

// K-major operand: rows are the M or N index, 16 columns per step lie 32 bytes apart in the atom.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t smem) {
  return kDescSwizzle128 | (64ull << 32) | (1ull << 16) | ((smem >> 4) & 0x3fff);
}
// MN-major operand: columns are the M or N index (blocks `block_bytes` apart), rows the product index.
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t smem, uint32_t block_bytes) {
  return kDescSwizzle128 | (64ull << 32) | (static_cast<uint64_t>(block_bytes >> 4) << 16) | ((smem >> 4) & 0x3fff);
}

// bf16 x bf16 -> fp32, 128 rows, n columns (a multiple of 16); B K-major, or MN-major when b_mn.
__device__ __forceinline__ uint32_t mma_desc(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
      "r"(static_cast<uint32_t>(add))
      : "memory");
}
// A from TMEM: 128 lanes, two bf16 per column.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
      "r"(static_cast<uint32_t>(add))
      : "memory");
}

// One lane of a converged warp.  Issuing warps stay converged and elect the lane only around the
// products, so that addresses and descriptors live in uniform registers: with a lane that runs alone
// they are moved there one by one, which costs several times the product's own issue.
__device__ __forceinline__ bool elect_lane() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(yes)::"memory");
  return yes != 0;
}

#define DLB_R4(m, r, i) m(r[i]), m(r[i + 1]), m(r[i + 2]), m(r[i + 3])
#define DLB_R16(m, r, i) DLB_R4(m, r, i), DLB_R4(m, r, i + 4), DLB_R4(m, r, i + 8), DLB_R4(m, r, i + 12)
#define DLB_OUT(x) "=r"(x)
#define DLB_IN(x) "r"(x)
#define DLB_INOUT(x) "+r"(x)

// 32 columns of this thread's lane, valid after tmem_loaded(r).
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,"
      "%31}, [%32];"
      : DLB_R16(DLB_OUT, r, 0), DLB_R16(DLB_OUT, r, 16)
      : "r"(addr));
}
// Waits for this thread's TMEM loads; the operand keeps uses of r behind the wait.
__device__ __forceinline__ void tmem_loaded(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : DLB_R16(DLB_INOUT, r, 0), DLB_R16(DLB_INOUT, r, 16)::"memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,"
      "%31,%32};" ::"r"(addr),
      DLB_R16(DLB_IN, r, 0), DLB_R16(DLB_IN, r, 16)
      : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : DLB_R16(DLB_OUT, r, 0)
      : "r"(addr));
}
__device__ __forceinline__ void tmem_loaded(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : DLB_R16(DLB_INOUT, r, 0)::"memory");
}
__device__ __forceinline__ void tmem_store8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), DLB_R4(DLB_IN, r, 0),
               DLB_R4(DLB_IN, r, 4)
               : "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two fp32 operations per instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a,b,c,d;\n\tmov.b64 a,{%2,%3};\n\tmov.b64 b,{%4,%5};\n\tmov.b64 c,{%6,%7};\n\t"
      "fma.rn.f32x2 d,a,b,c;\n\tmov.b64 {%0,%1},d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a,b,d;\n\tmov.b64 a,{%2,%3};\n\tmov.b64 b,{%4,%5};\n\tmul.rn.f32x2 d,a,b;\n\tmov.b64 {%0,%1},d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a,b,d;\n\tmov.b64 a,{%2,%3};\n\tmov.b64 b,{%4,%5};\n\tadd.rn.f32x2 d,a,b;\n\tmov.b64 {%0,%1},d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

}  // namespace dlb
