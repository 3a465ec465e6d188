// What the tensor-core attention kernels share: the change of a tile's scores, masks, and the list
// of key tiles that matter.
#pragma once

#include "attn_common.cuh"
#include "tcgen05.cuh"

namespace dlb {

constexpr int kTileRows = 128;                         // rows of an accumulator: one TMEM lane each
constexpr int kBlockBytes = kTileRows * 128;           // one 64-column block of a 128-row tile
constexpr int kLutPad = 160;                           // room on both sides of the bias by distance
constexpr int kMaxTiles = 4096;                        // key (or query) tiles a kernel can list
enum { kNoBias = 0, kSlope = 1, kTable = 2 };          // kTable: with or without slopes

// tanh(x) for |x| <= 1 as x * P(x^2), degree 6 in x^2: a least-squares fit of tanh(x) / x reweighted
// until the relative error was level, 5e-8 before fp32 rounding and 1.2e-7 with it.
__device__ __forceinline__ float2 tanh_small2(float2 x) {
  const float2 u = mul2(x, x);
  auto c = [](float v) { return make_float2(v, v); };
  float2 p = fma2(u, c(0.0010406870860606432f), c(-0.006202297285199165f));
  p = fma2(p, u, c(0.020288638770580292f));
  p = fma2(p, u, c(-0.053456228226423264f));
  p = fma2(p, u, c(0.13325180113315582f));
  p = fma2(p, u, c(-0.33332836627960205f));
  p = fma2(p, u, c(0.9999999403953552f));
  return mul2(p, x);
}

// tanh of N scores times `k`.  Scores well inside the cap (|x k| <= 1 in the whole warp, the usual
// case) take the polynomial on the fp32 pipes, 9 instructions for two; a warp with a larger one pays
// two special-function operations per score.
template <int N>
__device__ __forceinline__ void tanh_scores(float (&x)[N], float k) {
  float top = 0.f;
#pragma unroll
  for (int c = 0; c < N; c++) top = fmaxf(top, fabsf(x[c]));
  const bool small = top * fabsf(k) <= 1.f;  // false for NaN as well: fmaxf drops it, the slow side keeps it
  if (__all_sync(0xffffffffu, small)) {
    const float2 kk = make_float2(k, k);
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      const float2 t = tanh_small2(mul2(make_float2(x[c], x[c + 1]), kk));
      x[c] = t.x;
      x[c + 1] = t.y;
    }
  } else {
#pragma unroll
    for (int c = 0; c < N; c++) x[c] = tanh_score(x[c] * k);
  }
}

// Bias by distance of one head, times log2(e): lut[d + reach + kLutPad], constant outside +-reach.
__device__ __forceinline__ void fill_lut(float *lut, const AttnArgs &a, int h, int tid, int threads) {
  for (int e = tid; e < 2 * (a.reach + kLutPad) + 1; e += threads)
    lut[e] = table_entry(a, h, bucket_at(a, e - a.reach - kLutPad));
}
__host__ __device__ inline int lut_floats(int reach) { return 2 * (reach + kLutPad) + 4; }

// The tensor cores need 16-byte aligned rows, and a scale that keeps the order of the scores.
bool attn_mma_fits(const AttnArgs &a, bool backward);
int attn_fwd_mma(const AttnArgs &a, cudaStream_t st);
bool attn_bwd_mma_room(const AttnArgs &a);  // does its shared memory fit?
int attn_bwd_mma_keys(const AttnArgs &a, cudaStream_t st);
int attn_bwd_mma_queries(const AttnArgs &a, cudaStream_t st);

// Waits for copies or MMAs still in flight after another wait of the CTA gave up (bounded as well).
__device__ __forceinline__ void drain_wait(uint64_t *bar, unsigned parity) {
  const uint32_t addr = smem_u32(bar);
  const unsigned long long start = global_ns();
  for (;;) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (done || global_ns() - start > kWaitLimitNs) return;
  }
}

__device__ __forceinline__ int warp_min(int v) { return __reduce_min_sync(0xffffffffu, v); }
__device__ __forceinline__ int warp_max(int v) { return __reduce_max_sync(0xffffffffu, v); }

}  // namespace dlb
