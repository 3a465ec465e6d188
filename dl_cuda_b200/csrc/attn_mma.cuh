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

// Capped scores times log2(e), L tanh(k x) with L = cap * log2(e), k = scale / cap, as odd polynomials:
// least-squares fits of tanh(x) / x in x^2, reweighted until the relative error was level.
//   |k x| <= 0.25: degree 2, error 4.2e-7 of a score (5.0e-7 in fp32), powers of k and L folded into the
//                  coefficients (4 operations a score)
//   |k x| <= 1:    degree 6, error 7.2e-8 (1.6e-7 in fp32), 10 operations
// Anything larger takes two special-function operations per score.  A warp takes one road, for the largest of
// the scores that it holds at a time, which are others in the forward and in either pass of the backward:
// the same score may differ by 5.0e-7 of itself between them.  Roads of one accuracy would cost a degree
// more; against what bf16 leaves of a probability (2^-8) the difference is nothing.
struct CapCoef {
  float c0, c1, c2, k, out;
  bool folded;  // k^5 must not fall under fp32's range
};
__device__ __forceinline__ CapCoef cap_coef(float scale, float cap) {
  CapCoef c;
  c.k = scale / cap;
  c.out = cap * kLog2e;
  const float kk = c.k * c.k;
  c.c0 = 0.9999995827674866f * c.k * c.out;
  c.c1 = -0.3332189917564392f * kk * c.k * c.out;
  c.c2 = 0.12841492891311646f * kk * kk * c.k * c.out;
  c.folded = c.k > 1e-4f && c.k < 1e4f;
  return c;
}

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

__device__ __forceinline__ float2 tanh_to_1(float2 x) {
  const float2 u = mul2(x, x);
  float2 p = fma2(u, both(0.0010406870860606432f), both(-0.006202297285199165f));
  p = fma2(p, u, both(0.020288638770580292f));
  p = fma2(p, u, both(-0.053456228226423264f));
  p = fma2(p, u, both(0.13325180113315582f));
  p = fma2(p, u, both(-0.33332836627960205f));
  p = fma2(p, u, both(0.9999999403953552f));
  return mul2(p, x);
}

// Largest value, in four chains of three-operand maxima.
template <int N, bool ABS>
__device__ __forceinline__ float max_of(const float (&x)[N]) {
  constexpr int C = N < 8 ? 1 : 4;
  float top[C];
#pragma unroll
  for (int c = 0; c < C; c++) top[c] = ABS ? 0.f : -INFINITY;
#pragma unroll
  for (int e = 0; e < N; e += 2 * C)
#pragma unroll
    for (int c = 0; c < C; c++) {
      const float p = x[e + 2 * c], q = x[e + 2 * c + 1];
      top[c] = fmaxf(fmaxf(top[c], ABS ? fabsf(p) : p), ABS ? fabsf(q) : q);
    }
  if constexpr (C == 1) return top[0];
  else return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}

template <int N>
__device__ __forceinline__ void cap_scores(float (&x)[N], const CapCoef &c) {
  // fmaxf drops NaN: a NaN score stays one on every road
  const float top = max_of<N, true>(x) * c.k;
  if (c.folded && __all_sync(0xffffffffu, top <= 0.25f)) {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float2 v = make_float2(x[e], x[e + 1]), u = mul2(v, v);
      float2 p = fma2(u, both(c.c2), both(c.c1));
      p = fma2(p, u, both(c.c0));
      p = mul2(p, v);
      x[e] = p.x;
      x[e + 1] = p.y;
    }
  } else if (__all_sync(0xffffffffu, top <= 1.f)) {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float2 t = mul2(tanh_to_1(mul2(make_float2(x[e], x[e + 1]), both(c.k))), both(c.out));
      x[e] = t.x;
      x[e + 1] = t.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; e++) x[e] = tanh_score(x[e] * c.k) * c.out;
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
int attn_fwd_mma_splits(const AttnArgs &a);  // shares of the keys that attn_fwd_mma wants
int attn_fwd_mma(const AttnArgs &a, cudaStream_t st);
struct BwdMaps {
  CUtensorMap q, k, v, dout;
};
int make_bwd_maps(const AttnArgs &a, BwdMaps *maps);
int attn_bwd_mma_keys(const AttnArgs &a, const BwdMaps &maps, cudaStream_t st);
int attn_bwd_mma_queries(const AttnArgs &a, const BwdMaps &maps, cudaStream_t st);

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
