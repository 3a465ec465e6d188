// What the attention kernels share: the arguments as they travel to the GPU, who sees whom, and
// the score of a visible pair.  Scores are kept times log2(e), so that a probability is one exp2.
#pragma once

#include <climits>
#include <cmath>
#include <cstdint>

#include "common.cuh"

namespace dlb {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kHidesBelow = -1e30f;  // table entries under this hide their keys

// Lets a kernel use any amount of dynamic shared memory up to kMaxDynamicSmem (8 KB are left for static).
// The limit is a property of the kernel, not of a launch: set to each call's own need, a smaller call on
// one host thread would take it away from a larger one on another.
constexpr size_t kMaxDynamicSmem = 227 * 1024 - 8192;
template <typename K>
int allow_smem(K kern, size_t smem, const char *name) {
  DLB_REQUIRE(smem <= kMaxDynamicSmem, DLB_ERR_UNSUPPORTED, "%s: %zu bytes of shared memory", name, smem);
  if (smem <= 40 * 1024) return DLB_OK;  // 48 KB with the static are free to all
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMaxDynamicSmem));
  DLB_REQUIRE(e == cudaSuccess, DLB_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
  return DLB_OK;
}

// An address between two elements would fault in the kernel.
inline bool on_elements(const void *p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

struct Heads {
  void *ptr;
  long long batch, token, head;  // strides in elements
};

struct AttnArgs {
  int batch, heads, kv_heads, group, q_len, kv_len, dim, causal;
  float scale, cap;
  int buckets, reach;  // reach: max_distance of the bucket map
  const int *kv_lens, *q_start, *prefix, *q_docs, *kv_docs;
  const float *slopes, *table;
  const int *bucket_of;
  Heads q, k, v, o;
  float *lse;
  Heads dout, dq, dk, dv;  // backward only
  float *dtable;
  float *row_stats;        // backward: see stats_tile
  float *table_part;       // backward: [heads][parts][buckets]
  int table_parts;
  // forward split over the keys: partial outputs [split][b, h, i][dim] and {max, sum} [split][b, h, i]
  float *part_o;
  float2 *part_ml;
  int splits;
};

// Backward: what it needs of a query row, in tiles of 128 rows per (b, h): 128 times -lse * log2(e)
// (-infinity for a row that saw no key, and behind the last row: its probabilities are then
// exp2(s - infinity) = 0), then 128 times -delta.  1 KB a tile, on a 16-byte boundary for any q_len.
constexpr int kStatRows = 128;
__host__ __device__ inline int stat_tiles(int q_len) { return (q_len + kStatRows - 1) / kStatRows; }
__device__ __forceinline__ float *stats_tile(const AttnArgs &a, int b, int h, int tile) {
  return a.row_stats + ((static_cast<size_t>(b) * a.heads + h) * stat_tiles(a.q_len) + tile) * (2 * kStatRows);
}
// Backward: are these all the keys of a row (its probabilities, rebuilt from lse, add up to one), so that its
// score gradients add up to zero?  Not for a call over some of the keys with o and lse of all.  The sum may be
// off by twice what the rounding of lse makes of a probability, by what two kernels make of a score, and with
// bf16 by the roads of a cap (2^-21 of a score in each pass).  A share that lacks less of a row's weight than
// that passes for the whole, and what it lacks is lost in the same roundings.
template <typename T>
__device__ __forceinline__ bool row_is_whole(const AttnArgs &a, float sum, float minus_lse_log2) {
  const bool half = sizeof(T) == 2;
  const float limit = fmaf(fabsf(minus_lse_log2), 0x1p-22f * kLn2, half ? fmaf(a.cap, 0x1p-20f, 0x1p-15f) : 0x1p-18f);
  return fabsf(sum - 1.f) <= fminf(limit, 0x1p-10f);  // (lse = -infinity: the sum is 0)
}

__device__ __forceinline__ float2 stat_at(const AttnArgs &a, int b, int h, int i) {
  const float *t = stats_tile(a, b, h, i / kStatRows) + i % kStatRows;
  return make_float2(t[0], t[kStatRows]);
}

// Per batch: query i stands at start + i; keys from `end` on are reached by no query.
struct BatchView {
  int start, len, prefix, end;
};

__device__ __forceinline__ BatchView batch_view(const AttnArgs &a, int b) {
  BatchView v;
  v.start = a.q_start ? max(-(1 << 30), min(1 << 30, a.q_start[b])) : 0;
  v.len = a.kv_lens ? max(0, min(a.kv_len, a.kv_lens[b])) : a.kv_len;
  v.prefix = (a.causal && a.prefix) ? max(0, min(a.kv_len, a.prefix[b])) : 0;
  v.end = a.causal ? min(v.len, max(max(v.start + a.q_len, 0), v.prefix)) : v.len;
  return v;
}

// Keys [0, row_end) are visible to query i, as far as documents allow.
__device__ __forceinline__ int row_end(const AttnArgs &a, const BatchView &v, int i) {
  return a.causal ? min(v.len, max(v.start + i + 1, v.prefix)) : v.len;
}

// First query that sees key j (queries behind it see it too: row_end never falls with i).
__device__ __forceinline__ int first_query(const AttnArgs &a, const BatchView &v, int j) {
  return (!a.causal || j < v.prefix) ? 0 : max(0, j - v.start);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// tanh(x) = sign(x) * (1 - 2 / (1 + exp(2|x|))): near zero the difference cancels (absolute error
// about 1e-7), where cap * tanh(x / cap) would lose relative precision in small scores; there the
// odd series x - x^3/3 + 2x^5/15 - 17x^7/315 + 62x^9/2835 is used, whose first dropped term is under
// 1e-8 of x for |x| < 0.25.
__device__ __forceinline__ float tanh_score(float x) {
  const float ax = fabsf(x), x2 = x * x;
  const float e = ex2(ax * (2.f * kLog2e));
  const float far = copysignf(1.f - __fdividef(2.f, 1.f + e), x);
  float p = fmaf(x2, 62.f / 2835.f, -17.f / 315.f);
  p = fmaf(x2, p, 2.f / 15.f);
  p = fmaf(x2, p, -1.f / 3.f);
  const float near = fmaf(x * x2, p, x);
  return ax < 0.25f ? near : far;
}

// Table value of a bucket times log2(e), with the entries that hide their keys as -infinity.
__device__ __forceinline__ float table_entry(const AttnArgs &a, int h, int bucket) {
  const float t = a.table[h * a.buckets + bucket];
  return t < kHidesBelow ? -INFINITY : t * kLog2e;
}

__device__ __forceinline__ int bucket_at(const AttnArgs &a, int distance) {
  const int d = max(-a.reach, min(a.reach, distance)) + a.reach;
  return min(max(a.bucket_of[d], 0), a.buckets - 1);
}

}  // namespace dlb
