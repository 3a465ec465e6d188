// Attention on the fp32 pipes: every storage type, head width, stride and alignment.
//
// A CTA of 256 threads (16 x 16) works on tiles of 64 rows and 64 columns.  Thread (ty, tx) owns
// rows ty + 16a and columns tx + 16b (a, b < 4), so that a score costs head_dim multiply-adds fed by
// 8 16-byte shared loads per 64 of them; rows are padded by 16 bytes, which spreads the 8 rows a
// quarter warp reads over all banks.  A row's 16 threads are one half warp: its maximum and sum
// take four shuffles, and its probabilities pass through shared memory without a CTA barrier.
#pragma once

#include "attn_common.cuh"

namespace dlb {

constexpr int kGenTile = 64, kGenThreads = 256;

// Columns of the output that thread tx holds: groups of four adjacent ones, 64 apart (one or two
// adjacent ones for the narrow widths).
template <int DP>
struct GenCols {
  static constexpr int kCount = DP / 16;
  static constexpr int kAdjacent = kCount < 4 ? kCount : 4;
  __device__ __forceinline__ static int col(int tx, int n) { return (n / kAdjacent) * 64 + tx * kAdjacent + n % kAdjacent; }
};

// Tile row r -> source row address; rows at or beyond `rows` and columns beyond `dim` read as zero.
template <typename T, int DP, typename RowPtr>
__device__ __forceinline__ void gen_load_tile(float *dst, int rows, int dim, bool vec, RowPtr row_ptr) {
  constexpr int V = Store<T>::kPerVec;
  if (vec) {
    constexpr int per_row = DP / V;
    for (int e = threadIdx.x; e < kGenTile * per_row; e += kGenThreads) {
      const int r = e / per_row, c = (e % per_row) * V;
      float f[V];
#pragma unroll
      for (int i = 0; i < V; i++) f[i] = 0.f;
      if (r < rows && c < dim) Store<T>::unpack(ld_keep(row_ptr(r) + c), f);
#pragma unroll
      for (int i = 0; i < V; i += 4)
        *reinterpret_cast<float4 *>(dst + r * (DP + 4) + c + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
    }
  } else {
    for (int e = threadIdx.x; e < kGenTile * DP; e += kGenThreads) {
      const int r = e / DP, c = e % DP;
      dst[r * (DP + 4) + c] = (r < rows && c < dim) ? Store<T>::to_float(ld_co(row_ptr(r) + c)) : 0.f;
    }
  }
}

// out[a][b] = <x row ty + 16a, u row tx + 16b>
template <int DP>
__device__ __forceinline__ void gen_dot(float (&out)[4][4], const float *x, const float *u, int ty, int tx) {
#pragma unroll
  for (int a = 0; a < 4; a++)
#pragma unroll
    for (int b = 0; b < 4; b++) out[a][b] = 0.f;
#pragma unroll 4
  for (int d = 0; d < DP; d += 4) {
    float4 xv[4], uv[4];
#pragma unroll
    for (int a = 0; a < 4; a++) xv[a] = *reinterpret_cast<const float4 *>(x + (ty + 16 * a) * (DP + 4) + d);
#pragma unroll
    for (int b = 0; b < 4; b++) uv[b] = *reinterpret_cast<const float4 *>(u + (tx + 16 * b) * (DP + 4) + d);
#pragma unroll
    for (int a = 0; a < 4; a++)
#pragma unroll
      for (int b = 0; b < 4; b++) {
        out[a][b] = fmaf(xv[a].x, uv[b].x, out[a][b]);
        out[a][b] = fmaf(xv[a].y, uv[b].y, out[a][b]);
        out[a][b] = fmaf(xv[a].z, uv[b].z, out[a][b]);
        out[a][b] = fmaf(xv[a].w, uv[b].w, out[a][b]);
      }
  }
}

constexpr int kGenScoreStride = kGenTile + 4;

// acc[a][n] += sum_c w[row ty + 16a][c] * u[c][col n]
template <int DP>
__device__ __forceinline__ void gen_accumulate(float (&acc)[4][GenCols<DP>::kCount], const float *w, const float *u,
                                               int ty, int tx) {
  constexpr int N = GenCols<DP>::kCount, A = GenCols<DP>::kAdjacent;
#pragma unroll 2
  for (int c = 0; c < kGenTile; c += 4) {
    float wv[4][4];
#pragma unroll
    for (int a = 0; a < 4; a++) {
      const float4 t = *reinterpret_cast<const float4 *>(w + (ty + 16 * a) * kGenScoreStride + c);
      wv[a][0] = t.x; wv[a][1] = t.y; wv[a][2] = t.z; wv[a][3] = t.w;
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      float uv[N];
#pragma unroll
      for (int n = 0; n < N; n += A) {
        const float *src = u + (c + k) * (DP + 4) + GenCols<DP>::col(tx, n);
        if constexpr (A == 4) {
          const float4 t = *reinterpret_cast<const float4 *>(src);
          uv[n] = t.x; uv[n + 1] = t.y; uv[n + 2] = t.z; uv[n + 3] = t.w;
        } else if constexpr (A == 2) {
          const float2 t = *reinterpret_cast<const float2 *>(src);
          uv[n] = t.x; uv[n + 1] = t.y;
        } else {
          uv[n] = *src;
        }
      }
#pragma unroll
      for (int a = 0; a < 4; a++)
#pragma unroll
        for (int n = 0; n < N; n++) acc[a][n] = fmaf(wv[a][k], uv[n], acc[a][n]);
    }
  }
}

// Score (times log2 e) of a pair `distance` = j - p apart; also what its backward needs of the cap.
__device__ __forceinline__ float gen_score(const AttnArgs &a, float dot, int h, float slope, int distance, float *dcap) {
  float s;
  if (a.cap > 0.f) {
    const float t = tanh_score(dot * (a.scale / a.cap));
    s = t * (a.cap * kLog2e);
    *dcap = fmaf(-t, t, 1.f);
  } else {
    s = dot * (a.scale * kLog2e);
    *dcap = 1.f;
  }
  if (a.slopes) s -= slope * static_cast<float>(abs(distance));
  if (a.table) s += table_entry(a, h, bucket_at(a, distance));
  return s;
}

__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float half_warp_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Forward.  Tile rows are (query, head) pairs: with `pack` = group a tile holds 64 / group queries
// of all heads that share a key/value head (few queries: the cache is read once for the group),
// with pack = 1 it holds 64 queries of one head.  blockIdx.y is a share of the key tiles; with more
// than one share the partial results go to part_o / part_ml for attn_join_kernel.
template <typename T, int DP>
static __global__ void __launch_bounds__(kGenThreads)
attn_fwd_generic_kernel(const __grid_constant__ AttnArgs a, int pack, bool vec) {
  pdl_prologue();
  extern __shared__ __align__(16) float gen_smem[];
  float *qs = gen_smem, *ks = qs + kGenTile * (DP + 4), *vs = ks + kGenTile * (DP + 4), *ps = vs + kGenTile * (DP + 4);
  __shared__ int doc_tile[kGenTile];
  constexpr int N = GenCols<DP>::kCount;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int units = a.heads / pack;  // head, or key/value head when packed
  const int q_rows = a.q_len * pack, tiles = (q_rows + kGenTile - 1) / kGenTile;
  const int tile = tiles - 1 - static_cast<int>(blockIdx.x % tiles);  // long causal rows start first
  const int unit = (blockIdx.x / tiles) % units, b = blockIdx.x / (tiles * units);
  const int row0 = tile * kGenTile, rows = min(kGenTile, q_rows - row0);
  const int hk = pack > 1 ? unit : unit / a.group, h0 = pack > 1 ? unit * pack : unit;
  const BatchView view = batch_view(a, b);

  const T *qb = static_cast<const T *>(a.q.ptr) + b * a.q.batch + h0 * a.q.head;
  const T *kb = static_cast<const T *>(a.k.ptr) + b * a.k.batch + hk * a.k.head;
  const T *vb = static_cast<const T *>(a.v.ptr) + b * a.v.batch + hk * a.v.head;
  gen_load_tile<T, DP>(qs, rows, a.dim, vec, [&](int r) {
    const int x = row0 + r;
    return qb + static_cast<long long>(x / pack) * a.q.token + (x % pack) * a.q.head;
  });

  int pos[4], end[4], head[4], doc[4];
  float slope[4];
  int reach = 0;
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const int x = row0 + ty + 16 * r, i = x / pack;
    const bool valid = x < q_rows;
    head[r] = h0 + x % pack;
    pos[r] = view.start + i;
    end[r] = valid ? row_end(a, view, i) : 0;
    doc[r] = (a.q_docs && valid) ? a.q_docs[static_cast<long long>(b) * a.q_len + i] : 0;
    slope[r] = (a.slopes && valid) ? a.slopes[head[r]] * kLog2e : 0.f;
    reach = max(reach, end[r]);
  }
  // row_end never falls with the query: the last row's bound is the tile's.
  const int last = row_end(a, view, (row0 + rows - 1) / pack);
  const int key_tiles = (last + kGenTile - 1) / kGenTile;
  const int share = (key_tiles + a.splits - 1) / a.splits;
  const int t0 = min(key_tiles, static_cast<int>(blockIdx.y) * share), t1 = min(key_tiles, t0 + share);

  float acc[4][N], m[4], l[4];
#pragma unroll
  for (int r = 0; r < 4; r++) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int n = 0; n < N; n++) acc[r][n] = 0.f;
  }
  for (int t = t0; t < t1; t++) {
    const int j0 = t * kGenTile, keys = min(kGenTile, last - j0);
    __syncthreads();
    if (a.kv_docs) {
      if (threadIdx.x < kGenTile && threadIdx.x < keys)
        doc_tile[threadIdx.x] = a.kv_docs[static_cast<long long>(b) * a.kv_len + j0 + threadIdx.x];
      __syncthreads();
      bool any = false;  // does any row of the tile share a document with any of its keys?
      for (int c = tx; c < keys; c += 16)
#pragma unroll
        for (int r = 0; r < 4; r++) any |= (j0 + c < end[r]) && doc[r] == doc_tile[c];
      if (!__syncthreads_or(any)) continue;
    }
    gen_load_tile<T, DP>(ks, keys, a.dim, vec, [&](int r) { return kb + static_cast<long long>(j0 + r) * a.k.token; });
    gen_load_tile<T, DP>(vs, keys, a.dim, vec, [&](int r) { return vb + static_cast<long long>(j0 + r) * a.v.token; });
    __syncthreads();
    float s[4][4];
    gen_dot<DP>(s, qs, ks, ty, tx);
#pragma unroll
    for (int r = 0; r < 4; r++) {
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const int j = j0 + tx + 16 * c;
        bool seen = j < end[r];
        if (a.kv_docs) seen = seen && doc_tile[tx + 16 * c] == doc[r];
        float unused;
        s[r][c] = seen ? gen_score(a, s[r][c], head[r], slope[r], j - pos[r], &unused) : -INFINITY;
        top = fmaxf(top, s[r][c]);
      }
      top = fmaxf(m[r], half_warp_max(top));
      const float base = top == -INFINITY ? 0.f : top;
      const float keep = ex2(m[r] - base);
      m[r] = top;
      l[r] *= keep;
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const float p = ex2(s[r][c] - base);
        l[r] += p;
        ps[(ty + 16 * r) * kGenScoreStride + tx + 16 * c] = p;
      }
#pragma unroll
      for (int n = 0; n < N; n++) acc[r][n] *= keep;
    }
    __syncwarp();
    gen_accumulate<DP>(acc, ps, vs, ty, tx);
  }
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const float total = half_warp_sum(l[r]);
    const int x = row0 + ty + 16 * r;
    if (x >= q_rows) continue;
    const int i = x / pack;
    const size_t row = (static_cast<size_t>(b) * a.heads + head[r]) * a.q_len + i;
    if (a.splits > 1) {
      const size_t at = static_cast<size_t>(blockIdx.y) * a.batch * a.heads * a.q_len + row;
      if (tx == 0) a.part_ml[at] = make_float2(m[r], total);
#pragma unroll
      for (int n = 0; n < N; n++) {
        const int c = GenCols<DP>::col(tx, n);
        if (c < a.dim) a.part_o[at * a.dim + c] = acc[r][n];
      }
    } else {
      const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
      T *out = static_cast<T *>(a.o.ptr) + b * a.o.batch + static_cast<long long>(i) * a.o.token + head[r] * a.o.head;
#pragma unroll
      for (int n = 0; n < N; n++) {
        const int c = GenCols<DP>::col(tx, n);
        if (c < a.dim) out[c] = Store<T>::from_float(acc[r][n] * inv);
      }
      if (a.lse && tx == 0) a.lse[row] = total == 0.f ? -INFINITY : (m[r] + log2f(total)) * kLn2;
    }
  }
}

// Joins the shares of the keys: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.  One CTA per row: with
// one user there are few rows and many shares, which four warps then read side by side.
constexpr int kJoinThreads = 128, kMaxSplits = 256;

template <typename T>
static __global__ void __launch_bounds__(kJoinThreads) attn_join_kernel(const __grid_constant__ AttnArgs a) {
  pdl_prologue();
  __shared__ float weight[kMaxSplits], part[4][DLB_ATTN_MAX_HEAD_DIM], warp_value[4];
  const size_t rows = static_cast<size_t>(a.batch) * a.heads * a.q_len, row = blockIdx.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float2 ml[kMaxSplits / kJoinThreads];
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kMaxSplits / kJoinThreads; k++) {
    const int s = tid + k * kJoinThreads;
    ml[k] = s < a.splits ? a.part_ml[s * rows + row] : make_float2(-INFINITY, 0.f);
    m = fmaxf(m, ml[k].x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) warp_value[warp] = m;
  __syncthreads();
  m = fmaxf(fmaxf(warp_value[0], warp_value[1]), fmaxf(warp_value[2], warp_value[3]));
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
#pragma unroll
  for (int k = 0; k < kMaxSplits / kJoinThreads; k++) {
    const float w = ex2(ml[k].x - base);
    weight[tid + k * kJoinThreads] = w;
    l = fmaf(w, ml[k].y, l);
  }
  l = warp_sum(l);
  __syncthreads();
  if (lane == 0) warp_value[warp] = l;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = warp; s < a.splits; s += 4) {
    const float *src = a.part_o + (s * rows + row) * a.dim;
    const float w = weight[s];
#pragma unroll
    for (int n = 0; n < 4; n++)
      if (lane + 32 * n < a.dim) acc[n] = fmaf(w, src[lane + 32 * n], acc[n]);
  }
#pragma unroll
  for (int n = 0; n < 4; n++) part[warp][lane + 32 * n] = acc[n];
  __syncthreads();
  l = warp_value[0] + warp_value[1] + warp_value[2] + warp_value[3];
  const int i = row % a.q_len, h = (row / a.q_len) % a.heads, b = row / (static_cast<size_t>(a.q_len) * a.heads);
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  T *out = static_cast<T *>(a.o.ptr) + b * a.o.batch + i * a.o.token + h * a.o.head;
  if (tid < a.dim) out[tid] = Store<T>::from_float((part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid]) * inv);
  if (a.lse && tid == 0) a.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// Fills row_stats: -lse * log2(e) and -delta, delta = <dout_i, o_i> (= sum_j P_ij dP_ij).  One warp per row.
template <typename T>
static __global__ void __launch_bounds__(256) attn_row_stats_kernel(const __grid_constant__ AttnArgs a) {
  pdl_prologue();
  const int padded = stat_tiles(a.q_len) * kStatRows;
  const size_t rows = static_cast<size_t>(a.batch) * a.heads * padded;
  const size_t row = static_cast<size_t>(blockIdx.x) * 8 + threadIdx.x / 32;
  if (row >= rows) return;
  const int lane = threadIdx.x & 31;
  // heads innermost: neighbouring warps read neighbouring memory of [token, head] layouts
  const int h = row % a.heads, i = (row / a.heads) % padded, b = row / (static_cast<size_t>(padded) * a.heads);
  float sum = 0.f;
  if (i < a.q_len) {
    const T *o = static_cast<const T *>(a.o.ptr) + b * a.o.batch + i * a.o.token + h * a.o.head;
    const T *g = static_cast<const T *>(a.dout.ptr) + b * a.dout.batch + i * a.dout.token + h * a.dout.head;
    for (int c = lane; c < a.dim; c += 32) sum = fmaf(Store<T>::to_float(ld_co(o + c)), Store<T>::to_float(ld_co(g + c)), sum);
    sum = warp_sum(sum);
  }
  if (lane == 0) {
    float *at = stats_tile(a, b, h, i / kStatRows) + i % kStatRows;
    at[0] = i < a.q_len ? -a.lse[(static_cast<size_t>(b) * a.heads + h) * a.q_len + i] * kLog2e : -INFINITY;
    if (i < a.q_len && at[0] == INFINITY) at[0] = -INFINITY;  // lse = -infinity
    at[kStatRows] = -sum;
  }
}

// Backward.  The tile's 64 rows stay (keys and values when FOR_KEYS, else queries and output
// gradients), the other side streams by in tiles of 64 columns:
//   P = exp2(s - lse), dS = P (dP - delta);  FOR_KEYS: dV += P^T dO, dK += dS^T Q over the heads of
// the group, else dQ += dS K.  Each pass rebuilds the scores, so no sum crosses a CTA.
template <typename T, int DP, bool FOR_KEYS>
static __global__ void __launch_bounds__(kGenThreads)
attn_bwd_generic_kernel(const __grid_constant__ AttnArgs a, bool vec) {
  pdl_prologue();
  extern __shared__ __align__(16) float gen_smem[];
  constexpr int N = GenCols<DP>::kCount, kSlab = kGenTile * (DP + 4);
  float *xs = gen_smem, *ys = xs + kSlab, *us = ys + kSlab, *ws = us + kSlab;
  float *ds = ws + kSlab, *ps = ds + kGenTile * kGenScoreStride;
  float *sum_ds = ps + kGenTile * kGenScoreStride, *sum_p = sum_ds + a.buckets * kGenTile;
  __shared__ float2 col_stats[kGenTile];
  __shared__ int col_doc[kGenTile];
  const bool want_table = !FOR_KEYS && a.dtable != nullptr;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int len = FOR_KEYS ? a.kv_len : a.q_len, units = FOR_KEYS ? a.kv_heads : a.heads;
  const int tiles = (len + kGenTile - 1) / kGenTile;
  int tile = blockIdx.x % tiles;
  if (!FOR_KEYS) tile = tiles - 1 - tile;  // long causal rows first
  const int unit = (blockIdx.x / tiles) % units, b = blockIdx.x / (tiles * units);
  const int row0 = tile * kGenTile, rows = min(kGenTile, len - row0);
  const int hk = FOR_KEYS ? unit : unit / a.group;
  const BatchView view = batch_view(a, b);
  const int bound = FOR_KEYS ? min(rows, max(0, view.end - row0)) : rows;  // rows that hold numbers

  const T *kb = static_cast<const T *>(a.k.ptr) + b * a.k.batch + hk * a.k.head;
  const T *vb = static_cast<const T *>(a.v.ptr) + b * a.v.batch + hk * a.v.head;
  const T *q_all = static_cast<const T *>(a.q.ptr) + b * a.q.batch;
  const T *g_all = static_cast<const T *>(a.dout.ptr) + b * a.dout.batch;
  if (FOR_KEYS) {
    gen_load_tile<T, DP>(xs, bound, a.dim, vec, [&](int r) { return kb + static_cast<long long>(row0 + r) * a.k.token; });
    gen_load_tile<T, DP>(ys, bound, a.dim, vec, [&](int r) { return vb + static_cast<long long>(row0 + r) * a.v.token; });
  } else {
    gen_load_tile<T, DP>(xs, rows, a.dim, vec,
                         [&](int r) { return q_all + unit * a.q.head + static_cast<long long>(row0 + r) * a.q.token; });
    gen_load_tile<T, DP>(ys, rows, a.dim, vec,
                         [&](int r) { return g_all + unit * a.dout.head + static_cast<long long>(row0 + r) * a.dout.token; });
  }
  if (want_table)
    for (int e = threadIdx.x; e < 2 * a.buckets * kGenTile; e += kGenThreads) sum_ds[e] = 0.f;

  int row_doc[4], end[4];
  float2 row_stat[4];
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const int x = row0 + ty + 16 * r;
    const bool valid = ty + 16 * r < bound;
    const int *docs = FOR_KEYS ? a.kv_docs : a.q_docs;
    row_doc[r] = (docs && valid) ? docs[static_cast<long long>(b) * len + x] : 0;
    end[r] = (!FOR_KEYS && valid) ? row_end(a, view, x) : 0;
    row_stat[r] = (!FOR_KEYS && valid) ? stat_at(a, b, unit, x) : make_float2(-INFINITY, 0.f);
  }
  float acc_x[4][N], acc_y[4][N];
#pragma unroll
  for (int r = 0; r < 4; r++)
#pragma unroll
    for (int n = 0; n < N; n++) acc_x[r][n] = acc_y[r][n] = 0.f;

  const int last = FOR_KEYS ? a.q_len : row_end(a, view, row0 + rows - 1);
  const int first = FOR_KEYS ? (bound > 0 ? first_query(a, view, row0) / kGenTile : (a.q_len + kGenTile - 1) / kGenTile) : 0;
  const int t_end = (last + kGenTile - 1) / kGenTile;
  for (int g = 0; g < (FOR_KEYS ? a.group : 1); g++) {
    const int h = FOR_KEYS ? hk * a.group + g : unit;
    const float slope = a.slopes ? a.slopes[h] * kLog2e : 0.f;
    for (int t = first; t < t_end; t++) {
      const int c0 = t * kGenTile, cols = min(kGenTile, last - c0);
      __syncthreads();
      if (threadIdx.x < kGenTile) {
        const int c = threadIdx.x;
        const int *docs = FOR_KEYS ? a.q_docs : a.kv_docs;
        col_doc[c] = (docs && c < cols) ? docs[static_cast<long long>(b) * (FOR_KEYS ? a.q_len : a.kv_len) + c0 + c] : 0;
        if (FOR_KEYS)
          col_stats[c] = c < cols ? stat_at(a, b, h, c0 + c) : make_float2(-INFINITY, 0.f);
      }
      __syncthreads();
      if (a.kv_docs) {
        bool any = false;
        for (int c = tx; c < cols; c += 16)
#pragma unroll
          for (int r = 0; r < 4; r++) any |= ty + 16 * r < bound && row_doc[r] == col_doc[c];
        if (!__syncthreads_or(any)) continue;
      }
      if (FOR_KEYS) {
        gen_load_tile<T, DP>(us, cols, a.dim, vec, [&](int r) { return q_all + h * a.q.head + static_cast<long long>(c0 + r) * a.q.token; });
        gen_load_tile<T, DP>(ws, cols, a.dim, vec, [&](int r) { return g_all + h * a.dout.head + static_cast<long long>(c0 + r) * a.dout.token; });
      } else {
        gen_load_tile<T, DP>(us, cols, a.dim, vec, [&](int r) { return kb + static_cast<long long>(c0 + r) * a.k.token; });
        gen_load_tile<T, DP>(ws, cols, a.dim, vec, [&](int r) { return vb + static_cast<long long>(c0 + r) * a.v.token; });
      }
      __syncthreads();
      float s[4][4], dp[4][4];
      gen_dot<DP>(s, xs, us, ty, tx);
      gen_dot<DP>(dp, ys, ws, ty, tx);
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int c = 0; c < 4; c++) {
          const int row = row0 + ty + 16 * r, col = c0 + tx + 16 * c;
          const int i = FOR_KEYS ? col : row, j = FOR_KEYS ? row : col;
          bool seen = FOR_KEYS ? (ty + 16 * r < bound && tx + 16 * c < cols && j < row_end(a, view, i)) : j < end[r];
          if (a.kv_docs) seen = seen && row_doc[r] == col_doc[tx + 16 * c];
          const float2 stat = FOR_KEYS ? col_stats[tx + 16 * c] : row_stat[r];
          float dcap, p = 0.f, grad = 0.f;
          if (seen) {
            p = ex2(gen_score(a, s[r][c], h, slope, j - (view.start + i), &dcap) + stat.x);
            grad = p * (dp[r][c] + stat.y);
          } else {
            dcap = 0.f;
          }
          const int at = (ty + 16 * r) * kGenScoreStride + tx + 16 * c;
          ps[at] = p;
          ds[at] = grad;
          s[r][c] = dcap * a.scale;
        }
      __syncwarp();
      if (want_table) {
        // Rows' gradients of the scores add up to zero: what rounding left (in delta above all) is
        // taken off again in proportion to P when the buckets are summed, below.
        __syncthreads();
        if (threadIdx.x < kGenTile) {
          const int r = threadIdx.x;
          int now = -1;
          float part_ds = 0.f, part_p = 0.f;
          for (int c = 0; c < cols; c++) {
            const int n = bucket_at(a, c0 + c - (view.start + row0 + r));
            if (n != now) {
              if (now >= 0) {
                sum_ds[now * kGenTile + r] += part_ds;
                sum_p[now * kGenTile + r] += part_p;
              }
              now = n;
              part_ds = part_p = 0.f;
            }
            part_ds += ds[r * kGenScoreStride + c];
            part_p += ps[r * kGenScoreStride + c];
          }
          if (now >= 0) {
            sum_ds[now * kGenTile + r] += part_ds;
            sum_p[now * kGenTile + r] += part_p;
          }
        }
        __syncthreads();
      }
      if (FOR_KEYS) gen_accumulate<DP>(acc_y, ps, ws, ty, tx);
      // through the cap and the scale, into the gradient of <q, k>
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int c = 0; c < 4; c++) ds[(ty + 16 * r) * kGenScoreStride + tx + 16 * c] *= s[r][c];
      __syncwarp();
      gen_accumulate<DP>(acc_x, ds, us, ty, tx);
    }
  }
  const Heads &xo = FOR_KEYS ? a.dk : a.dq;
  T *dx = static_cast<T *>(xo.ptr) + b * xo.batch + unit * xo.head;
  T *dy = FOR_KEYS ? static_cast<T *>(a.dv.ptr) + b * a.dv.batch + unit * a.dv.head : nullptr;
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const int x = ty + 16 * r;
    if (x >= rows) continue;
#pragma unroll
    for (int n = 0; n < N; n++) {
      const int c = GenCols<DP>::col(tx, n);
      if (c >= a.dim) continue;
      dx[static_cast<long long>(row0 + x) * xo.token + c] = Store<T>::from_float(acc_x[r][n]);
      if (FOR_KEYS) dy[static_cast<long long>(row0 + x) * a.dv.token + c] = Store<T>::from_float(acc_y[r][n]);
    }
  }
  if (want_table) {
    __syncthreads();
    if (threadIdx.x < kGenTile) {
      const int r = threadIdx.x;
      float e = 0.f, p = 0.f;
      for (int n = 0; n < a.buckets; n++) {
        e += sum_ds[n * kGenTile + r];
        p += sum_p[n * kGenTile + r];
      }
      e = p > 0.f ? e / p : 0.f;
      for (int n = 0; n < a.buckets; n++) sum_ds[n * kGenTile + r] -= e * sum_p[n * kGenTile + r];
    }
    __syncthreads();
    float *part = a.table_part + (static_cast<size_t>(unit) * a.table_parts + b * tiles + tile) * a.buckets;
    for (int n = threadIdx.x; n < a.buckets; n += kGenThreads) {
      float sum = 0.f;
      for (int r = 0; r < kGenTile; r++) sum += sum_ds[n * kGenTile + r];
      part[n] = sum;
    }
  }
}

// dtable[h, n] = sum of the parts, in order.  One CTA per (head, bucket).
static __global__ void __launch_bounds__(128) attn_table_sum_kernel(const __grid_constant__ AttnArgs a) {
  pdl_prologue();
  __shared__ double warp_part[4];
  const int h = blockIdx.x / a.buckets, n = blockIdx.x % a.buckets;
  double sum = 0.0;
  for (int p = threadIdx.x; p < a.table_parts; p += 128)
    sum += a.table_part[(static_cast<size_t>(h) * a.table_parts + p) * a.buckets + n];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x / 32] = sum;
  __syncthreads();
  if (threadIdx.x == 0)
    a.dtable[h * a.buckets + n] = static_cast<float>(warp_part[0] + warp_part[1] + warp_part[2] + warp_part[3]);
}

}  // namespace dlb
