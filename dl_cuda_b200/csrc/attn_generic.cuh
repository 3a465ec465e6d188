// Attention in fp32 arithmetic: every storage type, head width, stride and alignment.
//
// The products run on the warp-level tensor path (mma.sync m16n8k8, tf32) with every operand split in
// two, x = hi + lo with 11 bits each: hi*hi + hi*lo + lo*hi leaves out 2^-21 of |x||y|.
// fp32 results are up to three times as far from the exact ones as those of plain fp32 arithmetic (2-norm at
// most 9e-7 over 210 random cases, 1.1e-6 for the gradient of a table); bf16 values need no lo, but take the
// same road.  Three such products run at 90 TFLOP/s where scalar multiply-adds reach 67 at best (both
// measured on a B200), and they need a quarter of the shared-memory reads: the 64x64 scalar tiles this
// replaces were bound by those.
//
// A CTA of eight warps keeps 16 * RG rows (RG groups of 16) and streams tiles of 64 rows past them; the
// 8 / RG warps of a row group take 8 * RG columns of a tile each and are joined at the end.  RG = 1 for
// few queries, 2 while 64-row tiles leave SMs idle, else 4.
//
// Fragments.  A product's inner index may run in any order: a lane loads 16 adjacent bytes of a row and
// uses them as two steps (columns 4c..4c+3 of 16); the probabilities of columns 2c, 2c + 1 stand where
// the second product wants inner indexes c and c + 4, so the streamed rows 2c, 2c + 1 are loaded for
// them, 16 bytes serving four 8-column tiles of the result.  Rows of a tile are multiples of 128 bytes
// with their 16-byte chunks permuted (chunk_at) so that both kinds of load hit every bank once.
//
// Measured, fp32: forward of 2 x 1000 tokens, 16 heads of 64, in packed documents 105 us (137 us with the
// scalar tiles); forward of 2 x 2048 tokens, causal, 546 us = 31 TFLOP/s, backward 1.75 ms = 25 TFLOP/s.
// The tensor pipe is busy for a third of the time: splitting operands and waiting for one product after
// another in few warps take the rest.
#pragma once

#include "attn_common.cuh"

namespace dlb {

constexpr int kGenThreads = 256, kGenCols = 64;  // threads; rows of a streamed tile

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// hi: x rounded to the 11 bits of tf32 (so that lo, exact, has either sign and errors average out); lo:
// the rest, cut to 11 bits where it is used.
__device__ __forceinline__ void split(float x, uint32_t &hi, uint32_t &lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}

template <int N>
struct Split {
  uint32_t hi[N], lo[N];
  Split() = default;
  __device__ __forceinline__ Split(const float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) split(x[i], hi[i], lo[i]);
  }
};

// d[t] += a b[t], b[t] the pair (b[2t], b[2t + 1]): the same term of all tiles side by side, so that a
// product seldom waits for the one before it on the same accumulator.
template <int N>
__device__ __forceinline__ void mma_3(float (&d)[N][4], const Split<4> &a, const float (&b)[2 * N]) {
  const Split<2 * N> s(b);
#pragma unroll
  for (int t = 0; t < N; t++) mma_tf32(d[t], a.lo, s.hi[2 * t], s.hi[2 * t + 1]);
#pragma unroll
  for (int t = 0; t < N; t++) mma_tf32(d[t], a.hi, s.lo[2 * t], s.lo[2 * t + 1]);
#pragma unroll
  for (int t = 0; t < N; t++) mma_tf32(d[t], a.hi, s.hi[2 * t], s.hi[2 * t + 1]);
}

// Place of 16-byte chunk `chunk` of row `row` in a tile with DP columns.
template <int DP>
__device__ __forceinline__ int chunk_at(int row, int chunk) {
  return row * DP + (chunk ^ ((row & 6) ^ ((row & 1) << 2))) * 4;
}

__device__ __forceinline__ void copy16_async(float *dst, const void *src, bool valid) {
  const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(dst)), bytes = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// Tile row r -> source row address; rows at or beyond `rows` and columns beyond `dim` read as zero.  fp32
// rows on 16-byte boundaries are copied asynchronously: the caller commits and waits.
template <typename T, int DP, typename RowPtr>
__device__ __forceinline__ void gen_load_tile(float *dst, int tile_rows, int rows, int dim, bool vec, RowPtr row_ptr) {
  constexpr int V = Store<T>::kPerVec;
  if (vec) {
    constexpr int per_row = DP / V;
    for (int e = threadIdx.x; e < tile_rows * per_row; e += kGenThreads) {
      const int r = e / per_row, c = (e % per_row) * V;
      const bool valid = r < rows && c < dim;
      if constexpr (V == 4) {
        copy16_async(dst + chunk_at<DP>(r, c / 4), valid ? row_ptr(r) + c : row_ptr(0), valid);
      } else {
        float f[V];
#pragma unroll
        for (int i = 0; i < V; i++) f[i] = 0.f;
        if (valid) Store<T>::unpack(ld_keep(row_ptr(r) + c), f);
#pragma unroll
        for (int i = 0; i < V; i += 4)
          *reinterpret_cast<float4 *>(dst + chunk_at<DP>(r, (c + i) / 4)) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
      }
    }
  } else {
    for (int e = threadIdx.x; e < tile_rows * DP; e += kGenThreads) {
      const int r = e / DP, c = e % DP;
      dst[chunk_at<DP>(r, c / 4) + c % 4] = (r < rows && c < dim) ? Store<T>::to_float(ld_co(row_ptr(r) + c)) : 0.f;
    }
  }
}

// out[t] = <rows x0 + g and x0 + g + 8 of x, row u0 + 8t + n of u> over `dim` columns.
template <int DP, int NT>
__device__ __forceinline__ void gen_dot(float (&out)[NT][4], const float *x, int x0, const float *u, int u0, int dim, int lane) {
  const int g = lane >> 2, c = lane & 3;
  float odd[NT][4];  // the second step of every 16 columns has sums of its own: shorter chains
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int e = 0; e < 4; e++) out[t][e] = odd[t][e] = 0.f;
  for (int d = 0; d < dim; d += 16) {
    const float4 p = *reinterpret_cast<const float4 *>(x + chunk_at<DP>(x0 + g, d / 4 + c));
    const float4 q = *reinterpret_cast<const float4 *>(x + chunk_at<DP>(x0 + g + 8, d / 4 + c));
    float b0[2 * NT], b1[2 * NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const float4 v = *reinterpret_cast<const float4 *>(u + chunk_at<DP>(u0 + 8 * t + g, d / 4 + c));
      b0[2 * t] = v.x;
      b0[2 * t + 1] = v.y;
      b1[2 * t] = v.z;
      b1[2 * t + 1] = v.w;
    }
    const Split<4> a0({p.x, q.x, p.y, q.y}), a1({p.z, q.z, p.w, q.w});
    const Split<2 * NT> s0(b0), s1(b1);
    // the same term of all sums side by side, as in mma_3
#pragma unroll
    for (int t = 0; t < NT; t++) {
      mma_tf32(out[t], a0.lo, s0.hi[2 * t], s0.hi[2 * t + 1]);
      mma_tf32(odd[t], a1.lo, s1.hi[2 * t], s1.hi[2 * t + 1]);
    }
#pragma unroll
    for (int t = 0; t < NT; t++) {
      mma_tf32(out[t], a0.hi, s0.lo[2 * t], s0.lo[2 * t + 1]);
      mma_tf32(odd[t], a1.hi, s1.lo[2 * t], s1.lo[2 * t + 1]);
    }
#pragma unroll
    for (int t = 0; t < NT; t++) {
      mma_tf32(out[t], a0.hi, s0.hi[2 * t], s0.hi[2 * t + 1]);
      mma_tf32(odd[t], a1.hi, s1.hi[2 * t], s1.hi[2 * t + 1]);
    }
  }
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int e = 0; e < 4; e++) out[t][e] += odd[t][e];
}

// acc[q][k] += w[t] . u rows u0 + 8t..: w as gen_dot left it.  acc[q][k], lane (g, c): rows g, g + 8 of
// columns 32q + 8c + k and 32q + 8c + 4 + k.  A tile's contribution is summed by itself and added to acc
// with a rounded addition: the tensor cores cut their sums off, and over a long row of tiles that adds
// up to a bias (1.3e-6 of dk over 1554 rows, against 4e-7 this way).
template <int DP, int NT>
__device__ __forceinline__ void gen_accumulate(float (&acc)[DP / 32][4][4], const float (&w)[NT][4], const float *u, int u0,
                                               int lane) {
  const int g = lane >> 2, c = lane & 3;
  Split<4> a[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) a[t] = Split<4>({w[t][0], w[t][2], w[t][1], w[t][3]});
#pragma unroll
  for (int q = 0; q < DP / 32; q++) {
    float sum[4][4] = {};
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int r = u0 + 8 * t + 2 * c;
      const float4 v0 = *reinterpret_cast<const float4 *>(u + chunk_at<DP>(r, 8 * q + g));
      const float4 v1 = *reinterpret_cast<const float4 *>(u + chunk_at<DP>(r + 1, 8 * q + g));
      mma_3<4>(sum, a[t], {v0.x, v1.x, v0.y, v1.y, v0.z, v1.z, v0.w, v1.w});
    }
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc[q][k][e] += sum[k][e];
  }
}

// Writes the lane's part of a 16-row result (times by[0] for row g, by[1] for row g + 8) to rows r0.. of
// a plain [rows][DP] buffer.
template <int DP>
__device__ __forceinline__ void gen_store_acc(float *dst, int r0, const float (&acc)[DP / 32][4][4], int lane) {
  const int g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int q = 0; q < DP / 32; q++)
#pragma unroll
    for (int x = 0; x < 2; x++) {
      float *row = dst + (r0 + g + 8 * x) * DP + 32 * q + 8 * c;
      *reinterpret_cast<float4 *>(row) = make_float4(acc[q][0][2 * x], acc[q][1][2 * x], acc[q][2][2 * x], acc[q][3][2 * x]);
      *reinterpret_cast<float4 *>(row + 4) =
          make_float4(acc[q][0][2 * x + 1], acc[q][1][2 * x + 1], acc[q][2][2 * x + 1], acc[q][3][2 * x + 1]);
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

__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// The next tile is copied while one is worked on, where two CTAs with two buffers each fit an SM; wider
// heads have one buffer, and the other CTA of the SM to fill the time.
template <int DP>
constexpr int kGenBuffers = DP <= 64 ? 2 : 1;
template <int DP, int RG>
constexpr size_t gen_fwd_smem() {
  return sizeof(float) * (16 * RG + kGenBuffers<DP> * 2 * kGenCols) * DP;
}

// Forward.  Tile rows are (query, head) pairs: with `pack` = group a tile holds 16 RG / group queries of
// all heads that share a key/value head (few queries: the cache is read once for the group), with
// pack = 1 it holds 16 RG queries of one head.  blockIdx.y is a share of the key tiles; with more than
// one share the partial results go to part_o / part_ml for attn_join_kernel.
template <typename T, int DP, int RG>
static __global__ void __launch_bounds__(kGenThreads, 2)
attn_fwd_generic_kernel(const __grid_constant__ AttnArgs a, int pack, bool vec) {
  pdl_prologue();
  extern __shared__ __align__(16) float gen_smem[];
  constexpr int kRows = 16 * RG, CG = 8 / RG, NT = RG;
  constexpr int NBUF = kGenBuffers<DP>, kSlab = kGenCols * DP;
  float *qs = gen_smem, *ring = qs + kRows * DP;  // then K and V tiles, in turn
  __shared__ int doc_tiles[2][kGenCols];
  __shared__ float m_s[CG][kRows], l_s[CG][kRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int r0 = (warp % RG) * 16, cg = warp / RG, c0 = cg * 8 * NT;  // this warp's rows and columns
  const int units = a.heads / pack;  // head, or key/value head when packed
  const int q_rows = a.q_len * pack, tiles = (q_rows + kRows - 1) / kRows;
  const int tile = tiles - 1 - static_cast<int>(blockIdx.x % tiles);  // long causal rows start first
  const int unit = (blockIdx.x / tiles) % units, b = blockIdx.x / (tiles * units);
  const int row0 = tile * kRows, rows = min(kRows, q_rows - row0);
  const int hk = pack > 1 ? unit : unit / a.group, h0 = pack > 1 ? unit * pack : unit;
  const BatchView view = batch_view(a, b);

  const T *qb = static_cast<const T *>(a.q.ptr) + b * a.q.batch + h0 * a.q.head;
  const T *kb = static_cast<const T *>(a.k.ptr) + b * a.k.batch + hk * a.k.head;
  const T *vb = static_cast<const T *>(a.v.ptr) + b * a.v.batch + hk * a.v.head;
  gen_load_tile<T, DP>(qs, kRows, rows, a.dim, vec, [&](int r) {
    const int x = row0 + r;
    return qb + static_cast<long long>(x / pack) * a.q.token + (x % pack) * a.q.head;
  });

  int pos[2], end[2], head[2], doc[2];
  float slope[2];
#pragma unroll
  for (int x = 0; x < 2; x++) {
    const int r = row0 + r0 + g + 8 * x, i = r / pack;
    const bool valid = r < q_rows;
    head[x] = h0 + r % pack;
    pos[x] = view.start + i;
    end[x] = valid ? row_end(a, view, i) : 0;
    doc[x] = (a.q_docs && valid) ? a.q_docs[static_cast<long long>(b) * a.q_len + i] : 0;
    slope[x] = (a.slopes && valid) ? a.slopes[head[x]] * kLog2e : 0.f;
  }
  // row_end never falls with the query: the last row's bound is the tile's.
  const int last = row_end(a, view, (row0 + rows - 1) / pack);
  const int key_tiles = (last + kGenCols - 1) / kGenCols;
  const int share = (key_tiles + a.splits - 1) / a.splits;
  const int t0 = min(key_tiles, static_cast<int>(blockIdx.y) * share), t1 = min(key_tiles, t0 + share);

  float acc[DP / 32][4][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int q = 0; q < DP / 32; q++)
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc[q][k][e] = 0.f;
  // First tile from t on that any row of this one shares a document with; its numbers go to doc_tiles[buf].
  auto next_tile = [&](int t, int buf) {
    if (!a.kv_docs) return t;
    for (; t < t1; t++) {
      const int j0 = t * kGenCols, keys = min(kGenCols, last - j0);
      __syncthreads();
      if (threadIdx.x < keys) doc_tiles[buf][threadIdx.x] = a.kv_docs[static_cast<long long>(b) * a.kv_len + j0 + threadIdx.x];
      __syncthreads();
      bool any = false;
      for (int j = c0 + c; j < min(keys, c0 + 8 * NT); j += 4)
#pragma unroll
        for (int x = 0; x < 2; x++) any |= (j0 + j < end[x]) && doc[x] == doc_tiles[buf][j];
      if (__syncthreads_or(any)) break;
    }
    return t;
  };
  auto load = [&](int t, int buf) {
    const int j0 = t * kGenCols, keys = min(kGenCols, last - j0);
    float *k = ring + buf * 2 * kSlab;
    gen_load_tile<T, DP>(k, kGenCols, keys, a.dim, vec, [&](int r) { return kb + static_cast<long long>(j0 + r) * a.k.token; });
    gen_load_tile<T, DP>(k + kSlab, kGenCols, keys, a.dim, vec, [&](int r) { return vb + static_cast<long long>(j0 + r) * a.v.token; });
  };
  int t = next_tile(t0, 0), buf = 0;
  if (NBUF == 2 && t < t1) load(t, 0);
  async_commit();
  while (t < t1) {
    int next = t1;
    if (NBUF == 2) {
      next = next_tile(t + 1, buf ^ 1);
      if (next < t1) load(next, buf ^ 1);
      async_commit();
      async_wait<1>();
    } else {
      load(t, 0);
      async_commit();
      async_wait<0>();
    }
    __syncthreads();
    const int j0 = t * kGenCols;
    const float *ks = ring + (NBUF == 2 ? buf : 0) * 2 * kSlab, *vs = ks + kSlab;
    const int *doc_tile = doc_tiles[NBUF == 2 ? buf : 0];
    float s[NT][4];
    gen_dot<DP, NT>(s, qs, r0, ks, c0, a.dim, lane);
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int x = e >> 1, col = c0 + 8 * n + 2 * c + (e & 1), j = j0 + col;
        bool seen = j < end[x];
        if (a.kv_docs) seen = seen && doc_tile[col] == doc[x];
        float unused;
        s[n][e] = seen ? gen_score(a, s[n][e], head[x], slope[x], j - pos[x], &unused) : -INFINITY;
        top[x] = fmaxf(top[x], s[n][e]);
      }
    float keep[2], base[2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
      top[x] = fmaxf(m[x], quad_max(top[x]));
      base[x] = top[x] == -INFINITY ? 0.f : top[x];
      keep[x] = ex2(m[x] - base[x]);
      m[x] = top[x];
      l[x] *= keep[x];
    }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        s[n][e] = ex2(s[n][e] - base[e >> 1]);
        l[e >> 1] += s[n][e];
      }
#pragma unroll
    for (int q = 0; q < DP / 32; q++)
#pragma unroll
      for (int k = 0; k < 4; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[q][k][e] *= keep[e >> 1];
    gen_accumulate<DP, NT>(acc, s, vs, c0, lane);
    __syncthreads();
    if (NBUF == 2) buf ^= 1;
    else next = next_tile(t + 1, 0);
    t = next;
  }
  // Join of the column groups, through the place of the K and V tiles: [column group][row][column].
  async_wait<0>();
  __syncthreads();
  float *ks = ring;
  gen_store_acc<DP>(ks, cg * kRows + r0, acc, lane);
#pragma unroll
  for (int x = 0; x < 2; x++) {
    l[x] = quad_sum(l[x]);
    if (c == 0) {
      m_s[cg][r0 + g + 8 * x] = m[x];
      l_s[cg][r0 + g + 8 * x] = l[x];
    }
  }
  __syncthreads();
  constexpr int kPer = kGenThreads / kRows;  // threads of a row
  const int r = threadIdx.x / kPer, part = threadIdx.x % kPer, x = row0 + r;
  if (x >= q_rows) return;
  float all = -INFINITY, total = 0.f, weight[CG];
#pragma unroll
  for (int k = 0; k < CG; k++) all = fmaxf(all, m_s[k][r]);
#pragma unroll
  for (int k = 0; k < CG; k++) {
    weight[k] = ex2(m_s[k][r] - (all == -INFINITY ? 0.f : all));
    total = fmaf(weight[k], l_s[k][r], total);
  }
  const int i = x / pack, h = h0 + x % pack;
  const size_t row = (static_cast<size_t>(b) * a.heads + h) * a.q_len + i;
  const bool whole = a.splits == 1;
  const size_t at = static_cast<size_t>(blockIdx.y) * a.batch * a.heads * a.q_len + row;
  const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
  T *out = static_cast<T *>(a.o.ptr) + b * a.o.batch + static_cast<long long>(i) * a.o.token + h * a.o.head;
  for (int col = part; col < a.dim; col += kPer) {
    float o = 0.f;
#pragma unroll
    for (int k = 0; k < CG; k++) o = fmaf(weight[k], ks[(k * kRows + r) * DP + col], o);
    if (whole) out[col] = Store<T>::from_float(o * inv);
    else a.part_o[at * a.dim + col] = o;
  }
  if (part == 0) {
    if (!whole) a.part_ml[at] = make_float2(all, total);
    else if (a.lse) a.lse[row] = total == 0.f ? -INFINITY : (all + log2f(total)) * kLn2;
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

// Fills row_stats: -lse * log2(e) and -delta, delta = <dout_i, o_i> (= sum_j P_ij dP_ij; from a bf16 output
// a first guess, see attn_bwd_generic).  A row is taken by LANES lanes with one 16-byte vector of each at a
// time, or by a warp element by element.
template <typename T, int LANES, bool VEC>
static __global__ void __launch_bounds__(256) attn_row_stats_kernel(const __grid_constant__ AttnArgs a) {
  pdl_prologue();
  const int padded = stat_tiles(a.q_len) * kStatRows;
  const size_t rows = static_cast<size_t>(a.batch) * a.heads * padded;
  const size_t row = static_cast<size_t>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
  const int lane = threadIdx.x % LANES;
  const bool there = row < rows;
  // heads innermost: neighbouring rows lie side by side in [token, head] layouts
  const int h = row % a.heads, i = (row / a.heads) % padded, b = row / (static_cast<size_t>(padded) * a.heads);
  float sum = 0.f;
  if (there && i < a.q_len) {
    const T *o = static_cast<const T *>(a.o.ptr) + b * a.o.batch + i * a.o.token + h * a.o.head;
    const T *g = static_cast<const T *>(a.dout.ptr) + b * a.dout.batch + i * a.dout.token + h * a.dout.head;
    if constexpr (VEC) {
      constexpr int V = Store<T>::kPerVec;
      for (int c = lane * V; c < a.dim; c += LANES * V) {
        float x[V], y[V];
        Store<T>::unpack(ld_keep(o + c), x);
        Store<T>::unpack(ld_keep(g + c), y);
#pragma unroll
        for (int e = 0; e < V; e++) sum = fmaf(x[e], y[e], sum);
      }
    } else {
      for (int c = lane; c < a.dim; c += LANES) sum = fmaf(Store<T>::to_float(ld_co(o + c)), Store<T>::to_float(ld_co(g + c)), sum);
    }
  }
#pragma unroll
  for (int k = LANES / 2; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
  if (there && lane == 0) {
    float *at = stats_tile(a, b, h, i / kStatRows) + i % kStatRows;
    at[0] = i < a.q_len ? -a.lse[(static_cast<size_t>(b) * a.heads + h) * a.q_len + i] * kLog2e : -INFINITY;
    if (i < a.q_len && at[0] == INFINITY) at[0] = -INFINITY;  // lse = -infinity
    at[kStatRows] = -sum;
  }
}

// Bytes behind the tiles that the sums for the table take: scores' gradients and probabilities of a tile,
// their sums per bucket and row in two halves of the columns, the bucket of every distance.
template <int RG>
__host__ __device__ inline size_t gen_table_bytes(const AttnArgs &a) {
  return a.dtable ? sizeof(float) * 2 * 16 * RG * (kGenCols + 1) + sizeof(float2) * 2 * a.buckets * 16 * RG +
                        (2 * a.reach + 1 + 15) / 16 * 16
                  : 0;
}
template <int DP, int RG>
constexpr int kBwdBuffers = DP == 128 && RG == 4 ? 1 : 2;  // what fits
template <int DP, int RG>
constexpr size_t gen_bwd_smem() {
  return sizeof(float) * (2 * 16 * RG + kBwdBuffers<DP, RG> * 2 * kGenCols) * DP;
}

// Backward.  16 RG rows stay (keys and values when FOR_KEYS, else queries and output gradients), the
// other side streams by in tiles of 64 rows:
//   P = exp2(s - lse), dS = P (dP - delta);  FOR_KEYS: dV += P^T dO, dK += dS^T Q over the heads of
// the group, else dQ += dS K.  Each pass rebuilds the scores, so no sum crosses a CTA.
// With bf16 storage delta comes from a rounded output; a row's dS add up to what that is off by, e, and the
// query pass takes e sum_j P_j k_j off dQ again and leaves delta + e to the key pass, a launch of its own
// then (attn_bwd_mma.cuh tells more).
template <typename T, int DP, int RG, bool FOR_KEYS>
__device__ __forceinline__ void attn_bwd_generic(const AttnArgs &a, bool vec, int block) {
  extern __shared__ __align__(16) float gen_smem[];
  constexpr int kRows = 16 * RG, CG = 8 / RG, NT = RG, kPitch = kGenCols + 1;
  constexpr int NBUF = kBwdBuffers<DP, RG>, kSlab = kGenCols * DP;
  float *xs = gen_smem, *ys = xs + kRows * DP, *ring = ys + kRows * DP;  // then U and W tiles, in turn
  float *ds_tile = ring + NBUF * 2 * kSlab, *p_tile = ds_tile + kRows * kPitch;                      // [row][column]
  float2 *sums = reinterpret_cast<float2 *>(p_tile + kRows * kPitch);                           // [half][bucket][row]
  unsigned char *bucket_lut = reinterpret_cast<unsigned char *>(sums + 2 * a.buckets * kRows);  // by distance
  __shared__ float2 col_stat_tiles[2][kGenCols];
  __shared__ int col_doc_tiles[2][kGenCols];
  constexpr bool kFixDelta = !FOR_KEYS && sizeof(T) == 2;
  __shared__ float2 row_sums[CG][kRows];
  const bool want_table = !FOR_KEYS && a.dtable != nullptr;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int r0 = (warp % RG) * 16, cg = warp / RG, w0 = cg * 8 * NT;  // this warp's rows and columns
  const int len = FOR_KEYS ? a.kv_len : a.q_len, units = FOR_KEYS ? a.kv_heads : a.heads;
  const int tiles = (len + kRows - 1) / kRows;
  int tile = block % tiles;
  if (!FOR_KEYS) tile = tiles - 1 - tile;  // long causal rows first
  const int unit = (block / tiles) % units, b = block / (tiles * units);
  const int row0 = tile * kRows, rows = min(kRows, len - row0);
  const int hk = FOR_KEYS ? unit : unit / a.group;
  const BatchView view = batch_view(a, b);
  const int bound = FOR_KEYS ? min(rows, max(0, view.end - row0)) : rows;  // rows that hold numbers

  const T *kb = static_cast<const T *>(a.k.ptr) + b * a.k.batch + hk * a.k.head;
  const T *vb = static_cast<const T *>(a.v.ptr) + b * a.v.batch + hk * a.v.head;
  const T *q_all = static_cast<const T *>(a.q.ptr) + b * a.q.batch;
  const T *g_all = static_cast<const T *>(a.dout.ptr) + b * a.dout.batch;
  if (FOR_KEYS) {
    gen_load_tile<T, DP>(xs, kRows, bound, a.dim, vec, [&](int r) { return kb + static_cast<long long>(row0 + r) * a.k.token; });
    gen_load_tile<T, DP>(ys, kRows, bound, a.dim, vec, [&](int r) { return vb + static_cast<long long>(row0 + r) * a.v.token; });
  } else {
    gen_load_tile<T, DP>(xs, kRows, rows, a.dim, vec,
                         [&](int r) { return q_all + unit * a.q.head + static_cast<long long>(row0 + r) * a.q.token; });
    gen_load_tile<T, DP>(ys, kRows, rows, a.dim, vec,
                         [&](int r) { return g_all + unit * a.dout.head + static_cast<long long>(row0 + r) * a.dout.token; });
  }
  if (want_table) {
    for (int e = threadIdx.x; e < 2 * a.buckets * kRows; e += kGenThreads) sums[e] = make_float2(0.f, 0.f);
    for (int e = threadIdx.x; e <= 2 * a.reach; e += kGenThreads) bucket_lut[e] = static_cast<unsigned char>(bucket_at(a, e - a.reach));
  }

  int row_doc[2], end[2];
  float2 row_stat[2];
#pragma unroll
  for (int x = 0; x < 2; x++) {
    const int r = r0 + g + 8 * x;
    const bool valid = r < bound;
    const int *docs = FOR_KEYS ? a.kv_docs : a.q_docs;
    row_doc[x] = (docs && valid) ? docs[static_cast<long long>(b) * len + row0 + r] : 0;
    end[x] = (!FOR_KEYS && valid) ? row_end(a, view, row0 + r) : 0;
    row_stat[x] = (!FOR_KEYS && valid) ? stat_at(a, b, unit, row0 + r) : make_float2(-INFINITY, 0.f);
  }
  float acc_x[DP / 32][4][4], acc_y[DP / 32][4][4], ds_sum[2] = {0.f, 0.f}, p_sum[2] = {0.f, 0.f};
#pragma unroll
  for (int q = 0; q < DP / 32; q++)
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc_x[q][k][e] = acc_y[q][k][e] = 0.f;

  const int last = FOR_KEYS ? a.q_len : row_end(a, view, row0 + rows - 1);
  const int t_end = (last + kGenCols - 1) / kGenCols;
  const int first = !FOR_KEYS ? 0 : bound > 0 ? first_query(a, view, row0) / kGenCols : t_end;
  // Steps are numbered over the heads of the group: step n * (t_end - first) + t - first.
  const int per_head = max(0, t_end - first), steps = per_head * (FOR_KEYS ? a.group : 1);
  // First step from `step` on that shares a document; its columns' numbers go to buffer `buf`.
  auto next_step = [&](int step, int buf) {
    for (; step < steps; step++) {
      const int h = FOR_KEYS ? hk * a.group + step / per_head : unit, c0 = (first + step % per_head) * kGenCols;
      const int cols = min(kGenCols, last - c0);
      if (a.kv_docs) __syncthreads();
      if (threadIdx.x < kGenCols) {
        const int k = threadIdx.x;
        const int *docs = FOR_KEYS ? a.q_docs : a.kv_docs;
        col_doc_tiles[buf][k] = (docs && k < cols) ? docs[static_cast<long long>(b) * (FOR_KEYS ? a.q_len : a.kv_len) + c0 + k] : 0;
        if (FOR_KEYS) col_stat_tiles[buf][k] = k < cols ? stat_at(a, b, h, c0 + k) : make_float2(-INFINITY, 0.f);
      }
      if (!a.kv_docs) break;
      __syncthreads();
      bool any = false;
      for (int k = w0 + c; k < min(cols, w0 + 8 * NT); k += 4)
#pragma unroll
        for (int x = 0; x < 2; x++) any |= r0 + g + 8 * x < bound && row_doc[x] == col_doc_tiles[buf][k];
      if (__syncthreads_or(any)) break;
    }
    return step;
  };
  auto load = [&](int step, int buf) {
    const int h = FOR_KEYS ? hk * a.group + step / per_head : unit, c0 = (first + step % per_head) * kGenCols;
    const int cols = min(kGenCols, last - c0);
    float *u = ring + buf * 2 * kSlab, *w = u + kSlab;
    if (FOR_KEYS) {
      gen_load_tile<T, DP>(u, kGenCols, cols, a.dim, vec,
                           [&](int r) { return q_all + h * a.q.head + static_cast<long long>(c0 + r) * a.q.token; });
      gen_load_tile<T, DP>(w, kGenCols, cols, a.dim, vec,
                           [&](int r) { return g_all + h * a.dout.head + static_cast<long long>(c0 + r) * a.dout.token; });
    } else {
      gen_load_tile<T, DP>(u, kGenCols, cols, a.dim, vec, [&](int r) { return kb + static_cast<long long>(c0 + r) * a.k.token; });
      gen_load_tile<T, DP>(w, kGenCols, cols, a.dim, vec, [&](int r) { return vb + static_cast<long long>(c0 + r) * a.v.token; });
    }
  };
  {
    int step = next_step(0, 0), buf = 0;
    if (NBUF == 2 && step < steps) load(step, 0);
    async_commit();
    while (step < steps) {
      int next = steps;
      if (NBUF == 2) {
        next = next_step(step + 1, buf ^ 1);
        if (next < steps) load(next, buf ^ 1);
        async_commit();
        async_wait<1>();
      } else {
        load(step, 0);
        async_commit();
        async_wait<0>();
      }
      __syncthreads();
      const int h = FOR_KEYS ? hk * a.group + step / per_head : unit, c0 = (first + step % per_head) * kGenCols;
      const int cols = min(kGenCols, last - c0);
      const float slope = a.slopes ? a.slopes[h] * kLog2e : 0.f;
      const float *us = ring + (NBUF == 2 ? buf : 0) * 2 * kSlab, *ws = us + kSlab;
      const float2 *col_stats = col_stat_tiles[NBUF == 2 ? buf : 0];
      const int *col_doc = col_doc_tiles[NBUF == 2 ? buf : 0];
      float p[NT][4], d[NT][4];
      gen_dot<DP, NT>(p, xs, r0, us, w0, a.dim, lane);
      gen_dot<DP, NT>(d, ys, r0, ws, w0, a.dim, lane);
#pragma unroll
      for (int k = 0; k < NT; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int x = e >> 1, r = r0 + g + 8 * x, cc = w0 + 8 * k + 2 * c + (e & 1);
          const int i = FOR_KEYS ? c0 + cc : row0 + r, j = FOR_KEYS ? row0 + r : c0 + cc;
          bool seen = FOR_KEYS ? (r < bound && cc < cols && j < row_end(a, view, i)) : j < end[x];
          if (a.kv_docs) seen = seen && row_doc[x] == col_doc[cc];
          const float2 stat = FOR_KEYS ? col_stats[cc] : row_stat[x];
          float dcap, prob = 0.f, grad = 0.f;
          if (seen) {
            prob = ex2(gen_score(a, p[k][e], h, slope, j - (view.start + i), &dcap) + stat.x);
            grad = prob * (d[k][e] + stat.y);
          } else {
            dcap = 0.f;
          }
          if (want_table) {
            ds_tile[r * kPitch + cc] = grad;
            p_tile[r * kPitch + cc] = prob;
          }
          if (kFixDelta) {
            ds_sum[x] += grad;
            p_sum[x] += prob;
          }
          p[k][e] = kFixDelta ? prob * dcap * a.scale : prob;
          d[k][e] = grad * dcap * a.scale;  // through the cap and the scale: the gradient of <q, k>
        }
      if (want_table) {
        __syncthreads();
        if (threadIdx.x < 2 * kRows) {  // a row's half tile per thread, one run of columns per bucket
          const int r = threadIdx.x % kRows, half = threadIdx.x / kRows, k0 = half * (kGenCols / 2);
          float2 *own = sums + half * a.buckets * kRows + r;
          int now = -1;
          float2 run = make_float2(0.f, 0.f);
          for (int k = k0; k < min(cols, k0 + kGenCols / 2); k++) {
            const int bucket = bucket_lut[max(-a.reach, min(a.reach, c0 + k - (view.start + row0 + r))) + a.reach];
            if (bucket != now) {
              if (now >= 0) {
                own[now * kRows].x += run.x;
                own[now * kRows].y += run.y;
              }
              now = bucket;
              run = make_float2(0.f, 0.f);
            }
            run.x += ds_tile[r * kPitch + k];
            run.y += p_tile[r * kPitch + k];
          }
          if (now >= 0) {
            own[now * kRows].x += run.x;
            own[now * kRows].y += run.y;
          }
        }
      }
      if (FOR_KEYS || kFixDelta) gen_accumulate<DP, NT>(acc_y, p, FOR_KEYS ? ws : us, w0, lane);
      gen_accumulate<DP, NT>(acc_x, d, us, w0, lane);
      __syncthreads();
      if (NBUF == 2) buf ^= 1;
      else next = next_step(step + 1, 0);
      step = next;
    }
    async_wait<0>();
  }
  if constexpr (kFixDelta) {
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const float2 sum = make_float2(quad_sum(ds_sum[x]), quad_sum(p_sum[x]));
      if (c == 0) row_sums[cg][r0 + g + 8 * x] = sum;
    }
    __syncthreads();
    float off[2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int k = 0; k < CG; k++) {
        sum.x += row_sums[k][r0 + g + 8 * x].x;
        sum.y += row_sums[k][r0 + g + 8 * x].y;
      }
      off[x] = row_is_whole<T>(a, sum.y, row_stat[x].x) ? sum.x : 0.f;
    }
#pragma unroll
    for (int q = 0; q < DP / 32; q++)
#pragma unroll
      for (int k = 0; k < 4; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc_x[q][k][e] = fmaf(-off[e >> 1], acc_y[q][k][e], acc_x[q][k][e]);
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const int r = r0 + g + 8 * x, i = row0 + r;
      if (c == 0 && cg == 0 && r < rows) stats_tile(a, b, unit, i / kStatRows)[kStatRows + i % kStatRows] = row_stat[x].y - off[x];
    }
  }
  float *us = ring;
  // Join of the column groups, through the place of the streamed tiles: [column group][row][column].
#pragma unroll
  for (int which = 0; which < (FOR_KEYS ? 2 : 1); which++) {
    __syncthreads();
    gen_store_acc<DP>(us, cg * kRows + r0, which ? acc_y : acc_x, lane);
    __syncthreads();
    const Heads &to = which ? a.dv : FOR_KEYS ? a.dk : a.dq;
    T *out = static_cast<T *>(to.ptr) + b * to.batch + unit * to.head;
    for (int e = threadIdx.x; e < rows * DP; e += kGenThreads) {
      const int r = e / DP, col = e % DP;
      if (col >= a.dim) continue;
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < CG; k++) sum += us[(k * kRows + r) * DP + col];
      out[static_cast<long long>(row0 + r) * to.token + col] = Store<T>::from_float(sum);
    }
  }
  if (want_table) {
    __syncthreads();
    if (threadIdx.x < kRows) {
      // The gradients of a whole row's scores add up to zero: what rounding left (in delta above all) is
      // taken off again in proportion to P.
      const int r = threadIdx.x;
      float e = 0.f, total = 0.f;
      for (int n = 0; n < a.buckets; n++) {
        float2 v = sums[n * kRows + r];
        const float2 other = sums[(a.buckets + n) * kRows + r];
        v.x += other.x;
        v.y += other.y;
        sums[n * kRows + r] = v;
        e += v.x;
        total += v.y;
      }
      e = r < rows && row_is_whole<T>(a, total, stat_at(a, b, unit, row0 + r).x) ? e / total : 0.f;
      for (int n = 0; n < a.buckets; n++) sums[n * kRows + r].x -= e * sums[n * kRows + r].y;
    }
    __syncthreads();
    float *part = a.table_part + (static_cast<size_t>(unit) * a.table_parts + b * tiles + tile) * a.buckets;
    for (int n = warp; n < a.buckets; n += kGenThreads / 32) {
      float sum = 0.f;
      for (int r = lane; r < kRows; r += 32) sum += sums[n * kRows + r].x;
      sum = warp_sum(sum);
      if (lane == 0) part[n] = sum;
    }
  }
}

// Both passes in one launch, or one of them: the first key_blocks CTAs make dK and dV, the others dQ and the
// table's parts.
template <typename T, int DP, int RG>
static __global__ void __launch_bounds__(kGenThreads, DP <= 64 ? 2 : 1)
attn_bwd_generic_kernel(const __grid_constant__ AttnArgs a, bool vec, int key_blocks) {
  pdl_prologue();
  if (static_cast<int>(blockIdx.x) < key_blocks) attn_bwd_generic<T, DP, RG, true>(a, vec, blockIdx.x);
  else attn_bwd_generic<T, DP, RG, false>(a, vec, blockIdx.x - key_blocks);
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
