// Attention of a few queries against a long cache (bf16): bound by reading K and V once.
//
// The queries of all heads that share a key/value head are the 16 rows of warp-level matrix products
// (mma.sync m16n8k16: with this few rows the products are free and the tensor memory of tcgen05, with
// its 128 lanes, would stand empty).  Nothing is staged in shared memory: a product's inner index may
// run in any order, so each lane loads 16 adjacent bytes of a K row and of the Q row and uses them as
// the fragments of two steps, and 16 adjacent bytes of V rows become the fragments of eight column
// tiles by byte permutations.  Every lane has its 16 loads of 16 keys in flight at once.
//
// The keys are split over CTAs (blockIdx.y) until the GPU is full several times, so that sequences of
// different lengths even out; the four warps of a CTA take every fourth 16 keys and are joined in
// shared memory, the CTAs by attn_join_kernel.
#include <algorithm>

#include "attn_mma.cuh"
#include "attn_step.cuh"

namespace dlb {
namespace {

constexpr int kStepWarps = 4, kStepThreads = 32 * kStepWarps, kStepRows = 16, kStepKeys = 16;

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// Word x of a 16-byte vector (x is a compile-time constant where this is used).
__device__ __forceinline__ uint32_t word(const uint4 &v, int x) { return x == 0 ? v.x : x == 1 ? v.y : x == 2 ? v.z : v.w; }

template <int NT>  // head_dim up to 32 * NT
__global__ void __launch_bounds__(kStepThreads, 3) attn_step_kernel(const __grid_constant__ AttnArgs a) {
  pdl_prologue();
  constexpr int NB = (NT + 1) / 2;  // blocks of 64 columns of V and O
  constexpr int W = NB * 64;
  __shared__ float out_s[kStepWarps][kStepRows][W + 4];
  __shared__ float m_s[kStepWarps][kStepRows], l_s[kStepWarps][kStepRows], r_s[kStepWarps][kStepRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int rows = a.q_len * a.group, row_tiles = (rows + kStepRows - 1) / kStepRows;
  const int tile = blockIdx.x % row_tiles, hk = (blockIdx.x / row_tiles) % a.kv_heads, b = blockIdx.x / (row_tiles * a.kv_heads);
  const BatchView view = batch_view(a, b);
  const int row_last = min(rows, (tile + 1) * kStepRows) - 1;
  const int last = row_end(a, view, row_last / a.group);  // row_end never falls with the query
  // this CTA's share of the keys, in multiples of what its warps take in one turn
  const int turn = kStepWarps * kStepKeys, turns = (last + turn - 1) / turn;
  const int share = (turns + a.splits - 1) / a.splits * turn;
  const int s0 = min(static_cast<long long>(last), static_cast<long long>(blockIdx.y) * share), s1 = min(last, s0 + share);

  int pos[2], end[2], head[2], doc[2];
  float slope[2], far_left[2];
  uint4 q[2][NT];
#pragma unroll
  for (int x = 0; x < 2; x++) {
    const int r = tile * kStepRows + g + 8 * x, i = r / a.group;
    const bool valid = r < rows;
    head[x] = hk * a.group + r % a.group;
    pos[x] = view.start + i;
    end[x] = valid ? row_end(a, view, i) : 0;
    doc[x] = (a.q_docs && valid) ? ld_co(a.q_docs + static_cast<long long>(b) * a.q_len + i) : 0;
    slope[x] = (a.slopes && valid) ? ld_co(a.slopes + head[x]) * kLog2e : 0.f;
    far_left[x] = (a.table && valid) ? table_entry(a, head[x], bucket_at(a, -a.reach)) : 0.f;
    const __nv_bfloat16 *src = static_cast<const __nv_bfloat16 *>(a.q.ptr) + b * a.q.batch + static_cast<long long>(i) * a.q.token +
                               head[x] * a.q.head;
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int col = (4 * t + c) * 8;
      q[x][t] = valid && col < a.dim ? ld_keep(src + col) : make_uint4(0, 0, 0, 0);
    }
  }
  const __nv_bfloat16 *kb = static_cast<const __nv_bfloat16 *>(a.k.ptr) + b * a.k.batch + hk * a.k.head;
  const __nv_bfloat16 *vb = static_cast<const __nv_bfloat16 *>(a.v.ptr) + b * a.v.batch + hk * a.v.head;
  const float inside = a.cap > 0.f ? a.scale / a.cap : 0.f, to_log2 = (a.cap > 0.f ? a.cap : a.scale) * kLog2e;
  const int far_to = min(view.start + (tile * kStepRows) / a.group, INT_MAX / 2) - a.reach;  // keys up to here are far left of all rows

  float acc[NB][8][4], m[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f}, sum_rounded[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < NB; n++)
#pragma unroll
    for (int t = 0; t < 8; t++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc[n][t][e] = 0.f;

  for (int j0 = s0 + warp * kStepKeys; j0 < s1; j0 += turn) {
    uint4 k[2][NT], v[NB][4];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int j = j0 + 8 * u + g;
      const __nv_bfloat16 *src = kb + static_cast<long long>(j) * a.k.token;
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const int col = (4 * t + c) * 8;
        k[u][t] = j < s1 && col < a.dim ? ld_stream(src + col) : make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int x = 0; x < 4; x++) {
        const int j = j0 + 2 * c + (x & 1) + 8 * (x >> 1), col = n * 64 + g * 8;
        v[n][x] = j < s1 && col < a.dim ? ld_stream(vb + static_cast<long long>(j) * a.v.token + col) : make_uint4(0, 0, 0, 0);
      }
    float s[2][4];  // [key tile][row g: keys 2c, 2c + 1; row g + 8: the same]
#pragma unroll
    for (int u = 0; u < 2; u++) {
#pragma unroll
      for (int e = 0; e < 4; e++) s[u][e] = 0.f;
#pragma unroll
      for (int t = 0; t < NT; t++) {
        mma16816(s[u], q[0][t].x, q[1][t].x, q[0][t].y, q[1][t].y, k[u][t].x, k[u][t].y);
        mma16816(s[u], q[0][t].z, q[1][t].z, q[0][t].w, q[1][t].w, k[u][t].z, k[u][t].w);
      }
    }
    const bool all_far = j0 + kStepKeys - 1 <= far_to;
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int x = e >> 1, j = j0 + 8 * u + 2 * c + (e & 1), d = j - pos[x];
        float y = s[u][e];
        if (a.cap > 0.f) y = tanh_score(y * inside);
        y *= to_log2;
        if (a.slopes) y = fmaf(-slope[x], static_cast<float>(abs(d)), y);
        if (a.table) y += all_far ? far_left[x] : table_entry(a, head[x], bucket_at(a, d));
        bool seen = j < end[x] && j < s1;
        if (a.kv_docs) seen = seen && ld_co(a.kv_docs + static_cast<long long>(b) * a.kv_len + j) == doc[x];
        s[u][e] = seen ? y : -INFINITY;
        top[x] = fmaxf(top[x], s[u][e]);
      }
    bool grow[2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
      top[x] = quad_max(top[x]);
      grow[x] = top[x] > m[x] + 8.f;
    }
    if (__any_sync(0xffffffffu, grow[0] || grow[1])) {
      float keep[2];
#pragma unroll
      for (int x = 0; x < 2; x++) {
        keep[x] = grow[x] ? ex2(m[x] - top[x]) : 1.f;
        if (grow[x]) m[x] = top[x];
        sum[x] *= keep[x];
        sum_rounded[x] *= keep[x];
      }
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int t = 0; t < 8; t++)
#pragma unroll
          for (int e = 0; e < 4; e++) acc[n][t][e] *= keep[e >> 1];
    }
    uint32_t p[2][2];  // [key tile][row]
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const float base = m[x] == -INFINITY ? 0.f : m[x];
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const float p0 = ex2(s[u][2 * x] - base), p1 = ex2(s[u][2 * x + 1] - base);
        p[u][x] = pack_bf16(p0, p1);
        sum[x] += p0 + p1;
        sum_rounded[x] += __uint_as_float(p[u][x] << 16) + __uint_as_float(p[u][x] & 0xffff0000u);
      }
    }
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int t = 0; t < 8; t++) {
        // column 64 n + 8 g + t of keys (2c, 2c + 1) and (2c + 8, 2c + 9)
        const uint32_t pick = t & 1 ? 0x7632 : 0x5410;
        const uint32_t b0 = __byte_perm(word(v[n][0], t / 2), word(v[n][1], t / 2), pick);
        const uint32_t b1 = __byte_perm(word(v[n][2], t / 2), word(v[n][3], t / 2), pick);
        mma16816(acc[n][t], p[0][0], p[0][1], p[1][0], p[1][1], b0, b1);
      }
  }
#pragma unroll
  for (int x = 0; x < 2; x++) {
    sum[x] = quad_sum(sum[x]);
    sum_rounded[x] = quad_sum(sum_rounded[x]);
    if (c == 0) {
      m_s[warp][g + 8 * x] = m[x];
      l_s[warp][g + 8 * x] = sum[x];
      r_s[warp][g + 8 * x] = sum_rounded[x];
    }
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int half = 0; half < 2; half++)  // columns 64 n + 16 c + 8 half + 0..7
#pragma unroll
        for (int t = 0; t < 8; t += 4)
          *reinterpret_cast<float4 *>(&out_s[warp][g + 8 * x][n * 64 + 16 * c + 8 * half + t]) =
              make_float4(acc[n][t][2 * x + half], acc[n][t + 1][2 * x + half], acc[n][t + 2][2 * x + half], acc[n][t + 3][2 * x + half]);
  }
  __syncthreads();
  // Join of the four warps: eight threads a row.
  const int r = threadIdx.x / 8, part = threadIdx.x % 8, rr = tile * kStepRows + r;
  if (rr >= rows) return;
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kStepWarps; w++) top = fmaxf(top, m_s[w][r]);
  const float base = top == -INFINITY ? 0.f : top;
  float weight[kStepWarps], l = 0.f, rounded = 0.f;
#pragma unroll
  for (int w = 0; w < kStepWarps; w++) {
    weight[w] = ex2(m_s[w][r] - base);
    l += weight[w] * l_s[w][r];
    rounded += weight[w] * r_s[w][r];
  }
  const int i = rr / a.group, h = hk * a.group + rr % a.group;
  const size_t row = (static_cast<size_t>(b) * a.heads + h) * a.q_len + i;
  const bool whole = a.splits == 1;
  // A share's output is kept for a quotient by the unrounded sum, which the join uses.
  const float to = rounded > 0.f || rounded != rounded ? (whole ? 1.f / rounded : l / rounded) : 0.f;
  const size_t at = static_cast<size_t>(blockIdx.y) * a.batch * a.heads * a.q_len + row;
  __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(a.o.ptr) + b * a.o.batch + static_cast<long long>(i) * a.o.token + h * a.o.head;
  for (int col = part * 8; col < a.dim; col += 64) {
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      o[e] = 0.f;
#pragma unroll
      for (int w = 0; w < kStepWarps; w++) o[e] = fmaf(weight[w], out_s[w][r][col + e], o[e]);
      o[e] *= to;
    }
    if (whole) {
      *reinterpret_cast<uint4 *>(out + col) = Store<__nv_bfloat16>::pack(o);
    } else {
      float4 *dst = reinterpret_cast<float4 *>(a.part_o + at * a.dim + col);
      dst[0] = make_float4(o[0], o[1], o[2], o[3]);
      dst[1] = make_float4(o[4], o[5], o[6], o[7]);
    }
  }
  if (part == 0) {
    if (!whole) a.part_ml[at] = make_float2(top, l);
    else if (a.lse) a.lse[row] = l == 0.f ? -INFINITY : (top + log2f(l)) * kLn2;
  }
}

}  // namespace

int attn_step_splits(int batch, int kv_heads, int rows, int kv_len) {
  // Three CTAs fit an SM; six times that many even out sequences of different lengths (64 users with
  // 4096 to 8192 keys: see the measurements beside the kernel), but a share keeps 256 keys.
  const long long ctas = static_cast<long long>(batch) * kv_heads * ceil_div(rows, kStepRows);
  const long long want = ceil_div(18ll * sm_count(), std::max(1ll, ctas));
  return static_cast<int>(std::max(1ll, std::min({want, static_cast<long long>(kv_len / 256), 256ll})));
}

int attn_step(const AttnArgs &a, cudaStream_t st) {
  const int rows = a.q_len * a.group;
  const dim3 grid(ceil_div(rows, kStepRows) * a.kv_heads * a.batch, a.splits);
  const int nt = ceil_div(a.dim, 32);
  auto kern = nt == 1 ? attn_step_kernel<1> : nt == 2 ? attn_step_kernel<2> : nt == 3 ? attn_step_kernel<3> : attn_step_kernel<4>;
  launch_pdl(kern, grid, dim3(kStepThreads), 0, st, a);
  DLB_LAUNCH_CHECK("attn_step");
  return DLB_OK;
}

}  // namespace dlb
