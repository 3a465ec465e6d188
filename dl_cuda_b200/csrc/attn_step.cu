// Attention of a few queries against a long cache (bf16): bound by reading K and V once.
//
// The queries of all heads that share a key/value head are the columns, 8 or 16, of warp-level matrix
// products (mma.sync m16n8k16: with this few the products are free, and the tensor memory of tcgen05,
// with its 128 lanes, would stand empty): S^T = K Q^T over 16 keys, O^T += V^T P^T over those keys.
// Nothing is staged in shared memory: a product's inner index may run in any order, so a lane loads 16
// adjacent bytes of a K row, and of the Q row, and uses them as the fragments of two steps; 16 adjacent
// bytes of four V rows become the fragments of four 16-column tiles by byte permutations.  Every lane
// has its 16 loads for 16 keys in flight at once.
//
// Probabilities are rounded to bf16 for O^T += V^T P^T, as in the forward of whole sequences, and the
// quotient's sum adds the rounded ones (1.8e-3 to 2.4e-3 from the exact output, of which its own rounding
// is 1.7e-3).
//
// The keys are split over CTAs (blockIdx.y) until the GPU is full several times, so that sequences of
// different lengths even out; the four warps of a CTA take every fourth 16 keys and are joined in
// shared memory, the CTAs by attn_join_kernel.
//
// Measured with 32 query heads on 8 key heads of 128 columns: 64 sequences of 4096 to 8192 keys 289 us,
// 5.4 TB/s of keys and values (0.82 of the copy peak; with a distance bias 292 us); one sequence of 65536
// keys 52 us, 5.1 TB/s.  Four rows of queries fill half of a product's eight columns, which costs nothing.
#include <algorithm>

#include "attn_mma.cuh"
#include "attn_step.cuh"

namespace dlb {
namespace {

constexpr int kStepWarps = 4, kStepThreads = 32 * kStepWarps, kStepKeys = 16;

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The 8x8 matrix of 16-bit values that the warp holds one row per four lanes, transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Over the eight lanes that hold a column (lane ids equal mod 4).
__device__ __forceinline__ float col_max(float v) {
#pragma unroll
  for (int o = 4; o < 32; o *= 2) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float col_sum(float v) {
#pragma unroll
  for (int o = 4; o < 32; o *= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Word x of a 16-byte vector (x is a compile-time constant where this is used).
__device__ __forceinline__ uint32_t word(const uint4 &v, int x) { return x == 0 ? v.x : x == 1 ? v.y : x == 2 ? v.z : v.w; }

// CTAs that share an SM: as many as leave a lane the registers for its loads (wide heads keep the next 16
// keys in flight beside the current 16: 5.1 -> 5.7 TB/s with three CTAs instead of four and no such
// loads; at 64 columns four CTAs with them are best).
constexpr int step_ctas_per_sm(int nt, int nr) { return nr == 2 ? 2 : nt > 2 ? 3 : 4; }

// NT: head_dim up to 32 * NT; NR: up to 8 * NR queries (rows of q x heads of the group) per CTA.
template <int NT, int NR>
__global__ void __launch_bounds__(kStepThreads, step_ctas_per_sm(NT, NR)) attn_step_kernel(const __grid_constant__ AttnArgs a) {
  pdl_prologue();
  constexpr int NB = (NT + 1) / 2;  // blocks of 64 columns of V and O
  constexpr int W = NB * 64, kRows = 8 * NR;
  __shared__ float out_s[kStepWarps][kRows][W + 4];
  __shared__ float m_s[kStepWarps][kRows], l_s[kStepWarps][kRows], r_s[kStepWarps][kRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int rows = a.q_len * a.group, row_tiles = (rows + kRows - 1) / kRows;
  const int tile = blockIdx.x % row_tiles, hk = (blockIdx.x / row_tiles) % a.kv_heads, b = blockIdx.x / (row_tiles * a.kv_heads);
  const BatchView view = batch_view(a, b);
  const int row_last = min(rows, (tile + 1) * kRows) - 1;
  const int last = row_end(a, view, row_last / a.group);  // row_end never falls with the query
  // this CTA's share of the keys, in multiples of what its warps take in one turn
  const int turn = kStepWarps * kStepKeys, turns = (last + turn - 1) / turn;
  const int share = (turns + a.splits - 1) / a.splits * turn;
  const int s0 = min(static_cast<long long>(last), static_cast<long long>(blockIdx.y) * share), s1 = min(last, s0 + share);

  // this lane's columns of S^T and O^T: rows 8y + 2c + x of the tile
  int pos[NR][2], end[NR][2], head[NR][2], doc[NR][2];
  float slope[NR][2], far_left[NR][2];
#pragma unroll
  for (int y = 0; y < NR; y++)
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const int r = tile * kRows + 8 * y + 2 * c + x, i = r / a.group;
      const bool valid = r < rows;
      head[y][x] = hk * a.group + r % a.group;
      pos[y][x] = view.start + i;
      end[y][x] = valid ? min(s1, row_end(a, view, i)) : 0;
      doc[y][x] = (a.q_docs && valid) ? ld_co(a.q_docs + static_cast<long long>(b) * a.q_len + i) : 0;
      slope[y][x] = (a.slopes && valid) ? ld_co(a.slopes + head[y][x]) * kLog2e : 0.f;
      far_left[y][x] = (a.table && valid) ? table_entry(a, head[y][x], bucket_at(a, -a.reach)) : 0.f;
    }
  uint4 q[NR][NT];  // row 8y + g
#pragma unroll
  for (int y = 0; y < NR; y++) {
    const int r = tile * kRows + 8 * y + g;
    const __nv_bfloat16 *src = static_cast<const __nv_bfloat16 *>(a.q.ptr) + b * a.q.batch +
                               static_cast<long long>(r / a.group) * a.q.token + (hk * a.group + r % a.group) * a.q.head;
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int col = (4 * t + c) * 8;
      q[y][t] = r < rows && col < a.dim ? ld_keep(src + col) : make_uint4(0, 0, 0, 0);
    }
  }
  const __nv_bfloat16 *kb = static_cast<const __nv_bfloat16 *>(a.k.ptr) + b * a.k.batch + hk * a.k.head;
  const __nv_bfloat16 *vb = static_cast<const __nv_bfloat16 *>(a.v.ptr) + b * a.v.batch + hk * a.v.head;
  const float to_log2 = a.cap > 0.f ? 1.f : a.scale * kLog2e;
  const CapCoef cap = a.cap > 0.f ? cap_coef(a.scale, a.cap) : CapCoef();
  const int far_to = view.start + (tile * kRows) / a.group - a.reach;  // keys up to here are beyond the reach of all rows

  float acc[NR][NB][4][4], m[NR][2], sum[NR][2], sum_rounded[NR][2];
#pragma unroll
  for (int y = 0; y < NR; y++) {
#pragma unroll
    for (int x = 0; x < 2; x++) {
      m[y][x] = -INFINITY;
      sum[y][x] = sum_rounded[y][x] = 0.f;
    }
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[y][n][t][e] = 0.f;
  }

  uint4 k[2][NT];
  auto load_k = [&](int j0) {
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
  };
  load_k(s0 + warp * kStepKeys);
  for (int j0 = s0 + warp * kStepKeys; j0 < s1; j0 += turn) {
    uint4 v[NB][4];
#pragma unroll
    for (int x = 0; x < 4; x++) {
      const int j = j0 + 2 * c + (x & 1) + 8 * (x >> 1);
      const __nv_bfloat16 *src = vb + static_cast<long long>(j) * a.v.token;
#pragma unroll
      for (int n = 0; n < NB; n++) {
        const int col = n * 64 + g * 8;
        v[n][x] = j < s1 && col < a.dim ? ld_stream(src + col) : make_uint4(0, 0, 0, 0);
      }
    }
    const bool all_far = j0 + kStepKeys - 1 <= far_to;
    float s[NR][4];  // {key g, key g + 8} x {row 2c, row 2c + 1}
    bool grow = false;
#pragma unroll
    for (int y = 0; y < NR; y++) {
#pragma unroll
      for (int e = 0; e < 4; e++) s[y][e] = 0.f;
#pragma unroll
      for (int t = 0; t < NT; t++) {
        mma16816(s[y], k[0][t].x, k[1][t].x, k[0][t].y, k[1][t].y, q[y][t].x, q[y][t].y);
        mma16816(s[y], k[0][t].z, k[1][t].z, k[0][t].w, k[1][t].w, q[y][t].z, q[y][t].w);
      }
    }
    load_k(j0 + turn);  // the next turn's keys are on their way while this one is finished
#pragma unroll
    for (int y = 0; y < NR; y++) {
      if (a.cap > 0.f) cap_scores(s[y], cap);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int x = e & 1, j = j0 + 8 * (e >> 1) + g, d = j - pos[y][x];
        float z = s[y][e] * to_log2;
        if (a.slopes) z = fmaf(-slope[y][x], static_cast<float>(abs(d)), z);
        if (a.table) z += all_far ? far_left[y][x] : table_entry(a, head[y][x], bucket_at(a, d));
        bool seen = j < end[y][x];
        if (a.kv_docs) seen = seen && ld_co(a.kv_docs + static_cast<long long>(b) * a.kv_len + j) == doc[y][x];
        s[y][e] = seen ? z : -INFINITY;
        grow = grow || s[y][e] > m[y][x] + 8.f;
      }
    }
    // The maximum a column's lanes share moves only when some score has outgrown it by 2^8.
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int y = 0; y < NR; y++)
#pragma unroll
        for (int x = 0; x < 2; x++) {
          const float top = fmaxf(m[y][x], col_max(fmaxf(s[y][x], s[y][x + 2])));
          const float keep = top > m[y][x] ? ex2(m[y][x] - top) : 1.f;
          m[y][x] = top;
          sum[y][x] *= keep;
          sum_rounded[y][x] *= keep;
#pragma unroll
          for (int n = 0; n < NB; n++)
#pragma unroll
            for (int t = 0; t < 4; t++) {
              acc[y][n][t][x] *= keep;
              acc[y][n][t][x + 2] *= keep;
            }
        }
    }
    uint32_t p[NR][2];  // fragments of P^T: keys 2c, 2c + 1 (and 8 more) of row g
#pragma unroll
    for (int y = 0; y < NR; y++) {
      const float base0 = m[y][0] == -INFINITY ? 0.f : m[y][0], base1 = m[y][1] == -INFINITY ? 0.f : m[y][1];
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const float p0 = ex2(s[y][2 * u] - base0), p1 = ex2(s[y][2 * u + 1] - base1);
        const uint32_t packed = pack_bf16(p0, p1);
        sum[y][0] += p0;
        sum[y][1] += p1;
        sum_rounded[y][0] += __uint_as_float(packed << 16);
        sum_rounded[y][1] += __uint_as_float(packed & 0xffff0000u);
        p[y][u] = transpose8x8(packed);
      }
    }
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int t = 0; t < 4; t++) {
        // columns 64 n + 8 g + 2 t (rows g of the fragment) and + 1 (rows g + 8)
        const uint32_t w0 = word(v[n][0], t), w1 = word(v[n][1], t), w2 = word(v[n][2], t), w3 = word(v[n][3], t);
        const uint32_t a0 = __byte_perm(w0, w1, 0x5410), a1 = __byte_perm(w0, w1, 0x7632);
        const uint32_t a2 = __byte_perm(w2, w3, 0x5410), a3 = __byte_perm(w2, w3, 0x7632);
#pragma unroll
        for (int y = 0; y < NR; y++) mma16816(acc[y][n][t], a0, a1, a2, a3, p[y][0], p[y][1]);
      }
  }
#pragma unroll
  for (int y = 0; y < NR; y++)
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const float l = col_sum(sum[y][x]), rounded = col_sum(sum_rounded[y][x]);
      const int r = 8 * y + 2 * c + x;
      if (g == 0) {
        m_s[warp][r] = m[y][x];
        l_s[warp][r] = l;
        r_s[warp][r] = rounded;
      }
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int t = 0; t < 4; t += 2)  // columns 64 n + 8 g + 2 t .. 2 t + 3
          *reinterpret_cast<float4 *>(&out_s[warp][r][n * 64 + 8 * g + 2 * t]) =
              make_float4(acc[y][n][t][x], acc[y][n][t][x + 2], acc[y][n][t + 1][x], acc[y][n][t + 1][x + 2]);
    }
  __syncthreads();
  // Join of the four warps: 16 or 8 threads a row.
  constexpr int kParts = kStepThreads / kRows;
  const int r = threadIdx.x / kParts, part = threadIdx.x % kParts, rr = tile * kRows + r;
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
  for (int col = part * 8; col < a.dim; col += kParts * 8) {
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

namespace {
// Rows of a CTA: one fragment of 8 where they all fit it, else two.
int step_rows(int rows) { return rows <= 8 ? 8 : 16; }
}  // namespace

int attn_step_splits(int batch, int kv_heads, int rows, int kv_len, int dim) {
  // Four rounds of CTAs even out sequences of different lengths; where that would leave a share less than
  // 1024 keys, as many rounds as it does not, or, under two, just one (of shares down to 128 keys): a last
  // round that is nearly empty costs as much as a full one (one user, 65536 keys: 76 us with 1.15 rounds).
  const long long ctas = std::max(1ll, static_cast<long long>(batch) * kv_heads * ceil_div(rows, step_rows(rows)));
  const long long fill = static_cast<long long>(step_ctas_per_sm(ceil_div(dim, 32), step_rows(rows) / 8)) * sm_count();
  const long long even = std::min(ceil_div(4 * fill, ctas), kv_len / 1024ll);
  const long long one_round = std::min(fill / ctas, kv_len / 128ll);
  return static_cast<int>(std::max(1ll, std::min(even * ctas >= 2 * fill ? even : one_round, 256ll)));
}

int attn_step(const AttnArgs &a, cudaStream_t st) {
  const int rows = a.q_len * a.group, per_cta = step_rows(rows), nt = ceil_div(a.dim, 32);
  const dim3 grid(ceil_div(rows, per_cta) * a.kv_heads * a.batch, a.splits);
  auto launch = [&](auto kern) -> int {
    launch_pdl(kern, grid, dim3(kStepThreads), 0, st, a);
    DLB_LAUNCH_CHECK("attn_step");
    return DLB_OK;
  };
  if (per_cta == 8)
    return nt == 1   ? launch(attn_step_kernel<1, 1>)
           : nt == 2 ? launch(attn_step_kernel<2, 1>)
           : nt == 3 ? launch(attn_step_kernel<3, 1>)
                     : launch(attn_step_kernel<4, 1>);
  return nt == 1   ? launch(attn_step_kernel<1, 2>)
         : nt == 2 ? launch(attn_step_kernel<2, 2>)
         : nt == 3 ? launch(attn_step_kernel<3, 2>)
                   : launch(attn_step_kernel<4, 2>);
}

}  // namespace dlb
