// Attention backward on the tensor cores (bf16): one kernel in two roles.
//
// A CTA keeps 128 rows X, Y (FOR_KEYS: a tile of K and V; else of Q and dO) and streams the other side
// U, W (Q and dO of every head of the group; else K and V) past them in tiles of 128 rows:
//     S = X U^T, G = Y W^T (TMEM) -> P = 2^(s - lse), D = P (G - delta), times the cap's derivative
//     FOR_KEYS: dV += P W, dK += D U;   else dQ += D U, R += P U        (TMEM, scaled at the end)
// with P and D written over S and G as bf16 (P of the query pass beside D).  The row threads take the
// exponentials of S while the tensor cores make G and the last tile's dK, and D while they make dV and the
// next S.  TMEM holds S, G and the sums; for heads up to 64 wide it has room for more, and S does not wait
// for P: the key pass keeps P beside S, the query pass two S where its ring has four stages to feed them.
//
// P and D are rounded to bf16, the operand type of the next product (in two parts these products would
// double); sums, delta, row statistics and the gradient of the table are fp32.
//
// Tiles of 64 columns with two buffers each were slower (889 instead of 811 us for both passes over 4096
// x 4096 tokens, 32 heads of 128; 908 us since R is made): a product of 128 x 64 takes the tensor cores as
// long as one of 128 x 128, 65 cycles for 16 inner columns, so S and G cost twice as much.  What bounds the key pass now, by the
// clock: 2800 cycles a tile, of which P takes 1430 (1024 of them are the special-function units' 16 a
// clock) and dV with the next S, which cannot start before P is complete, 1260; the tensor cores are busy
// for 2048.
//
// Two passes rebuild S and G twice: 8 products of 2 * dim flop per pair where a single pass would need
// 5.  In return no sum crosses a CTA: no fp32 copy of dQ in memory, no atomics, the same bits every time.
//
// delta.  <dout, o> from the bf16 output is off by its rounding, which moves every D of a row the same way:
// where values have a common part (o large, D small) that is far more than D's own rounding.  The query
// pass therefore takes it as a first guess only.  Its rows add up D in fp32; with the true delta a row's D
// add up to zero, so the sum e is what the guess is off by, and
//     dQ = scale (sum_j D_ij k_j - e_i R_i),  R_i = sum_j P_ij k_j (times the cap's derivative)
// at the price of one product; delta + e goes to the key pass, which runs second.  (A row whose P do not add
// up to one has o and lse of more keys than the call's: its guess stays.)  dq and dk of 70 causal
// tokens come from 2.7e-3 to 2.35e-3 of the exact ones (the output's and D's own rounding make 2.35e-3),
// both passes over 4096 tokens, 32 heads of 128 on 8, causal with a cap, from 537 to 576 us.
#pragma once

#include <algorithm>

#include "attn_mma.cuh"

namespace dlb {

constexpr int kStatsBytes = 2 * kStatRows * sizeof(float);
static_assert(kStatRows == kTileRows, "a stage takes one tile of row statistics");

// PARTS threads share a row's 128 columns: four, or two where the sums for the table leave no room for
// more.  Registers with PARTS = 4: launched with 96 each (640 * 96 = 61440); the row warps go up to 104,
// the four others down to 64 (512 * 104 + 128 * 64 = 61440).
constexpr int kBwdRowRegs = 104, kBwdOtherRegs = 64;
template <int PARTS>
struct BwdWarps {
  static constexpr int kRows = 4 * PARTS, kLoad = kRows, kMma = kRows + 1;
  static constexpr int kThreads = PARTS == 4 ? 640 : 320;
};

template <int NB, int ST>
struct BwdShape {
  static constexpr int kX = 0, kY = NB * kBlockBytes, kRing = 2 * NB * kBlockBytes;
  static constexpr int kStage = 2 * NB * kBlockBytes;
  static constexpr int kStats = kRing + ST * kStage, kRest = kStats + ST * kStatsBytes;
};

// Where in the padded tables a warp's 16 pairs from distance d0 on (FOR_KEYS: back) lie when all its
// rows' pairs are beyond the reach; -1 when some are not (then all are near enough for the padding).
template <bool FOR_KEYS>
__device__ __forceinline__ int far_side(const AttnArgs &a, int d0) {
  const int lo = FOR_KEYS ? d0 - 15 : d0, hi = FOR_KEYS ? d0 : d0 + 15;
  const bool left = hi <= -a.reach, right = lo >= a.reach;
  if (!__all_sync(0xffffffffu, left || right)) return -1;
  return left ? 0 : 2 * (a.reach + kLutPad);
}

// {-lse * log2(e), -delta} of query x (row `row` of tile `tile`), delta = <dout_x, o_x> by the PARTS threads
// of the row (a first guess, see above), and its place in row_stats filled; rows behind the last query get
// {-infinity, 0}.
template <int NB, int PARTS>
__device__ __forceinline__ float2 make_row_stats(const AttnArgs &a, int b, int h, int tile, int x, int part, int row, bool valid,
                                                 float (*delta_part)[kTileRows]) {
  float sum = 0.f, lse = -INFINITY;
  if (valid) {
    using S = Store<__nv_bfloat16>;
    const __nv_bfloat16 *o = static_cast<const __nv_bfloat16 *>(a.o.ptr) + b * a.o.batch + static_cast<long long>(x) * a.o.token + h * a.o.head;
    const __nv_bfloat16 *g = static_cast<const __nv_bfloat16 *>(a.dout.ptr) + b * a.dout.batch +
                             static_cast<long long>(x) * a.dout.token + h * a.dout.head;
    constexpr int kLoads = NB * kBlockCols / (8 * PARTS);  // all in flight at once
    uint4 ov[kLoads], gv[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; k++) {
      const int c = (k * PARTS + part) * 8;
      ov[k] = c < a.dim ? ld_keep(o + c) : make_uint4(0, 0, 0, 0);
      gv[k] = c < a.dim ? ld_keep(g + c) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int k = 0; k < kLoads; k++) {
      float u[8], v[8];
      S::unpack(ov[k], u);
      S::unpack(gv[k], v);
#pragma unroll
      for (int e = 0; e < 8; e++) sum = fmaf(u[e], v[e], sum);
    }
    lse = ld_co(a.lse + (static_cast<size_t>(b) * a.heads + h) * a.q_len + x);
  }
  delta_part[part][row] = sum;
  named_bar_sync(1, 128 * PARTS);
  sum = 0.f;
#pragma unroll
  for (int k = 0; k < PARTS; k++) sum += delta_part[k][row];
  const float2 stat = make_float2(lse == -INFINITY ? -INFINITY : -lse * kLog2e, -sum);
  if (part == 0) {
    float *to = stats_tile(a, b, h, tile) + row;
    to[0] = stat.x;
    to[kStatRows] = stat.y;
  }
  return stat;
}

// Bytes behind the ring: bias by distance, bucket by distance, sums of the score gradients per part, bucket
// and row (a thread's own, so that no order is left to chance), tile flags.  The gradient of the table is
// made by the key pass: its delta is exact, so that nothing has to be taken off a row's sums afterwards.
struct BwdRest {
  int lut, buckets, sums, flags, total;
};
__host__ __device__ inline BwdRest bwd_rest(const AttnArgs &a, bool for_keys, int parts) {
  const int tiles = ((for_keys ? a.q_len : a.kv_len) + kTileRows - 1) / kTileRows;
  const int slots = for_keys && a.dtable != nullptr ? a.buckets * parts * kTileRows : 0;
  BwdRest r;
  r.lut = 0;
  r.buckets = r.lut + (a.table ? 4 * lut_floats(a.reach) : 0);
  r.sums = r.buckets + (slots ? (lut_floats(a.reach) + 15) / 16 * 16 : 0);
  r.flags = r.sums + slots * 4;
  r.total = r.flags + (tiles + 15) / 16 * 16;
  return r;
}

template <int NB, int ST, int PARTS, bool FOR_KEYS, bool CAP, int BIAS>
static __global__ void __launch_bounds__(BwdWarps<PARTS>::kThreads, 1)
attn_bwd_mma_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ BwdMaps maps, unsigned int *timeouts) {
  using Shape = BwdShape<NB, ST>;
  constexpr int kBwdLoadWarp = BwdWarps<PARTS>::kLoad, kBwdMmaWarp = BwdWarps<PARTS>::kMma;
  constexpr int kBwdThreads = BwdWarps<PARTS>::kThreads, kRowThreads = 128 * PARTS;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  unsigned char *ring = smem + Shape::kRing;
  const BwdRest rest = bwd_rest(a, FOR_KEYS, PARTS);
  float *lut = reinterpret_cast<float *>(smem + Shape::kRest + rest.lut);
  unsigned char *bucket_lut = smem + Shape::kRest + rest.buckets;
  float *sums = reinterpret_cast<float *>(smem + Shape::kRest + rest.sums);  // [part][bucket][row]
  unsigned char *flags = smem + Shape::kRest + rest.flags;
  __shared__ uint64_t x_full, full[ST], empty[ST], s_full[2], g_full, p_full[2], d_full, v_full, acc_full, drain;
  __shared__ uint32_t tmem_slot;
  __shared__ int dead_flag, doc_range[2];
  __shared__ float delta_part[FOR_KEYS ? 1 : PARTS][kTileRows], d_part[FOR_KEYS ? 1 : PARTS][kTileRows];
  __shared__ float p_part[FOR_KEYS ? 1 : PARTS][kTileRows];
  __shared__ __align__(16) int doc_tile[kTileRows];
  volatile int *dead = &dead_flag;
  // s_full and p_full come in pairs, used in turn: with two S the tensor cores may finish the next tile's
  // before a row thread has seen this one's.
  // TMEM: S 0, G 128, dK or dQ 256; then dV 384 and P over S or at 448, or the second S at 384 and R at
  // 320 (heads up to 64 wide), or R at 384
  constexpr bool kTwoS = !FOR_KEYS && ST >= 4, kOwnP = FOR_KEYS && NB == 1;
  constexpr uint32_t kAccX = 256, kAccY = !FOR_KEYS && NB == 1 ? 320 : 384, kG = 128;
  constexpr uint32_t kPStep = kOwnP ? 8 : 16;  // columns of P per 16 of S
  const bool table_sums = BIAS == kTable && FOR_KEYS && a.dtable != nullptr;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    mbar_init(&x_full, 1);
    for (int s = 0; s < ST; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int t = 0; t < 2; t++) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4 * PARTS);
    }
    mbar_init(&g_full, 1);
    mbar_init(&v_full, 1);
    mbar_init(&d_full, 4 * PARTS);
    mbar_init(&acc_full, 1);
    mbar_init(&drain, 1);
    dead_flag = 0;
    mbar_fence_init();
  }
  if (warp == kBwdMmaWarp) tmem_alloc(&tmem_slot, 512);
  if (tid == kBwdLoadWarp * 32) {
    prefetch_map(&(FOR_KEYS ? maps.k : maps.q));
    prefetch_map(&(FOR_KEYS ? maps.v : maps.dout));
    prefetch_map(&(FOR_KEYS ? maps.q : maps.k));
    prefetch_map(&(FOR_KEYS ? maps.dout : maps.v));
  }
  pdl_prologue();

  // Tiles are the slowest index, those with most work under a causal mask first.
  const int len = FOR_KEYS ? a.kv_len : a.q_len, units = FOR_KEYS ? a.kv_heads : a.heads;
  const int tiles = (len + kTileRows - 1) / kTileRows;
  int tile = blockIdx.x / (units * a.batch);
  if (!FOR_KEYS) tile = tiles - 1 - tile;
  const int unit = blockIdx.x % units, b = (blockIdx.x / units) % a.batch;
  const int hk = FOR_KEYS ? unit : unit / a.group, heads_here = FOR_KEYS ? a.group : 1;
  const int row0 = tile * kTileRows, row_last = min(len, row0 + kTileRows) - 1;
  const BatchView view = batch_view(a, b);

  // flags[n]: 1 when some row of the tile meets stream tile n, 3 when every row meets all of it.
  int stream_end, from = 0;  // stream rows [from, stream_end) matter
  int full_from = 0, full_end;
  if (FOR_KEYS) {
    stream_end = row0 < view.end ? a.q_len : 0;
    from = first_query(a, view, row0);
    full_from = first_query(a, view, row_last);
    full_end = row0 + kTileRows <= view.end ? a.q_len : 0;
  } else {
    stream_end = row_end(a, view, row_last);
    full_end = row_end(a, view, row0);
  }
  const int n_tiles = (stream_end + kTileRows - 1) / kTileRows;
  if (a.q_docs) {
    const int *docs = (FOR_KEYS ? a.kv_docs : a.q_docs) + static_cast<long long>(b) * len;
    if (warp == 0) {
      int lo = INT_MAX, hi = INT_MIN;
      for (int r = row0 + lane; r <= row_last; r += 32) {
        const int d = ld_co(docs + r);
        lo = min(lo, d);
        hi = max(hi, d);
      }
      lo = warp_min(lo);
      hi = warp_max(hi);
      if (lane == 0) {
        doc_range[0] = lo;
        doc_range[1] = hi;
      }
    }
    __syncthreads();
  }
  const int *stream_docs = a.q_docs ? (FOR_KEYS ? a.q_docs : a.kv_docs) + static_cast<long long>(b) * (FOR_KEYS ? a.q_len : a.kv_len)
                                    : nullptr;
  for (int n = warp; n < n_tiles; n += kBwdThreads / 32) {
    const int c0 = n * kTileRows;
    bool active = c0 + kTileRows > from, whole = c0 >= full_from && c0 + kTileRows <= full_end;
    if (stream_docs) {
      int lo = INT_MAX, hi = INT_MIN;
      for (int c = c0 + lane; c < min(stream_end, c0 + kTileRows); c += 32) {
        const int d = ld_co(stream_docs + c);
        lo = min(lo, d);
        hi = max(hi, d);
      }
      lo = warp_min(lo);
      hi = warp_max(hi);
      active = active && lo <= doc_range[1] && doc_range[0] <= hi;
      whole = whole && lo == hi && doc_range[0] == doc_range[1] && lo == doc_range[0];
    }
    if (lane == 0) flags[n] = active ? (whole ? 3 : 1) : 0;
  }
  if (BIAS == kTable && !FOR_KEYS) fill_lut(lut, a, unit, tid, kBwdThreads);
  if (table_sums) {
    for (int e = tid; e < 2 * (a.reach + kLutPad) + 1; e += kBwdThreads)
      bucket_lut[e] = static_cast<unsigned char>(bucket_at(a, e - a.reach - kLutPad));
    for (int e = tid; e < PARTS * a.buckets * kTileRows; e += kBwdThreads) sums[e] = 0.f;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp < kBwdLoadWarp) {
    if (PARTS == 4) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kBwdRowRegs));
    const int part = warp >> 2, row = tid & 127, x = row0 + row;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    constexpr int kCols = kTileRows / PARTS, kChunks = kCols / 16;  // this thread's columns, 16 at a time
    const uint32_t s_base = tmem + lane_base + part * kCols, g_at = s_base + kG;
    const uint32_t p_at = kOwnP ? tmem + lane_base + 448 + part * (kCols / 2) : s_base;
    const bool valid = x < len && (!FOR_KEYS || x < view.end);
    const int row_doc = (a.q_docs && valid) ? ld_co((FOR_KEYS ? a.kv_docs : a.q_docs) + static_cast<long long>(b) * len + x) : 0;
    // Stream rows [see_from, see_end) are visible to this row, as far as documents allow.
    const int see_from = !valid ? INT_MAX : FOR_KEYS ? first_query(a, view, x) : 0;
    const int see_end = !valid ? 0 : FOR_KEYS ? a.q_len : row_end(a, view, x);
    // The query pass, which runs first, makes its rows' statistics itself and leaves them to the key pass.
    const float2 row_stat = FOR_KEYS ? make_float2(-INFINITY, 0.f) : make_row_stats<NB, PARTS>(a, b, unit, tile, x, part, row, valid, delta_part);
    const float to_log2 = CAP ? 1.f : a.scale * kLog2e;
    const CapCoef cap = CAP ? cap_coef(a.scale, a.cap) : CapCoef();
    const float2 uncap = both(CAP ? 1.f / cap.out : 0.f);
    const int tail = !FOR_KEYS && view.end % kTileRows && view.end < a.kv_len ? view.end / kTileRows : -1;
    int bucket_now = 0;
    float bucket_sum = 0.f;
    auto flush_bucket = [&](int next) {
      sums[(part * a.buckets + bucket_now) * kTileRows + row] += bucket_sum;
      bucket_sum = 0.f;
      bucket_now = next;
    };
    float2 d_sum[2] = {both(0.f), both(0.f)}, p_sum = both(0.f);  // of this thread's D and P, for e
    int it = -1;
    for (int g = 0; g < heads_here; g++) {
      const int h = FOR_KEYS ? hk * a.group + g : unit;
      const float slope = (BIAS != kNoBias && a.slopes) ? ld_co(a.slopes + h) * kLog2e : 0.f;
      if (BIAS == kTable && FOR_KEYS) {
        // this head's bias by distance, once all row threads are past the last head's tiles
        named_bar_sync(1, kRowThreads);
        fill_lut(lut, a, h, tid, kRowThreads);
        named_bar_sync(1, kRowThreads);
      }
      for (int n = 0; n < n_tiles; n++) {
        const int f = flags[n];
        if (!f) continue;
        it++;
        const int c0 = n * kTileRows, s = it % ST;
        const bool by_doc = f != 3 && stream_docs;
        int col_doc = 0;
        if (by_doc && part == 0) col_doc = ld_co(stream_docs + min(c0 + row, (FOR_KEYS ? a.q_len : a.kv_len) - 1));
        if (FOR_KEYS) mbar_wait(&full[s], (it / ST) & 1, dead, timeouts);  // the stage's statistics
        mbar_wait(&s_full[it & 1], (it >> 1) & 1, dead, timeouts);
        if (by_doc) {  // the tile's document numbers
          named_bar_sync(2, kRowThreads);
          if (part == 0) doc_tile[row] = col_doc;
          named_bar_sync(2, kRowThreads);
        }
        tc_fence_after();
        const float *stats = reinterpret_cast<const float *>(smem + Shape::kStats + s * kStatsBytes) + part * kCols;
        // Probabilities, from S alone.  A chunk's P and D go over the first 8 columns of its own S and G.
        const uint32_t s_at = s_base + (kTwoS && (it & 1) ? 384 : 0);
        float p[kCols], capped[CAP ? kCols : 1];  // P, P times the cap's derivative
#pragma unroll
        for (int q = 0; q < kChunks; q++) {
          const int e0 = q * 16, c1 = c0 + part * kCols + e0;
          uint32_t sr[16];
          tmem_load16(s_at + e0, sr);
          tmem_loaded(sr);
          float x16[16];
#pragma unroll
          for (int e = 0; e < 16; e++) x16[e] = __uint_as_float(sr[e]);
          if (CAP) cap_scores(x16, cap);
          const int d0 = FOR_KEYS ? x - (view.start + c1) : c1 - (view.start + x);  // distance j - p at e = 0
          const float *lut_at = lut + d0 + a.reach + kLutPad;
          const int far_at = BIAS == kTable ? far_side<FOR_KEYS>(a, d0) : 0;
          const float far_bias = BIAS == kTable && far_at >= 0 ? lut[far_at] : 0.f;
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            float4 l4 = make_float4(row_stat.x, row_stat.x, row_stat.x, row_stat.x);
            if (FOR_KEYS) l4 = *reinterpret_cast<const float4 *>(stats + e0 + e);
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
              float2 shift = k ? make_float2(l4.z, l4.w) : make_float2(l4.x, l4.y);
              if (BIAS == kTable) {
                const float2 bias = far_at >= 0 ? both(far_bias)
                                    : FOR_KEYS  ? make_float2(lut_at[-(e + k)], lut_at[-(e + k + 1)])
                                                : make_float2(lut_at[e + k], lut_at[e + k + 1]);
                shift = add2(shift, bias);
              }
              if (BIAS == kSlope || (BIAS == kTable && a.slopes)) {
                const float d = static_cast<float>(d0), f0 = static_cast<float>(e + k), f1 = static_cast<float>(e + k + 1);
                shift.x = fmaf(-slope, fabsf(FOR_KEYS ? d - f0 : d + f0), shift.x);
                shift.y = fmaf(-slope, fabsf(FOR_KEYS ? d - f1 : d + f1), shift.y);
              }
              const float2 v = make_float2(x16[e + k], x16[e + k + 1]);
              const float2 y = CAP ? add2(v, shift) : fma2(v, both(to_log2), shift);
              p[e0 + e + k] = ex2(y.x);
              p[e0 + e + k + 1] = ex2(y.y);
            }
          }
          if (f != 3) {
            if (stream_docs) {
#pragma unroll
              for (int e = 0; e < 16; e += 4) {
                const int4 d = *reinterpret_cast<const int4 *>(&doc_tile[part * kCols + e0 + e]);
                const int same[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
                for (int k = 0; k < 4; k++)
                  if (same[k] != row_doc) p[e0 + e + k] = 0.f;
              }
            }
            // Hidden: columns in front of the first query that sees the key (behind the last query
            // -lse = -infinity has done it), or behind the last key that the query sees.
            const int cut = FOR_KEYS ? see_from - c1 : see_end - c1;
#pragma unroll
            for (int e = 0; e < 16; e++)
              if (FOR_KEYS ? e < cut : e >= cut) p[e0 + e] = 0.f;
            if (CAP) {  // a hidden score may be NaN, and the cap's derivative of it
#pragma unroll
              for (int e = 0; e < 16; e++)
                if (p[e0 + e] == 0.f) x16[e] = 0.f;
            }
          }
          if (CAP) {
#pragma unroll
            for (int e = 0; e < 16; e += 2) {  // d tanh = 1 - tanh^2
              const float2 t = mul2(make_float2(x16[e], x16[e + 1]), uncap);
              const float2 c = mul2(make_float2(p[e0 + e], p[e0 + e + 1]), fma2(make_float2(-t.x, -t.y), t, both(1.f)));
              capped[CAP ? e0 + e : 0] = c.x;
              capped[CAP ? e0 + e + 1 : 0] = c.y;
            }
          }
          if (FOR_KEYS) {
            uint32_t packed[8];
#pragma unroll
            for (int e = 0; e < 8; e++) packed[e] = pack_bf16(p[e0 + 2 * e], p[e0 + 2 * e + 1]);
            if (kOwnP && q == 0 && it > 0) mbar_wait(&v_full, (it - 1) & 1, dead, timeouts);  // the last P has been used
            tmem_store8(p_at + q * kPStep, packed);
          }
        }
        if (FOR_KEYS) tmem_stored();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[it & 1]);  // (S has been read, also where P is of no use)

        auto through_cap = [&](int e) {
          return CAP ? make_float2(capped[CAP ? e : 0], capped[CAP ? e + 1 : 0]) : make_float2(p[e], p[e + 1]);
        };
        mbar_wait(&g_full, it & 1, dead, timeouts);
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < kChunks; q++) {
          const int e0 = q * 16, c1 = c0 + part * kCols + e0;
          uint32_t gr[16];
          tmem_load16(g_at + e0, gr);
          tmem_loaded(gr);
          float dp[16];
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            float4 d4 = make_float4(row_stat.y, row_stat.y, row_stat.y, row_stat.y);
            if (FOR_KEYS) d4 = *reinterpret_cast<const float4 *>(stats + kTileRows + e0 + e);
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
              const float2 minus = k ? make_float2(d4.z, d4.w) : make_float2(d4.x, d4.y);
              const float2 d2 = add2(make_float2(__uint_as_float(gr[e + k]), __uint_as_float(gr[e + k + 1])), minus);
              dp[e + k] = d2.x;
              dp[e + k + 1] = d2.y;
            }
          }
          if (f != 3) {  // what is hidden may have met anything in V
#pragma unroll
            for (int e = 0; e < 16; e++) dp[e] = p[e0 + e] == 0.f ? 0.f : dp[e];
          }
          if (table_sums) {
            // One run of columns per bucket: its sum stays in a register until the bucket changes.
            const int d0 = x - (view.start + c1), far_at = far_side<FOR_KEYS>(a, d0);
            if (far_at >= 0) {
              const int n_now = bucket_lut[far_at];
              if (n_now != bucket_now) flush_bucket(n_now);
              float2 t[2] = {both(0.f), both(0.f)};
#pragma unroll
              for (int e = 0; e < 16; e += 2)
                t[e >> 1 & 1] = fma2(make_float2(p[e0 + e], p[e0 + e + 1]), make_float2(dp[e], dp[e + 1]), t[e >> 1 & 1]);
              const float2 u = add2(t[0], t[1]);
              bucket_sum += u.x + u.y;
            } else {
              const unsigned char *at = bucket_lut + d0 + a.reach + kLutPad;
#pragma unroll
              for (int e = 0; e < 16; e++) {
                const int n_now = at[-e];
                if (n_now != bucket_now) flush_bucket(n_now);
                bucket_sum = fmaf(p[e0 + e], dp[e], bucket_sum);
              }
            }
          }
          uint32_t packed[8];
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float2 d2 = make_float2(dp[2 * e], dp[2 * e + 1]), y = mul2(through_cap(e0 + 2 * e), d2);
            if (!FOR_KEYS) {
              const float2 p2 = make_float2(p[e0 + 2 * e], p[e0 + 2 * e + 1]);
              d_sum[e & 1] = fma2(p2, d2, d_sum[e & 1]);
              p_sum = add2(p_sum, p2);
            }
            packed[e] = pack_bf16(y.x, y.y);
          }
          tmem_store8(g_at + e0, packed);
          if (!FOR_KEYS) {  // beside D
#pragma unroll
            for (int e = 0; e < 8; e++) {
              const float2 y = through_cap(e0 + 2 * e);
              packed[e] = pack_bf16(y.x, y.y);
            }
            tmem_store8(g_at + e0 + 8, packed);
          }
        }
        if (n == tail) {
          // Rows of K that no query reaches may hold anything, and 0 * NaN is NaN.
          const int first = view.end - c0;
          for (int e = part * 128 + row; e < (kTileRows - first) * NB * 8; e += kRowThreads) {
            const int r = first + e / (NB * 8), q = e % (NB * 8);
            *reinterpret_cast<uint4 *>(ring + s * Shape::kStage + (q / 8) * kBlockBytes + r * 128 + (q % 8) * 16) =
                make_uint4(0, 0, 0, 0);
          }
          fence_async_smem();
        }
        tmem_stored();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&d_full);
      }
      if (table_sums) {  // this head's part of its table's gradient; the sums start anew
        flush_bucket(0);
        named_bar_sync(1, kRowThreads);
        float *to = a.table_part + (static_cast<size_t>(h) * a.table_parts + b * tiles + tile) * a.buckets;
        for (int n = warp; n < a.buckets; n += BwdWarps<PARTS>::kRows) {
          float v = 0.f;
#pragma unroll
          for (int k = 0; k < PARTS; k++)
            for (int r = lane; r < kTileRows; r += 32) {
              float &slot = sums[(k * a.buckets + n) * kTileRows + r];
              v += slot;
              slot = 0.f;
            }
          v = warp_sum(v);
          if (lane == 0) to[n] = v;
        }
        // (the next head's sums wait for the barriers around its bias by distance)
      }
    }
    float off = 0.f;  // what delta was off by
    if constexpr (!FOR_KEYS) {
      const float2 sum = add2(d_sum[0], d_sum[1]);
      d_part[part][row] = sum.x + sum.y;
      p_part[part][row] = p_sum.x + p_sum.y;
      named_bar_sync(1, kRowThreads);
      float total = 0.f;
#pragma unroll
      for (int k = 0; k < PARTS; k++) {
        off += d_part[k][row];
        total += p_part[k][row];
      }
      if (!row_is_whole<__nv_bfloat16>(a, total, row_stat.x)) off = 0.f;
      if (part == 0) stats_tile(a, b, unit, tile)[kStatRows + row] = row_stat.y - off;
    }
    mbar_wait(&acc_full, 0, dead, timeouts);
    tc_fence_after();
    // FOR_KEYS: the first half of the row warps stores dK, the other dV; else all share the columns of dQ.
    constexpr int kSharers = FOR_KEYS ? PARTS / 2 : PARTS;
    const bool second = FOR_KEYS && part >= PARTS / 2;
    const Heads &to = !FOR_KEYS ? a.dq : second ? a.dv : a.dk;
    const float by = second ? 1.f : a.scale;
    const uint32_t acc_at = tmem + lane_base + (second ? kAccY : kAccX);
    __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(to.ptr) + b * to.batch + static_cast<long long>(x) * to.token + unit * to.head;
    for (int c = 32 * (part % kSharers); c < a.dim; c += 32 * kSharers) {
      uint32_t o[32];
      if (it >= 0) {
        tmem_load32(acc_at + c, o);
        tmem_loaded(o);
        if constexpr (!FOR_KEYS) {
          uint32_t r[32];
          tmem_load32(tmem + lane_base + kAccY + c, r);
          tmem_loaded(r);
#pragma unroll
          for (int e = 0; e < 32; e++) o[e] = __float_as_uint(fmaf(-off, __uint_as_float(r[e]), __uint_as_float(o[e])));
        }
      }
#pragma unroll
      for (int e = 0; e < 32; e += 8) {
        uint32_t v[4];
#pragma unroll
        for (int k = 0; k < 4; k++)
          v[k] = it < 0 ? 0u : pack_bf16(__uint_as_float(o[e + 2 * k]) * by, __uint_as_float(o[e + 2 * k + 1]) * by);
        if (x < len && c + e < a.dim) *reinterpret_cast<uint4 *>(out + c + e) = make_uint4(v[0], v[1], v[2], v[3]);
      }
    }
    tc_fence_before();
  } else {
    if (PARTS == 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kBwdOtherRegs));
    if (warp == kBwdLoadWarp) {
      if (lane == 0) {
        const int x_head = FOR_KEYS ? hk : unit;
        mbar_expect_tx(&x_full, 2 * NB * kBlockBytes);
        for (int c = 0; c < NB; c++) {
          tma_load_rows(smem + Shape::kX + c * kBlockBytes, &(FOR_KEYS ? maps.k : maps.q), &x_full, c * kBlockCols, row0, x_head, b);
          tma_load_rows(smem + Shape::kY + c * kBlockBytes, &(FOR_KEYS ? maps.v : maps.dout), &x_full, c * kBlockCols, row0, x_head, b);
        }
        int it = 0;
        for (int g = 0; g < heads_here && !*dead; g++) {
          const int head = FOR_KEYS ? hk * a.group + g : hk;  // of the streamed tensors
          for (int n = 0; n < n_tiles; n++) {
            if (!flags[n]) continue;
            const int s = it % ST;
            const unsigned use = it / ST;
            if (use) mbar_wait(&empty[s], (use - 1) & 1, dead, timeouts);
            if (*dead) break;
            unsigned char *stage = ring + s * Shape::kStage;
            mbar_expect_tx(&full[s], Shape::kStage + (FOR_KEYS ? kStatsBytes : 0));
            for (int c = 0; c < NB; c++) {
              tma_load_rows(stage + c * kBlockBytes, &(FOR_KEYS ? maps.q : maps.k), &full[s], c * kBlockCols, n * kTileRows, head, b);
              tma_load_rows(stage + (NB + c) * kBlockBytes, &(FOR_KEYS ? maps.dout : maps.v), &full[s], c * kBlockCols, n * kTileRows, head, b);
            }
            if (FOR_KEYS)
              bulk_load(smem + Shape::kStats + s * kStatsBytes, stats_tile(a, b, head, n), kStatsBytes, &full[s]);
            it++;
          }
        }
        if (*dead) {  // no copy may be in flight when the CTA ends
          drain_wait(&x_full, 0);
          for (int i = max(0, it - ST); i < it; i++) drain_wait(&full[i % ST], (i / ST) & 1);
        }
      }
    } else if (warp == kBwdMmaWarp) {
      const int k_steps = (a.dim + 15) / 16, n_cols = k_steps * 16;
      const uint32_t idesc_s = mma_desc(kTileRows, false), idesc_acc = mma_desc(n_cols, true);
      const uint64_t xd = desc_k_major(smem_u32(smem + Shape::kX)), yd = desc_k_major(smem_u32(smem + Shape::kY));
      const uint64_t u_desc = desc_k_major(smem_u32(ring)), u_desc_mn = desc_mn_major(smem_u32(ring), kBlockBytes);
      constexpr uint32_t kStageStep = Shape::kStage >> 4, kW = (NB * kBlockBytes) >> 4;  // in descriptor units
      auto scores = [&](uint32_t to, uint64_t ad, uint64_t bd, uint64_t *bar) {
        if (elect_lane()) {
#pragma unroll
          for (int k = 0; k < NB * 4; k++) {
            const int at = (k / 4) * (kBlockBytes >> 4) + (k % 4) * 2;
            if (k < k_steps) mma_ss(tmem + to, ad + at, bd + at, idesc_s, k > 0);
          }
          tc_commit(bar);
        }
        __syncwarp();
      };
      auto accumulate = [&](uint32_t to, uint32_t from, uint32_t step, uint64_t bd, bool add, uint64_t *bar) {
        if (elect_lane()) {
#pragma unroll
          for (int k = 0; k < kTileRows / 16; k++)
            mma_ts(tmem + to, tmem + from + k * step, bd + k * (2048 >> 4), idesc_acc, add || k > 0);
          if (bar) tc_commit(bar);
        }
        __syncwarp();
      };
      auto make_s = [&](int it) {
        mbar_wait(&full[it % ST], (it / ST) & 1, dead, timeouts);
        scores(kTwoS && (it & 1) ? 384 : 0, xd, u_desc + (it % ST) * kStageStep, &s_full[it & 1]);
      };
      auto make_g = [&](int it) { scores(kG, yd, u_desc + (it % ST) * kStageStep + kW, &g_full); };
      auto add_dv = [&](int it) {  // P of tile `it` is there
        accumulate(kAccY, kOwnP ? 448 : 0, kPStep, u_desc_mn + (it % ST) * kStageStep + kW, it > 0, kOwnP ? &v_full : nullptr);
      };
      auto add_x = [&](int it) {  // dK, or dQ and R, when D of tile `it` is there
        mbar_wait(&d_full, it & 1, dead, timeouts);
        tc_fence_after();
        const uint64_t ud = u_desc_mn + (it % ST) * kStageStep;
        if (!FOR_KEYS) accumulate(kAccY, kG + 8, 16, ud, it > 0, nullptr);
        accumulate(kAccX, kG, 16, ud, it > 0, &empty[it % ST]);
      };
      auto wait_p = [&](int it) {  // S of tile `it` has been read, its P is there
        mbar_wait(&p_full[it & 1], (it >> 1) & 1, dead, timeouts);
        tc_fence_after();
      };
      mbar_wait(&x_full, 0, dead, timeouts);
      int total = 0;
      for (int n = 0; n < n_tiles; n++) total += flags[n] != 0;
      total *= heads_here;
      if (kTwoS && total > 0) make_s(0);
      for (int it = 0; it < total && !*dead; it++) {
        if (kTwoS) {
          if (it > 0) add_x(it - 1);
          make_g(it);
          if (it + 1 < total) {
            if (it > 0) wait_p(it - 1);
            make_s(it + 1);
          }
        } else if (ST > 1) {
          if (it > 0) {
            wait_p(it - 1);
            if (FOR_KEYS && !kOwnP) add_dv(it - 1);
          }
          make_s(it);
          if (it > 0) {
            if (FOR_KEYS && kOwnP) add_dv(it - 1);
            add_x(it - 1);
          }
          make_g(it);
        } else {  // one stage: the next tile comes when the last is done with
          if (it > 0) {
            wait_p(it - 1);
            if (FOR_KEYS) add_dv(it - 1);
            add_x(it - 1);
          }
          make_s(it);
          make_g(it);
        }
      }
      if (total > 0) {
        if (kTwoS && total > 1) wait_p(total - 2);
        wait_p(total - 1);
        if (FOR_KEYS) add_dv(total - 1);
        add_x(total - 1);
      }
      if (elect_lane()) tc_commit(&acc_full);
      __syncwarp();
      if (*dead) {
        if (elect_lane()) tc_commit(&drain);
        __syncwarp();
        drain_wait(&drain, 0);
      }
    }
  }
  __syncthreads();
  if (warp == kBwdMmaWarp) {
    tc_fence_after();
    tmem_free(tmem, 512);
  }
}

// What the sums of the most buckets and the longest map leave room for.
constexpr int kMostSums = 4 * DLB_ATTN_MAX_BUCKETS * kTileRows * 2;  // two parts
constexpr int kMostLuts = 5 * (2 * (DLB_ATTN_MAX_DISTANCE + kLutPad) + 4) + 16;
static_assert(1024 + BwdShape<1, 2>::kRest + kMostSums + kMostLuts + kMaxTiles <= kMaxDynamicSmem, "any table must fit");
static_assert(1024 + BwdShape<2, 1>::kRest + kMostSums + kMostLuts + kMaxTiles <= kMaxDynamicSmem, "any table must fit");

template <bool FOR_KEYS>
int bwd_mma_launch(const AttnArgs &a, const BwdMaps &maps, cudaStream_t st) {
  const char *name = FOR_KEYS ? "attn_bwd_mma (keys)" : "attn_bwd_mma (queries)";
  unsigned int *timeouts = wait_timeouts_counter();
  DLB_REQUIRE(timeouts != nullptr, DLB_ERR_NO_DEVICE, "%s: no CUDA device", name);
  auto launch = [&](auto kern, int ring_end, int parts) -> int {
    const size_t smem = 1024 + ring_end + bwd_rest(a, FOR_KEYS, parts).total;
    if (int rc = allow_smem(kern, smem, name)) return rc;
    const int grid = ceil_div(FOR_KEYS ? a.kv_len : a.q_len, kTileRows) * (FOR_KEYS ? a.kv_heads : a.heads) * a.batch;
    launch_pdl(kern, dim3(grid), dim3(parts == 4 ? BwdWarps<4>::kThreads : BwdWarps<2>::kThreads), smem, st, a, maps, timeouts);
    DLB_LAUNCH_CHECK(name);
    return DLB_OK;
  };
  const bool cap = a.cap > 0.f;
#define DLB_PICK(NB, ST, PARTS, BIAS)                                                                            \
  (cap ? launch(attn_bwd_mma_kernel<NB, ST, PARTS, FOR_KEYS, true, BIAS>, BwdShape<NB, ST>::kRest, PARTS)        \
       : launch(attn_bwd_mma_kernel<NB, ST, PARTS, FOR_KEYS, false, BIAS>, BwdShape<NB, ST>::kRest, PARTS))
  if constexpr (FOR_KEYS) {
    if (a.dtable) {
      // The sums for the table cost stages of the ring; the last shape holds the most buckets there can be.
      auto fits = [&](int ring_end, int parts) { return 1024 + ring_end + bwd_rest(a, true, parts).total <= kMaxDynamicSmem; };
      if (a.dim <= kBlockCols) {
        if (fits(BwdShape<1, 4>::kRest, 4)) return DLB_PICK(1, 4, 4, kTable);
        if (fits(BwdShape<1, 2>::kRest, 4)) return DLB_PICK(1, 2, 4, kTable);
        return DLB_PICK(1, 2, 2, kTable);
      }
      if (fits(BwdShape<2, 2>::kRest, 4)) return DLB_PICK(2, 2, 4, kTable);
      if (fits(BwdShape<2, 1>::kRest, 4)) return DLB_PICK(2, 1, 4, kTable);
      return DLB_PICK(2, 1, 2, kTable);
    }
  }
  if (a.dim <= kBlockCols) {
    if (a.table) return DLB_PICK(1, 4, 4, kTable);
    return a.slopes ? DLB_PICK(1, 4, 4, kSlope) : DLB_PICK(1, 4, 4, kNoBias);
  }
  if (a.table) return DLB_PICK(2, 2, 4, kTable);
  return a.slopes ? DLB_PICK(2, 2, 4, kSlope) : DLB_PICK(2, 2, 4, kNoBias);
#undef DLB_PICK
}

}  // namespace dlb
