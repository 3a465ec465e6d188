// Attention forward on the tensor cores (bf16).
//
// A CTA owns two tiles of 128 queries of one head and walks over the tiles of 128 keys that any of
// them sees.  One warp copies K and V tiles into a ring (TMA), one issues the products, and each
// query tile has eight warps for its softmax:
//     S = Q K^T (TMEM, fp32) -> scores s -> P = 2^(s - m) (bf16, written over S) -> O += P V
// The two query tiles take turns: while one's softmax runs, the other's products do.  O stays in TMEM.
// Exponentials are taken against a reference that moves only when a score leaves its range of 2^32, so
// no maximum stands between a score and its exponential, and O is hardly ever rescaled; keys are walked
// from where the queries stand outwards, so that a distance bias shows its largest scores at once (from
// the far end of a prefix, every tile moved the reference: 64 instead of 53 us for 3 x 1531 tokens).
// Probabilities are rounded to bf16, the operand type of the second product: in two bf16 parts they would
// need that product twice.  The sum behind the quotient adds the ROUNDED ones, so that a row's weights add
// up to one exactly as the product sees them (one prompt's output 1.9e-3 instead of 2.3e-3 from the exact
// one, 1.9e-3 to 2.4e-3 over 150 random cases, of which the output's own rounding is 1.7e-3); lse comes from
// the unrounded ones.
//
// Measured (4096 tokens, 32 heads of 128 on 8 key heads): 268 us, 1.03 PFLOP/s, of the 1.66 that the
// library's plain product reaches; causal 147 us, causal with a cap 184 us (205 us from a cold L2).
// By the clock a pair of tiles takes 3500 cycles where the tensor cores need 2470 of issue: a tile's own
// chain of scores, softmax (1700 cycles a tile, half of which are exponentials) and product is what remains,
// since TMEM has no room for a second S.
// Taking a quarter of the exponentials as polynomials on the fp32 pipes changed nothing (275 us).
#include <algorithm>

#include "attn_mma.cuh"

namespace dlb {
namespace {

// Eight softmax warps per query tile: a row belongs to two threads, 64 of a tile's 128 keys each.  (With
// one thread a row, two warps a scheduler, nothing covered the latencies: 288 instead of 272 us
// for 4096 x 4096 tokens, 32 heads of 128.)
constexpr int kLoadWarp = 16, kMmaWarp = 17, kFwdThreads = 640, kHalf = kTileRows / 2;
// Registers: launched with 96 each (640 * 96 = 61440); the softmax warps go up to 104, the four others
// down to 64 (512 * 104 + 128 * 64 = 61440).
constexpr int kSoftmaxRegs = 104, kOtherRegs = 64;
// A row's exponentials are taken against a reference m that its scores (in powers of two) have to stay
// within 2^32 of from above; fp32 sums and bf16 probabilities bear that with room to spare, and the
// reference divides out.  It starts at 0, which serves most rows from end to end.
constexpr float kReach = 32.f;
// A sum under this may have lost weights to underflow (or has none): 2^26 times the smallest it can hold.
constexpr float kNothing = 1e-30f;

template <int NB>
struct FwdShape {
  static constexpr int kStages = NB == 2 ? 2 : 3;
  static constexpr int kTileBytes = NB * kBlockBytes;
  static constexpr int kRing = 2 * kTileBytes;                       // behind the two Q tiles
  static constexpr int kLut = kRing + 2 * kStages * kTileBytes;      // K ring, V ring
};

struct FwdMaps {
  CUtensorMap q, k, v;
};

// Barrier of a query tile's 256 softmax threads that also tells whether any of them says yes.
__device__ __forceinline__ bool any_of_group(int id, bool yes) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbarrier.cta.red.or.pred q, %1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(id), "r"(static_cast<uint32_t>(yes))
      : "memory");
  return any != 0;
}

template <int NB, bool CAP, int BIAS>
__global__ void __launch_bounds__(kFwdThreads, 1)
attn_fwd_mma_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ FwdMaps maps, unsigned int *timeouts) {
  using Shape = FwdShape<NB>;
  constexpr int ST = Shape::kStages;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  unsigned char *ks = smem + Shape::kRing, *vs = ks + ST * Shape::kTileBytes;
  float *lut = reinterpret_cast<float *>(smem + Shape::kLut);
  unsigned char *flags = smem + Shape::kLut + (BIAS == kTable ? sizeof(float) * lut_floats(a.reach) : 0);
  __shared__ uint64_t q_full, k_full[ST], k_empty[ST], v_full[ST], v_empty[ST], s_full[2], p_full[2], o_full[2], drain;
  __shared__ uint32_t tmem_slot;
  __shared__ int dead_flag;
  __shared__ int doc_range[4];
  __shared__ __align__(16) int doc_tile[2][kTileRows];
  __shared__ float redo_top[2][2][kTileRows], redo_sum[2][2][kTileRows];  // [query tile][half][row]
  volatile int *dead = &dead_flag;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    mbar_init(&q_full, 1);
    for (int s = 0; s < ST; s++) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int t = 0; t < 2; t++) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 8);
      mbar_init(&o_full[t], 1);
    }
    mbar_init(&drain, 1);
    dead_flag = 0;
    mbar_fence_init();
  }
  if (warp == kMmaWarp) tmem_alloc(&tmem_slot, 512);
  if (tid == kLoadWarp * 32) {
    prefetch_map(&maps.q);
    prefetch_map(&maps.k);
    prefetch_map(&maps.v);
  }
  pdl_prologue();

  // Pairs of query tiles are the slowest index, last pair first: long causal rows start early, and the
  // heads that share keys run at the same time.
  const int pairs = (a.q_len + 2 * kTileRows - 1) / (2 * kTileRows), per_pair = a.heads * a.batch;
  const int pair = pairs - 1 - static_cast<int>(blockIdx.x) / per_pair;
  const int h = blockIdx.x % a.heads, b = (blockIdx.x / a.heads) % a.batch, hk = h / a.group;
  const int row0 = pair * 2 * kTileRows;
  const BatchView view = batch_view(a, b);

  // flags[n]: bit 2t: tile t sees some of key tile n; bit 2t + 1: every row of it sees all of it.
  int first_end[2], last_end[2];
#pragma unroll
  for (int t = 0; t < 2; t++) {
    const int r0 = row0 + t * kTileRows, r1 = min(a.q_len, r0 + kTileRows) - 1;
    first_end[t] = r0 < a.q_len ? row_end(a, view, r0) : 0;
    last_end[t] = r0 < a.q_len ? row_end(a, view, r1) : 0;
  }
  const int n_tiles = (max(last_end[0], last_end[1]) + kTileRows - 1) / kTileRows;
  // This CTA's share of them (blockIdx.y), from the tile where the queries stand to the first, then on
  // from there: the nearest keys first.
  const int share = (n_tiles + a.splits - 1) / a.splits;
  const int n_first = min(n_tiles, static_cast<int>(blockIdx.y) * share), n_last = min(n_tiles, n_first + share);
  const int n_count = n_last - n_first;
  const int here = max(n_first, min(n_last - 1, (view.start + min(a.q_len, row0 + 2 * kTileRows) - 1) / kTileRows));
  auto walk = [&](int k) { return k <= here - n_first ? here - k : n_first + k; };
  if (a.q_docs) {
    if (warp < 2) {
      int lo = INT_MAX, hi = INT_MIN;
      for (int r = row0 + warp * kTileRows + lane; r < min(a.q_len, row0 + (warp + 1) * kTileRows); r += 32) {
        const int d = ld_co(a.q_docs + static_cast<long long>(b) * a.q_len + r);
        lo = min(lo, d);
        hi = max(hi, d);
      }
      lo = warp_min(lo);
      hi = warp_max(hi);
      if (lane == 0) {
        doc_range[2 * warp] = lo;
        doc_range[2 * warp + 1] = hi;
      }
    }
    __syncthreads();
  }
  for (int n = n_first + warp; n < n_last; n += kFwdThreads / 32) {
    const int j0 = n * kTileRows;
    int lo = 0, hi = 0;
    if (a.kv_docs) {
      lo = INT_MAX;
      hi = INT_MIN;
      for (int j = j0 + lane; j < min(view.end, j0 + kTileRows); j += 32) {
        const int d = ld_co(a.kv_docs + static_cast<long long>(b) * a.kv_len + j);
        lo = min(lo, d);
        hi = max(hi, d);
      }
      lo = warp_min(lo);
      hi = warp_max(hi);
    }
    int f = 0;
#pragma unroll
    for (int t = 0; t < 2; t++) {
      bool active = j0 < last_end[t], full = j0 + kTileRows <= first_end[t];
      if (a.kv_docs) {
        const int qlo = doc_range[2 * t], qhi = doc_range[2 * t + 1];
        active = active && lo <= qhi && qlo <= hi;
        full = full && lo == hi && qlo == qhi && lo == qlo;
      }
      if (active) f |= (full ? 3 : 1) << (2 * t);
    }
    if (lane == 0) flags[n] = static_cast<unsigned char>(f);
  }
  if (BIAS == kTable) fill_lut(lut, a, h, tid, kFwdThreads);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp < kLoadWarp) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int t = warp >> 3, half = warp >> 2 & 1, row = (warp & 3) * 32 + lane, i = row0 + t * kTileRows + row;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lane_base + t * 128 + half * kHalf;  // this thread's scores
    const uint32_t p_at = tmem + lane_base + t * 128 + half * (kHalf / 2), o_at = tmem + lane_base + 256 + t * 128;
    const bool valid = i < a.q_len;
    const int end = valid ? row_end(a, view, i) : 0, pos = view.start + i;
    const int doc = (a.q_docs && valid) ? ld_co(a.q_docs + static_cast<long long>(b) * a.q_len + i) : 0;
    const float slope = (BIAS != kNoBias && a.slopes) ? ld_co(a.slopes + h) * kLog2e : 0.f;
    const float to_log2 = CAP ? 1.f : a.scale * kLog2e;
    const CapCoef cap = CAP ? cap_coef(a.scale, a.cap) : CapCoef();
    constexpr bool kRaw = !CAP && BIAS == kNoBias;  // the exponent straight from the products
    const int tail = view.end % kTileRows && view.end < a.kv_len ? view.end / kTileRows : -1;

    // Scores of 32 keys from j1 on, masked; times to_log2 still to come when kRaw.
    auto scores = [&](float (&x)[32], int c, int j1, bool whole) {
      uint32_t raw[32];
      tmem_load32(s_at + c * 32, raw);
      tmem_loaded(raw);
#pragma unroll
      for (int e = 0; e < 32; e++) x[e] = __uint_as_float(raw[e]);
      if (CAP) cap_scores(x, cap);
      if (BIAS != kNoBias) {
        const int d0 = j1 - pos;
        const float d = static_cast<float>(d0);
        const bool slopes = BIAS == kSlope || a.slopes;
        bool far = true;
        const float *at = lut + d0 + a.reach + kLutPad;
        float base = 0.f;
        if (BIAS == kTable) {
          // Either the warp's pairs are all beyond the reach, or all within 31 + 31 of it on either side,
          // where the padded table covers every index.
          const bool left = d0 + 31 <= -a.reach, right = d0 >= a.reach;
          far = __all_sync(0xffffffffu, left || right);
          if (far) base = left ? lut[0] : lut[2 * (a.reach + kLutPad)];
        }
        if (far && !slopes) {
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 y = fma2(make_float2(x[e], x[e + 1]), both(to_log2), both(base));
            x[e] = y.x;
            x[e + 1] = y.y;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float2 bias = BIAS == kTable && !far ? make_float2(at[e], at[e + 1]) : both(base);
            if (slopes) {
              bias.x = fmaf(-slope, fabsf(d + static_cast<float>(e)), bias.x);
              bias.y = fmaf(-slope, fabsf(d + static_cast<float>(e + 1)), bias.y);
            }
            const float2 y = fma2(make_float2(x[e], x[e + 1]), both(to_log2), bias);
            x[e] = y.x;
            x[e + 1] = y.y;
          }
        }
      }
      if (!whole) {
        const int room = end - j1;
        if (a.kv_docs) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const int4 k = *reinterpret_cast<const int4 *>(&doc_tile[t][half * kHalf + c * 32 + e]);
            x[e] = k.x == doc ? x[e] : -INFINITY;
            x[e + 1] = k.y == doc ? x[e + 1] : -INFINITY;
            x[e + 2] = k.z == doc ? x[e + 2] : -INFINITY;
            x[e + 3] = k.w == doc ? x[e + 3] : -INFINITY;
          }
        }
        if (room < 32) {
#pragma unroll
          for (int e = 0; e < 32; e++) x[e] = e < room ? x[e] : -INFINITY;
        }
      }
    };

    float m = 0.f, sum = 0.f, sum_rounded = 0.f;
    bool settled = false;  // the row has weight, or a reference of its own
    int it = -1, done = 0;
    for (int k = 0; k < n_count; k++) {
      const int n = walk(k);
      const int f = flags[n];
      if (!f) continue;
      it++;
      if (!(f >> (2 * t) & 1)) continue;
      const int j0 = n * kTileRows, j1 = j0 + half * kHalf;
      const bool whole = f >> (2 * t + 1) & 1;
      int key_doc = 0;
      if (!whole && a.kv_docs && half == 0)
        key_doc = ld_co(a.kv_docs + static_cast<long long>(b) * a.kv_len + min(j0 + row, a.kv_len - 1));
      mbar_wait(&s_full[t], done & 1, dead, timeouts);
      if (!whole && a.kv_docs) {  // the tile's document numbers; the last use of the old ones lies behind a barrier
        if (half == 0) doc_tile[t][row] = key_doc;
        named_bar_sync(2 + t, 256);
      }
      tc_fence_after();
      // One pass over the scores against the reference, which the keys so far fit.  Only if some row's
      // sum says that it may not (too large, or nothing left of visible keys) the maximum is taken, the
      // reference moved where that is out of its range, what has been summed rescaled, and the pass repeated.
      // (A sum above 2^32 of many weights that are all below it repeats the pass and moves nothing: the
      // result is the same, the softmax of such a tile takes three times as long.)
      uint32_t packed[32];
      float2 part, part_rounded;
      for (int pass = 0;; pass++) {
        float2 l[2] = {both(0.f), both(0.f)}, r[2] = {both(0.f), both(0.f)};
#pragma unroll
        for (int c = 0; c < 2; c++) {
          float x[32];
          scores(x, c, j1 + c * 32, whole);
          const float2 minus = both(-m);
#pragma unroll
          for (int e = 0; e < 16; e++) {
            const float2 v = make_float2(x[2 * e], x[2 * e + 1]);
            const float2 y = kRaw ? fma2(v, both(to_log2), minus) : add2(v, minus);
            const float2 p = make_float2(ex2(y.x), ex2(y.y));
            const uint32_t w = pack_bf16(p.x, p.y);
            packed[c * 16 + e] = w;
            l[e & 1] = add2(l[e & 1], p);
            r[e & 1] = add2(r[e & 1], make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)));
          }
        }
        part = add2(l[0], l[1]);
        part_rounded = add2(r[0], r[1]);
        const float total = part.x + part.y;
        if (total >= kNothing) settled = true;
        const bool misfit = !(total <= 4294967296.f) || (!settled && end > j1);
        if (!any_of_group(4 + t, misfit) || pass == 1) break;
        float top = -INFINITY;
        for (int c = 0; c < 2; c++) {
          float x[32];
          scores(x, c, j1 + c * 32, whole);
          top = fmaxf(top, max_of<32, false>(x));
        }
        if (kRaw) top *= to_log2;
        redo_top[t][half][row] = top;
        redo_sum[t][half][row] = sum;
        named_bar_sync(2 + t, 256);
        top = fmaxf(top, redo_top[t][half ^ 1][row]);
        const float row_sum = sum + redo_sum[t][half ^ 1][row];
        named_bar_sync(2 + t, 256);
        const bool above = top > m + kReach, below = row_sum < kNothing && top < m - kReach && top > -INFINITY;
        const float keep = above ? ex2(m - top) : below ? 0.f : 1.f;
        if (above || below) m = top;
        settled = settled || row_sum >= kNothing || top > -INFINITY;
        sum *= keep;
        sum_rounded *= keep;
        if (done > 0) {
          for (int c = half * 32; c < a.dim; c += 64) {
            uint32_t o[32];
            tmem_load32(o_at + c, o);
            tmem_loaded(o);
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float2 y = mul2(make_float2(__uint_as_float(o[e]), __uint_as_float(o[e + 1])), both(keep));
              o[e] = __float_as_uint(y.x);
              o[e + 1] = __float_as_uint(y.y);
            }
            tmem_store32(o_at + c, o);
          }
        }
      }
      // All of the tile's scores have been read (any_of_group is a barrier): P may go over them.
      tmem_store32(p_at, packed);
      sum += part.x + part.y;
      sum_rounded += part_rounded.x + part_rounded.y;
      if (n == tail) {
        // Rows of V behind the last key any query reaches may hold anything, and 0 * NaN is NaN.
        const int s = it % ST;
        mbar_wait(&v_full[s], (it / ST) & 1, dead, timeouts);
        const int from = view.end - j0;
        for (int e = half * 128 + row; e < (kTileRows - from) * NB * 8; e += 256) {
          const int r = from + e / (NB * 8), x = e % (NB * 8);
          *reinterpret_cast<uint4 *>(vs + s * Shape::kTileBytes + (x / 8) * kBlockBytes + r * 128 + (x % 8) * 16) =
              make_uint4(0, 0, 0, 0);
        }
        fence_async_smem();
      }
      tmem_stored();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[t]);
      done++;
    }
    redo_top[t][half][row] = sum_rounded;
    redo_sum[t][half][row] = sum;
    named_bar_sync(2 + t, 256);
    sum += redo_sum[t][half ^ 1][row];
    sum_rounded += redo_top[t][half ^ 1][row];
    if (done > 0) mbar_wait(&o_full[t], 0, dead, timeouts);
    tc_fence_after();
    const bool whole_row = a.splits == 1, any = sum_rounded > 0.f || sum_rounded != sum_rounded;
    // A share's output is kept for a quotient by the unrounded sum, which the join uses.
    const float by = !any ? 0.f : whole_row ? 1.f / sum_rounded : sum / sum_rounded;
    const size_t at = (static_cast<size_t>(b) * a.heads + h) * a.q_len + i;
    const size_t part_at = static_cast<size_t>(blockIdx.y) * a.batch * a.heads * a.q_len + at;
    __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(a.o.ptr) + b * a.o.batch + static_cast<long long>(i) * a.o.token + h * a.o.head;
    for (int c = half * 32; c < a.dim; c += 64) {
      uint32_t o[32];
      if (done > 0) {
        tmem_load32(o_at + c, o);
        tmem_loaded(o);
      }
#pragma unroll
      for (int e = 0; e < 32; e += 8) {
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; k++) f[k] = by == 0.f ? 0.f : __uint_as_float(o[e + k]) * by;
        if (!valid || c + e >= a.dim) continue;
        if (whole_row) {
          *reinterpret_cast<uint4 *>(out + c + e) = Store<__nv_bfloat16>::pack(f);
        } else {
          float4 *to = reinterpret_cast<float4 *>(a.part_o + part_at * a.dim + c + e);
          to[0] = make_float4(f[0], f[1], f[2], f[3]);
          to[1] = make_float4(f[4], f[5], f[6], f[7]);
        }
      }
    }
    if (!whole_row) {
      if (valid && half == 0) a.part_ml[part_at] = make_float2(sum == 0.f ? -INFINITY : m, sum);
    } else if (a.lse && valid && half == 0) {
      a.lse[at] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * kLn2;
    }
    tc_fence_before();
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kLoadWarp) {
      if (lane == 0) {
        const int q_tiles = row0 + kTileRows < a.q_len ? 2 : 1;
        mbar_expect_tx(&q_full, q_tiles * Shape::kTileBytes);
        for (int t = 0; t < q_tiles; t++)
          for (int c = 0; c < NB; c++)
            tma_load_rows(smem + (t * NB + c) * kBlockBytes, &maps.q, &q_full, c * kBlockCols, row0 + t * kTileRows, h, b);
        int it = 0;
        for (int k = 0; k < n_count; k++) {
          const int n = walk(k);
          if (!flags[n]) continue;
          const int s = it % ST;
          const unsigned use = it / ST;
          if (use) mbar_wait(&k_empty[s], (use - 1) & 1, dead, timeouts);
          if (*dead) break;
          mbar_expect_tx(&k_full[s], Shape::kTileBytes);
          for (int c = 0; c < NB; c++)
            tma_load_rows(ks + (s * NB + c) * kBlockBytes, &maps.k, &k_full[s], c * kBlockCols, n * kTileRows, hk, b);
          if (use) mbar_wait(&v_empty[s], (use - 1) & 1, dead, timeouts);
          if (*dead) {
            drain_wait(&k_full[s], use & 1);
            break;
          }
          mbar_expect_tx(&v_full[s], Shape::kTileBytes);
          for (int c = 0; c < NB; c++)
            tma_load_rows(vs + (s * NB + c) * kBlockBytes, &maps.v, &v_full[s], c * kBlockCols, n * kTileRows, hk, b);
          it++;
        }
        // The CTA must not end with copies in flight: after a wait that gave up they are waited for here.
        if (*dead) {
          drain_wait(&q_full, 0);
          for (int i = max(0, it - ST); i < it; i++) {
            drain_wait(&k_full[i % ST], (i / ST) & 1);
            drain_wait(&v_full[i % ST], (i / ST) & 1);
          }
        }
      }
    } else if (warp == kMmaWarp) {
      const int k_steps = (a.dim + 15) / 16, n_cols = k_steps * 16;
      const uint32_t idesc_s = mma_desc(kTileRows, false), idesc_o = mma_desc(n_cols, true);
      const uint64_t q_desc = desc_k_major(smem_u32(smem)), k_desc = desc_k_major(smem_u32(ks));
      const uint64_t v_desc = desc_mn_major(smem_u32(vs), kBlockBytes);
      constexpr uint32_t kTileStep = Shape::kTileBytes >> 4;  // in descriptor units
      bool pending[2] = {false, false}, started[2] = {false, false};
      unsigned p_phase[2] = {0, 0};
      auto issue_pv = [&](int t, int s) {  // O_t += P_t V(stage s)
        mbar_wait(&p_full[t], p_phase[t], dead, timeouts);
        p_phase[t] ^= 1;
        tc_fence_after();
        const uint64_t vd = v_desc + s * kTileStep;
        if (elect_lane()) {
#pragma unroll
          for (int k = 0; k < kTileRows / 16; k++)
            mma_ts(tmem + 256 + t * 128, tmem + t * 128 + k * 8, vd + k * (2048 >> 4), idesc_o, started[t] || k > 0);
        }
        __syncwarp();
        started[t] = true;
        pending[t] = false;
      };
      auto commit = [&](uint64_t *bar) {
        if (elect_lane()) tc_commit(bar);
        __syncwarp();
      };
      mbar_wait(&q_full, 0, dead, timeouts);
      int it = 0;
      for (int k = 0; k < n_count; k++) {
        const int n = walk(k);
        const int f = flags[n];
        if (!f) continue;
        const int s = it % ST, before = (it + ST - 1) % ST;
        mbar_wait(&k_full[s], (it / ST) & 1, dead, timeouts);
        if (it > 0) mbar_wait(&v_full[before], ((it - 1) / ST) & 1, dead, timeouts);
#pragma unroll
        for (int t = 0; t < 2; t++) {
          if (pending[t]) issue_pv(t, before);
          if (f >> (2 * t) & 1) {
            const uint64_t qd = q_desc + t * kTileStep, kd = k_desc + s * kTileStep;
            if (elect_lane()) {
#pragma unroll
              for (int k = 0; k < NB * 4; k++) {
                const int at = (k / 4) * (kBlockBytes >> 4) + (k % 4) * 2;
                if (k < k_steps) mma_ss(tmem + t * 128, qd + at, kd + at, idesc_s, k > 0);
              }
              tc_commit(&s_full[t]);
            }
            __syncwarp();
            pending[t] = true;
          }
        }
        commit(&k_empty[s]);
        if (it > 0) commit(&v_empty[before]);
        it++;
      }
      if (it > 0) {
        const int s = (it - 1) % ST;
        mbar_wait(&v_full[s], ((it - 1) / ST) & 1, dead, timeouts);
#pragma unroll
        for (int t = 0; t < 2; t++) {
          if (pending[t]) issue_pv(t, s);
          if (started[t]) commit(&o_full[t]);
        }
      }
      if (*dead) {
        commit(&drain);
        drain_wait(&drain, 0);
      }
    }
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_free(tmem, 512);
  }
}

}  // namespace

int make_heads_map(CUtensorMap *map, const void *ptr, int dim, int tokens, int heads, int batch, long long token_stride,
                   long long head_stride, long long batch_stride, int rows) {
  using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                              const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<Encode> cached{nullptr};
  Encode encode = cached.load(std::memory_order_acquire);
  if (encode == nullptr) {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found) != cudaSuccess || fn == nullptr)
      return -1;
    encode = reinterpret_cast<Encode>(fn);
    cached.store(encode, std::memory_order_release);
  }
  // A stride of a dimension with one entry is never used: any valid value will do.
  const cuuint64_t row = 16ull * ((dim * 2 + 15) / 16);
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(tokens), static_cast<cuuint64_t>(heads),
                              static_cast<cuuint64_t>(batch)};
  const cuuint64_t strides[3] = {tokens > 1 ? 2ull * token_stride : row, heads > 1 ? 2ull * head_stride : row,
                                 batch > 1 ? 2ull * batch_stride : row};
  const cuuint32_t box[4] = {kBlockCols, static_cast<cuuint32_t>(rows), 1, 1}, ones[4] = {1, 1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(ptr), dims, strides, box, ones,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

namespace {

// A tensor map wants positive strides in multiples of 16 bytes under 2^40; stores want the same grid.
bool grid16(const Heads &h, int tokens, int heads, int batch) {
  auto ok = [](int n, long long s) { return n <= 1 || (s > 0 && s % 8 == 0 && s < (1ll << 38)); };
  return aligned16(h.ptr) && ok(tokens, h.token) && ok(heads, h.head) && ok(batch, h.batch);
}

}  // namespace

bool attn_mma_fits(const AttnArgs &a, bool backward) {
  if (a.dim % 8 != 0 || !(a.scale > 0.f) || a.q_len <= 0 || a.kv_len <= 0) return false;
  if (a.kv_len > kMaxTiles * kTileRows || a.q_len > kMaxTiles * kTileRows) return false;
  if (!grid16(a.q, a.q_len, a.heads, a.batch) || !grid16(a.o, a.q_len, a.heads, a.batch)) return false;
  if (!grid16(a.k, a.kv_len, a.kv_heads, a.batch) || !grid16(a.v, a.kv_len, a.kv_heads, a.batch)) return false;
  if (!backward) return true;
  return grid16(a.dout, a.q_len, a.heads, a.batch) && grid16(a.dq, a.q_len, a.heads, a.batch) &&
         grid16(a.dk, a.kv_len, a.kv_heads, a.batch) && grid16(a.dv, a.kv_len, a.kv_heads, a.batch);
}

int attn_fwd_mma_splits(const AttnArgs &a) {
  // Few queries against many keys: shares of the key tiles fill the GPU once, of four tiles at least.
  const long long ctas = static_cast<long long>(ceil_div(a.q_len, 2 * kTileRows)) * a.heads * a.batch;
  return static_cast<int>(std::max(1ll, std::min({sm_count() / ctas, ceil_div(a.kv_len, kTileRows) / 4ll, 256ll})));
}

int attn_fwd_mma(const AttnArgs &a, cudaStream_t st) {
  FwdMaps maps;
  int rc = make_heads_map(&maps.q, a.q.ptr, a.dim, a.q_len, a.heads, a.batch, a.q.token, a.q.head, a.q.batch, kTileRows);
  if (!rc) rc = make_heads_map(&maps.k, a.k.ptr, a.dim, a.kv_len, a.kv_heads, a.batch, a.k.token, a.k.head, a.k.batch, kTileRows);
  if (!rc) rc = make_heads_map(&maps.v, a.v.ptr, a.dim, a.kv_len, a.kv_heads, a.batch, a.v.token, a.v.head, a.v.batch, kTileRows);
  DLB_REQUIRE(rc == 0, DLB_ERR_CUDA, "attn_fwd: tensor map refused (%d)", rc);
  unsigned int *timeouts = wait_timeouts_counter();
  DLB_REQUIRE(timeouts != nullptr, DLB_ERR_NO_DEVICE, "attn_fwd: no CUDA device");
  const int tiles = ceil_div(a.kv_len, kTileRows);
  auto launch = [&](auto kern, int blocks) -> int {
    const size_t smem = 1024 + (blocks == 2 ? FwdShape<2>::kLut : FwdShape<1>::kLut) +
                        (a.table ? sizeof(float) * lut_floats(a.reach) : 0) + ceil_div(tiles, 16) * 16;
    if (int rc = allow_smem(kern, smem, "attn_fwd")) return rc;
    const int grid = ceil_div(a.q_len, 2 * kTileRows) * a.heads * a.batch;
    launch_pdl(kern, dim3(grid, a.splits), dim3(kFwdThreads), smem, st, a, maps, timeouts);
    DLB_LAUNCH_CHECK("attn_fwd_mma");
    return DLB_OK;
  };
  const int bias = a.table ? kTable : a.slopes ? kSlope : kNoBias;
#define DLB_PICK(NB)                                                                                   \
  (a.cap > 0.f ? (bias == kTable   ? launch(attn_fwd_mma_kernel<NB, true, kTable>, NB)                 \
                  : bias == kSlope ? launch(attn_fwd_mma_kernel<NB, true, kSlope>, NB)                 \
                                   : launch(attn_fwd_mma_kernel<NB, true, kNoBias>, NB))               \
               : (bias == kTable   ? launch(attn_fwd_mma_kernel<NB, false, kTable>, NB)                \
                  : bias == kSlope ? launch(attn_fwd_mma_kernel<NB, false, kSlope>, NB)                \
                                   : launch(attn_fwd_mma_kernel<NB, false, kNoBias>, NB)))
  return a.dim <= kBlockCols ? DLB_PICK(1) : DLB_PICK(2);
#undef DLB_PICK
}

}  // namespace dlb
