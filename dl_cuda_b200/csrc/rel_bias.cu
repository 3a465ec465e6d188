// Learned relative position bias by buckets for programs that hold scores as a matrix: the add in
// front of the softmax, and the gradient of the table.  Over 2 x 16 heads of 2048 x 2048 fp32 the add takes
// 161 us (6.6 TB/s, the copy peak), the gradient 115 us (4.7 TB/s).  A thread's and a CTA's sums are fp32,
// 4 bytes of shared memory for each of 256 threads and each bucket, the sum of the CTAs fp64: 2e-7 from the
// exact gradient.
#include <algorithm>
#include <cmath>

#include "attn_common.cuh"

namespace dlb {
namespace {

constexpr int kBiasThreads = 256;

struct BiasArgs {
  const void *in;  // scores (may be NULL) or dscores
  const float *table;
  const int *bucket_of;
  void *out;
  float *part;
  int batch, heads, q_len, kv_len, start, buckets, reach;
};

__device__ __forceinline__ int bias_bucket(const BiasArgs &a, int distance) {
  const int d = max(-a.reach, min(a.reach, distance)) + a.reach;
  return min(max(a.bucket_of[d], 0), a.buckets - 1);
}

// A row is taken by one warp, 16 bytes a lane and four such loads in flight; a row that starts off the
// 16-byte grid (odd kv_len) has up to V - 1 single elements in front and behind.
template <typename T>
struct RowCut {
  static constexpr int V = Store<T>::kPerVec;
  int head, vectors, tail;  // elements in front, 16-byte vectors, elements behind
  __device__ __forceinline__ RowCut(const T *row, int n, bool vec) {
    head = vec ? min(n, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / static_cast<int>(sizeof(T))) : n;
    vectors = (n - head) / V;
    tail = n - head - vectors * V;
  }
};

constexpr int kBiasRows = 32;  // rows of a CTA: four per warp

template <typename T>
__global__ void __launch_bounds__(kBiasThreads) rel_bias_fwd_kernel(const __grid_constant__ BiasArgs a, bool vec) {
  pdl_prologue();
  extern __shared__ float by_distance[];
  constexpr int V = Store<T>::kPerVec, kInFlight = 4;
  const int row_tiles = (a.q_len + kBiasRows - 1) / kBiasRows;
  const int tile = blockIdx.x % row_tiles, h = (blockIdx.x / row_tiles) % a.heads, b = blockIdx.x / (row_tiles * a.heads);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int d = threadIdx.x; d <= 2 * a.reach; d += kBiasThreads)
    by_distance[d] = a.table[h * a.buckets + bias_bucket(a, d - a.reach)];
  __syncthreads();
  const int i1 = min(a.q_len, (tile + 1) * kBiasRows);
  for (int i = tile * kBiasRows + warp; i < i1; i += kBiasThreads / 32) {
    const size_t row = (static_cast<size_t>(b) * a.heads + h) * a.q_len + i;
    const T *src = a.in ? static_cast<const T *>(a.in) + row * a.kv_len : nullptr;
    T *dst = static_cast<T *>(a.out) + row * a.kv_len;
    const int shift = a.reach - (a.start + i);  // by_distance of column j is at j + shift, within 0..2 reach
    auto bias_at = [&](int j) { return by_distance[max(0, min(2 * a.reach, j + shift))]; };
    const RowCut<T> cut(dst, a.kv_len, vec);
    for (int e = lane; e < cut.head + cut.tail; e += 32) {
      const int j = e < cut.head ? e : cut.vectors * V + e;
      dst[j] = Store<T>::from_float((src ? Store<T>::to_float(ld_co(src + j)) : 0.f) + bias_at(j));
    }
    for (int v0 = lane; v0 < cut.vectors; v0 += 32 * kInFlight) {
      uint4 x[kInFlight];
#pragma unroll
      for (int k = 0; k < kInFlight; k++) {
        const int v = v0 + 32 * k;
        x[k] = src && v < cut.vectors ? ld_stream(src + cut.head + v * V) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < kInFlight; k++) {
        const int v = v0 + 32 * k, j = cut.head + v * V;
        if (v >= cut.vectors) break;
        float f[V];
        Store<T>::unpack(x[k], f);
        if (j + V - 1 + shift <= 0 || j + shift >= 2 * a.reach) {  // beyond the reach: one value
          const float far = bias_at(j);
#pragma unroll
          for (int e = 0; e < V; e++) f[e] += far;
        } else {
#pragma unroll
          for (int e = 0; e < V; e++) f[e] += bias_at(j + e);
        }
        st_stream(dst + j, Store<T>::pack(f));
      }
    }
  }
}

// part[h][cta][bucket]: a CTA takes rows of one head of all batches.  What lies beyond the reach has one
// bucket on either side and is summed in two registers; nearer elements go to a column of their own
// thread per bucket in shared memory.
template <typename T>
__global__ void __launch_bounds__(kBiasThreads) rel_bias_bwd_kernel(const __grid_constant__ BiasArgs a, int parts) {
  pdl_prologue();
  extern __shared__ float sums[];  // [buckets][threads], then the bucket of every distance
  constexpr int V = Store<T>::kPerVec, kInFlight = 4, kWarps = kBiasThreads / 32;
  unsigned char *bucket_lut = reinterpret_cast<unsigned char *>(sums + a.buckets * kBiasThreads);
  const int part = blockIdx.x % parts, h = blockIdx.x / parts, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  for (int n = 0; n < a.buckets; n++) sums[n * kBiasThreads + tid] = 0.f;
  for (int d = tid; d <= 2 * a.reach; d += kBiasThreads) bucket_lut[d] = static_cast<unsigned char>(bias_bucket(a, d - a.reach));
  __syncthreads();
  float left = 0.f, right = 0.f;
  const long long rows = static_cast<long long>(a.batch) * a.q_len;
  for (long long r = static_cast<long long>(part) * kWarps + warp; r < rows; r += static_cast<long long>(parts) * kWarps) {
    const int b = r / a.q_len, i = r % a.q_len;
    const T *src = static_cast<const T *>(a.in) + ((static_cast<size_t>(b) * a.heads + h) * a.q_len + i) * a.kv_len;
    const int shift = a.reach - (a.start + i);
    auto add = [&](int j, float x) { sums[bucket_lut[max(0, min(2 * a.reach, j + shift))] * kBiasThreads + tid] += x; };
    const RowCut<T> cut(src, a.kv_len, true);
    for (int e = lane; e < cut.head + cut.tail; e += 32) {
      const int j = e < cut.head ? e : cut.vectors * V + e;
      add(j, Store<T>::to_float(ld_co(src + j)));
    }
    for (int v0 = lane; v0 < cut.vectors; v0 += 32 * kInFlight) {
      uint4 x[kInFlight];
#pragma unroll
      for (int k = 0; k < kInFlight; k++) {
        const int v = v0 + 32 * k;
        x[k] = v < cut.vectors ? ld_stream(src + cut.head + v * V) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < kInFlight; k++) {
        const int v = v0 + 32 * k, j = cut.head + v * V;
        if (v >= cut.vectors) break;
        float f[V];
        Store<T>::unpack(x[k], f);
        const bool far_left = j + V - 1 + shift <= 0, far_right = j + shift >= 2 * a.reach;
        if (far_left || far_right) {
          float s = 0.f;
#pragma unroll
          for (int e = 0; e < V; e++) s += f[e];
          if (far_left) left += s;
          else right += s;
        } else {
#pragma unroll
          for (int e = 0; e < V; e++) add(j + e, f[e]);
        }
      }
    }
  }
  sums[bucket_lut[0] * kBiasThreads + tid] += left;
  sums[bucket_lut[2 * a.reach] * kBiasThreads + tid] += right;
  __syncthreads();
  for (int n = warp; n < a.buckets; n += kWarps) {
    float s = 0.f;
    for (int t = lane; t < kBiasThreads; t += 32) s += sums[n * kBiasThreads + t];
    s = warp_sum(s);
    if (lane == 0) a.part[(static_cast<size_t>(h) * parts + part) * a.buckets + n] = s;
  }
}

__global__ void __launch_bounds__(128) rel_bias_sum_kernel(const float *part, float *out, int parts, int buckets) {
  pdl_prologue();
  __shared__ double warp_part[4];
  const int h = blockIdx.x / buckets, n = blockIdx.x % buckets;
  double sum = 0.0;
  for (int p = threadIdx.x; p < parts; p += 128) sum += ld_co(part + (static_cast<size_t>(h) * parts + p) * buckets + n);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x / 32] = sum;
  __syncthreads();
  if (threadIdx.x == 0) out[blockIdx.x] = static_cast<float>(warp_part[0] + warp_part[1] + warp_part[2] + warp_part[3]);
}

int check_shape(const char *call, int batch, int heads, int q_len, int kv_len, int q_start, int buckets, int reach, int dtype) {
  DLB_REQUIRE(batch >= 0 && heads >= 0 && q_len >= 0 && kv_len >= 0 && buckets > 0 && reach >= 0, DLB_ERR_INVALID_ARG,
              "%s: batch=%d heads=%d q_len=%d kv_len=%d buckets=%d max_distance=%d", call, batch, heads, q_len, kv_len,
              buckets, reach);
  DLB_REQUIRE(dtype == DLB_F32 || dtype == DLB_BF16, DLB_ERR_INVALID_ARG, "%s: dtype=%d", call, dtype);
  DLB_REQUIRE(buckets <= DLB_ATTN_MAX_BUCKETS && reach <= DLB_ATTN_MAX_DISTANCE, DLB_ERR_UNSUPPORTED,
              "%s: buckets=%d (at most %d), max_distance=%d (at most %d)", call, buckets, DLB_ATTN_MAX_BUCKETS, reach,
              DLB_ATTN_MAX_DISTANCE);
  constexpr int kMax = 1 << 29;
  DLB_REQUIRE(q_len <= kMax && kv_len <= kMax && q_start >= -2 * kMax && q_start <= 2 * kMax, DLB_ERR_UNSUPPORTED,
              "%s: q_len=%d kv_len=%d q_start=%d", call, q_len, kv_len, q_start);
  DLB_REQUIRE(static_cast<long long>(batch) * heads * q_len < (1ll << 31), DLB_ERR_UNSUPPORTED,
              "%s: batch=%d heads=%d q_len=%d make too many rows", call, batch, heads, q_len);
  return DLB_OK;
}

// Row groups of a head: enough CTAs for six per SM, with a row for each warp.
int bias_parts(int batch, int heads, int q_len) {
  const long long rows = static_cast<long long>(batch) * q_len;
  return static_cast<int>(std::max(1ll, std::min<long long>(ceil_div(rows, 8ll), ceil_div(6 * sm_count(), std::max(heads, 1)))));
}

// Can 16-byte accesses be used between the ragged ends of rows?  What is read and written has to have the
// same place within 16 bytes.
bool rows_can_be_cut(const void *p, const void *q) {
  return q == nullptr || reinterpret_cast<uintptr_t>(p) % 16 == reinterpret_cast<uintptr_t>(q) % 16;
}
int esize_of(int dtype) { return dtype == DLB_F32 ? 4 : 2; }

}  // namespace
}  // namespace dlb

using namespace dlb;

extern "C" int dlb_rel_bucket_map_host(int32_t *h_bucket_of, int buckets, int max_distance, int both_directions) {
  DLB_REQUIRE(h_bucket_of != nullptr, DLB_ERR_INVALID_ARG, "rel_bucket_map: null pointer");
  const int each = both_directions ? buckets / 2 : buckets;
  const int own = each / 2;  // distances with a bucket of their own
  DLB_REQUIRE(buckets > 0 && own >= 1 && (!both_directions || buckets % 2 == 0) && max_distance > own, DLB_ERR_INVALID_ARG,
              "rel_bucket_map: buckets=%d max_distance=%d both_directions=%d", buckets, max_distance, both_directions);
  DLB_REQUIRE(buckets <= DLB_ATTN_MAX_BUCKETS && max_distance <= DLB_ATTN_MAX_DISTANCE, DLB_ERR_UNSUPPORTED,
              "rel_bucket_map: buckets=%d (at most %d), max_distance=%d (at most %d)", buckets, DLB_ATTN_MAX_BUCKETS,
              max_distance, DLB_ATTN_MAX_DISTANCE);
  const int wide = each - own;
  auto of = [&](int distance) {
    if (distance < own) return distance;
    // log spacing; 1e-9 puts a border that falls on a whole distance into the upper bucket whatever log rounds to
    const double at = std::log(static_cast<double>(distance) / own) / std::log(static_cast<double>(max_distance) / own) * wide;
    return own + std::min(wide - 1, static_cast<int>(std::floor(at + 1e-9)));
  };
  for (int r = -max_distance; r <= max_distance; r++)
    h_bucket_of[r + max_distance] = both_directions ? (r <= 0 ? of(-r) : each + of(r)) : of(std::max(-r, 0));
  return DLB_OK;
}

extern "C" int dlb_rel_bias_fwd(const void *scores, const float *table, const int32_t *bucket_of, void *out, int batch,
                                int heads, int q_len, int kv_len, int q_start, int buckets, int max_distance, int dtype,
                                void *stream) {
  if (int st = check_shape("rel_bias_fwd", batch, heads, q_len, kv_len, q_start, buckets, max_distance, dtype)) return st;
  if (batch == 0 || heads == 0 || q_len == 0 || kv_len == 0) return DLB_OK;
  DLB_REQUIRE(table && bucket_of && out, DLB_ERR_INVALID_ARG, "rel_bias_fwd: null pointer");
  DLB_REQUIRE(on_elements(scores, esize_of(dtype)) && on_elements(out, esize_of(dtype)) && on_elements(table, 4) && on_elements(bucket_of, 4),
              DLB_ERR_INVALID_ARG, "rel_bias_fwd: an address is not on an element");
  BiasArgs a = {scores, table, bucket_of, out, nullptr, batch, heads, q_len, kv_len, q_start, buckets, max_distance};
  const bool vec = rows_can_be_cut(out, scores);
  const dim3 grid(ceil_div(q_len, kBiasRows) * heads * batch);
  const size_t smem = sizeof(float) * (2 * max_distance + 1);
  auto kern = dtype == DLB_F32 ? rel_bias_fwd_kernel<float> : rel_bias_fwd_kernel<__nv_bfloat16>;
  launch_pdl(kern, grid, dim3(kBiasThreads), smem, as_stream(stream), a, vec);
  DLB_LAUNCH_CHECK("rel_bias_fwd");
  return DLB_OK;
}

extern "C" size_t dlb_rel_bias_bwd_workspace_bytes(int batch, int heads, int q_len, int kv_len, int buckets) {
  if (check_shape("rel_bias_bwd", batch, heads, q_len, kv_len, 0, buckets, 0, DLB_F32) != DLB_OK) return 0;
  return sizeof(float) * static_cast<size_t>(heads) * bias_parts(batch, heads, q_len) * buckets;
}

extern "C" int dlb_rel_bias_bwd(const void *dscores, const int32_t *bucket_of, float *dtable, void *workspace,
                                size_t workspace_bytes, int batch, int heads, int q_len, int kv_len, int q_start,
                                int buckets, int max_distance, int dtype, void *stream) {
  if (int st = check_shape("rel_bias_bwd", batch, heads, q_len, kv_len, q_start, buckets, max_distance, dtype)) return st;
  if (heads == 0) return DLB_OK;
  const bool empty = batch == 0 || q_len == 0 || kv_len == 0;
  DLB_REQUIRE((dscores || empty) && bucket_of && dtable, DLB_ERR_INVALID_ARG, "rel_bias_bwd: null pointer");
  DLB_REQUIRE(on_elements(dscores, esize_of(dtype)) && on_elements(dtable, 4) && on_elements(bucket_of, 4), DLB_ERR_INVALID_ARG,
              "rel_bias_bwd: an address is not on an element");
  const size_t need = dlb_rel_bias_bwd_workspace_bytes(batch, heads, q_len, kv_len, buckets);
  DLB_REQUIRE(workspace != nullptr && workspace_bytes >= need && aligned16(workspace), DLB_ERR_WORKSPACE,
              "rel_bias_bwd: workspace of %zu bytes (16-byte aligned) needed, %zu given", need, workspace_bytes);
  const int parts = bias_parts(batch, heads, q_len);
  BiasArgs a = {dscores, nullptr, bucket_of, nullptr, static_cast<float *>(workspace), batch, heads, q_len, kv_len,
                q_start, buckets, max_distance};
  const size_t smem = sizeof(float) * buckets * kBiasThreads + 2 * max_distance + 1;
  auto kern = dtype == DLB_F32 ? rel_bias_bwd_kernel<float> : rel_bias_bwd_kernel<__nv_bfloat16>;
  if (int rc = allow_smem(kern, smem, "rel_bias_bwd")) return rc;
  launch_pdl(kern, dim3(heads * parts), dim3(kBiasThreads), smem, as_stream(stream), a, parts);
  DLB_LAUNCH_CHECK("rel_bias_bwd");
  launch_pdl(rel_bias_sum_kernel, dim3(heads * buckets), dim3(128), 0, as_stream(stream),
             static_cast<const float *>(a.part), dtable, parts, buckets);
  DLB_LAUNCH_CHECK("rel_bias_sum");
  return DLB_OK;
}
