// A paged key-value cache: writing new rows, attention of new tokens over it, and its eviction.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"
#include "sample_key.cuh"

namespace wgpt {

constexpr int kErrCache = 5;  // the error word's value for page ids, lengths and row offsets out of range

// The descriptor of a cache as the kernels take it.
struct PagedView {
  void *k, *v;
  const uint32_t *table;
  int *lengths;
  long long page_stride, position_stride, head_stride;
  uint32_t n_pages, page_size;
  int page_shift;  // log2 of the page size, or -1 where it is no power of two
  int n_kv, hs, n_seq, table_stride, max_length;
  int *err;
};

// The new tokens' rows: sequence s has rows starts[s] .. starts[s+1] - 1, or `per` rows each.
struct NewRows {
  const int *starts;
  int n_rows, per;
};

__device__ __forceinline__ int paged_length(const PagedView &c, int s) {
  const int L = __ldcg(c.lengths + s);
  if (L >= 0 && L <= c.max_length) return L;
  *c.err = kErrCache;
  return L < 0 ? 0 : c.max_length;
}

// Rows [first, first + n) of sequence s, inside [0, n_rows) whatever starts says.
__device__ __forceinline__ void new_rows(const PagedView &c, const NewRows &r, int s, int &first, int &n) {
  if (r.starts == nullptr) {
    first = s * r.per;
    n = r.per;
    return;
  }
  const int a = __ldcg(r.starts + s), b = __ldcg(r.starts + s + 1);
  first = min(max(a, 0), r.n_rows);
  n = min(max(b, first), r.n_rows) - first;
  if (a != first || b != first + n) *c.err = kErrCache;
}

// Where a position's rows begin (elements into a pool), or -1 and the error word.
__device__ __forceinline__ long long paged_offset(const PagedView &c, int s, int pos) {
  const uint32_t index = (uint32_t)pos / c.page_size;
  const uint32_t page = __ldcg(c.table + (size_t)s * c.table_stride + index);
  if (page >= c.n_pages) {
    *c.err = kErrCache;
    return -1;
  }
  return (long long)page * c.page_stride + (long long)((uint32_t)pos - index * c.page_size) * c.position_stride;
}

// The sequence that row belongs to, or -1: a warp counts the sequences that end at or before it, 32 at a time.
__device__ __forceinline__ int sequence_of(const PagedView &c, const NewRows &r, int row, int lane) {
  if (r.starts == nullptr) return row / r.per;
  int count = 0;
  for (int s = lane; s < c.n_seq; s += kWarp) count += __ldcg(r.starts + s + 1) <= row ? 1 : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) count += __shfl_xor_sync(0xffffffffu, count, o);
  return count < c.n_seq ? count : -1;
}

template <typename T>
struct Pack4;  // four elements
template <>
struct Pack4<float> {
  float4 v;
  __device__ __forceinline__ static Pack4 of(float4 f) { return {f}; }
};
template <>
struct Pack4<__half> {
  uint2 v;
  __device__ __forceinline__ static Pack4 of(float4 f) {
    const __half2 a = __floats2half2_rn(f.x, f.y), b = __floats2half2_rn(f.z, f.w);
    return {make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b))};
  }
};
template <>
struct Pack4<__nv_bfloat16> {
  uint2 v;
  __device__ __forceinline__ static Pack4 of(float4 f) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(f.x, f.y), b = __floats2bfloat162_rn(f.z, f.w);
    return {make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b))};
  }
};

// ------------------------------------------------------------------------------------------ new rows into the pages
// A CTA takes whole rows; four values a thread and step, k and v side by side.
constexpr int kAppendThreads = 128;

template <typename T>
__global__ void __launch_bounds__(kAppendThreads)
paged_append_kernel(PagedView c, NewRows r, const float *__restrict__ k, const float *__restrict__ v, long long ld) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int per_head = c.hs / 4, n4 = c.n_kv * per_head;
  for (int row = blockIdx.x; row < r.n_rows; row += gridDim.x) {
    const int s = sequence_of(c, r, row, lane);
    if (s < 0) continue;
    int first, n;
    new_rows(c, r, s, first, n);
    const int pos = paged_length(c, s) - n + (row - first);
    if ((unsigned)(row - first) >= (unsigned)n || pos < 0) continue;
    const long long at = paged_offset(c, s, pos);
    if (at < 0) continue;
    const float4 *k4 = reinterpret_cast<const float4 *>(k + (long long)row * ld);
    const float4 *v4 = reinterpret_cast<const float4 *>(v + (long long)row * ld);
    for (int i = threadIdx.x; i < n4; i += kAppendThreads) {
      const int h = i / per_head;
      const long long to = at + (long long)h * c.head_stride + (i - h * per_head) * 4;
      const float4 a = __ldcg(k4 + i), b = __ldcg(v4 + i);
      *reinterpret_cast<Pack4<T> *>(static_cast<T *>(c.k) + to) = Pack4<T>::of(a);
      *reinterpret_cast<Pack4<T> *>(static_cast<T *>(c.v) + to) = Pack4<T>::of(b);
    }
  }
}

// ------------------------------------------------------------------------------------------ selection
// The need-th largest of n 32-bit keys by a CTA of NT threads: digits of 11, 11 and 10 bits from the top, a histogram of each
// digit among the keys that share the digits found so far. Returns the key, and in `ties` how many keys equal to it belong
// to the need largest. hist: 2048 counters in shared memory, warp_sums: NT / 32, found: 3.
template <int NT, typename Key>
__device__ uint32_t radix_threshold(Key key, int n, int need, uint32_t *hist, uint32_t *warp_sums, uint32_t *found,
                                    int &ties) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t prefix = 0, mask = 0, left = (uint32_t)need;
#pragma unroll 1
  for (int pass = 0; pass < 3; pass++) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass < 2 ? 2048 : 1024;
    for (int i = tid; i < 2048; i += NT) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += NT) {
      const uint32_t k = key(i);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    // from the largest digit down: thread t holds 2048 / NT digits next to one another
    constexpr int PT = 2048 / NT;
    uint32_t mine = 0;
#pragma unroll
    for (int u = 0; u < PT; u++) mine += hist[2047 - (tid * PT + u)];
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) warp_sums[warp] = upto;
    __syncthreads();
    for (int w = 0; w < warp; w++) upto += warp_sums[w];
    uint32_t before = upto - mine;
    if (before < left && left <= upto) {
#pragma unroll
      for (int u = 0; u < PT; u++) {
        const uint32_t d = 2047 - (tid * PT + u), cnt = hist[d];
        if (before < left && left <= before + cnt) {
          found[0] = d;
          found[1] = left - before;
        }
        before += cnt;
      }
    }
    __syncthreads();
    prefix |= found[0] << shift;
    mask |= (uint32_t)(bins - 1) << shift;
    left = found[1];
    __syncthreads();
  }
  ties = (int)left;
  return prefix;
}

// ------------------------------------------------------------------------------------------ eviction
struct PagedEvict {
  PagedView from, to;
  int keep, recent;
  const float *weights;
  float *weights_to;
  int *kept;
  long long ld, ld_to;
};

// Order-preserving bits of a weight; NaN is the largest.
__device__ __forceinline__ uint32_t weight_key(float w) { return isnan(w) ? 0xFFFFFFFFu : value_key(w); }

// One CTA per sequence: the weight that the last position to stay has, then the positions that stay, in order.
constexpr int kEvictThreads = 1024;

__global__ void __launch_bounds__(kEvictThreads) paged_select_kernel(PagedEvict e) {
  __shared__ uint32_t hist[2048], warp_sums[32], found[2];
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int L = paged_length(e.from, s), n = min(L, e.keep);
  const float *w = e.weights + (long long)s * e.ld;
  int *kept = e.kept + (long long)s * e.keep;
  float *wt = e.weights_to ? e.weights_to + (long long)s * e.ld_to : nullptr;
  const int old = L > e.keep ? L - e.recent : 0, need = e.keep - e.recent;
  int out = 0;
  if (old > 0 && need > 0) {
    int ties;
    const uint32_t t = radix_threshold<kEvictThreads>([&](int i) { return weight_key(__ldcg(w + i)); }, old, need, hist,
                                                      warp_sums, found, ties);
    int eq0 = 0, gt0 = 0;  // equal to and above the threshold so far
    for (int base = 0; base < old; base += kEvictThreads) {
      const int i = base + tid;
      const float x = i < old ? __ldcg(w + i) : 0.f;
      const uint32_t k = i < old ? weight_key(x) : 0u;
      const bool gt = i < old && k > t, eq = i < old && k == t;
      const unsigned below = (1u << lane) - 1u, mg = __ballot_sync(0xffffffffu, gt), me = __ballot_sync(0xffffffffu, eq);
      if (lane == 0) warp_sums[warp] = (uint32_t)__popc(me) << 16 | (uint32_t)__popc(mg);
      __syncthreads();
      uint32_t before = 0, all = 0;
      for (int q = 0; q < 32; q++) {
        const uint32_t x2 = warp_sums[q];
        before += q < warp ? x2 : 0u;
        all += x2;
      }
      const int g = gt0 + (int)(before & 0xffffu) + __popc(mg & below), q = eq0 + (int)(before >> 16) + __popc(me & below);
      if (gt || (eq && q < ties)) {
        const int at = g + min(q, ties);
        kept[at] = i;
        if (wt) wt[at] = x;
      }
      gt0 += (int)(all & 0xffffu);
      eq0 += (int)(all >> 16);
      __syncthreads();
    }
    out = need;
  }
  for (int i = out + tid; i < n; i += kEvictThreads) {
    const int from = L - n + i;  // the newest, or all of a sequence that stays whole
    kept[i] = from;
    if (wt) wt[i] = __ldcg(w + from);
  }
  for (int i = n + tid; i < e.keep; i += kEvictThreads) {
    kept[i] = -1;
    if (wt) wt[i] = 0.f;
  }
  if (tid == 0) e.to.lengths[s] = n;
}

// Copies what stays. A warp takes a position: its rows of all heads in both pools, 16 bytes a lane.
__global__ void __launch_bounds__(256) paged_gather_kernel(PagedEvict e, int elem) {
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.y, lane = threadIdx.x & 31, n = min(paged_length(e.from, s), e.keep);
  const int chunks = e.from.hs * elem / 16, all = chunks * e.from.n_kv;
  for (int i = blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += gridDim.x * 8) {
    const long long a = paged_offset(e.from, s, __ldcg(e.kept + (long long)s * e.keep + i)), b = paged_offset(e.to, s, i);
    if (a < 0 || b < 0) continue;
    for (int j = lane; j < all; j += 32) {
      const int h = j / chunks, x = (j - h * chunks) * 16;
      const long long at = (a + h * e.from.head_stride) * elem + x, to = (b + h * e.to.head_stride) * elem + x;
      const uint4 kk = __ldcg(reinterpret_cast<const uint4 *>(static_cast<const char *>(e.from.k) + at));
      const uint4 vv = __ldcg(reinterpret_cast<const uint4 *>(static_cast<const char *>(e.from.v) + at));
      *reinterpret_cast<uint4 *>(static_cast<char *>(e.to.k) + to) = kk;
      *reinterpret_cast<uint4 *>(static_cast<char *>(e.to.v) + to) = vv;
    }
  }
}

}  // namespace wgpt
