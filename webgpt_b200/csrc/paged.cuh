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
// A warp takes a row. Three round trips to memory find its place (its sequence, that one's length, the page), so the first values
// of k and v are asked for ahead of them.
constexpr int kAppendThreads = 256, kAppendAhead = 6;

template <typename T>
__global__ void __launch_bounds__(kAppendThreads)
paged_append_kernel(const __grid_constant__ PagedView c, NewRows r, const float *__restrict__ k, const float *__restrict__ v, long long ld) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, row = blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
  if (row >= r.n_rows) return;
  const int per_head = c.hs / 4, n4 = c.n_kv * per_head;
  const float4 *k4 = reinterpret_cast<const float4 *>(k + (long long)row * ld);
  const float4 *v4 = reinterpret_cast<const float4 *>(v + (long long)row * ld);
  float4 a[kAppendAhead], b[kAppendAhead];
  auto ask = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kAppendAhead; u++) {
      const int i = i0 + lane + 32 * u;
      if (i < n4) {
        a[u] = __ldcg(k4 + i);
        b[u] = __ldcg(v4 + i);
      }
    }
  };
  ask(0);
  const int s = sequence_of(c, r, row, lane);
  if (s < 0) return;
  int first, n;
  new_rows(c, r, s, first, n);
  const int pos = paged_length(c, s) - n + (row - first);
  if ((unsigned)(row - first) >= (unsigned)n || pos < 0) return;
  const long long at = paged_offset(c, s, pos);
  if (at < 0) return;
  for (int i0 = 0; i0 < n4; i0 += 32 * kAppendAhead) {
    if (i0 > 0) ask(i0);
#pragma unroll
    for (int u = 0; u < kAppendAhead; u++) {
      const int i = i0 + lane + 32 * u;
      if (i >= n4) continue;
      const int h = i / per_head;
      const long long to = at + (long long)h * c.head_stride + (i - h * per_head) * 4;
      *reinterpret_cast<Pack4<T> *>(static_cast<T *>(c.k) + to) = Pack4<T>::of(a[u]);
      *reinterpret_cast<Pack4<T> *>(static_cast<T *>(c.v) + to) = Pack4<T>::of(b[u]);
    }
  }
}

// ------------------------------------------------------------------------------------------ selection
// The need-th largest of all 32-bit keys of a cluster of C CTAs (or of one) of NT threads: digits of 11, 11 and 10 bits from the
// top, a histogram of each digit among the keys that share the digits found so far, added up over the cluster. key(u) is a
// thread's u-th key of n, there(u) whether it has one. Returns the key, and in `ties` how many keys equal to it belong to the
// need largest. hist: 2 * 2048 counters in shared memory at the same place in every CTA, warp_sums: NT / 32, found: 2.
template <int NT, typename Key, typename There>
__device__ uint32_t radix_threshold(Key key, There there, int n, int need, int C, uint32_t *hist2, uint32_t *warp_sums,
                                    uint32_t *found, int &ties) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t prefix = 0, mask = 0, left = (uint32_t)need;
#pragma unroll 1
  for (int pass = 0; pass < 3; pass++) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t bins = pass < 2 ? 2048 : 1024;
    uint32_t *hist = hist2 + (pass & 1) * 2048;  // a neighbour may still read the other
    for (int i = tid; i < 2048; i += NT) hist[i] = 0;
    __syncthreads();
#pragma unroll 4
    for (int u = 0; u < n; u++) {
      const uint32_t k = there(u) ? key(u) : 0u;
      if (there(u) && (k & mask) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1u);
    }
    if (C > 1) {
      cluster_arrive();
      cluster_wait();
    } else {
      __syncthreads();
    }
    // from the largest digit down: a thread holds 2048 / NT digits next to one another
    constexpr int PT = 2048 / NT;
    uint32_t count[PT], mine = 0;
#pragma unroll
    for (int u = 0; u < PT; u++) {
      const uint32_t d = 2047 - (tid * PT + u);
      count[u] = 0;
      if (C == 1) {
        count[u] = hist[d];
      } else {
        for (int q = 0; q < C; q++) count[u] += __float_as_uint(dsmem_ld(dsmem_addr(hist + d, q)));
      }
      mine += count[u];
    }
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
        if (before < left && left <= before + count[u]) {
          found[0] = 2047 - (tid * PT + u);
          found[1] = left - before;
        }
        before += count[u];
      }
    }
    __syncthreads();
    prefix |= found[0] << shift;
    mask |= (bins - 1) << shift;
    left = found[1];
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

// A cluster per sequence, each CTA with a stretch of its positions: the weight that the last position to stay has, then the
// positions that stay, in order. A thread of a stretch takes groups of four positions, 1024 groups from one of its to the next.
constexpr int kEvictThreads = 1024, kEvictCluster = 8;

__global__ void __launch_bounds__(kEvictThreads) paged_select_kernel(const __grid_constant__ PagedEvict e) {
  __shared__ uint32_t hist[2 * 2048], warp_sums[32], found[2];
  __shared__ float above[kEvictCluster], equal[kEvictCluster];  // of the CTAs' stretches, as bits
  uint32_t C;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(C));
  const int rank = (int)cluster_ctarank(), s = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const int L = paged_length(e.from, s), n = min(L, e.keep);
  const float *w = e.weights + (long long)s * e.ld;
  int *kept = e.kept + (long long)s * e.keep;
  float *wt = e.weights_to ? e.weights_to + (long long)s * e.ld_to : nullptr;
  const int old = L > e.keep ? L - e.recent : 0, need = e.keep - e.recent;
  const int all = (int)C * kEvictThreads, me = rank * kEvictThreads + tid;
  int out = 0;
  if (old > 0 && need > 0) {  // the same for the whole cluster
    const int share = ((old + (int)C - 1) / (int)C + 3) / 4 * 4, beg = min(old, rank * share), end = min(old, beg + share);
    const int rounds = (end - beg + 4 * kEvictThreads - 1) / (4 * kEvictThreads);
    auto at = [&](int u) { return beg + (u >> 2) * 4 * kEvictThreads + 4 * tid + (u & 3); };
    auto there = [&](int u) { return at(u) < end; };
    auto next_to = [&](int u) { return beg + u * kEvictThreads + tid; };  // where the order does not matter
    int ties;
    const uint32_t t = radix_threshold<kEvictThreads>([&](int u) { return weight_key(__ldcg(w + next_to(u))); },
                                                      [&](int u) { return next_to(u) < end; }, 4 * rounds, need, (int)C, hist,
                                                      warp_sums, found, ties);
    // how many lie above the threshold and on it, in the stretches before this one
    int gt = 0, eq = 0;
#pragma unroll 4
    for (int u = 0; u < 4 * rounds; u++)
      if (next_to(u) < end) {
        const uint32_t k = weight_key(__ldcg(w + next_to(u)));
        gt += k > t ? 1 : 0;
        eq += k == t ? 1 : 0;
      }
    int gt0 = 0, eq0 = 0;
    if (C > 1) {
      gt = __reduce_add_sync(0xffffffffu, gt);
      eq = __reduce_add_sync(0xffffffffu, eq);
      __syncthreads();
      if (lane == 0) {
        hist[2048 + warp] = gt;  // a neighbour may still read the first half
        hist[2080 + warp] = eq;
      }
      __syncthreads();
      if (tid < (int)C) {  // to every CTA
        uint32_t g = 0, q = 0;
        for (int i = 0; i < kEvictThreads / 32; i++) {
          g += hist[2048 + i];
          q += hist[2080 + i];
        }
        dsmem_st(dsmem_addr(&above[rank], tid), __uint_as_float(g));
        dsmem_st(dsmem_addr(&equal[rank], tid), __uint_as_float(q));
      }
      cluster_arrive();
      cluster_wait();
      for (int i = 0; i < rank; i++) {
        gt0 += (int)__float_as_uint(above[i]);
        eq0 += (int)__float_as_uint(equal[i]);
      }
    }
    for (int u0 = 0; u0 < 4 * rounds; u0 += 4) {
      float x[4];
      uint32_t k[4];
      int g = 0, q = 0;
#pragma unroll
      for (int u = 0; u < 4; u++) {
        x[u] = there(u0 + u) ? __ldcg(w + at(u0 + u)) : 0.f;
        k[u] = weight_key(x[u]);
        g += there(u0 + u) && k[u] > t ? 1 : 0;
        q += there(u0 + u) && k[u] == t ? 1 : 0;
      }
      uint32_t mine = (uint32_t)q << 16 | (uint32_t)g, upto = mine, sum = 0;  // 4096 positions: both fit 16 bits
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      __syncthreads();
      if (lane == 31) warp_sums[warp] = upto;
      __syncthreads();
      upto -= mine;
      const uint32_t ws = warp_sums[lane];
      upto += __reduce_add_sync(0xffffffffu, lane < warp ? ws : 0u);
      sum = __reduce_add_sync(0xffffffffu, ws);
      int gi = gt0 + (int)(upto & 0xffffu), qi = eq0 + (int)(upto >> 16);
#pragma unroll
      for (int u = 0; u < 4; u++) {
        if (!there(u0 + u)) continue;
        const bool is_gt = k[u] > t, is_eq = k[u] == t;
        if (is_gt || (is_eq && qi < ties)) {
          const int to = gi + min(qi, ties);
          kept[to] = at(u0 + u);
          if (wt) wt[to] = x[u];
        }
        gi += is_gt ? 1 : 0;
        qi += is_eq ? 1 : 0;
      }
      gt0 += (int)(sum & 0xffffu);
      eq0 += (int)(sum >> 16);
    }
    out = need;
  }
  for (int i = out + me; i < n; i += all) {
    const int from = L - n + i;  // the newest, or all of a sequence that stays whole
    kept[i] = from;
    if (wt) wt[i] = __ldcg(w + from);
  }
  for (int i = n + me; i < e.keep; i += all) {
    kept[i] = -1;
    if (wt) wt[i] = 0.f;
  }
  if (C > 1) {  // shared memory stays until the others have read it; lengths may be one array
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  if (me == 0) e.to.lengths[s] = n;
}

// Copies what stays. A warp takes a position: its rows of all heads in both pools, 16 bytes a lane.
__global__ void __launch_bounds__(256) paged_gather_kernel(const __grid_constant__ PagedEvict e, int elem) {
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
