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

// Rows [first, first + n) of sequence s, inside [0, n_rows) whatever starts says. Whether starts goes on from s to s + 1: sequences
// share no rows where it always does.
__device__ __forceinline__ bool new_rows(const PagedView &c, const NewRows &r, int s, int &first, int &n) {
  if (r.starts == nullptr) {
    first = s * r.per;
    n = r.per;
    return true;
  }
  const int a = __ldcg(r.starts + s), b = __ldcg(r.starts + s + 1);
  first = min(max(a, 0), r.n_rows);
  n = min(max(b, first), r.n_rows) - first;
  if (a != first || b != first + n) *c.err = kErrCache;
  return a <= b;
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
// of k and v are asked for ahead of them. Bound by latency for one row (12 heads of 64: 4.1 us, an empty kernel's time) and by bytes for
// prompts: 16 of up to 1021 rows of 12 heads of 64 in f32, written in f16 (83 MB): 19 us, 4.3 TB/s; a thread's pieces asked for only
// when the place is known took 38. Each value is rounded once, to the cache's type, which is what the cache is.
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
// top, a histogram of each digit among the keys that share the digits found so far, added up over the cluster. each(f) calls f
// with every key of this thread. Returns the key, and in `ties` how many keys equal to it belong to the need largest.
// hist2: 2 * 2048 counters in shared memory at the same place in every CTA, total: 2048 likewise, warp_sums: NT / 32, found: 2. C: 8 at
// most, a power of two.
template <int NT, typename Each>
__device__ uint32_t radix_threshold(Each each, int need, int C, int rank, uint32_t *hist2, uint32_t *total, uint32_t *warp_sums, uint32_t *found, int &ties) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t prefix = 0, mask = 0, left = (uint32_t)need;
#pragma unroll 1
  for (int pass = 0; pass < 3; pass++) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t bins = pass < 2 ? 2048 : 1024;
    uint32_t *hist = hist2 + (pass & 1) * 2048;  // a neighbour may still read the other
    for (int i = tid; i < 2048; i += NT) hist[i] = 0;
    __syncthreads();
    each([&](uint32_t k) {
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1u);
    });
    if (C > 1) {  // every CTA adds up its share of the digits over the cluster and tells all of them
      cluster_arrive();
      cluster_wait();
      const int share = 2048 / C;
      for (int i = tid; i < share; i += NT) {
        const int d = rank * share + i;
        float part[8];
        uint32_t sum = 0;
#pragma unroll
        for (int q = 0; q < 8; q++) part[q] = dsmem_ld(dsmem_addr(hist + d, q < C ? q : 0));
#pragma unroll
        for (int q = 0; q < 8; q++) sum += q < C ? __float_as_uint(part[q]) : 0u;
        for (int q = 0; q < C; q++) dsmem_st(dsmem_addr(total + d, q), __uint_as_float(sum));
      }
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
      count[u] = C > 1 ? total[d] : hist[d];
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
    upto += __reduce_add_sync(0xffffffffu, lane < warp && lane < NT / 32 ? warp_sums[lane] : 0u);
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
// positions that stay, in order. A thread's u-th position of a round is u * 1024 + its number, so that a round's flags lie in order
// as [u][warp][lane]; a stretch of one round (131072 positions a sequence) stays in registers. Bound by its chain of histograms,
// barriers and scans: about 11 us for one CTA of 1024 positions, 19 for clusters with 32768 each, where every CTA reading all
// eight histograms took 28.
constexpr int kEvictThreads = 1024, kEvictCluster = 8, kEvictVals = 16, kEvictRound = kEvictThreads * kEvictVals;

__global__ void __launch_bounds__(kEvictThreads) paged_select_kernel(const __grid_constant__ PagedEvict e) {
  __shared__ uint32_t hist[2 * 2048], total[2048], warp_sums[32], found[2];
  __shared__ uint32_t flags[2][kEvictVals * 32];                // above the threshold and on it, of every 32 positions of a round
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
    const int share = (old + (int)C - 1) / (int)C, beg = min(old, rank * share), end = min(old, beg + share);
    const int rounds = (end - beg + kEvictRound - 1) / kEvictRound;
    float x[kEvictVals];
    auto fetch = [&](int round) {
#pragma unroll
      for (int u = 0; u < kEvictVals; u++) {
        const int i = beg + round * kEvictRound + u * kEvictThreads + tid;
        x[u] = i < end ? __ldcg(w + i) : 0.f;
      }
    };
    auto there = [&](int round, int u) { return beg + round * kEvictRound + u * kEvictThreads + tid < end; };
    auto past = [&](int round, int u) { return beg + round * kEvictRound + u * kEvictThreads >= end; };  // the same for all threads
    if (rounds == 1) fetch(0);
    auto each = [&](auto f) {
      for (int round = 0; round < rounds; round++) {
        if (rounds > 1) fetch(round);
#pragma unroll
        for (int u = 0; u < kEvictVals; u++) {
          if (past(round, u)) break;
          if (there(round, u)) f(weight_key(x[u]));
        }
      }
    };
    int ties;
    const uint32_t t = radix_threshold<kEvictThreads>(each, need, (int)C, rank, hist, total, warp_sums, found, ties);
    int gt0 = 0, eq0 = 0;  // above the threshold and on it, before the round at hand
    if (C > 1) {           // in the stretches before this one
      int gt = 0, eq = 0;
      each([&](uint32_t k) {
        gt += k > t ? 1 : 0;
        eq += k == t ? 1 : 0;
      });
      gt = __reduce_add_sync(0xffffffffu, gt);
      eq = __reduce_add_sync(0xffffffffu, eq);
      if (lane == 0) {
        flags[0][warp] = gt;
        flags[1][warp] = eq;
      }
      __syncthreads();
      if (warp == 0) {
        const uint32_t g = __reduce_add_sync(0xffffffffu, flags[0][lane]), q = __reduce_add_sync(0xffffffffu, flags[1][lane]);
        if (lane < (int)C) {  // to every CTA
          dsmem_st(dsmem_addr(&above[rank], lane), __uint_as_float(g));
          dsmem_st(dsmem_addr(&equal[rank], lane), __uint_as_float(q));
        }
      }
      cluster_arrive();
      cluster_wait();
      for (int i = 0; i < rank; i++) {
        gt0 += (int)__float_as_uint(above[i]);
        eq0 += (int)__float_as_uint(equal[i]);
      }
    }
    for (int round = 0; round < rounds; round++) {
      if (rounds > 1) fetch(round);
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kEvictVals; u++) {
        if (past(round, u)) {
          if (lane < 2) flags[lane][u * 32 + warp] = 0;
          continue;
        }
        const uint32_t k = weight_key(x[u]);
        const uint32_t g = __ballot_sync(0xffffffffu, there(round, u) && k > t), q = __ballot_sync(0xffffffffu, there(round, u) && k == t);
        if (lane == 0) {
          flags[0][u * 32 + warp] = g;
          flags[1][u * 32 + warp] = q;
        }
      }
      __syncthreads();
      // every warp adds up the counts before its own flags: lane l those of the l-th sixteen
      uint32_t mine = 0;  // both counts: up to 16384 each
      const int first = lane * kEvictVals;
#pragma unroll
      for (int i0 = 0; i0 < kEvictVals; i0++) {
        const int i = first + ((i0 + lane) & (kEvictVals - 1));  // in an order that spreads over the banks
        mine += (uint32_t)__popc(flags[1][i]) << 16 | (uint32_t)__popc(flags[0][i]);
      }
      uint32_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      const uint32_t sum = __shfl_sync(0xffffffffu, upto, 31);
      upto -= mine;
#pragma unroll
      for (int u = 0; u < kEvictVals; u++) {
        if (past(round, u)) break;
        const int at = u * 32 + warp, of = at / kEvictVals;
        // what lies before the lane's sixteen that `at` belongs to, and inside them before it
        const uint32_t base = __shfl_sync(0xffffffffu, upto, of);
        const int j = of * kEvictVals + (lane & (kEvictVals - 1));
        const uint32_t in = j < at && lane < kEvictVals ? (uint32_t)__popc(flags[1][j]) << 16 | (uint32_t)__popc(flags[0][j]) : 0u;
        const uint32_t before = base + __reduce_add_sync(0xffffffffu, in);
        const uint32_t g = flags[0][at], q = flags[1][at], below = (1u << lane) - 1u;
        const int gi = gt0 + (int)(before & 0xffffu) + __popc(g & below), qi = eq0 + (int)(before >> 16) + __popc(q & below);
        if ((g >> lane & 1u) || ((q >> lane & 1u) && qi < ties)) {
          const int to = gi + min(qi, ties);
          kept[to] = beg + round * kEvictRound + u * kEvictThreads + tid;
          if (wt) wt[to] = x[u];
        }
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

constexpr int kGatherAhead = 4;

// Copies what stays. A warp takes a position: its rows of all heads in both pools, 16 bytes a lane, four of each pool in flight. Bound by
// bytes: 8 users, 8191 of 32768 positions each of 8 heads of 128 in f16 (537 MB both ways) 89 us, 6.0 TB/s.
__global__ void __launch_bounds__(256) paged_gather_kernel(const __grid_constant__ PagedEvict e, int elem) {
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.y, lane = threadIdx.x & 31, n = min(paged_length(e.from, s), e.keep);
  const int chunks = e.from.hs * elem / 16, all = chunks * e.from.n_kv;
  for (int i = blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += gridDim.x * 8) {
    const long long a = paged_offset(e.from, s, __ldcg(e.kept + (long long)s * e.keep + i)), b = paged_offset(e.to, s, i);
    if (a < 0 || b < 0) continue;
    for (int j0 = lane; j0 < all; j0 += 32 * kGatherAhead) {
      uint4 kk[kGatherAhead], vv[kGatherAhead];
#pragma unroll
      for (int u = 0; u < kGatherAhead; u++) {
        const int j = j0 + 32 * u, h = j / chunks;
        const long long at = (a + h * e.from.head_stride) * elem + (j - h * chunks) * 16;
        if (j < all) {
          kk[u] = __ldcg(reinterpret_cast<const uint4 *>(static_cast<const char *>(e.from.k) + at));
          vv[u] = __ldcg(reinterpret_cast<const uint4 *>(static_cast<const char *>(e.from.v) + at));
        }
      }
#pragma unroll
      for (int u = 0; u < kGatherAhead; u++) {
        const int j = j0 + 32 * u, h = j / chunks;
        const long long to = (b + h * e.to.head_stride) * elem + (j - h * chunks) * 16;
        if (j < all) {
          *reinterpret_cast<uint4 *>(static_cast<char *>(e.to.k) + to) = kk[u];
          *reinterpret_cast<uint4 *>(static_cast<char *>(e.to.v) + to) = vv[u];
        }
      }
    }
  }
}

}  // namespace wgpt
