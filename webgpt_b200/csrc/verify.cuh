// Verification of drafted tokens against the target's probabilities (speculative sampling), from given random numbers.
#pragma once
#include "common.cuh"
#include "paged.cuh"
#include "sample_key.cuh"

namespace wgpt {

constexpr int kErrRow = 6;     // the error word's value for a row of logits without a distribution
constexpr int kErrDrafts = 7;  // for a number of drafts out of range
constexpr uint32_t kNoId = 0xFFFFFFFFu;

struct Verify {
  int n_seq, n_draft, V, top_k, chunks;
  const float *target, *draft;
  long long ld_target, ld_draft;
  const uint32_t *draft_ids;
  const int *n_drafted;
  double temperature;
  const double *uniforms;
  uint32_t *ids_out;
  int *n_accepted;
  int *err;
  float2 *partial;   // (largest, sum) of each chunk of each row: [n_seq][2 * n_draft + 1][chunks]
  float *list_value; // top_k > 0: each row's kept logits, largest first, and their ids, [n_seq][2 * n_draft + 1][top_k]
  int *list_id;
};

__device__ __forceinline__ int drafted(const Verify &a, int s) {
  const int n = a.n_drafted ? __ldcg(a.n_drafted + s) : a.n_draft;
  if (n >= 0 && n <= a.n_draft) return n;
  *a.err = kErrDrafts;
  return n < 0 ? 0 : a.n_draft;
}

// Row r of a sequence: r <= n_draft are the target's, n_draft + 1 + i the draft's i-th.
__device__ __forceinline__ const float *logits_row(const Verify &a, int s, int r) {
  return r <= a.n_draft ? a.target + ((long long)s * (a.n_draft + 1) + r) * a.ld_target
                        : a.draft + ((long long)s * a.n_draft + (r - a.n_draft - 1)) * a.ld_draft;
}
// Whether a row decides anything: the target's behind every draft and behind the last, the draft's of every draft.
__device__ __forceinline__ bool row_wanted(const Verify &a, int r, int n) {
  return r <= a.n_draft ? r <= n : r - a.n_draft - 1 < n;
}
__device__ __forceinline__ float logit(const float *p) {
  const float x = __ldcg(p);
  return isnan(x) ? -INFINITY : x;
}

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The largest value of each chunk of a row and the sum of exp((x - largest) / temperature) over it.
constexpr int kVerifyChunk = 8192, kVerifyThreads = 256;

__global__ void __launch_bounds__(kVerifyThreads) verify_sums_kernel(Verify a) {
  __shared__ float red[2][kVerifyThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.z, r = blockIdx.y, tid = threadIdx.x;
  if (!row_wanted(a, r, drafted(a, s))) return;
  const float *x = logits_row(a, s, r);
  const int beg = blockIdx.x * kVerifyChunk, end = min(a.V, beg + kVerifyChunk);
  float m = -INFINITY;
  for (int i = beg + tid; i < end; i += kVerifyThreads) m = fmaxf(m, logit(x + i));
  m = warp_max(m);
  if ((tid & 31) == 0) red[0][tid >> 5] = m;
  __syncthreads();
  for (int w = 0; w < kVerifyThreads / 32; w++) m = fmaxf(m, red[0][w]);
  const float inv = (float)(1.0 / a.temperature);
  float sum = 0.f;
  if (m > -INFINITY)
    for (int i = beg + tid; i < end; i += kVerifyThreads) sum += expf((logit(x + i) - m) * inv);
  sum = warp_sum(sum);
  if ((tid & 31) == 0) red[1][tid >> 5] = sum;
  __syncthreads();
  if (tid == 0) {
    sum = 0.f;
    for (int w = 0; w < kVerifyThreads / 32; w++) sum += red[1][w];
    a.partial[((long long)s * (2 * a.n_draft + 1) + r) * a.chunks + blockIdx.x] = make_float2(m, sum);
  }
}

// top_k > 0: the kept logits of a row in descending order, by one CTA.
constexpr int kListThreads = 1024;

__global__ void __launch_bounds__(kListThreads) verify_list_kernel(Verify a) {
  __shared__ uint32_t hist[2048], warp_sums[32], found[2], count[2];
  __shared__ unsigned long long kept[128];
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.y, r = blockIdx.x, tid = threadIdx.x;
  if (!row_wanted(a, r, drafted(a, s))) return;
  const float *x = logits_row(a, s, r);
  int ties;
  const uint32_t t = radix_threshold<kListThreads>([&](int i) { return value_key(logit(x + i)); }, a.V, a.top_k, hist,
                                                   warp_sums, found, ties);
  if (tid < 2) count[tid] = 0;
  __syncthreads();
  for (int i = tid; i < a.V; i += kListThreads) {
    const float v = logit(x + i);
    if (value_key(v) > t) kept[atomicAdd(&count[0], 1u)] = sample_key(v, i);
  }
  __syncthreads();
  // of the values at the threshold, the lowest indices
  const int above = a.top_k - ties, lane = tid & 31, warp = tid >> 5;
  int eq0 = 0;
  for (int base = 0; base < a.V && eq0 < ties; base += kListThreads) {
    const int i = base + tid;
    const float v = i < a.V ? logit(x + i) : 0.f;
    const bool eq = i < a.V && value_key(v) == t;
    const unsigned me = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) warp_sums[warp] = __popc(me);
    __syncthreads();
    int before = eq0, all = 0;
    for (int q = 0; q < 32; q++) {
      before += q < warp ? (int)warp_sums[q] : 0;
      all += (int)warp_sums[q];
    }
    before += __popc(me & ((1u << lane) - 1u));
    if (eq && before < ties) kept[above + before] = sample_key(v, i);
    eq0 += all;
    __syncthreads();
  }
  __syncthreads();
  if (tid < a.top_k) {
    const unsigned long long mine = kept[tid];
    int rank = 0;
    for (int j = 0; j < a.top_k; j++) rank += kept[j] > mine ? 1 : 0;
    const long long at = ((long long)s * (2 * a.n_draft + 1) + r) * a.top_k + rank;
    a.list_value[at] = sample_key_value(mine);
    a.list_id[at] = sample_key_index(mine);
  }
}

// ids_out and n_accepted of a sequence, once `accepted` and the drawn id are known.
__device__ __forceinline__ void write_ids(const Verify &a, int s, int accepted, uint32_t drawn) {
  for (int i = threadIdx.x; i <= a.n_draft; i += blockDim.x)
    a.ids_out[(long long)s * (a.n_draft + 1) + i] =
        i < accepted ? __ldcg(a.draft_ids + (long long)s * a.n_draft + i) : i == accepted ? drawn : kNoId;
  if (threadIdx.x == 0) a.n_accepted[s] = accepted;
}

// The accept step and the draw over the whole vocabulary, one CTA per sequence.
constexpr int kDrawThreads = 1024;

__global__ void __launch_bounds__(kDrawThreads) verify_draw_kernel(Verify a) {
  __shared__ int first_rejected, hit;
  __shared__ double red[32], red2[32];
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = drafted(a, s);
  if (tid == 0) {
    first_rejected = n;
    hit = a.V;
  }
  __syncthreads();
  const float2 *part = a.partial + (long long)s * (2 * a.n_draft + 1) * a.chunks;
  // (largest, sum) of a row, by a warp
  auto row_stats = [&](int r, float &m, double &z) {
    m = -INFINITY;
    for (int c = lane; c < a.chunks; c += 32) m = fmaxf(m, __ldcg(part + r * a.chunks + c).x);
    m = warp_max(m);
    z = 0.0;
    for (int c = lane; c < a.chunks; c += 32) {
      const float2 p = __ldcg(part + r * a.chunks + c);
      if (p.x > -INFINITY) z += (double)p.y * exp(((double)p.x - (double)m) / a.temperature);
    }
    z = warp_sum64(z);
  };
  for (int i = warp; i < n; i += kDrawThreads / 32) {
    float m, mq = 0.f;
    double z, zq = 1.0;
    row_stats(i, m, z);
    if (a.draft) row_stats(a.n_draft + 1 + i, mq, zq);
    if (lane == 0) {
      const uint32_t x = __ldcg(a.draft_ids + (long long)s * a.n_draft + i);
      bool ok = false;
      if (x >= (uint32_t)a.V) {
        *a.err = 1;
      } else if (!isinf(m) && !isinf(mq)) {
        const double p = exp(((double)logit(logits_row(a, s, i) + x) - (double)m) / a.temperature) / z;
        const double q = a.draft ? exp(((double)logit(logits_row(a, s, a.n_draft + 1 + i) + x) - (double)mq) / a.temperature) / zq : 1.0;
        ok = __ldcg(a.uniforms + (long long)s * (a.n_draft + 1) + i) * q < p;
      }
      if (!ok) atomicMin(&first_rejected, i);
    }
  }
  __syncthreads();
  const int at = first_rejected;
  const float *x = logits_row(a, s, at), *y = nullptr;
  float m, mq = 0.f;
  double z, zq;
  row_stats(at, m, z);
  uint32_t only = kNoId;
  bool rest = at < n;
  if (rest) {
    if (a.draft) {
      y = logits_row(a, s, a.n_draft + 1 + at);
      row_stats(a.n_draft + 1 + at, mq, zq);
      if (isinf(mq)) {
        if (tid == 0) *a.err = kErrRow;
        rest = false;
      }
    } else {
      only = __ldcg(a.draft_ids + (long long)s * a.n_draft + at);
    }
  }
  if (isinf(m)) {
    if (tid == 0) *a.err = kErrRow;
    write_ids(a, s, at, 0u);
    return;
  }
  auto block_sum = [&](double v, double *buf) {
    v = warp_sum64(v);
    if (lane == 0) buf[warp] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < 32; w++) v += buf[w];
    return v;
  };
  auto e = [&](const float *row, float top, int i) { return exp(((double)logit(row + i) - (double)top) / a.temperature); };
  // a warp takes V / 32 ids next to one another
  const int share = (a.V + 31) / 32, beg = min(a.V, warp * share), end = min(a.V, beg + share);
  double sx = 0.0, sy = 0.0;
  for (int i = beg + lane; i < end; i += 32) {
    sx += e(x, m, i);
    if (rest && y) sy += e(y, mq, i);
  }
  z = block_sum(sx, red);
  zq = block_sum(sy, red2);
  __syncthreads();
  const double u = __ldcg(a.uniforms + (long long)s * (a.n_draft + 1) + a.n_draft);
  for (int attempt = 0; attempt < 2; attempt++) {
    auto weight = [&](int i) {
      const double p = e(x, m, i) / z;
      if (!rest) return p;
      const double q = y ? e(y, mq, i) / zq : (uint32_t)i == only ? 1.0 : 0.0;
      return p > q ? p - q : 0.0;
    };
    double mine = 0.0;
    for (int i = beg + lane; i < end; i += 32) mine += weight(i);
    const double total = block_sum(mine, red);
    if (total > 0.0) {
      double before = 0.0;
      for (int w = 0; w < warp; w++) before += red[w];
      const double goal = u * total;
      // only the warp in whose share the running sum passes the goal, and the last one with anything in it
      if (before + red[warp] > goal && before <= goal) {
        int last = -1;  // the share's sum was rounded in another order: it may pass the goal where the running sum does not
        bool found = false;
        for (int i0 = beg; i0 < end; i0 += 32) {
          const int i = i0 + lane;
          double w = i < end ? weight(i) : 0.0, run = w;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += up;
          }
          const unsigned past = __ballot_sync(0xffffffffu, i < end && before + run > goal);
          if (past) {
            if (lane == 0) atomicMin(&hit, i0 + __ffs(past) - 1);
            found = true;
            break;
          }
          const unsigned some = __ballot_sync(0xffffffffu, w > 0.0);
          if (some) last = i0 + 31 - __clz(some);
          before += __shfl_sync(0xffffffffu, run, 31);
        }
        if (!found && last >= 0 && lane == 0) atomicMin(&hit, last);
      }
      break;
    }
    rest = false;
    __syncthreads();
  }
  __syncthreads();
  write_ids(a, s, at, (uint32_t)min(hit, a.V - 1));
}

// The same over the kept lists, one CTA per sequence.
__global__ void __launch_bounds__(128) verify_draw_list_kernel(Verify a) {
  __shared__ int first_rejected;
  __shared__ double w_list[128];
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.top_k;
  const int n = drafted(a, s);
  if (tid == 0) first_rejected = n;
  __syncthreads();
  const long long base = (long long)s * (2 * a.n_draft + 1) * K;
  const float *lv = a.list_value + base;
  const int *li = a.list_id + base;
  auto top_of = [&](int r) { return __ldcg(lv + r * K); };
  // the sum of a row's exponentials, by a warp, in the order of the list
  auto row_sum = [&](int r) {
    double z = 0.0;
    const double m = top_of(r);
    for (int j0 = 0; j0 < K; j0 += 32) {
      const double v = j0 + lane < K ? exp(((double)__ldcg(lv + r * K + j0 + lane) - m) / a.temperature) : 0.0;
      for (int j = 0; j < 32; j++) z += __shfl_sync(0xffffffffu, v, j);
    }
    return z;
  };
  auto share_of = [&](int r, uint32_t id, double z) {  // an id's probability in row r, by a warp
    double p = 0.0;
    for (int j = lane; j < K; j += 32)
      if ((uint32_t)__ldcg(li + r * K + j) == id) p = exp(((double)__ldcg(lv + r * K + j) - (double)top_of(r)) / a.temperature) / z;
    return warp_sum64(p);
  };
  for (int i = warp; i < n; i += 4) {
    const uint32_t x = __ldcg(a.draft_ids + (long long)s * a.n_draft + i);
    bool ok = false;
    if (x >= (uint32_t)a.V) {
      if (lane == 0) *a.err = 1;
    } else if (!isinf(top_of(i)) && !(a.draft && isinf(top_of(a.n_draft + 1 + i)))) {
      const double p = share_of(i, x, row_sum(i));
      const double q = a.draft ? share_of(a.n_draft + 1 + i, x, row_sum(a.n_draft + 1 + i)) : 1.0;
      ok = __ldcg(a.uniforms + (long long)s * (a.n_draft + 1) + i) * q < p;
    }
    if (!ok && lane == 0) atomicMin(&first_rejected, i);
  }
  __syncthreads();
  const int at = first_rejected;
  const double m = top_of(at);
  if (isinf(m)) {
    if (tid == 0) *a.err = kErrRow;
    write_ids(a, s, at, 0u);
    return;
  }
  bool rest = at < n;
  const int rq = a.n_draft + 1 + at;
  if (rest && a.draft && isinf(top_of(rq))) {
    if (tid == 0) *a.err = kErrRow;
    rest = false;
  }
  const double z = row_sum(at), zq = rest && a.draft ? row_sum(rq) : 1.0;
  const double u = __ldcg(a.uniforms + (long long)s * (a.n_draft + 1) + a.n_draft);
  double p = 0.0, w = 0.0;
  if (tid < K) {
    const uint32_t id = (uint32_t)__ldcg(li + at * K + tid);
    p = exp(((double)__ldcg(lv + at * K + tid) - m) / a.temperature) / z;
    w = p;
    if (rest) {
      double q = 0.0;
      if (a.draft) {
        for (int j = 0; j < K; j++)
          if ((uint32_t)__ldcg(li + rq * K + j) == id) q = exp(((double)__ldcg(lv + rq * K + j) - (double)top_of(rq)) / a.temperature) / zq;
      } else {
        q = id == __ldcg(a.draft_ids + (long long)s * a.n_draft + at) ? 1.0 : 0.0;
      }
      w = p > q ? p - q : 0.0;
    }
    w_list[tid] = w;
  }
  if (!__syncthreads_or(w > 0.0)) {
    if (tid < K) w_list[tid] = p;
    __syncthreads();
  }
  // all threads add the list up alike, left to right
  double total = 0.0, run = 0.0;
  for (int j = 0; j < K; j++) total += w_list[j];
  int pick = K - 1;
  for (int j = 0; j < K; j++) {
    run += w_list[j];
    if (run > u * total) {
      pick = j;
      break;
    }
  }
  write_ids(a, s, at, (uint32_t)__ldcg(li + at * K + pick));
}

}  // namespace wgpt
