// Verification of drafted tokens against the target's probabilities (speculative sampling), from given random numbers.
#pragma once
#include "common.cuh"
#include "paged.cuh"
#include "sample_key.cuh"

namespace wgpt {

constexpr int kErrRow = 6;     // the error word's value for a row of logits without a distribution
constexpr int kErrDrafts = 7;  // for a number of drafts out of range
constexpr uint32_t kNoId = 0xFFFFFFFFu;
constexpr int kMaxDraft = 64;

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

// The largest value of each chunk of a row and the sum of exp((x - largest) / temperature) over it; a chunk is in registers
// between the two. Decides whether drafts are accepted: each exponential is good to 2^-22, their sum to a few 1e-8.
constexpr int kVerifyThreads = 256, kVerifyVals = 16, kVerifyChunk = kVerifyThreads * kVerifyVals;

__global__ void __launch_bounds__(kVerifyThreads) verify_sums_kernel(const __grid_constant__ Verify a) {
  __shared__ float red[kVerifyThreads / 32];
  __shared__ double red64[kVerifyThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.z, r = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int beg = blockIdx.x * kVerifyChunk;
  if (!row_wanted(a, r, drafted(a, s))) return;
  const float *x = logits_row(a, s, r) + beg;
  const int n = min(a.V - beg, kVerifyChunk);
  float v[kVerifyVals], m = -INFINITY;
#pragma unroll
  for (int u = 0; u < kVerifyVals; u++) v[u] = tid + u * kVerifyThreads < n ? __ldcg(x + tid + u * kVerifyThreads) : -INFINITY;
#pragma unroll
  for (int u = 0; u < kVerifyVals; u++) m = fmaxf(m, v[u]);  // NaN is passed over
  m = warp_max(m);
  if (lane == 0) red[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kVerifyThreads / 32; w++) m = fmaxf(m, red[w]);
  const float c = (float)(1.4426950408889634 / a.temperature);
  float sum = 0.f;
#pragma unroll
  for (int u = 0; u < kVerifyVals; u++) {
    const float e = exp2f((v[u] - m) * c);
    sum += v[u] > -INFINITY ? e : 0.f;
  }
  double sum64 = warp_sum64((double)sum);
  if (lane == 0) red64[warp] = sum64;
  __syncthreads();
  if (tid == 0) {
    sum64 = 0.0;
    for (int w = 0; w < kVerifyThreads / 32; w++) sum64 += red64[w];
    a.partial[((long long)s * (2 * a.n_draft + 1) + r) * a.chunks + blockIdx.x] = make_float2(m, (float)sum64);
  }
}

// e^(x / temperature) of x <= 0 in double precision, to about 1e-15: x / temperature = (64 n + j + f) ln 2 / 64 with |f| <= 1/2, so
// that it is 2^n 2^(j/64) e^(f ln 2 / 64), the second from a table and the third by its series (table-driven exponentials, Tang 1989).
// scale: 64 / (ln 2 temperature).
__device__ __forceinline__ double exp_of(double x, double scale, const double *table) {
  const double t = x * scale;
  const double shifted = t + 6755399441055744.0;  // 1.5 * 2^52: the integer nearest to t in the low word
  const int n = __double2loint(shifted);
  const double f = t - (shifted - 6755399441055744.0);
  constexpr double z = 0.010830424696249145;  // ln 2 / 64
  double p = fma(f, z * z * z * z * z / 120.0, z * z * z * z / 24.0);
  p = fma(p, f, z * z * z / 6.0);
  p = fma(p, f, z * z / 2.0);
  p = fma(p, f, z);
  p = fma(p, f, 1.0);
  const double y = table[n & 63] * p;
  return t < -65000.0 ? 0.0 : __hiloint2double(__double2hiint(y) + ((n >> 6) << 20), __double2loint(y));  // 2^-1015 and below: 0
}

// top_k > 0: the kept logits of a row in descending order, by one CTA. Each thread's largest key (of the value, among equals of the
// lowest index) is a candidate for the bound: the top_k-th largest of them is a key that at least top_k keys reach, all of them in
// the top_k threads that hold one. Those read their share again; what reaches the bound is ranked by counting.
constexpr int kListThreads = 1024;

__global__ void __launch_bounds__(kListThreads) verify_list_kernel(const __grid_constant__ Verify a, int cap) {
  extern __shared__ __align__(16) unsigned long long cand[];  // [cap], cap = top_k * ceil(V / kListThreads)
  __shared__ int count;
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.y, r = blockIdx.x, tid = threadIdx.x;
  if (!row_wanted(a, r, drafted(a, s))) return;
  const float *x = logits_row(a, s, r);
  unsigned long long best = 0ull;
  for (int i0 = 0; i0 < a.V; i0 += 16 * kListThreads) {
    float v[16];
#pragma unroll
    for (int u = 0; u < 16; u++) {
      const int i = i0 + tid + u * kListThreads;
      v[u] = i < a.V ? logit(x + i) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 16; u++) {
      const int i = i0 + tid + u * kListThreads;
      const unsigned long long k = i < a.V ? sample_key(v[u], i) : 0ull;
      best = k > best ? k : best;
    }
  }
  if (tid == 0) count = 0;
  // the bound, bit by bit: the value's, and where several threads have that value, the index's
  const int holders = min(a.V, kListThreads);
  unsigned long long bound = 1ull;
  if (holders > a.top_k) {
    bound = 0ull;
    for (int bit = 63; bit >= 32; bit--) {
      const unsigned long long trial = bound | 1ull << bit;
      if (__syncthreads_count(best >= trial) >= a.top_k) bound = trial;
    }
    if (__syncthreads_count(best >= bound) > a.top_k)
      for (int bit = 31; bit >= 0; bit--) {
        const unsigned long long trial = bound | 1ull << bit;
        if (__syncthreads_count(best >= trial) >= a.top_k) bound = trial;
      }
  }
  __syncthreads();
  if (best >= bound)
    for (int i0 = tid; i0 < a.V; i0 += 16 * kListThreads) {
      float v[16];
#pragma unroll
      for (int u = 0; u < 16; u++) v[u] = i0 + u * kListThreads < a.V ? logit(x + i0 + u * kListThreads) : 0.f;
#pragma unroll
      for (int u = 0; u < 16; u++) {
        const int i = i0 + u * kListThreads;
        if (i >= a.V) continue;
        const unsigned long long k = sample_key(v[u], i);
        if (k >= bound) {
          const int at = atomicAdd(&count, 1);
          if (at < cap) cand[at] = k;
        }
      }
    }
  __syncthreads();
  const int n = min(count, cap);
  const long long to = ((long long)s * (2 * a.n_draft + 1) + r) * a.top_k;
  for (int i = tid; i < n; i += kListThreads) {
    const unsigned long long mine = cand[i];
    int rank = 0;
    for (int j = 0; j < n; j++) rank += cand[j] > mine ? 1 : 0;
    if (rank < a.top_k) {
      a.list_value[to + rank] = sample_key_value(mine);
      a.list_id[to + rank] = sample_key_index(mine);
    }
  }
}

// ids_out and n_accepted of a sequence, once `accepted` and the drawn id are known.
__device__ __forceinline__ void write_ids(const Verify &a, int s, int accepted, uint32_t drawn) {
  for (int i = threadIdx.x; i <= a.n_draft; i += blockDim.x)
    a.ids_out[(long long)s * (a.n_draft + 1) + i] =
        i < accepted ? __ldcg(a.draft_ids + (long long)s * a.n_draft + i) : i == accepted ? drawn : kNoId;
  if (threadIdx.x == 0) a.n_accepted[s] = accepted;
}

// The accept step and the draw over the whole vocabulary, a cluster of CTAs per sequence. The draw needs running sums good to
// far below the smallest probability, so its exponentials are in double precision: those of the target's row, and of the draft's if a
// draft was not accepted. Every warp takes a stretch of ids; the sums of the stretches say in which one the running sum passes the
// number, and that warp adds its stretch up id by id. A lane keeps its exponentials where they fit kVals registers.
constexpr int kDrawThreads = 512, kDrawWarps = kDrawThreads / 32, kDrawCluster = 8;

template <int kVals>
__global__ void __launch_bounds__(kDrawThreads) verify_draw_kernel(const __grid_constant__ Verify a) {
  __shared__ int first_rejected, hit;
  __shared__ float s_max[2 * kMaxDraft + 1];
  __shared__ double s_sum[2 * kMaxDraft + 1];
  __shared__ double table[64];
  __shared__ double sums[3][kDrawCluster][kDrawWarps];  // of every warp of the cluster: the target's, the draft's, what is drawn from
  uint32_t C;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(C));
  const int rank = (int)cluster_ctarank(), s = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cluster_arrive_relaxed();
  if (tid < 64) table[tid] = exp2(tid / 64.0);
  pdl_launch_dependents();
  pdl_wait();
  const int n = drafted(a, s), rows = 2 * a.n_draft + 1;
  if (tid == 0) {
    first_rejected = n;
    hit = a.V;
  }
  // every CTA finds the first draft that is not accepted: (largest, sum) of the rows, a warp each
  const float2 *part = a.partial + (long long)s * rows * a.chunks;
  for (int r = warp; r < rows; r += kDrawWarps) {
    if (!row_wanted(a, r, n) || (r > a.n_draft && !a.draft)) continue;
    float m = -INFINITY;
    for (int c = lane; c < a.chunks; c += 32) m = fmaxf(m, __ldcg(part + r * a.chunks + c).x);
    m = warp_max(m);
    double z = 0.0;
    for (int c = lane; c < a.chunks; c += 32) {
      const float2 p = __ldcg(part + r * a.chunks + c);
      if (p.x > -INFINITY) z += (double)p.y * exp(((double)p.x - (double)m) / a.temperature);
    }
    z = warp_sum64(z);
    if (lane == 0) {
      s_max[r] = m;
      s_sum[r] = z;
    }
  }
  __syncthreads();
  if (tid < n) {
    const int i = tid, rq = a.n_draft + 1 + i;
    const uint32_t x = __ldcg(a.draft_ids + (long long)s * a.n_draft + i);
    bool ok = false;
    if (x >= (uint32_t)a.V) {
      *a.err = 1;
    } else if (!isinf(s_max[i]) && !(a.draft && isinf(s_max[rq]))) {
      const double p = exp(((double)logit(logits_row(a, s, i) + x) - (double)s_max[i]) / a.temperature) / s_sum[i];
      const double q = a.draft ? exp(((double)logit(logits_row(a, s, rq) + x) - (double)s_max[rq]) / a.temperature) / s_sum[rq] : 1.0;
      ok = __ldcg(a.uniforms + (long long)s * (a.n_draft + 1) + i) * q < p;
    }
    if (!ok) atomicMin(&first_rejected, i);
  }
  __syncthreads();
  const int at = first_rejected;
  const float *x = logits_row(a, s, at), *y = nullptr;
  const double m = s_max[at], scale = 64.0 / (0.6931471805599453 * a.temperature);
  double mq = 0.0;
  uint32_t only = kNoId;
  bool rest = at < n;
  if (rest && a.draft) {
    y = logits_row(a, s, a.n_draft + 1 + at);
    mq = s_max[a.n_draft + 1 + at];
    if (isinf(mq)) {
      if (tid == 0) *a.err = kErrRow;
      rest = false;
    }
  } else if (rest) {
    only = __ldcg(a.draft_ids + (long long)s * a.n_draft + at);
  }
  const bool none = isinf(m);
  const int stretch = (a.V + (int)C * kDrawWarps - 1) / ((int)C * kDrawWarps);
  const int beg = min(a.V, (rank * kDrawWarps + warp) * stretch), end = min(a.V, beg + stretch);
  auto ex = [&](int i) { return exp_of((double)logit(x + i) - m, scale, table); };
  auto ey = [&](int i) { return exp_of((double)logit(y + i) - mq, scale, table); };
  const bool two = rest && y != nullptr;
  double vx[kVals > 0 ? kVals : 1], vy[kVals > 0 ? kVals : 1];
  // a sum of every warp to every CTA, behind one barrier of the cluster
  auto tell = [&](int which, double v) {
    v = warp_sum64(v);
    if (lane < (int)C) dsmem_st64(dsmem_addr(&sums[which][rank][warp], lane), (unsigned long long)__double_as_longlong(v));
  };
  auto total_of = [&](int which) {
    double v = 0.0;
    for (int q = 0; q < (int)C; q++)
      for (int w = 0; w < kDrawWarps; w++) v += sums[which][q][w];
    return v;
  };
  cluster_wait();  // the others run
  double zx = 1.0, zq = 1.0;
  if (!none) {
    double sx = 0.0, sy = 0.0;
    if constexpr (kVals > 0) {
#pragma unroll
      for (int u = 0; u < kVals; u++) {
        const int i = beg + lane + 32 * u;
        vx[u] = i < end ? ex(i) : 0.0;
        vy[u] = two && i < end ? ey(i) : 0.0;
        sx += vx[u];
        sy += vy[u];
      }
    } else {
      for (int i = beg + lane; i < end; i += 32) {
        sx += ex(i);
        if (two) sy += ey(i);
      }
    }
    tell(0, sx);
    if (two) tell(1, sy);
  }
  cluster_arrive();
  cluster_wait();
  const double u01 = __ldcg(a.uniforms + (long long)s * (a.n_draft + 1) + a.n_draft);
  int which = 0;
  if (!none) {
    zx = total_of(0);
    if (two) zq = total_of(1);
  }
  const double ix = 1.0 / zx, iq = 1.0 / zq;
  // what an id counts: e / sum, less the draft's (or less all of it at the drafted id), none below zero
  auto weight = [&](double e, double f, int i) {
    const double p = e * ix, q = two ? f * iq : (uint32_t)i == only ? 1.0 : 0.0;
    return rest ? fmax(p - q, 0.0) : e;
  };
  if (rest && !none) {
    double sr = 0.0;
    if constexpr (kVals > 0) {
#pragma unroll
      for (int u = 0; u < kVals; u++) {
        const int i = beg + lane + 32 * u;
        if (i < end) sr += weight(vx[u], vy[u], i);
      }
    } else {
      for (int i = beg + lane; i < end; i += 32) sr += weight(ex(i), two ? ey(i) : 0.0, i);
    }
    tell(2, sr);
  }
  cluster_arrive();
  cluster_wait();
  double total = zx;
  if (rest && !none) {
    total = total_of(2);
    which = 2;
    if (!(total > 0.0)) {  // nothing is left: drawn from the target's row itself
      rest = false;
      total = zx;
      which = 0;
    }
  }
  if (!none) {
    const double goal = u01 * total;
    double before = 0.0;
    for (int q = 0; q < rank; q++)
      for (int w = 0; w < kDrawWarps; w++) before += sums[which][q][w];
    for (int w = 0; w < warp; w++) before += sums[which][rank][w];
    // the warp in whose stretch the running sum passes the goal; its id goes to the first CTA
    if (before + sums[which][rank][warp] > goal && before <= goal) {
      int last = -1, found = -1;  // the stretch's sum was rounded in another order: it may pass the goal where the running sum does not
      for (int i0 = beg; i0 < end && found < 0; i0 += 32) {
        const int i = i0 + lane;
        const double w = i < end ? weight(ex(i), two ? ey(i) : 0.0, i) : 0.0;
        double run = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double up = __shfl_up_sync(0xffffffffu, run, o);
          if (lane >= o) run += up;
        }
        const unsigned past = __ballot_sync(0xffffffffu, i < end && before + run > goal);
        if (past) found = i0 + __ffs(past) - 1;
        const unsigned some = __ballot_sync(0xffffffffu, w > 0.0);
        if (some) last = i0 + 31 - __clz(some);
        before += __shfl_sync(0xffffffffu, run, 31);
      }
      if (found < 0) found = last;
      if (lane == 0 && found >= 0) dsmem_st(dsmem_addr(&hit, 0), __int_as_float(found));
    }
  }
  cluster_arrive();
  cluster_wait();
  if (rank != 0) return;
  if (none && tid == 0) *a.err = kErrRow;
  write_ids(a, s, at, none ? 0u : (uint32_t)min(hit, a.V - 1));
}

// The same over the kept lists, one CTA per sequence.
__global__ void __launch_bounds__(128) verify_draw_list_kernel(const __grid_constant__ Verify a) {
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
