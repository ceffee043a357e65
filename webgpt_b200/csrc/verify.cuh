// Verification of drafted tokens against the target's probabilities (speculative sampling), from given random numbers.
#pragma once
#include "common.cuh"
#include "paged_attention.cuh"
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
  double2 *list_sum; // top_k > 0: each row's sum of exponentials and the drafted id's probability, [n_seq][2 * n_draft + 1]
  float *list_value; // each row's kept logits, largest first, and their ids, [n_seq][2 * n_draft + 1][top_k]
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

// The largest value of each chunk of a row and the sum of exp((x - largest) / temperature) over it, a warp a chunk: every lane has its
// own running maximum until the end. Decides whether drafts are accepted: each exponential is good to 2^-22, their sum to a few 1e-8.
// Bound by bytes: 64 users with up to 4 drafts over 50257 ids (85 MB) 20 us, 4.3 TB/s, launch and ragged ends included.
constexpr int kVerifyThreads = 256, kVerifyVals = 16, kVerifyTurns = 4, kVerifyChunk = 32 * kVerifyVals * kVerifyTurns;

__global__ void __launch_bounds__(kVerifyThreads) verify_sums_kernel(const __grid_constant__ Verify a) {
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.z, r = blockIdx.y, lane = threadIdx.x & 31, chunk = blockIdx.x * (kVerifyThreads / 32) + (threadIdx.x >> 5);
  if (chunk >= a.chunks || !row_wanted(a, r, drafted(a, s))) return;
  const float *x = logits_row(a, s, r) + (long long)chunk * kVerifyChunk + lane;
  const int n = min(a.V - chunk * kVerifyChunk, kVerifyChunk) - lane;
  const float c = (float)(1.4426950408889634 / a.temperature);
  float v[kVerifyVals], next[kVerifyVals], m = -INFINITY, sum = 0.f;
#pragma unroll
  for (int u = 0; u < kVerifyVals; u++) next[u] = 32 * u < n ? __ldcg(x + 32 * u) : -INFINITY;
#pragma unroll
  for (int t = 0; t < kVerifyTurns; t++) {
    if (t * 32 * kVerifyVals >= n + lane) break;  // the same for the warp
    float top = m;
#pragma unroll
    for (int u = 0; u < kVerifyVals; u++) top = fmaxf(top, v[u] = fmaxf(next[u], -INFINITY));  // NaN counts as -infinity
    if (t + 1 < kVerifyTurns) {
#pragma unroll
      for (int u = 0; u < kVerifyVals; u++) {
        const int i = 32 * (u + (t + 1) * kVerifyVals);
        next[u] = i < n ? __ldcg(x + i) : -INFINITY;
      }
    }
    if (top == -INFINITY) continue;
    sum *= exp2_of((m - top) * c);
    m = top;
#pragma unroll
    for (int u = 0; u < kVerifyVals; u++) sum += exp2_of((v[u] - m) * c);
  }
  const float top = warp_max(m);
  double all = m > -INFINITY ? (double)(sum * exp2_of((m - top) * c)) : 0.0;
  all = warp_sum64(all);
  if (lane == 0) a.partial[((long long)s * (2 * a.n_draft + 1) + r) * a.chunks + chunk] = make_float2(top, (float)all);
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

// top_k > 0: the kept logits of a row in descending order, their sum of exponentials and the drafted id's probability, by one CTA.
// The largest values of 128 groups of threads give a bound, the top_k-th largest of them, that at least top_k values reach; what
// reaches it is mostly little more than that, and is ranked by counting. A row made so that more reach it than the list holds goes
// by the threads' largest keys (of the value, among equals of the lowest index) instead: what reaches the top_k-th largest of
// those lies in top_k threads' shares. One round over the row and one over a few threads' shares of it: with the draw 20 us for 16
// users with 5 drafts and 40 kept logits (29 MB), where a CTA reads its 200 KB at what one SM gets.
constexpr int kListThreads = 1024, kListGroups = 128, kListCap = 1536, kListVals = 28;

__global__ void __launch_bounds__(kListThreads) verify_list_kernel(const __grid_constant__ Verify a, int cap) {
  extern __shared__ __align__(16) unsigned long long cand[];  // [cap], cap >= kListCap and top_k * ceil(V / kListThreads)
  __shared__ __align__(16) float group[kListGroups];
  __shared__ unsigned long long top[128];
  __shared__ double ev[128];
  __shared__ int count, n_shares;
  __shared__ short shares[kListThreads];
  __shared__ float s_bound;
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.y, r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.top_k;
  if (!row_wanted(a, r, drafted(a, s))) return;
  const float *x = logits_row(a, s, r);
  float m = -INFINITY;
  for (int i0 = tid; i0 < a.V; i0 += kListVals * kListThreads) {
    float v[kListVals];
#pragma unroll
    for (int u = 0; u < kListVals; u++) v[u] = i0 + u * kListThreads < a.V ? __ldcg(x + i0 + u * kListThreads) : -INFINITY;
#pragma unroll
    for (int u = 0; u < kListVals; u++) m = fmaxf(m, v[u]);  // NaN is passed over
  }
  const float own = m;
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((lane & 7) == 0) group[tid >> 3] = m;
  if (tid == 0) {
    count = n_shares = 0;
    s_bound = -INFINITY;
  }
  __syncthreads();
  if (tid < kListGroups) {
    const float mine = group[tid];
    int above = 0, upto = 0;
#pragma unroll 8
    for (int j = 0; j < kListGroups / 4; j++) {
      const float4 g = reinterpret_cast<const float4 *>(group)[j];
      above += (g.x > mine ? 1 : 0) + (g.y > mine ? 1 : 0) + (g.z > mine ? 1 : 0) + (g.w > mine ? 1 : 0);
      upto += (g.x >= mine ? 1 : 0) + (g.y >= mine ? 1 : 0) + (g.z >= mine ? 1 : 0) + (g.w >= mine ? 1 : 0);
    }
    if (above < K && K <= upto) s_bound = mine;  // equal ones write the same
  }
  __syncthreads();
  // the threads' shares that something at the bound lies in, a warp a share
  const float bound = s_bound;
  if (own >= bound) shares[atomicAdd(&n_shares, 1)] = (short)tid;
  __syncthreads();
  const int per_thread = (a.V + kListThreads - 1) / kListThreads;
  for (int j = warp; j < n_shares; j += kListThreads / 32) {
    const int share = shares[j];
#pragma unroll 2
    for (int u = lane; u < per_thread; u += 32) {
      const int i = share + u * kListThreads;
      if (i >= a.V) continue;
      const float y = logit(x + i);
      if (y >= bound) {
        const int at = atomicAdd(&count, 1);
        if (at < cap) cand[at] = sample_key(y, i);
      }
    }
  }
  __syncthreads();
  if (count > cap) {  // the same for all
    unsigned long long best = 0ull, least = 0ull;
    for (int i = tid; i < a.V; i += kListThreads) {
      const unsigned long long k = sample_key(logit(x + i), i);
      best = k > best ? k : best;
    }
    for (int bit = 63; bit >= 0; bit--) {
      const unsigned long long trial = least | 1ull << bit;
      if (__syncthreads_count(best >= trial) >= K) least = trial;
    }
    __syncthreads();
    if (tid == 0) count = 0;
    __syncthreads();
    if (best >= least)
      for (int i = tid; i < a.V; i += kListThreads) {
        const unsigned long long k = sample_key(logit(x + i), i);
        if (k >= least) {
          const int at = atomicAdd(&count, 1);
          if (at < cap) cand[at] = k;
        }
      }
    __syncthreads();
  }
  const int n = min(count, cap);
  const long long row = (long long)s * (2 * a.n_draft + 1) + r, to = row * K;
  for (int i = tid; i < n; i += kListThreads) {
    const unsigned long long mine = cand[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; j++) rank += cand[j] > mine ? 1 : 0;
    if (rank < K) {
      top[rank] = mine;
      a.list_value[to + rank] = sample_key_value(mine);
      a.list_id[to + rank] = sample_key_index(mine);
    }
  }
  __syncthreads();
  if (tid < K) ev[tid] = exp(((double)sample_key_value(top[tid]) - (double)sample_key_value(top[0])) / a.temperature);
  __syncthreads();
  if (warp == 0) {
    double z = 0.0, p = 0.0;
    const int i = r <= a.n_draft ? r : r - a.n_draft - 1;
    const uint32_t id = i < a.n_draft ? __ldcg(a.draft_ids + (long long)s * a.n_draft + i) : kNoId;
    for (int j = lane; j < K; j += 32) {
      z += ev[j];
      if ((uint32_t)sample_key_index(top[j]) == id) p = ev[j];
    }
    z = warp_sum64(z);
    p = warp_sum64(p);
    if (lane == 0) a.list_sum[row] = make_double2(z, p / z);
  }
}

// ids_out and n_accepted of a sequence, once `accepted` and the drawn id are known.
template <int NT>
__device__ __forceinline__ void write_ids(const Verify &a, int s, int accepted, uint32_t drawn, int tid) {
  for (int i = tid; i <= a.n_draft; i += NT)
    a.ids_out[(long long)s * (a.n_draft + 1) + i] =
        i < accepted ? __ldcg(a.draft_ids + (long long)s * a.n_draft + i) : i == accepted ? drawn : kNoId;
  if (tid == 0) a.n_accepted[s] = accepted;
}

// The accept step and the draw over the whole vocabulary, a cluster of CTAs per sequence. The draw needs running sums good to
// far below the smallest probability, so its exponentials are in double precision: those of the target's row, and of the draft's if a
// draft was not accepted, each by its row's sum, which the accept step has (good to a few 1e-8; the same for rows that are the same,
// so that nothing is left of them). Every warp takes a stretch of ids; the sums of the stretches say in which one the running sum passes the
// number, and that warp adds its stretch up id by id. A lane keeps its exponentials where they fit kVals registers. Bound by latency
// (logits, exponentials, two barriers of the cluster): one user with 4 drafts 15 us with the sums, 64 users 51; the FP64 pipe is
// busy a fifth of the time. Going over the rows a second time for their own sums took 64.
constexpr int kDrawThreads = 512, kDrawWarps = kDrawThreads / 32, kDrawCluster = 8;

template <int kVals>
__global__ void __launch_bounds__(kDrawThreads, kVals > 0 ? 1 : 2) verify_draw_kernel(const __grid_constant__ Verify a) {
  __shared__ int first_rejected;
  __shared__ float s_max[2 * kMaxDraft + 1];
  __shared__ double s_sum[2 * kMaxDraft + 1];
  __shared__ double table[64];
  __shared__ double sums[2][kDrawCluster][kDrawWarps];  // of every warp of the cluster: the target's, what a draft leaves of it
  uint32_t C;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(C));
  const int rank = (int)cluster_ctarank(), s = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < 2 * kDrawCluster * kDrawWarps; i += kDrawThreads) (&sums[0][0][0])[i] = 0.0;  // of CTAs that are not there too
  cluster_arrive();
  if (tid < 64) table[tid] = exp2(tid / 64.0);
  pdl_launch_dependents();
  pdl_wait();
  const double u01 = __ldcg(a.uniforms + (long long)s * (a.n_draft + 1) + a.n_draft);
  const int n = drafted(a, s), rows = 2 * a.n_draft + 1;
  if (tid == 0) first_rejected = n;
  __syncthreads();
  // every CTA finds the first draft that is not accepted: (largest, sum) of the rows, a warp each
  const double scale = 64.0 / (0.6931471805599453 * a.temperature);
  const float2 *part = a.partial + (long long)s * rows * a.chunks;
  for (int r = warp; r < rows; r += kDrawWarps) {
    if (!row_wanted(a, r, n) || (r > a.n_draft && !a.draft)) continue;
    float m = -INFINITY;
    for (int c = lane; c < a.chunks; c += 32) m = fmaxf(m, __ldcg(part + r * a.chunks + c).x);
    m = warp_max(m);
    double z = 0.0;
    for (int c = lane; c < a.chunks; c += 32) {
      const float2 p = __ldcg(part + r * a.chunks + c);
      if (p.x > -INFINITY) z += (double)p.y * exp_of((double)p.x - (double)m, scale, table);
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
      const double p = exp_of((double)logit(logits_row(a, s, i) + x) - (double)s_max[i], scale, table) / s_sum[i];
      const double q = a.draft ? exp_of((double)logit(logits_row(a, s, rq) + x) - (double)s_max[rq], scale, table) / s_sum[rq] : 1.0;
      ok = __ldcg(a.uniforms + (long long)s * (a.n_draft + 1) + i) * q < p;
    }
    if (!ok) atomicMin(&first_rejected, i);
  }
  __syncthreads();
  const int at = first_rejected;
  const float *x = logits_row(a, s, at), *y = nullptr;
  const double m = s_max[at];
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
  const bool two = rest && y != nullptr;
  constexpr int kLook = kVals > 0 ? kVals : 4, kPick = 4;
  double vx[kVals > 0 ? kVals : 1];
  // a lane's logits of ids i0, i0 + 32, ...: -infinity, which counts nothing, behind the stretch
  auto fetch = [&](int i0, auto &lx, auto &ly) {
#pragma unroll
    for (int u = 0; u < (int)(sizeof(lx) / sizeof(float)); u++) {
      const int i = i0 + 32 * u;
      lx[u] = i < end ? logit(x + i) : -INFINITY;
      ly[u] = two && rest && i < end ? logit(y + i) : -INFINITY;
    }
  };
  // what an id counts: its exponential; where a draft was turned down that by its row's sum, less the draft's (or less all of it
  // at the drafted id), none below zero
  const double ix = none ? 0.0 : 1.0 / s_sum[at], iq = two ? 1.0 / s_sum[a.n_draft + 1 + at] : 0.0;
  auto weight = [&](float lx, float ly, int i) {
    const double e = exp_of((double)lx - m, scale, table);
    if (!rest) return e;
    const double q = two ? __dmul_rn(exp_of((double)ly - mq, scale, table), iq) : (uint32_t)i == only ? 1.0 : 0.0;
    return fmax(__dmul_rn(e, ix) - q, 0.0);  // rounded alike, so that equal rows leave zeros
  };
  // every warp's sum over its stretch, told to every CTA, behind one barrier of the cluster
  auto add_up = [&]() {
    double sum = 0.0;
    if (!none) {
      if constexpr (kVals > 0) {
        float lx[kVals], ly[kVals];
        fetch(beg + lane, lx, ly);
#pragma unroll
        for (int u = 0; u < kVals; u++) {
          if (beg + 32 * u >= end) break;
          sum += vx[u] = weight(lx[u], ly[u], beg + lane + 32 * u);
        }
      } else {
        for (int i0 = beg + lane; i0 < end; i0 += 32 * kLook) {
          float lx[kLook], ly[kLook];
          fetch(i0, lx, ly);
#pragma unroll
          for (int u = 0; u < kLook; u++) sum += weight(lx[u], ly[u], i0 + 32 * u);
        }
      }
      sum = warp_sum64(sum);
      if (lane < (int)C)
        dsmem_st64(dsmem_addr(&sums[rest ? 1 : 0][rank][warp], lane), (unsigned long long)__double_as_longlong(sum));
    }
    cluster_arrive();
    cluster_wait();
  };
  // of all warps' sums: what lies before each, and their total; every warp for itself, four sums a lane
  constexpr int kAll = kDrawCluster * kDrawWarps, kPer = kAll / 32;
  double upto[kPer], from;
  auto prefixes = [&]() {
    const double *v = &sums[rest ? 1 : 0][0][0] + lane * kPer;
    double sum = 0.0;
#pragma unroll
    for (int u = 0; u < kPer; u++) upto[u] = sum += v[u];
    from = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, from, o);
      if (lane >= o) from += up;
    }
    const double total = __shfl_sync(0xffffffffu, from, 31);
    from = __shfl_up_sync(0xffffffffu, from, 1);
    if (lane == 0) from = 0.0;
    return total;
  };
  cluster_wait();  // the others run
  add_up();
  double total = prefixes();
  if (rest && !(total > 0.0)) {  // nothing is left, in the whole cluster's eyes: drawn from the target's row itself
    rest = false;
    add_up();
    total = prefixes();
  }
  if (!none) {
    // the last stretch with anything in it that begins at or below the goal has the id (rounding may put the beginning of an empty
    // one there); one warp adds it up
    const double goal = u01 * total, *of = &sums[rest ? 1 : 0][0][0] + lane * kPer;
    int mine = -1;
#pragma unroll
    for (int u = 0; u < kPer; u++)
      if ((u == 0 ? from : from + upto[u - 1]) <= goal && of[u] > 0.0) mine = lane * kPer + u;
    const int owner = __reduce_max_sync(0xffffffffu, mine);
    if (owner == rank * kDrawWarps + warp) {
      double before = 0.0;
#pragma unroll
      for (int u = 0; u < kPer; u++)
        if (mine == owner && owner == lane * kPer + u) before = u == 0 ? from : from + upto[u - 1];
      before = __shfl_sync(0xffffffffu, before, owner / kPer);
      int last = -1, found = -1;  // the stretch's sum was rounded in another order: it may pass the goal where the running sum does not
      auto look = [&](int i0, double w) {  // 32 ids
        double run = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double up = __shfl_up_sync(0xffffffffu, run, o);
          if (lane >= o) run += up;
        }
        const unsigned past = __ballot_sync(0xffffffffu, i0 + lane < end && before + run > goal);
        found = past ? i0 + __ffs(past) - 1 : last;  // the row's sum, rounded in another order, passed the goal
      };
      // 32 ids at a time: first the sums of some such rows, then the one in which the goal is passed, id by id
      auto rows_of = [&](int i0, double (&w)[kPick]) {
        double sum[kPick];
#pragma unroll
        for (int u = 0; u < kPick; u++) sum[u] = w[u];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
          for (int u = 0; u < kPick; u++) sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], o);
#pragma unroll
        for (int u = 0; u < kPick; u++) {
          if (found >= 0 || sum[u] == 0.0) continue;
          last = i0 + 32 * u + 31 - __clz(__ballot_sync(0xffffffffu, w[u] > 0.0));
          if (before + sum[u] > goal) look(i0 + 32 * u, w[u]);
          before += sum[u];
        }
      };
      if constexpr (kVals > 0) {
#pragma unroll
        for (int h = 0; h < kVals; h += kPick) {
          double w[kPick];
#pragma unroll
          for (int u = 0; u < kPick; u++) w[u] = beg + 32 * (h + u) < end ? vx[h + u] : 0.0;
          if (found < 0) rows_of(beg + 32 * h, w);
        }
      } else {
        for (int i0 = beg; i0 < end && found < 0; i0 += 32 * kPick) {
          double w[kPick];
          float lx[kPick], ly[kPick];
          fetch(i0 + lane, lx, ly);
#pragma unroll
          for (int u = 0; u < kPick; u++) w[u] = weight(lx[u], ly[u], i0 + lane + 32 * u);
          rows_of(i0, w);
        }
      }
      write_ids<32>(a, s, at, (uint32_t)(found < 0 ? last : found), lane);
    } else if (owner < 0 && rank == 0 && warp == 0) {  // a number that is none
      write_ids<32>(a, s, at, (uint32_t)(a.V - 1), lane);
    }
  } else if (rank == 0 && warp == 0) {
    if (lane == 0) *a.err = kErrRow;
    write_ids<32>(a, s, at, 0u, lane);
  }
}

// The same over the kept lists, one CTA per sequence.
__global__ void __launch_bounds__(128) verify_draw_list_kernel(const __grid_constant__ Verify a) {
  __shared__ int first_rejected, s_pick;
  __shared__ double w_list[128];
  __shared__ float vq[128];
  __shared__ int iq[128];
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.x, tid = threadIdx.x, K = a.top_k;
  const double u01 = __ldcg(a.uniforms + (long long)s * (a.n_draft + 1) + a.n_draft);
  const int n = drafted(a, s);
  if (tid == 0) first_rejected = n;
  __syncthreads();
  const long long base = (long long)s * (2 * a.n_draft + 1);
  auto top_of = [&](int r) { return __ldcg(a.list_value + (base + r) * K); };
  if (tid < n) {
    const int i = tid, rq = a.n_draft + 1 + i;
    const uint32_t x = __ldcg(a.draft_ids + (long long)s * a.n_draft + i);
    bool ok = false;
    if (x >= (uint32_t)a.V) {
      *a.err = 1;
    } else if (!isinf(top_of(i)) && !(a.draft && isinf(top_of(rq)))) {
      const double p = __ldcg(a.list_sum + base + i).y, q = a.draft ? __ldcg(a.list_sum + base + rq).y : 1.0;
      ok = __ldcg(a.uniforms + (long long)s * (a.n_draft + 1) + i) * q < p;
    }
    if (!ok) atomicMin(&first_rejected, i);
  }
  __syncthreads();
  const int at = first_rejected, rq = a.n_draft + 1 + at;
  const double m = top_of(at);
  if (isinf(m)) {
    if (tid == 0) *a.err = kErrRow;
    write_ids<128>(a, s, at, 0u, tid);
    return;
  }
  bool rest = at < n;
  double mq = 0.0, zq = 1.0;
  if (rest && a.draft) {
    mq = top_of(rq);
    zq = __ldcg(a.list_sum + base + rq).x;
    if (isinf(mq)) {
      if (tid == 0) *a.err = kErrRow;
      rest = false;
    }
    if (tid < K) {
      vq[tid] = __ldcg(a.list_value + (base + rq) * K + tid);
      iq[tid] = __ldcg(a.list_id + (base + rq) * K + tid);
    }
  }
  const double z = __ldcg(a.list_sum + base + at).x;
  const uint32_t id = tid < K ? (uint32_t)__ldcg(a.list_id + (base + at) * K + tid) : kNoId;
  double p = 0.0, w = 0.0;
  __syncthreads();
  if (tid < K) {
    p = exp(((double)__ldcg(a.list_value + (base + at) * K + tid) - m) / a.temperature) / z;
    w = p;
    if (rest) {
      double q = 0.0;
      if (a.draft) {
        int j = -1;
#pragma unroll 8
        for (int i = 0; i < K; i++)
          if ((uint32_t)iq[i] == id) j = i;
        if (j >= 0) q = exp(((double)vq[j] - mq) / a.temperature) / zq;
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
  // the running sums of the list, four entries a lane
  if (tid < 32) {
    double run[4], from = 0.0;
#pragma unroll
    for (int u = 0; u < 4; u++) run[u] = from += 4 * tid + u < K ? w_list[4 * tid + u] : 0.0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, from, o);
      if (tid >= o) from += up;
    }
    const double goal = u01 * __shfl_sync(0xffffffffu, from, 31);
    from = __shfl_up_sync(0xffffffffu, from, 1);
    if (tid == 0) from = 0.0;
    int pick = 127, last = -1;
#pragma unroll
    for (int u = 3; u >= 0; u--) {
      if (from + run[u] > goal) pick = 4 * tid + u;
      if (4 * tid + u < K && w_list[4 * tid + u] > 0.0) last = max(last, 4 * tid + u);
    }
    pick = __reduce_min_sync(0xffffffffu, pick);
    last = __reduce_max_sync(0xffffffffu, last);
    if (tid == 0) s_pick = min(pick, last);
  }
  __syncthreads();
  write_ids<128>(a, s, at, (uint32_t)__ldcg(a.list_id + (base + at) * K + s_pick), tid);
}

}  // namespace wgpt
