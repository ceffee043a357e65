// Verification of drafted tokens against the target's probabilities (speculative sampling), from given random numbers.
#pragma once
#include <cfloat>

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
// own running maximum until the end. Tells whether a draft is accepted wherever the answer is not close (kUnsure).
// Bound by bytes: 64 users with up to 4 drafts over 50257 ids (85 MB) 20 us, 4.3 TB/s, launch and ragged ends included.
constexpr int kVerifyThreads = 256, kVerifyVals = 16, kVerifyTurns = 4, kVerifyChunk = 32 * kVerifyVals * kVerifyTurns;

__global__ void __launch_bounds__(kVerifyThreads) verify_sums_kernel(const __grid_constant__ Verify a) {
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.z, r = blockIdx.y, lane = threadIdx.x & 31, chunk = blockIdx.x * (kVerifyThreads / 32) + (threadIdx.x >> 5);
  if (chunk >= a.chunks || !row_wanted(a, r, drafted(a, s))) return;
  const float *x = logits_row(a, s, r) + (long long)chunk * kVerifyChunk + lane;
  const int n = min(a.V - chunk * kVerifyChunk, kVerifyChunk) - lane;
  const float c = (float)fmin(1.4426950408889634 / a.temperature, (double)FLT_MAX);  // finite: zero times it is zero
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

// The accept step and the draw over the whole vocabulary, a cluster of CTAs per sequence, in double precision.
// Accepting: u q < p is decided by the sums in f32 unless the two sides are within kUnsure of one another; both rows are
// added up in double precision by the cluster then, for one in some 30 000 drafts.
// The draw needs running sums good to far below the smallest probability: those of e_p where all drafts were accepted, else of
// max(e_p / Z_p - e_q / Z_q, 0), here times Z_p Z_q. The rows' sums Z would have to be known first; but they hardly change which ids
// count. So the ids are told apart by the f32 sums (a difference of two logits against a border), and the same round adds up both
// rows and, over the ids that count, both rows again: Z_q sum e_p - Z_p sum e_q of a stretch is off by the ids on the wrong side alone, which are
// few and whose terms are within the f32 sums' error of zero. Where little is left (kLeft) that might still be seen, and a second round
// tells them apart by the good sums. Equal rows have equal sums and leave zeros.
// Every warp takes a stretch of ids; the sums of the stretches say in which one the running sum passes the number, and the warps of
// its CTA add that stretch up id by id, a row of 32 ids each.
// Bound by latency (logits, exponentials, three barriers of the cluster): one user with 4 drafts over 50257 ids 15.0 us with the sums, 64 users
// 43.5.
constexpr int kDrawThreads = 512, kDrawWarps = kDrawThreads / 32, kDrawCluster = 8;
// A row's sum in f32 is off by less than 1e-5 of itself: 70 roundings of a lane's additions and of its five rescalings (2^-24 each), six
// exponentials (2^-22), and three roundings in each exponent's argument, (largest - logit) / temperature, whose mean over the
// distribution is below ln V <= 21. Both sums of a draft's two rows: 2e-5.
constexpr double kUnsure = 1.0 / 32768;
constexpr double kLeft = 1.0 / 16;
constexpr double kNoise = 1.5e-14;  // a difference below this much of its terms is their rounding: nothing

// A row's sum of exponentials in double precision, by the whole cluster of C CTAs; every thread gets it. A lane has the ids i0, i0 + 32,
// ... below end; places: a number for each warp of the cluster, the same in every CTA, those of CTAs that are not there zero.
__device__ __noinline__ double draw_row_sum(const float *x, float top, int i0, int end, double scale, const double *table, double *places,
                                            int place, int C, int lane) {
  double sum = 0.0;
  for (int i = i0; i < end; i += 32) sum += exp_of((double)logit(x + i) - (double)top, scale, table);
  sum = warp_sum64(sum);
  if (lane < C) dsmem_st64(dsmem_addr(places + place, lane), (unsigned long long)__double_as_longlong(sum));
  cluster_arrive();
  cluster_wait();
  sum = 0.0;
  for (int i = lane; i < kDrawCluster * kDrawWarps; i += 32) sum += places[i];
  sum = warp_sum64(sum);
  cluster_arrive();  // before the places are written again
  cluster_wait();
  return sum;
}

// kLook: logits of a row that a lane asks for at once.
template <int kLook, int kCtas>
__global__ void __launch_bounds__(kDrawThreads, kCtas) verify_draw_kernel(const __grid_constant__ Verify a) {
  __shared__ int first_rejected, s_last;
  __shared__ unsigned s_unsure[2];  // drafts that the sums in f32 do not decide
  __shared__ float s_max[2 * kMaxDraft + 1];
  __shared__ double s_sum[2 * kMaxDraft + 1];
  __shared__ double table[64];
  // of every warp of the cluster, for each round: the target's row, the draft's, and both over the ids that count
  __shared__ double sums[2][4][kDrawCluster][kDrawWarps];
  __shared__ double s_row[2][32];  // sums of rows of 32 ids
  __shared__ double s_found[4];    // total, the rows' sums, what lies before the stretch that has the id
  __shared__ int s_owner;
  uint32_t C;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(C));
  const int rank = (int)cluster_ctarank(), s = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < 8 * kDrawCluster * kDrawWarps; i += kDrawThreads) (&sums[0][0][0][0])[i] = 0.0;  // of CTAs that are not there too
  cluster_arrive();
  if (tid < 64) table[tid] = exp2(tid / 64.0);
  pdl_launch_dependents();
  pdl_wait();
  const double u01 = __ldcg(a.uniforms + (long long)s * (a.n_draft + 1) + a.n_draft);
  const int n = drafted(a, s), rows = 2 * a.n_draft + 1;
  if (tid == 0) first_rejected = n;
  __syncthreads();
  const int stretch = (a.V + (int)C * kDrawWarps - 1) / ((int)C * kDrawWarps);
  const int beg = min(a.V, (rank * kDrawWarps + warp) * stretch), end = min(a.V, beg + stretch);
  // every CTA finds the first draft that is not accepted: (largest, sum) of the rows, a warp each
  const double scale = fmin(64.0 / (0.6931471805599453 * a.temperature), DBL_MAX);
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
  auto weight_of = [&](int r, uint32_t id) { return exp_of((double)logit(logits_row(a, s, r) + id) - (double)s_max[r], scale, table); };
  if (tid < 64) {
    const int i = tid, rq = a.n_draft + 1 + i;
    bool open = false;
    if (i < n) {
      const uint32_t x = __ldcg(a.draft_ids + (long long)s * a.n_draft + i);
      bool ok = false;
      if (x >= (uint32_t)a.V) {
        *a.err = 1;
      } else if (!isinf(s_max[i]) && !(a.draft && isinf(s_max[rq]))) {
        // u q < p with both sides times Z_p Z_q
        const double p = weight_of(i, x) * (a.draft ? s_sum[rq] : 1.0),
                     uq = __ldcg(a.uniforms + (long long)s * (a.n_draft + 1) + i) * (a.draft ? weight_of(rq, x) : 1.0) * s_sum[i];
        ok = uq < p;
        open = p > 0.0 && fabs(uq - p) <= kUnsure * p;
      }
      if (!ok && !open) atomicMin(&first_rejected, i);
    }
    const unsigned all = __ballot_sync(0xffffffffu, open);
    if (lane == 0) s_unsure[warp] = all;
  }
  __syncthreads();
  int at = first_rejected;
  cluster_wait();  // the others run
  auto row_sum = [&](int r) {
    return draw_row_sum(logits_row(a, s, r), s_max[r], beg + lane, end, scale, table, &sums[0][0][0][0], rank * kDrawWarps + warp, (int)C, lane);
  };
  unsigned long long unsure = (unsigned long long)s_unsure[1] << 32 | s_unsure[0];
  for (; unsure != 0; unsure &= unsure - 1) {  // the same for the whole cluster
    const int i = __ffsll((long long)unsure) - 1;
    if (i >= at) break;
    const uint32_t x = __ldcg(a.draft_ids + (long long)s * a.n_draft + i);
    const int rq = a.n_draft + 1 + i;
    const double p = weight_of(i, x) * (a.draft ? row_sum(rq) : 1.0), q = (a.draft ? weight_of(rq, x) : 1.0) * row_sum(i);
    if (!(__ldcg(a.uniforms + (long long)s * (a.n_draft + 1) + i) * q < p)) at = i;
  }
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
  const bool none = isinf(m), two = rest && y != nullptr;
  auto exp_x = [&](float l) { return exp_of((double)l - m, scale, table); };
  auto exp_y = [&](float l) { return exp_of((double)l - mq, scale, table); };
  double zp = none ? 1.0 : s_sum[at], zq = two ? s_sum[a.n_draft + 1 + at] : 1.0;
  // an id counts where its target's logit is further above its draft's than this: e_p z_q > e_q z_p
  const float border = two && !none ? (float)(m - mq + a.temperature * (double)logf((float)zp / (float)zq)) : 0.f;
  // every warp's sums over its stretch, told to every CTA, behind one barrier of the cluster
  int round = 0;
  auto add_up = [&]() {
    double sum[4] = {0.0, 0.0, 0.0, 0.0};
    if (!none) {
      float lx[kLook], ly[kLook], next_x[kLook], next_y[kLook];
      auto fetch = [&](int i0) {  // -infinity, which counts nothing, behind the stretch
#pragma unroll
        for (int u = 0; u < kLook; u++) {
          const int i = i0 + 32 * u;
          next_x[u] = i < end ? logit(x + i) : -INFINITY;
          next_y[u] = two && i < end ? logit(y + i) : -INFINITY;
        }
      };
      fetch(beg + lane);
      for (int i0 = beg + lane; i0 - lane < end; i0 += 32 * kLook) {
#pragma unroll
        for (int u = 0; u < kLook; u++) {
          lx[u] = next_x[u];
          ly[u] = next_y[u];
        }
        fetch(i0 + 32 * kLook);
        double e[kLook], f[kLook];
#pragma unroll
        for (int u = 0; u < kLook; u++) sum[0] += e[u] = exp_x(lx[u]);
        if (two) {
#pragma unroll
          for (int u = 0; u < kLook; u++) sum[1] += f[u] = exp_y(ly[u]);
#pragma unroll
          for (int u = 0; u < kLook; u++) {
            const bool in = round == 0 ? lx[u] - ly[u] > border : __dmul_rn(e[u], zq) > __dmul_rn(f[u], zp);
            sum[2] += in ? e[u] : 0.0;
            sum[3] += in ? f[u] : 0.0;
          }
        } else if (rest) {
#pragma unroll
          for (int u = 0; u < kLook; u++) sum[2] += (uint32_t)(i0 + 32 * u) == only ? 0.0 : e[u];
        }
      }
      if (two) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
          for (int k = 0; k < 4; k++) sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], o);
      } else {
        sum[0] = warp_sum64(sum[0]);
        if (rest) sum[2] = warp_sum64(sum[2]);
      }
      if (lane < (int)C) {
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (k == 0 || two || (rest && k == 2))
            dsmem_st64(dsmem_addr(&sums[round][k][rank][warp], lane), (unsigned long long)__double_as_longlong(sum[k]));
      }
    }
    cluster_arrive();
    cluster_wait();
  };
  // Of all warps' sums, by one warp, four sums a lane: their total, and the last stretch with anything in it that begins at or below
  // number * total, which has the id (rounding may put the beginning of an empty one there); -1: a number that is none. The other warps
  // doing the same would keep it from the FP64 pipe.
  constexpr int kAll = kDrawCluster * kDrawWarps, kPer = kAll / 32;
  auto before_lane = [&](double upto) {  // no difference: a tiny sum ahead of a large one is not to be lost
    const double x = __shfl_up_sync(0xffffffffu, upto, 1);
    return lane > 0 ? x : 0.0;
  };
  auto find = [&]() {
    const double *v = &sums[round][0][0][0] + lane * kPer;
    const double *v2 = v + (rest ? 2 * kAll : 0);
    double of[kPer], ahead[kPer], up2[kPer], up3[kPer], run2 = 0.0, run3 = 0.0;
#pragma unroll
    for (int u = 0; u < kPer; u++) {
      up2[u] = run2;
      run2 += v2[u];
    }
    double before2 = run2, total;
    if (two && rest) {
      zp = zq = 0.0;
#pragma unroll
      for (int u = 0; u < kPer; u++) {
        up3[u] = run3;
        run3 += v[3 * kAll + u];
        zp += v[u];
        zq += v[kAll + u];
      }
      double before3 = run3;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double a2 = __shfl_up_sync(0xffffffffu, before2, o), a3 = __shfl_up_sync(0xffffffffu, before3, o);
        if (lane >= o) {
          before2 += a2;
          before3 += a3;
        }
        zp += __shfl_xor_sync(0xffffffffu, zp, o);
        zq += __shfl_xor_sync(0xffffffffu, zq, o);
      }
      total = __shfl_sync(0xffffffffu, before2, 31) * zq - __shfl_sync(0xffffffffu, before3, 31) * zp;
      before2 = before_lane(before2);
      before3 = before_lane(before3);
      bool left = false;
#pragma unroll
      for (int u = 0; u < kPer; u++) {
        const double p = v2[u] * zq, w = p - v[3 * kAll + u] * zp;
        of[u] = w > kNoise * p ? w : 0.0;
        left = left || of[u] > 0.0;
        ahead[u] = (before2 + up2[u]) * zq - (before3 + up3[u]) * zp;
      }
      if (!__any_sync(0xffffffffu, left)) total = 0.0;
    } else {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double a2 = __shfl_up_sync(0xffffffffu, before2, o);
        if (lane >= o) before2 += a2;
      }
      total = __shfl_sync(0xffffffffu, before2, 31);
      before2 = before_lane(before2);
#pragma unroll
      for (int u = 0; u < kPer; u++) {
        of[u] = v2[u];
        ahead[u] = before2 + up2[u];
      }
    }
    int mine = -1;
    double from = 0.0;
#pragma unroll
    for (int u = 0; u < kPer; u++)
      if (ahead[u] <= u01 * total && of[u] > 0.0) {
        mine = lane * kPer + u;
        from = ahead[u];
      }
    const int owner = __reduce_max_sync(0xffffffffu, mine);
    if (lane == 0) {
      s_found[0] = total;
      s_found[1] = zp;
      s_found[2] = zq;
      s_owner = owner;
    }
    if (owner >= 0 && mine == owner) s_found[3] = from;
  };
  double total;
  for (bool added = false;;) {  // the same for the whole cluster
    if (!added) add_up();
    added = true;
    if (warp == 0) find();
    __syncthreads();
    total = s_found[0];
    zp = s_found[1];
    zq = s_found[2];
    if (two && rest && !none && round == 0 && total < kLeft * zp * zq) {  // again, with the good sums
      round = 1;
      added = false;
    } else if (rest && !(total > 0.0)) {  // nothing is left: drawn from the target's row itself
      rest = false;
    } else {
      break;
    }
    __syncthreads();  // before the places are written again
  }
  if (none) {
    if (rank == 0 && warp == 0) {
      if (lane == 0) *a.err = kErrRow;
      write_ids<32>(a, s, at, 0u, lane);
    }
    return;
  }
  const double goal = u01 * total;
  const int owner = s_owner;
  if (owner < 0) {
    if (rank == 0 && warp == 0) write_ids<32>(a, s, at, (uint32_t)(a.V - 1), lane);
    return;
  }
  if (owner / kDrawWarps != rank) return;
  double before = s_found[3];
  if (tid == 0) s_last = owner * stretch;  // an id whatever rounding does in very long stretches
  // The stretch's rows of 32 ids, two a warp at a time: their sums, then, in the first whose running sum passes the goal, id by
  // id. The stretch's sum was rounded in another order and may pass the goal where the running sum does not: the last id that counts then.
  constexpr int kRows = 2;
  static_assert(kRows * kDrawWarps == 32, "a lane a row");
  const int own_end = min(a.V, (owner + 1) * stretch);
  for (int i0 = owner * stretch, turn = 0; i0 < own_end; i0 += 32 * 32, turn ^= 1) {
    double w[kRows], sum[kRows];
    float lx[kRows], ly[kRows];
#pragma unroll
    for (int u = 0; u < kRows; u++) {
      const int i = i0 + 32 * (u * kDrawWarps + warp) + lane;
      lx[u] = i < own_end ? logit(x + i) : -INFINITY;
      ly[u] = two && i < own_end ? logit(y + i) : -INFINITY;
    }
#pragma unroll
    for (int u = 0; u < kRows; u++) {
      w[u] = exp_x(lx[u]);
      if (rest && two)
        w[u] = fmax(__dmul_rn(w[u], zq) - __dmul_rn(exp_y(ly[u]), zp), 0.0);
      else if (rest && (uint32_t)(i0 + 32 * (u * kDrawWarps + warp) + lane) == only)
        w[u] = 0.0;
      sum[u] = w[u];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int u = 0; u < kRows; u++) sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], o);
    if (lane == 0)
      for (int u = 0; u < kRows; u++) s_row[turn][u * kDrawWarps + warp] = sum[u];
    __syncthreads();
    const double row = s_row[turn][lane];
    double run = row;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    const unsigned full = __ballot_sync(0xffffffffu, row > 0.0), past = __ballot_sync(0xffffffffu, row > 0.0 && before + run > goal);
    const int hit = past ? __ffs(past) - 1 : 31 - __clz(full);  // a row; -1: all are empty
    const double above = __shfl_sync(0xffffffffu, run - row, hit & 31);
#pragma unroll
    for (int u = 0; u < kRows; u++) {
      if (hit != u * kDrawWarps + warp) continue;
      const int first = i0 + 32 * hit;
      int id = first + 31 - __clz(__ballot_sync(0xffffffffu, w[u] > 0.0));
      if (past) {
        double r = w[u];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double up = __shfl_up_sync(0xffffffffu, r, o);
          if (lane >= o) r += up;
        }
        const unsigned in = __ballot_sync(0xffffffffu, w[u] > 0.0 && before + above + r > goal);
        if (in) id = first + __ffs(in) - 1;
        write_ids<32>(a, s, at, (uint32_t)id, lane);
      } else if (lane == 0) {
        s_last = id;
      }
    }
    if (past) return;  // the same for the whole CTA
    before += __shfl_sync(0xffffffffu, run, 31);
  }
  __syncthreads();
  if (warp == 0) write_ids<32>(a, s, at, (uint32_t)s_last, lane);
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
