// Attention over a paged cache of half-precision values for more than eight rows that share a head of the cache (grouped heads,
// drafts, prompts), head sizes up to 128, on tcgen05: the mathematics, the equal shares and the joining of
// paged_attention_kernel. There every warp's path of loading fragments, eight rows at a time, is what bounds such calls.
//
// Keys are the instruction's 128 lanes and query rows its columns: S^T = K Q^T from shared memory (the key tile as it lies, the
// queries as the sum of two half or three bfloat16 values, whose columns lie beside one another: the tile's bytes, which every
// instruction reads again, are what an instruction of few columns takes), so that a softmax thread has one key and up to 16
// rows. Its probabilities, split the same way, go back to shared memory as the second operand of O^T = V^T P^T, whose first is
// the value tile as it lies, MN-major; there a thread has one dimension and those rows. A tile's O is added to f32 sums in
// registers, so that nothing is accumulated across tiles in tensor memory, whose additions cut off.
//
// A row's maximum would have to be found across the lanes. The exponents are taken relative to a reference instead, a whole
// number at or above the first tile's maximum, that is raised only when some score of a tile is more than 2^kSlack above it: one vote
// a tile, and the maxima across lanes only then.
//   four warps for every 16 rows: softmax and sums;
//   one warp    issues the MMAs: the next tile's scores before this tile's values;
//   four warps  fill a ring of tiles by cp.async, 32 rows each, in the order in which they are used up: K0 K1 V0 K2 V1 ...
// Every wait is bounded; on expiry *err = 3 and the result is void. A row that meets an infinity or NaN is computed again by a warp,
// which may take longer than a wait's polls: a wait begins anew as long as such a warp, or one that looks for its next sequence, gets on.
// Measured, 8 heads of 128, f16, 8 users with up to 5 tokens of 4 rows each: up to 8192 positions (192 MB) 48 us, 4.0 TB/s, of which
// some 25 are the beginning (7), the change from one group to the next and the joins; up to 32768 (663 MB) 117 us, 5.7 TB/s. A tile of
// 64 KB takes a CTA 1.4 us then, which is its share of the copy rate.
#pragma once
#include "paged_attention.cuh"
#include "tcgen05.cuh"

namespace wgpt {

constexpr int kTcKeys = 128, kTcBlock = kTcKeys * 128, kTcRows = 16;  // positions of a tile; bytes of 64 dimensions of one; rows of a softmax thread
constexpr float kSlack = 8.f;

// For each of 16 values the warp's result of f: lanes 2 r and 2 r + 1 get that of value r. Halves of what is left are exchanged, so
// that 16 shuffles do what 80 would.
template <typename F>
__device__ __forceinline__ float warp_each16(const float (&x)[16], int lane, F f) {
  float a[8], b[4], c[2];
  const bool h16 = lane & 16, h8 = lane & 8, h4 = lane & 4, h2 = lane & 2;
#pragma unroll
  for (int i = 0; i < 8; i++) a[i] = f(h16 ? x[i + 8] : x[i], __shfl_xor_sync(0xffffffffu, h16 ? x[i] : x[i + 8], 16));
#pragma unroll
  for (int i = 0; i < 4; i++) b[i] = f(h8 ? a[i + 4] : a[i], __shfl_xor_sync(0xffffffffu, h8 ? a[i] : a[i + 4], 8));
#pragma unroll
  for (int i = 0; i < 2; i++) c[i] = f(h4 ? b[i + 2] : b[i], __shfl_xor_sync(0xffffffffu, h4 ? b[i] : b[i + 2], 4));
  const float d = f(h2 ? c[1] : c[0], __shfl_xor_sync(0xffffffffu, h2 ? c[0] : c[1], 2));
  return f(d, __shfl_xor_sync(0xffffffffu, d, 1));
}

// HB: blocks of 64 dimensions; N: rows of a row tile
template <typename T, int HB, int N>
struct TcShape {
  static constexpr int kTerms = std::is_same<T, __half>::value ? 2 : 3;
  static constexpr int kGroups = N / kTcRows, kSoft = 128 * kGroups, kThreads = kSoft + 32 + 128;
  static constexpr int kStage = HB * kTcBlock;
  static constexpr int kCols = kTerms * N;  // columns of an instruction: the rows' terms beside one another, so that the tile is read once
  static constexpr int kPTile = (kCols + 63) / 64 * kTcBlock, kP = 2 * kPTile, kQ = HB * kCols * 128;
  static constexpr uint32_t kTmem = 4 * kCols <= 128 ? 128 : 4 * kCols <= 256 ? 256 : 512;  // scores and values of two tiles each
  static constexpr int kFit = (int)(((216 << 10) - kP - kQ) / kStage);
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr int kSmem = 1024 + kStages * kStage + kP + kQ;
  static_assert(kStages >= 4, "");
};

// 16 consecutive 32-bit columns of each term, the terms `apart` columns from one another, added up, the last term first.
template <int TERMS>
__device__ __forceinline__ void tmem_ld_terms(uint32_t taddr, uint32_t apart, float (&v)[16]) {
  uint32_t a[16], b[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%32];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%33];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]),
        "=r"(a[8]), "=r"(a[9]), "=r"(a[10]), "=r"(a[11]), "=r"(a[12]), "=r"(a[13]), "=r"(a[14]), "=r"(a[15]),
        "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3]), "=r"(b[4]), "=r"(b[5]), "=r"(b[6]), "=r"(b[7]),
        "=r"(b[8]), "=r"(b[9]), "=r"(b[10]), "=r"(b[11]), "=r"(b[12]), "=r"(b[13]), "=r"(b[14]), "=r"(b[15])
      : "r"(taddr + (TERMS - 1) * apart), "r"(taddr + (TERMS - 2) * apart)
      : "memory");
#pragma unroll
  for (int j = 0; j < 16; j++) v[j] = __uint_as_float(a[j]) + __uint_as_float(b[j]);
  if constexpr (TERMS == 3) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]),
          "=r"(a[8]), "=r"(a[9]), "=r"(a[10]), "=r"(a[11]), "=r"(a[12]), "=r"(a[13]), "=r"(a[14]), "=r"(a[15])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int j = 0; j < 16; j++) v[j] += __uint_as_float(a[j]);
  }
}

template <typename T, int HB, int N>
__global__ void __launch_bounds__((TcShape<T, HB, N>::kThreads), 1) paged_attention_tc_kernel(const __grid_constant__ PagedAttention a) {
  using S = TcShape<T, HB, N>;
  constexpr int TERMS = S::kTerms, NS = S::kStages, R = kTcRows, SOFT = S::kSoft, WARPS = SOFT / 32;
  constexpr float kLift = TERMS == 2 ? 7.f : 0.f;  // probabilities up to 2^(kSlack + kLift), in a half's range
  extern __shared__ uint8_t tc_raw[];
  uint8_t *stages = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(tc_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *Ps = stages + NS * S::kStage, *Qs = Ps + S::kP;
  __shared__ uint64_t full[NS], empty[NS], q_ready, s_done[2], p_ready[2], o_done[2], drained;
  __shared__ uint32_t tmem_slot, s_sum[S::kThreads / 32];
  __shared__ int abort_word, s_last;
  __shared__ unsigned int s_progress, s_odd;  // how far work has come that the others cannot see; rows that came out non-finite
  __shared__ PagedPart s_part[3];  // the softmax warps' part and the next, and a place for the first
  __shared__ __align__(16) float s_qscale[N], s_max[4][N], s_l[N], s_m[N];
  __shared__ int s_lo[N], s_hi[N];
  __shared__ long long s_row[N], s_out[N];  // where the rows' scores and results begin
  __shared__ float4 s_red[SOFT];
  __shared__ float s_red_sum[SOFT];
  volatile int *abort_flag = &abort_word;
  volatile unsigned int *progress = &s_progress;
  const PagedView &c = a.c;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, hs = c.hs;
  if (tid == 0) {
    for (int i = 0; i < NS; i++) {
      mbar_init(&full[i], 128);
      mbar_init(&empty[i], 1);
    }
    mbar_init(&q_ready, WARPS);
    for (int i = 0; i < 2; i++) {
      mbar_init(&s_done[i], 1);
      mbar_init(&p_ready[i], WARPS);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(&drained, 1);
    abort_word = 0;
    s_progress = s_odd = 0;
    fence_async_smem();
  }
  if (warp == WARPS) tmem_alloc(&tmem_slot, S::kTmem);
  if (hs & 63)  // what lies behind a row's end takes part in products: zeros
    for (int i = tid; i < NS * S::kStage / 16; i += S::kThreads) reinterpret_cast<uint4 *>(stages)[i] = make_uint4(0, 0, 0, 0);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_launch_dependents();  // behind the allocation: the next kernel's CTAs may want tensor memory too
  pdl_wait();

  uint32_t per = 1, x1 = 0;
  PagedPart first;
  const bool any = paged_first(a, first, kTcKeys, s_sum, &s_part[2], per, x1);
  // A wait that has run out makes all others return at once: every role runs to its end.
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    if (!*abort_flag && !mbar_wait(bar, parity & 1, TC_POLLS)) {
      unsigned int seen;
      do {
        seen = *progress;
      } while (!*abort_flag && !mbar_wait(bar, parity & 1, TC_POLLS) && *progress != seen);
      if (!mbar_wait(bar, parity & 1, 1)) *abort_flag = 1;
    }
    __syncwarp();
  };

  if (any && warp < WARPS) {
    // ------------------------------------------------------------------ softmax and sums
    const int quad = warp & 3, r0 = (warp >> 2) * R;  // of the tensor memory's lanes; this thread's rows
    const uint32_t lanes = tmem + ((uint32_t)(32 * quad) << 16) + r0;
    const int key = tid & 127;  // of a tile, and the dimension whose sums this thread has
    uint32_t tile = 0;    // of all parts
    auto meet = [] { asm volatile("barrier.cta.sync 1, %0;" ::"n"(SOFT) : "memory"); };
    auto some = [&](bool x) -> bool {  // in any thread of the four warps
      int r;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
          : "=r"(r)
          : "r"((int)x), "n"(SOFT)
          : "memory");
      return r != 0;
    };
    if (tid == 0) s_part[0] = first;
    meet();
    for (int turn = 0;; turn ^= 1) {
      const PagedPart &w = s_part[turn];
      const int rows = w.g.rows, n_tiles = w.n_tiles;
      const long long q_at = lane < rows ? row_offset(a, w, lane, a.ld_q) : -1;  // of the row that is this lane's number
      // ---- the queries: K-major rows of 128 bytes, 16-byte pieces swizzled
      if (n_tiles > 0) {
        constexpr int kMine = N / WARPS;  // rows of a warp, their loads in flight together
        float v[kMine][2 * HB];
#pragma unroll
        for (int y = 0; y < kMine; y++) {
          const int r = warp + y * WARPS;
          const long long at = __shfl_sync(0xffffffffu, q_at, r);
#pragma unroll
          for (int i = 0; i < HB; i++) {
            const int d = 2 * lane + 64 * i;
            const float2 f = at >= 0 && d < hs ? __ldcg(reinterpret_cast<const float2 *>(a.q + at + d)) : make_float2(0.f, 0.f);
            v[y][2 * i] = f.x;
            v[y][2 * i + 1] = f.y;
          }
        }
#pragma unroll
        for (int y = 0; y < kMine; y++) {
          const int r = warp + y * WARPS;
          int e = 0;
          if constexpr (TERMS == 2) {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 2 * HB; i++) top = fmaxf(top, fabsf(v[y][i]));
            top = warp_max(top);
            e = row_exponent(top);
          }
#pragma unroll
          for (int i = 0; i < HB; i++) {
            float f0 = v[y][2 * i] * pow2_of(-e), f1 = v[y][2 * i + 1] * pow2_of(-e);
#pragma unroll
            for (int t = 0; t < TERMS; t++)
              *reinterpret_cast<uint32_t *>(Qs + ((i * TERMS + t) * N + r) * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) =
                  split2<T>(f0, f1);
          }
          if (lane == 0) s_qscale[r] = a.scale2 * pow2_of(e);
        }
      }
      if (tid < N) {
        int lo = 0, hi = 0;
        if (tid < rows) {
          row_range(a, w.q, (w.g.r0 + tid) / a.group, lo, hi);
          s_out[tid] = row_offset(a, w, tid, a.ld_out);
        }
        s_lo[tid] = lo;
        s_hi[tid] = hi;
        if (a.scores) s_row[tid] = row_index(a, w, tid) * c.max_length;
      }
      fence_async_smem();
      meet();
      if (n_tiles > 0 && lane == 0) mbar_arrive(&q_ready);
      // the next part, by one thread while the first scores are on their way
      const bool more = paged_more(a, w, x1);
      if (more && tid == SOFT - 1) paged_next(a, s_part[turn ^ 1], w, x1, kTcKeys, &s_progress);
      __syncwarp();
      float m[R], l[R], o[R];
#pragma unroll
      for (int r = 0; r < R; r++) {
        m[r] = -INFINITY;
        l[r] = 0.f;
        o[r] = 0.f;
      }
      int pos = w.q.begin + w.u0 * kTcKeys + key;
      const uint32_t *table = c.table + (size_t)w.g.s * c.table_stride;
      auto page_of = [&](int p) -> uint32_t {  // asked for a tile ahead
        if (p < w.g.lowest || p >= w.g.highest) return 0xFFFFFFFFu;
        return __ldcg(table + (c.page_shift >= 0 ? (uint32_t)p >> c.page_shift : (uint32_t)p / c.page_size));
      };
      uint32_t page = 0u, page_next = n_tiles > 0 ? page_of(pos) : 0u;
      auto add_values = [&](uint32_t i) {  // of tile i
        wait(&o_done[i & 1], i >> 1);
        tc_fence_after();
        float v[R];
        tmem_ld_terms<TERMS>(lanes + S::kCols * (2 + (i & 1)), N, v);
#pragma unroll
        for (int r = 0; r < R; r++) o[r] += v[r];
      };
      for (int t = 0; t < n_tiles; t++, tile++, pos += kTcKeys) {
        page = page_next;
        page_next = t + 1 < n_tiles ? page_of(pos + kTcKeys) : 0u;
        wait(&s_done[tile & 1], tile >> 1);
        tc_fence_after();
        float x[R];
        tmem_ld_terms<TERMS>(lanes + S::kCols * (tile & 1), N, x);
        const int pos0 = pos - key;
        const bool whole = pos0 >= w.g.inner_low && pos0 + kTcKeys <= w.g.inner_high;
#pragma unroll
        for (int r = 0; r < R; r += 4) {
          const float4 qs = *reinterpret_cast<const float4 *>(s_qscale + r0 + r);
          x[r] *= qs.x;
          x[r + 1] *= qs.y;
          x[r + 2] *= qs.z;
          x[r + 3] *= qs.w;
        }
        const bool there = page < c.n_pages;
        if (!whole || !there) {
#pragma unroll
          for (int r = 0; r < R; r++)
            if (!(there && pos >= s_lo[r0 + r] && pos < s_hi[r0 + r])) x[r] = -INFINITY;
        }
        if (a.scores) {
#pragma unroll
          for (int r = 0; r < R; r++)
            if (r0 + r < rows && pos >= s_lo[r0 + r] && pos < s_hi[r0 + r]) a.scores[s_row[r0 + r] + pos] = x[r];
        }
        bool far = false;
#pragma unroll
        for (int r = 0; r < R; r++) far |= x[r] > m[r] + kSlack;
        __syncwarp();
        bool added = t == 0;  // the last tile's values
        if (some(far)) {  // raise the references of the rows that need it
          if (!added) add_values(tile - 1);
          added = true;
          const float most = warp_each16(x, lane, [](float u, float v) { return fmaxf(u, v); });
          if ((lane & 1) == 0) s_max[quad][r0 + lane / 2] = most;
          meet();
#pragma unroll
          for (int r = 0; r < R; r++) {
            const float top = ceilf(fmaxf(fmaxf(s_max[0][r0 + r], s_max[1][r0 + r]), fmaxf(s_max[2][r0 + r], s_max[3][r0 + r])));
            if (top > m[r]) {
              const float f = exp2f(m[r] - top);
              l[r] *= f;
              o[r] *= f;
              m[r] = top;
            }
          }
          meet();  // before the maxima are written again
        }
        // ---- probabilities: MN-major rows of 128 bytes, a key each, 16-byte pieces of eight rows swizzled
#pragma unroll
        for (int g = 0; g < R / 8; g++) {
          uint32_t words[TERMS][4];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int r = 8 * g + 2 * i;
            float p0 = x[r] == -INFINITY ? 0.f : exp2_of(x[r] - (m[r] - kLift));
            float p1 = x[r + 1] == -INFINITY ? 0.f : exp2_of(x[r + 1] - (m[r + 1] - kLift));
            l[r] += p0;
            l[r + 1] += p1;
#pragma unroll
            for (int u = 0; u < TERMS; u++) words[u][i] = split2<T>(p0, p1);
          }
#pragma unroll
          for (int u = 0; u < TERMS; u++) {
            const int at = (u * N + r0) / 8 + g;  // of the row's 16-byte pieces
            *reinterpret_cast<uint4 *>(Ps + (tile & 1) * S::kPTile + at / 8 * kTcBlock + key * 128 + (((at & 7) ^ (key & 7)) << 4)) =
                make_uint4(words[u][0], words[u][1], words[u][2], words[u][3]);
          }
        }
        fence_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[tile & 1]);
        if (!added) add_values(tile - 1);  // while this tile's are made
      }
      if (n_tiles > 0) add_values(tile - 1);
      tc_fence_before();
      // ---- the rows' sums over the keys
      const float down = kLift != 0.f ? 1.f / 128.f : 1.f;
      uint32_t odd = 0;
      const float mine_sum = warp_each16(l, lane, [](float u, float v) { return u + v; });
      if ((lane & 1) == 0) s_max[quad][r0 + lane / 2] = mine_sum;
#pragma unroll
      for (int r = 0; r < R; r++) {
        o[r] *= down;
        if (r0 + r < rows && key < hs && !(fabsf(o[r]) < INFINITY)) odd |= 1u << (r0 + r);
        if (key == r) s_m[r0 + r] = m[r];
      }
      meet();
      if (tid < N) {
        s_l[tid] = ((s_max[0][tid] + s_max[1][tid]) + (s_max[2][tid] + s_max[3][tid])) * down;
        if (tid < rows && !(fabsf(s_l[tid]) < INFINITY)) odd |= 1u << tid;
      }
      __syncwarp();
      float *values = reinterpret_cast<float *>(Ps);  // the probabilities' place: the products that read them are done
      if (odd != 0) atomicOr(&s_odd, odd);
      if (some(odd != 0)) {  // each such row from what it sees alone, a warp a row
        odd = s_odd;
        uint32_t mine = 0;
        int turn_of = 0;
        for (uint32_t left = odd; left != 0; left &= left - 1)
          if (turn_of++ % WARPS == warp) mine |= left & -left;
        paged_rows_apart<T, kTcKeys, 2 * HB>(a, w, 0, 1, mine, lane, values, s_m, s_l, &s_progress);
        meet();
#pragma unroll
        for (int r = 0; r < R; r++)
          if ((odd >> (r0 + r) & 1u) && key < hs) o[r] = values[(r0 + r) * hs + key];
        if (tid == 0) s_odd = 0;
        meet();
      }
      // ---- the result, or this part of it
      const int first_cta = paged_first_cta(a, w, per), last_cta = (int)((w.end - 1) / per), parts = last_cta - first_cta + 1;
      float *slot = a.partial + (2ll * blockIdx.x + ((int)blockIdx.x == first_cta ? 1 : 0)) * paged_slot(N, hs);
      if (parts == 1) {
        if (tid < N) s_max[0][tid] = s_l[tid] != 0.f ? 1.f / s_l[tid] : 0.f;
        meet();
#pragma unroll
        for (int r = 0; r < R; r++)
          if (r0 + r < rows && key < hs) a.out[s_out[r0 + r] + key] = o[r] * s_max[0][r0 + r];
      } else {
        float *to = slot + r0 * hs + key;
#pragma unroll
        for (int r = 0; r < R; r++, to += hs)
          if (r0 + r < rows && key < hs) __stcg(to, o[r]);
      }
      if (tid < rows) {
        if (parts > 1) {
          __stcg(slot + N * hs + tid, s_m[tid]);
          __stcg(slot + N * hs + N + tid, s_l[tid]);
        } else if (a.stats) {
          a.stats[row_index(a, w, tid)] = s_m[tid] + log2f(s_l[tid]);
        }
      }
      if (parts > 1) paged_join(a, w, first_cta, parts, N, tid, SOFT, meet, s_red, s_red_sum, values, S::kP / 8, s_out, &s_last);
      if (!more) break;
      meet();
    }
  } else if (any && warp == WARPS) {
    // ------------------------------------------------------------------ products: the whole warp runs this, one lane issues
    constexpr uint32_t kType = TERMS == 2 ? 0u : (1u << 7) | (1u << 10);
    constexpr uint32_t idesc_s = f16_idesc(128, S::kCols) | kType, idesc_o = idesc_s | (1u << 15) | (1u << 16);  // values and probabilities: MN-major
    const uint32_t st0 = umma_desc_lo(smem_addr(stages)), p0 = umma_desc_lo(smem_addr(Ps)), q0 = umma_desc_lo(smem_addr(Qs));
    uint32_t tile = 0, use = 0, part = 0;  // of all parts: tiles, stages used up, parts with tiles
    auto scores = [&](uint32_t i) {
      const uint32_t st = use % NS;
      wait(&full[st], use / NS);
      fence_async_smem();
      tc_fence_after();
      const uint32_t d = tmem + S::kCols * (i & 1), k = st0 + st * (S::kStage >> 4);
#pragma unroll
      for (int b = 0; b < HB; b++)
#pragma unroll
        for (int s = 0; s < 4; s++)
          umma1_f16(d, k + b * (kTcBlock >> 4) + 2 * s, q0 + b * (S::kCols * 128 >> 4) + 2 * s, idesc_s, b > 0 || s > 0 ? 1u : 0u);
      umma_commit_elect(&s_done[i & 1]);
      umma_commit_elect(&empty[st]);
      use++;
    };
    PagedPart w = first;
    for (;;) {
      const int n_tiles = w.n_tiles;
      if (n_tiles > 0) {
        wait(&q_ready, part++);
        scores(tile);
        for (int t = 0; t < n_tiles; t++, tile++) {
          if (t + 1 < n_tiles) scores(tile + 1);
          const uint32_t st = use % NS;
          wait(&full[st], use / NS);
          wait(&p_ready[tile & 1], tile >> 1);
          fence_async_smem();
          tc_fence_after();
          // 16 keys a step; the block of dimensions from 64 on, and that of columns from 64 on, lie kTcBlock further (with one
          // block of dimensions, it is taken twice)
          const uint32_t v = (st0 + st * (S::kStage >> 4)) | (HB > 1 ? (uint32_t)(kTcBlock >> 4) << 16 : 0u);
          const uint32_t p = (p0 + (tile & 1) * (S::kPTile >> 4)) | (S::kCols > 64 ? (uint32_t)(kTcBlock >> 4) << 16 : 0u);
#pragma unroll
          for (int s = 0; s < kTcKeys / 16; s++)
            umma1_f16(tmem + S::kCols * (2 + (tile & 1)), v + s * (2048 >> 4), p + s * (2048 >> 4), idesc_o, s > 0 ? 1u : 0u);
          umma_commit_elect(&o_done[tile & 1]);
          umma_commit_elect(&empty[st]);
          use++;
        }
      }
      if (!paged_more(a, w, x1)) break;
      const PagedPart before = w;
      paged_next(a, w, before, x1, kTcKeys, lane == 0 ? &s_progress : nullptr);
    }
    if (*abort_flag) {  // what has been issued ends before its operands go
      umma_commit_elect(&drained);
      mbar_wait(&drained, 0, TC_POLLS);
    }
  } else if (any) {
    // ------------------------------------------------------------------ copies
    constexpr int kLanes = 8 * HB, kAtOnce = 32 / kLanes;  // lanes that share a row
    const int lw = warp - WARPS - 1, piece = lane % kLanes, sub = lane / kLanes;
    const bool mine = piece * 8 < hs;  // 8 values a piece
    const uint32_t st0 = smem_addr(stages) + (piece >> 3) * kTcBlock + (32 * lw + sub) * 128;
    uint32_t fills = 0, swizzle[8 / kAtOnce];
#pragma unroll
    for (int i = 0; i < 8 / kAtOnce; i++) swizzle[i] = ((piece & 7) ^ ((i * kAtOnce + sub) & 7)) << 4;
    auto fill = [&](const T *from, long long at, bool plain) {
      const uint32_t st = fills % NS;
      wait(&empty[st], fills / NS + 1);  // the first use of a stage waits for nothing
      const uint32_t to = st0 + st * S::kStage;
      if (plain) {  // one address per 16 positions, the others at a fixed distance
        uint32_t dst[8 / kAtOnce];  // the swizzle repeats every eight rows
#pragma unroll
        for (int i = 0; i < 8 / kAtOnce; i++) dst[i] = to + swizzle[i];
        const long long step = (long long)kAtOnce * c.position_stride * 2;
#pragma unroll
        for (int b = 0; b < 2; b++) {
          const char *p = reinterpret_cast<const char *>(from + __shfl_sync(0xffffffffu, at, 16 * b) + (long long)sub * c.position_stride) + piece * 16;
          if (mine) {
#pragma unroll
            for (int i = 0; i < 16 / kAtOnce; i++) {
              cp_async16(dst[i % (8 / kAtOnce)] + (16 * b + i * kAtOnce) * 128, p);
              p += step;
            }
          }
        }
      } else {
#pragma unroll 4
        for (int i = 0; i < 32 / kAtOnce; i++) {
          const long long x = __shfl_sync(0xffffffffu, at, i * kAtOnce + sub);
          if (mine)
            cp_async16_or_zero(to + i * kAtOnce * 128 + (((piece & 7) ^ ((i * kAtOnce + sub) & 7)) << 4),
                               reinterpret_cast<const char *>(from + (x < 0 ? 0 : x)) + piece * 16, x >= 0);
        }
      }
      // arrives when this thread's copies have landed; the warp that issues the products fences them for the async proxy (a fence
      // here would wait for every copy in flight)
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(&full[st])) : "memory");
      fills++;
    };
    PagedPart w = first;
    for (;;) {
      const T *k = static_cast<const T *>(c.k) + w.g.kvh * c.head_stride, *v = static_cast<const T *>(c.v) + w.g.kvh * c.head_stride;
      const uint32_t *table = c.table + (size_t)w.g.s * c.table_stride;
      int pos = w.q.begin + w.u0 * kTcKeys + 32 * lw + lane;
      uint32_t page = 0xFFFFFFFFu, slot = 0;
      auto look_up = [&]() {
        page = 0xFFFFFFFFu;
        if (pos >= w.g.lowest && pos < w.g.highest) {
          const uint32_t index = c.page_shift >= 0 ? (uint32_t)pos >> c.page_shift : (uint32_t)pos / c.page_size;
          slot = (uint32_t)pos - index * c.page_size;
          page = __ldcg(table + index);
        }
      };
      if (w.n_tiles > 0) look_up();
      long long before_at = -1;
      bool before_plain = false;
      for (int t = 0; t <= w.n_tiles; t++) {
        long long at = -1;
        bool plain = false;
        if (t < w.n_tiles) {
          if (page < c.n_pages)
            at = (long long)page * c.page_stride + (long long)slot * c.position_stride;
          else if (pos >= w.g.lowest && pos < w.g.highest)
            *c.err = kErrCache;
          plain = c.page_size % 16 == 0 && __all_sync(0xffffffffu, at >= 0);
          pos += kTcKeys;
          if (t + 1 < w.n_tiles) look_up();
          fill(k, at, plain);
        }
        if (t > 0) fill(v, before_at, before_plain);
        before_at = at;
        before_plain = plain;
      }
      if (!paged_more(a, w, x1)) break;
      const PagedPart before = w;
      paged_next(a, w, before, x1, kTcKeys, lane == 0 ? &s_progress : nullptr);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  __syncthreads();
  if (tid == 0 && *abort_flag) atomicExch(c.err, 3);
  if (warp == WARPS) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kTmem);
  }
}

}  // namespace wgpt
