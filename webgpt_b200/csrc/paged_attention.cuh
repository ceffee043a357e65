// Attention of new tokens over a paged cache.
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(c s_ij - m_i),  s_ij = q_i . k_j,  c = scale / ln 2,  m_i = max_j c s_ij
// in one pass over the keys, with the running maximum and sum in f32 (sums and values are multiplied by 2^(old - new maximum)
// when it moves). Exponentials are ex2.approx, good to 2^-22; CUDA's exp2f promises two units in the last place, which is as much.
//
// What bounds it is the cache's bytes: a row of K and V is read once for all the query rows that share it (the heads of its
// group, times the new tokens), at most a row tile of them; and for small calls a chain of about 7 us: lengths, pages, the first
// tiles, merge, join. Measured: one token of 12 heads of 64 over 200 f32 positions 7.5 us; 16 users of 25 heads over up to 1024
// f32 positions (118 MB) 29 us, 4.0 TB/s; one user of 8 heads of 128 with 4 rows each over 131072 bf16 positions (537 MB) 98 us,
// 5.5 TB/s; 32 users of 12 heads of 64 over up to 4097 f16 positions (261 MB) 56 us, 4.7 TB/s. All (sequence, head of the cache, row tile) groups lie behind one
// another as units of a few tiles of positions; every CTA takes as many units as any other, whatever the lengths are, so a CTA
// may hold the end of one group, whole ones, and the beginning of another. A group that is shared is joined by the CTA that
// finishes last, in the order of the positions.
//
// Inside a CTA the key groups (of one warp, or of several with eight rows each) take a tile of each unit and do not meet until
// the group ends: each has a ring of tiles in shared memory that cp.async fills, K and V tiles in turn. While a group's results
// are put together the first tiles of the next one are on their way.
#pragma once
#include <type_traits>

#include "paged.cuh"

namespace wgpt {

__device__ __forceinline__ float paged_value(const float *p) { return __ldcg(p); }
__device__ __forceinline__ float paged_value(const __half *p) { return __half2float(__ldcg(p)); }
__device__ __forceinline__ float paged_value(const __nv_bfloat16 *p) { return __bfloat162float(__ldcg(p)); }

constexpr int kPagedKeyGroups = 4, kPagedWarps = 8, kPagedRows = 32;  // at most, in a CTA

struct PagedAttention {
  PagedView c;
  NewRows r;
  int n_head, group, window;
  float scale2;  // scale / ln 2
  const float *q;
  float *out;
  long long ld_q, ld_out;
  int key_groups, row_warps, rows;  // of a CTA: key groups of row_warps warps; rows of a row tile
  int least;             // fewest units a CTA takes
  int extra;             // units that the beginning and end of a group count as
  int ahead;             // whether the results of a group leave room for the next one's first tiles
  float *partial;        // [2 * CTAs][paged_slot(rows, hs)]
  unsigned int *join;    // a counter per CTA, zero on entry and left zero
  int row0, row1;        // the rows of this launch: [row0, row1)
  float *scores, *stats; // [(row1 - row0) * n_head][max_length] and [(row1 - row0) * n_head], in units of log 2, or NULL
  unsigned int *skip;    // whether the call does nothing, for the kernel that adds the weights up; or NULL
};

// Quotients that the chain ahead of the first copy waits for: mostly by one.
__device__ __forceinline__ uint32_t quotient(uint32_t x, uint32_t by) { return by == 1 ? x : x / by; }

// A sequence's share of the work.
struct PagedSeq {
  int first, n, L, begin;  // rows, length, position of the first unit
  int tiles, units;        // row tiles, units of each and what is added to them
};

// A sequence's rows in this launch, and how many positions there are up to the last of them: one whose last rows come later is as much
// shorter. Returns what new_rows does.
__device__ __forceinline__ bool launch_rows(const PagedAttention &a, int s, int &first, int &n, int &L) {
  const bool on = new_rows(a.c, a.r, s, first, n);
  const int end = first + n, to = min(end, a.row1);
  L = max(0, paged_length(a.c, s) - (end - to));
  first = max(first, a.row0);
  n = max(0, to - first);
  return on;
}

__device__ __forceinline__ PagedSeq paged_seq(const PagedAttention &a, int s, int unit, bool *in_order = nullptr) {
  PagedSeq q;
  const bool on = launch_rows(a, s, q.first, q.n, q.L);
  if (in_order) *in_order = on;
  const int lowest = a.window > 0 ? max(0, q.L - q.n + 1 - a.window) : 0;
  q.begin = min(lowest, q.L) & ~(unit - 1);
  q.tiles = q.n * a.group <= a.rows ? (q.n > 0 ? 1 : 0) : (q.n * a.group + a.rows - 1) / a.rows;
  q.units = a.extra + max(1, (q.L - q.begin + unit - 1) >> (__ffs(unit) - 1));  // one even if there is nothing to see: the rows are set to zero
  return q;
}
__device__ __forceinline__ uint32_t paged_work(const PagedAttention &a, const PagedSeq &q) {
  return (uint32_t)q.tiles * (uint32_t)q.units * (uint32_t)a.c.n_kv;
}

// What a part of a group leaves for the others: the rows' values, maxima and sums.
__host__ __device__ constexpr int paged_slot(int rows, int hs) { return rows * hs + (2 * rows + 3) / 4 * 4; }

// The row tile that a CTA works on.
struct PagedGroup {
  int s, kvh, r0, rows;    // sequence, head of the cache, first row of the tile (token * group + head in the group), rows
  int lowest, highest;     // positions that some row sees: [lowest, highest)
  int inner_low, inner_high;  // positions that every row sees
};

// A CTA's part of it, and where the sequence's work begins.
struct PagedPart {
  PagedSeq q;
  PagedGroup g;
  uint32_t seq_begin, begin, end, next;  // of the sequence, of the group; the unit behind this part
  int u0, n_tiles;                       // units of the group
};

__device__ __forceinline__ void row_range(const PagedAttention &a, const PagedSeq &q, int token, int &lo, int &hi) {
  hi = max(0, q.L - q.n + token + 1);
  lo = a.window > 0 ? max(0, hi - a.window) : 0;
}
__device__ __forceinline__ long long row_offset(const PagedAttention &a, const PagedPart &w, int r, long long ld) {
  const int token = (int)quotient(w.g.r0 + r, a.group), head = w.g.kvh * a.group + (w.g.r0 + r) - token * a.group;
  return (long long)(w.q.first + token) * ld + (long long)head * a.c.hs;
}
__device__ __forceinline__ long long row_index(const PagedAttention &a, const PagedPart &w, int r) {
  const int token = (int)quotient(w.g.r0 + r, a.group), head = w.g.kvh * a.group + (w.g.r0 + r) - token * a.group;
  return (long long)(w.q.first - a.row0 + token) * a.n_head + head;
}

// Every group begins with a.extra units that have no positions: what it takes to load its queries and to put its results together,
// which a CTA with the end of one group and the beginning of another does twice. A share that ends among them leaves the group to
// the next CTA.
__device__ __forceinline__ bool paged_more(const PagedAttention &a, const PagedPart &w, uint32_t end) { return w.next + a.extra < end; }
__device__ __forceinline__ int paged_first_cta(const PagedAttention &a, const PagedPart &w, uint32_t per) {
  return (int)((w.begin + a.extra) / per);
}

// The part that begins at unit x of sequence s, up to unit end at most; q and seq_begin are the sequence's.
__device__ __forceinline__ void paged_part(const PagedAttention &a, PagedPart &w, const PagedSeq &q, int s, uint32_t seq_begin, uint32_t x,
                                           uint32_t end, int unit) {
  const uint32_t gi = quotient(x - seq_begin, (uint32_t)q.units);
  w.q = q;
  w.seq_begin = seq_begin;
  w.begin = seq_begin + gi * (uint32_t)q.units;
  w.end = w.begin + (uint32_t)q.units;
  w.next = min(end, w.end);
  w.g.s = s;
  w.g.kvh = (int)quotient(gi, (uint32_t)q.tiles);
  w.g.r0 = (int)(gi - (uint32_t)w.g.kvh * (uint32_t)q.tiles) * a.rows;
  w.g.rows = min(a.rows, q.n * a.group - w.g.r0);
  const int first = q.n == 1 ? 0 : (int)quotient(w.g.r0, a.group), last = q.n == 1 ? 0 : (int)quotient(w.g.r0 + w.g.rows - 1, a.group);
  row_range(a, q, first, w.g.lowest, w.g.inner_high);
  row_range(a, q, last, w.g.inner_low, w.g.highest);
  // units that no row of the tile sees are left out
  const int shift = __ffs(unit) - 1;
  w.u0 = max(max(0, (int)(x - w.begin) - a.extra), (w.g.lowest - q.begin) >> shift);
  w.n_tiles = max(0, min((int)(w.next - w.begin) - a.extra, (w.g.highest - q.begin + unit - 1) >> shift) - w.u0);
}

// A CTA's units [.., end) of all there are and the part they begin with, by all its threads, every one of which gets it: false if
// there are none. Nor are there any where the row offsets decrease somewhere: rows would be counted for several sequences, more of them
// than the caller's bound on the units allows for. sums: a number for each warp; place: a part.
__device__ __forceinline__ bool paged_first(const PagedAttention &a, PagedPart &to, int unit, uint32_t *sums, PagedPart *place, uint32_t &per,
                                            uint32_t &end) {
  const int threads = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n_seq = a.c.n_seq;
  PagedSeq q;
  bool bad = false;
  auto weight_of = [&](int s) -> uint32_t {
    if (s >= n_seq) return 0;
    bool in_order;
    q = paged_seq(a, s, unit, &in_order);
    bad = bad || !in_order;
    return paged_work(a, q);
  };
  auto skipped = [&](bool skip) {
    if (a.skip && blockIdx.x == 0 && tid == 0) *a.skip = skip ? 1u : 0u;
    return skip;
  };
  auto before_lane = [&](uint32_t mine) {  // sum over the lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, mine, o);
      if (lane >= o) mine += x;
    }
    return mine;
  };
  if (n_seq <= 32) {  // every warp for itself, a sequence a lane
    const uint32_t mine = weight_of(lane), upto = before_lane(mine), total = __shfl_sync(0xffffffffu, upto, 31);
    if (skipped(__any_sync(0xffffffffu, bad))) return false;
    per = max((uint32_t)a.least, (total + gridDim.x - 1) / gridDim.x);
    const uint32_t x0 = blockIdx.x * per;  // the caller sees to it that it does not pass 2^32
    end = min(total, x0 + per);
    if (x0 >= end) return false;
    const int s = __ffs(__ballot_sync(0xffffffffu, x0 < upto)) - 1;
    PagedSeq of;
    of.first = __shfl_sync(0xffffffffu, q.first, s);
    of.n = __shfl_sync(0xffffffffu, q.n, s);
    of.L = __shfl_sync(0xffffffffu, q.L, s);
    of.begin = __shfl_sync(0xffffffffu, q.begin, s);
    of.tiles = __shfl_sync(0xffffffffu, q.tiles, s);
    of.units = __shfl_sync(0xffffffffu, q.units, s);
    paged_part(a, to, of, s, __shfl_sync(0xffffffffu, upto - mine, s), x0, end, unit);
    return end > to.begin + a.extra;
  }
  auto scan = [&](uint32_t mine, uint32_t &all) {  // sum over the threads before this one, and over all
    const uint32_t upto = before_lane(mine);
    __syncthreads();
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    const uint32_t of = lane < threads / 32 ? sums[lane] : 0u;
    all = __reduce_add_sync(0xffffffffu, of);
    return upto - mine + __reduce_add_sync(0xffffffffu, lane < warp ? of : 0u);
  };
  uint32_t total = 0, mine = 0, before = 0;
  for (int s0 = 0; s0 < n_seq; s0 += threads) {
    uint32_t all;
    mine = weight_of(s0 + tid);
    before = total + scan(mine, all);
    total += all;
  }
  if (skipped(__syncthreads_or(bad))) return false;
  per = max((uint32_t)a.least, (total + gridDim.x - 1) / gridDim.x);
  const uint32_t x0 = blockIdx.x * per, x1 = min(total, x0 + per);  // the caller sees to it that neither passes 2^32
  if (x0 >= x1) return false;
  end = x1;
  uint32_t sum = 0;
  for (int s0 = 0; s0 < n_seq && sum <= x0; s0 += threads) {
    uint32_t all;
    mine = weight_of(s0 + tid);
    before = sum + scan(mine, all);
    if (before <= x0 && x0 < before + mine) paged_part(a, *place, q, s0 + tid, before, x0, x1, unit);
    sum += all;
  }
  __syncthreads();
  to = *place;
  return end > to.begin + a.extra;
}

// The part behind `w`, which ends before unit `end`. May not be `w` itself. progress, or NULL: goes on with every sequence passed over.
__device__ __forceinline__ void paged_next(const PagedAttention &a, PagedPart &to, const PagedPart &w, uint32_t end, int unit,
                                           unsigned int *progress = nullptr) {
  uint32_t seq_begin = w.seq_begin;
  PagedSeq q = w.q;
  int s = w.g.s;
  while (w.next >= seq_begin + paged_work(a, q)) {
    seq_begin += paged_work(a, q);
    q = paged_seq(a, ++s, unit);
    if (progress) atomicAdd(progress, 1u);
  }
  paged_part(a, to, q, s, seq_begin, w.next, end, unit);
}

// Copies 16 bytes, or writes zeros where there is nothing to copy.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t to, const void *from, bool there) {
  const int bytes = there ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

// The power of two that brings a row's largest magnitude near 2^13, the middle of a half's range, as its exponent; a row that has an
// infinity or no value but zero stays.
__device__ __forceinline__ int row_exponent(float top) {
  const int e = (__float_as_int(top) >> 23) - 127 - 13;  // top >= 0
  return top > 0.f && top < INFINITY ? max(e, -126) : 0;
}
__device__ __forceinline__ float pow2_of(int e) { return __int_as_float((127 + e) << 23); }  // |e| <= 126

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What the kernel of a type, a (padded) head size and a number of rows takes of shared memory. f32: products on the CUDA cores, RT
// rows a warp; else on the tensor cores, eight rows a warp.
template <typename T, int HSP, int RT, int STAGES>
struct PagedShape {
  static constexpr bool kWide = sizeof(T) == 4;
  static constexpr int kTerms = kWide ? 1 : std::is_same<T, __half>::value ? 2 : 3;  // values that a query or probability is split into
  static constexpr int kPitch = HSP * (int)sizeof(T) + 16;  // of a row in shared memory: 16-byte pieces of 8 rows meet all banks
  static constexpr int kTile = HSP * (int)sizeof(T) <= 256 ? 32 : 16;  // positions of a tile
  static constexpr int kTileBytes = kTile * kPitch;
  static constexpr int kQPitch = kWide ? HSP * 4 : HSP * 2 + 16;
  static constexpr int kStages = STAGES;  // tiles of a ring
  static constexpr int kRing = kStages * kTileBytes;
  static constexpr int kPBytes = kWide ? RT * kTile * 4 : 0;  // a warp's probabilities of a tile
  __host__ __device__ static constexpr int q_bytes(int rows) { return rows * kTerms * kQPitch; }
  __host__ __device__ static constexpr int smem(int key_groups, int rows) { return q_bytes(rows) + key_groups * (kPBytes + kRing); }
  __host__ __device__ static constexpr bool ahead(int rows, int hs) { return rows * hs * 4 <= kTileBytes; }
  __host__ __device__ static constexpr bool fits(int rows, int hs) { return rows * hs * 4 <= kRing; }
};

// The values of 16 bytes of a row.
__device__ __forceinline__ void paged_values(const float *p, float (&v)[4]) {
  const float4 f = __ldcg(reinterpret_cast<const float4 *>(p));
  v[0] = f.x;
  v[1] = f.y;
  v[2] = f.z;
  v[3] = f.w;
}
template <typename T>
__device__ __forceinline__ void paged_values(const T *p, float (&v)[8]) {
  const uint4 u = __ldcg(reinterpret_cast<const uint4 *>(p));
  const uint32_t word[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    float2 f;
    if constexpr (std::is_same<T, __half>::value)
      f = __half22float2(*reinterpret_cast<const __half2 *>(&word[i]));
    else
      f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&word[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// Rows of a tile that came out non-finite (an infinity or NaN in V, in a key, in q, also where a row's mask leaves it out: zero times
// infinity), a bit each: the same again by one warp, each row from what it sees alone. Leaves the row's maximum, sum and values as
// the fast path does. A lane takes a position for the scores and some dimensions for the values. PIECES: of 32 dimensions. progress, or
// NULL: goes on with every 32 positions, for those who wait. One user of 131072 f16 positions, 8 heads of 128 with 16 rows each, all of
// which meet an infinity: 8.3 ms, 0.11 without it; 34 with a round trip to memory for every few positions.
template <typename T, int TILE, int PIECES>
__device__ __noinline__ void paged_rows_apart(const PagedAttention &a, const PagedPart &w, int key_group, int key_groups, uint32_t rows,
                                              int lane, float *o_out, float *m_out, float *l_out, unsigned int *progress) {
  constexpr int kBlock = TILE < 32 ? TILE : 32, kWide = 16 / (int)sizeof(T), kAtOnce = 8 / PIECES;
  const PagedView &c = a.c;
  const PagedSeq &q = w.q;
  const PagedGroup &g = w.g;
  const T *k = static_cast<const T *>(c.k) + g.kvh * c.head_stride, *v = static_cast<const T *>(c.v) + g.kvh * c.head_stride;
  for (; rows != 0; rows &= rows - 1) {
    const int r = __ffs(rows) - 1;
    int lo, hi;
    row_range(a, q, (g.r0 + r) / a.group, lo, hi);
    const float *x = a.q + row_offset(a, w, r, a.ld_q);
    float o[PIECES], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < PIECES; i++) o[i] = 0.f;
    for (int u = w.u0; u < w.u0 + w.n_tiles; u++) {
      const int base = q.begin + (u * key_groups + key_group) * TILE;
      for (int b = base; b < base + TILE; b += kBlock) {
        if (max(b, lo) >= min(b + kBlock, hi)) continue;
        const bool seen = lane < kBlock && b + lane >= lo && b + lane < hi;
        const long long at = seen ? paged_offset(c, g.s, b + lane) : -1;
        // loads without branches, so that they are on their way together: what is not there is read from somewhere else
        const T *key = k + max(at, 0ll);
        float d = 0.f;
#pragma unroll 1
        for (int i = 0; i < PIECES; i++) {
          const float qi = lane + 32 * i < c.hs ? __ldcg(x + lane + 32 * i) : 0.f;
          float kk[32 / kWide][kWide];
#pragma unroll
          for (int y = 0; y < 32 / kWide; y++) paged_values(key + min(32 * i + kWide * y, c.hs - kWide), kk[y]);
#pragma unroll
          for (int y = 0; y < 32 / kWide; y++)
#pragma unroll
            for (int e = 0; e < kWide; e++) {
              const float qe = __shfl_sync(0xffffffffu, qi, kWide * y + e);
              d = 32 * i + kWide * y < c.hs ? fmaf(qe, kk[y][e], d) : d;
            }
        }
        const float sc = at >= 0 ? d * a.scale2 : -INFINITY;
        if (a.scores && seen) a.scores[row_index(a, w, r) * c.max_length + b + lane] = sc;
        const float nm = fmaxf(m, warp_max(sc)), f = m == nm ? 1.f : exp2f(m - nm), p = sc == -INFINITY ? 0.f : exp2f(sc - nm);
        const uint32_t live = __ballot_sync(0xffffffffu, sc != -INFINITY);
        l = l * f + warp_sum(p);
        m = nm;
#pragma unroll
        for (int i = 0; i < PIECES; i++) o[i] *= f;
#pragma unroll 1
        for (int j = 0; j < kBlock; j += kAtOnce) {
          float vv[kAtOnce][PIECES];
#pragma unroll
          for (int y = 0; y < kAtOnce; y++) {
            const T *value = v + max(__shfl_sync(0xffffffffu, at, j + y), 0ll);
#pragma unroll
            for (int i = 0; i < PIECES; i++) vv[y][i] = paged_value(value + min(lane + 32 * i, c.hs - 1));
          }
#pragma unroll
          for (int y = 0; y < kAtOnce; y++) {
            const float pj = __shfl_sync(0xffffffffu, p, j + y);
            const bool in = live >> (j + y) & 1u;
#pragma unroll
            for (int i = 0; i < PIECES; i++) o[i] = in ? fmaf(pj, vv[y][i], o[i]) : o[i];
          }
        }
        if (progress && lane == 0) atomicAdd(progress, 1u);
      }
    }
#pragma unroll
    for (int i = 0; i < PIECES; i++)
      if (lane + 32 * i < c.hs) o_out[r * c.hs + lane + 32 * i] = o[i];
    if (lane == 0) {
      m_out[r] = m;
      l_out[r] = l;
    }
  }
}

// A key group's ring: fills tiles of K and of V in turn. Every warp of the group holds a copy and brings its share of the rows.
template <typename T, int HSP, int RT, int STAGES>
struct PagedRing {
  using S = PagedShape<T, HSP, RT, STAGES>;
  static constexpr int kTile = S::kTile;
  static constexpr int kPerRow = HSP * (int)sizeof(T) / 16;          // 16-byte pieces of a row
  static constexpr int kLanes = kPerRow < 32 ? kPerRow : 32;         // lanes that share a row
  static constexpr int kAtOnce = 32 / kLanes, kWidth = kPerRow / kLanes;
  const PagedView &c;
  const T *k, *v;      // this head's rows of page 0
  const uint32_t *table;
  uint32_t base;       // shared-memory address of the ring
  uint32_t *ok;        // [kStages] which of a tile's positions are there
  int lowest, highest, pos, unit, lane, share, of, next;
  uint32_t page, slot; // of this lane's position of the next tile to fill
  long long at;        // where this lane's position of the tile at hand begins, or -1
  bool plain;          // the tile at hand: all of its positions are there, and 16 from a multiple of 16 on share a page

  __device__ __forceinline__ PagedRing(const PagedView &c_, uint32_t base_, uint32_t *ok_, int lane_, int unit_, int share_, int of_)
      : c(c_), base(base_), ok(ok_), unit(unit_), lane(lane_), share(share_), of(of_) {}

  __device__ __forceinline__ void look_up() {  // the page of this lane's position, asked for a tile ahead
    page = 0xFFFFFFFFu;
    slot = 0;
    if (pos >= lowest && pos < highest) {
      const uint32_t index = c.page_shift >= 0 ? (uint32_t)pos >> c.page_shift : (uint32_t)pos / c.page_size;
      slot = (uint32_t)pos - index * c.page_size;
      page = __ldcg(table + index);
    }
  }
  // Begins at position `first` (a multiple of 16) of a part, with the first tiles on their way. The ring is empty.
  __device__ __forceinline__ void begin(const PagedPart &w, int first) {
    k = static_cast<const T *>(c.k) + w.g.kvh * c.head_stride;
    v = static_cast<const T *>(c.v) + w.g.kvh * c.head_stride;
    table = c.table + (size_t)w.g.s * c.table_stride;
    lowest = w.g.lowest;
    highest = w.g.highest;
    pos = first + (lane & (kTile - 1));
    next = 0;
    if (w.n_tiles > 0) look_up();
#pragma unroll
    for (int h = 0; h < STAGES - 1; h++) fill((h & 1) == 0, h < 2 * w.n_tiles);
  }
  // Fills the next stage with a tile of keys or of values, and commits it.
  __device__ __forceinline__ void fill(bool keys, bool any) {
    const int stage = next;
    next = next + 1 == S::kStages ? 0 : next + 1;
    if (any) {
      if (keys) {
        at = -1;
        if (page < c.n_pages)
          at = (long long)page * c.page_stride + (long long)slot * c.position_stride;
        else if (pos >= lowest && pos < highest)
          *c.err = kErrCache;
        const uint32_t there = __ballot_sync(0xffffffffu, at >= 0);
        plain = c.page_size % 16 == 0 && there == 0xffffffffu;
        if (lane == 0 && share == 0) ok[stage] = there;
        pos += unit;
        look_up();
      }
      const T *from = keys ? k : v;
      const uint32_t to = base + stage * S::kTileBytes + lane / kLanes * S::kPitch + lane % kLanes * 16;
      if (plain && of == 1) {  // one address per 16 positions, the others at a fixed distance
        const long long step = (long long)kAtOnce * c.position_stride * (int)sizeof(T);
#pragma unroll
        for (int b = 0; b < kTile / 16; b++) {
          const char *p = reinterpret_cast<const char *>(from + __shfl_sync(0xffffffffu, at, 16 * b) + lane / kLanes * c.position_stride) + lane % kLanes * 16;
#pragma unroll
          for (int i = 0; i < 16 / kAtOnce; i++) {
#pragma unroll
            for (int w = 0; w < kWidth; w++)
              if ((lane % kLanes + w * 32) * 16 < c.hs * (int)sizeof(T))
                cp_async16(to + (16 * b + i * kAtOnce) * S::kPitch + w * 512, p + w * 512);
            p += step;
          }
        }
      } else {
#pragma unroll 2
        for (int i = share; i < kTile / kAtOnce; i += of) {
          const long long x = __shfl_sync(0xffffffffu, at, i * kAtOnce + lane / kLanes);
#pragma unroll
          for (int w = 0; w < kWidth; w++) {
            const int piece = (lane % kLanes + w * 32) * 16;
            if (piece < c.hs * (int)sizeof(T))
              cp_async16_or_zero(to + i * kAtOnce * S::kPitch + w * 512, reinterpret_cast<const char *>(from + (x < 0 ? 0 : x)) + piece, x >= 0);
          }
        }
      }
    }
    cp_async_commit();
  }
};

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two values rounded to the 16-bit type, packed, and what is left of them.
template <typename T>
__device__ __forceinline__ uint32_t split2(float &x, float &y) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    x -= f.x;
    y -= f.y;
    return *reinterpret_cast<const uint32_t *>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const float2 f = __bfloat1622float2(h);
    x -= f.x;
    y -= f.y;
    return *reinterpret_cast<const uint32_t *>(&h);
  }
}


// Joins a group's parts once this CTA's lies in its slot: the CTA that finishes last does, in the order of the positions. By
// `threads` threads that meet in sync(); red and red_sum: a place for each of them; factor: twice `places` values; out_at:
// where the rows' results go.
template <typename Sync>
__device__ __forceinline__ void paged_join(const PagedAttention &a, const PagedPart &w, int first_cta, int parts, int ROWS, int tid,
                                           int threads, Sync sync, float4 *red, float *red_sum, float *factor, int places, const long long *out_at, int *is_last) {
  const int hs = a.c.hs, quads = hs / 4, items = w.g.rows * quads, slot_floats = paged_slot(ROWS, hs);
  sync();
  if (tid == 0) {  // its fences stand for all threads', on their side of the barriers
    __threadfence();
    const unsigned int done = atomicAdd(a.join + first_cta, 1u);
    *is_last = done == (unsigned)parts - 1;
    if (*is_last) a.join[first_cta] = 0;
    __threadfence();
  }
  sync();
  if (!*is_last) return;
  auto part_of = [&](int k) { return a.partial + (2ll * (first_cta + k) + (k == 0 ? 1 : 0)) * slot_floats; };
  const int rows = w.g.rows, n = parts * rows;
  const bool table = n <= places;  // else every thread computes the factors that it needs
  float *sums = factor + places;
  if (table) {
    for (int i = tid; i < n; i += threads) {
      const int k = i / rows, r = i - k * rows;
      factor[i] = __ldcg(part_of(k) + ROWS * hs + r);
      sums[i] = __ldcg(part_of(k) + ROWS * hs + ROWS + r);
    }
    sync();
    // a warp a row, or a thread where there are few parts
    const int of = parts > 8 ? 32 : 1, lane = parts > 8 ? tid & 31 : 0;
    for (int r = tid / of; r < rows; r += threads / of) {
      float top = -INFINITY, sum = 0.f;
      for (int k = lane; k < parts; k += of) top = fmaxf(top, factor[k * rows + r]);
      if (of > 1) top = warp_max(top);
      for (int k = lane; k < parts; k += of) {
        const float m = factor[k * rows + r], l = sums[k * rows + r], f = m == -INFINITY && l == 0.f ? 0.f : exp2f(m - top);
        factor[k * rows + r] = f;
        sum += f * l;
      }
      if (of > 1) sum = warp_sum(sum);
      if (lane == 0) {
        sums[r] = sum != 0.f ? 1.f / sum : 0.f;  // the first part's places: this row's, read already
        if (a.stats) a.stats[row_index(a, w, r)] = top + log2f(sum);
      }
    }
    sync();
  }
  // Where a row tile has few values, several threads share a quad and take every so many parts. A part's values are a round trip
  // away, so that what counts is how many are asked for at once: eight, or four of two quads.
  const int share = items >= threads ? 1 : threads / items;
  if (table && items > threads) {
    for (int i = tid; i < items; i += 2 * threads) {
      const int at[2] = {i, min(i + threads, items - 1)}, r[2] = {at[0] / quads, at[1] / quads};
      float4 v[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
      for (int k0 = 0; k0 < parts; k0 += 4) {
        float4 o[4][2];
#pragma unroll
        for (int x = 0; x < 4; x++) {
          const float4 *part = reinterpret_cast<const float4 *>(part_of(min(k0 + x, parts - 1)));
          o[x][0] = __ldcg(part + at[0]);
          o[x][1] = __ldcg(part + at[1]);
        }
#pragma unroll
        for (int x = 0; x < 4; x++)
          if (k0 + x < parts) {
#pragma unroll
            for (int y = 0; y < 2; y++) {
              const float f = factor[(k0 + x) * rows + r[y]];
              v[y].x += f * o[x][y].x;
              v[y].y += f * o[x][y].y;
              v[y].z += f * o[x][y].z;
              v[y].w += f * o[x][y].w;
            }
          }
      }
#pragma unroll
      for (int y = 0; y < 2; y++) {
        const float inv = sums[r[y]];
        if (i + y * threads < items)
          reinterpret_cast<float4 *>(a.out + out_at[r[y]])[at[y] - r[y] * quads] = make_float4(v[y].x * inv, v[y].y * inv, v[y].z * inv, v[y].w * inv);
      }
    }
    return;
  }
  for (int i0 = 0; i0 < items; i0 += threads) {
    const int i = share > 1 ? tid % items : i0 + tid, sh = share > 1 ? tid / items : 0;
    const bool live = i < items && sh < share;
    const int r = live ? i / quads : 0;
    float top = -INFINITY, sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) {
      if (!table)
        for (int k = 0; k < parts; k++) top = fmaxf(top, __ldcg(part_of(k) + ROWS * hs + r));
      for (int k0 = sh; k0 < parts; k0 += 8 * share) {
        float4 o[8];
        float fs[8];
#pragma unroll
        for (int x = 0; x < 8; x++) {
          const int k = min(k0 + x * share, parts - 1);
          const float *part = part_of(k);
          o[x] = __ldcg(reinterpret_cast<const float4 *>(part) + i);
          if (table) {
            fs[x] = factor[k * rows + r];
          } else {
            const float m = __ldcg(part + ROWS * hs + r), l = __ldcg(part + ROWS * hs + ROWS + r);
            fs[x] = m == -INFINITY && l == 0.f ? 0.f : exp2f(m - top);
            if (k0 + x * share < parts) sum += fs[x] * l;
          }
        }
#pragma unroll
        for (int x = 0; x < 8; x++)
          if (k0 + x * share < parts) {
            v.x += fs[x] * o[x].x;
            v.y += fs[x] * o[x].y;
            v.z += fs[x] * o[x].z;
            v.w += fs[x] * o[x].w;
          }
      }
    }
    if (share > 1) {
      red[tid] = v;
      red_sum[tid] = sum;
      sync();
      if (tid < items)
        for (int y = 1; y < share; y++) {
          const float4 o = red[y * items + tid];
          v.x += o.x;
          v.y += o.y;
          v.z += o.z;
          v.w += o.w;
          sum += red_sum[y * items + tid];
        }
    }
    if (live && sh == 0) {
      const float inv = table ? sums[r] : sum != 0.f ? 1.f / sum : 0.f;
      if (table || sum != 0.f) v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
      reinterpret_cast<float4 *>(a.out + out_at[r])[i - r * quads] = v;
      if (a.stats && !table && i == r * quads) a.stats[row_index(a, w, r)] = top + log2f(sum);
    }
  }
}

// f32: RT rows a warp on the CUDA cores, a lane one key of a tile for the scores and four dimensions for the values. 16-bit types: eight
// rows a warp on mma.sync. Scores and sums are f32; a query is the sum of two half or three bfloat16 values, good to 2^-22 or
// 2^-24 of its row's largest, a probability likewise, and the cache's values go in as they are: products of them are exact.
template <typename T, int HSP, int RT, int STAGES>
__global__ void __launch_bounds__(sizeof(T) == 4 ? 128 : 32 * kPagedWarps, sizeof(T) == 4 ? (HSP <= 64 ? 3 : HSP <= 128 ? 2 : 1) : HSP <= 128 ? 2 : 1)
paged_attention_kernel(const __grid_constant__ PagedAttention a) {
  using S = PagedShape<T, HSP, RT, STAGES>;
  constexpr int TERMS = S::kTerms, D = S::kStages, kTile = S::kTile;
  constexpr int MAXROWS = S::kWide ? RT : kPagedRows;
  // f32: a lane holds four dimensions of kQuads pieces of a row; where 16 lanes hold a row, the halves of the warp take even and odd keys
  constexpr int kQuads = HSP <= 128 ? 1 : HSP / 128, kHalves = HSP <= 64 ? 2 : 1;
  constexpr float kLift = std::is_same<T, __half>::value ? 14.f : 0.f;  // probabilities are held times 2^14, in the middle of a half's range
  extern __shared__ __align__(16) unsigned char paged_smem[];
  __shared__ float s_m[kPagedKeyGroups][MAXROWS], s_l[kPagedKeyGroups][MAXROWS], s_qscale[MAXROWS];
  __shared__ int s_lo[MAXROWS], s_hi[MAXROWS];
  __shared__ long long s_row[MAXROWS], s_out[MAXROWS];  // where the rows' scores and results begin
  __shared__ uint32_t s_ok[kPagedKeyGroups][D];
  __shared__ uint32_t s_sum[kPagedWarps];
  __shared__ PagedPart s_part[2];
  __shared__ int s_last, s_more;
  __shared__ float4 s_red[S::kWide ? 128 : 32 * kPagedWarps];
  __shared__ float s_red_sum[S::kWide ? 128 : 32 * kPagedWarps];
  const PagedView &c = a.c;
  const int KG = a.key_groups, RW = S::kWide ? 1 : a.row_warps, ROWS = S::kWide ? RT : a.rows, threads = blockDim.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hs = c.hs, unit = KG * kTile;
  const int kg = S::kWide ? warp : warp / RW, rw = S::kWide ? 0 : warp - kg * RW;
  unsigned char *q_smem = paged_smem, *rings = paged_smem + S::q_bytes(ROWS) + KG * S::kPBytes, *ring_smem = rings + kg * S::kRing;
  float *p_smem = reinterpret_cast<float *>(paged_smem + S::q_bytes(ROWS)) + warp * RT * kTile;
  const int o_at = a.ahead ? (D - 1) * S::kTileBytes : 0;  // a key group's results, in its ring
  float *o_smem = reinterpret_cast<float *>(ring_smem + o_at);
  auto meet = [&]() {  // the warps of a key group
    __syncwarp();
    if (RW > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + kg), "r"(32 * RW) : "memory");
  };
  pdl_launch_dependents();
  // where 32 does not divide the head size, what lies behind a row takes part in products: zeros, times zeros of the query's
  const bool padded = !S::kWide && (hs & 31) != 0;
  auto clear = [&](unsigned char *from, int bytes) {
    for (int i = rw * 32 + lane; i < bytes / 16; i += 32 * RW) reinterpret_cast<uint4 *>(from)[i] = make_uint4(0, 0, 0, 0);
    meet();
  };
  if (padded) clear(ring_smem, S::kRing);
  pdl_wait();

  // ---- this CTA's units: [.., x1)
  uint32_t per, x1;
  {
    PagedPart first;
    if (!paged_first(a, first, unit, s_sum, &s_part[1], per, x1)) return;
    if (tid == 0) s_part[0] = first;
  }
  __syncthreads();

  PagedRing<T, HSP, RT, STAGES> ring(c, smem_addr(ring_smem), s_ok[kg], lane, unit, rw, RW);
  auto start = [&](const PagedPart &w) { ring.begin(w, w.q.begin + (w.u0 * KG + kg) * kTile); };
  start(s_part[0]);
  for (int turn = 0;; turn ^= 1) {
    const PagedPart &w = s_part[turn];
    const PagedGroup &g = w.g;
    // ---- the next part, by a thread that has no query to load first
    if (tid == threads - 1) {
      s_more = paged_more(a, w, x1);
      if (s_more) paged_next(a, s_part[turn ^ 1], w, x1, unit);
    }
    // ---- the queries
    if constexpr (S::kWide) {
      float4 *q4 = reinterpret_cast<float4 *>(q_smem);
      for (int i = tid; i < ROWS * (HSP / 4); i += threads) {
        const int r = i / (HSP / 4), d = i % (HSP / 4);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < g.rows && 4 * d < hs) v = __ldcg(reinterpret_cast<const float4 *>(a.q + row_offset(a, w, r, a.ld_q)) + d);
        q4[i] = v;
      }
    } else {
      constexpr int kAtOnce = 2;  // rows of a warp whose loads are in flight together: eight rows a row warp, two key groups or more
      for (int rr = warp; rr < ROWS; rr += threads / 32 * kAtOnce) {
        float v[kAtOnce][HSP / 32];
#pragma unroll
        for (int y = 0; y < kAtOnce; y++) {
          const int r = rr + y * (threads / 32);
          const float *row = r < g.rows ? a.q + row_offset(a, w, r, a.ld_q) : nullptr;
#pragma unroll
          for (int i = 0; i < HSP / 64; i++) {
            const int d = 2 * lane + 64 * i;
            const float2 f = row && d < hs ? __ldcg(reinterpret_cast<const float2 *>(row + d)) : make_float2(0.f, 0.f);
            v[y][2 * i] = f.x;
            v[y][2 * i + 1] = f.y;
          }
        }
#pragma unroll
        for (int y = 0; y < kAtOnce; y++) {
          const int r = rr + y * (threads / 32);
          if (r >= ROWS) break;
          int e = 0;
          if constexpr (TERMS == 2) {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < HSP / 32; i++) top = fmaxf(top, fabsf(v[y][i]));
            top = warp_max(top);
            e = row_exponent(top);
          }
#pragma unroll
          for (int i = 0; i < HSP / 64; i++) {
            float f0 = v[y][2 * i] * pow2_of(-e), f1 = v[y][2 * i + 1] * pow2_of(-e);
#pragma unroll
            for (int t = 0; t < TERMS; t++)
              *reinterpret_cast<uint32_t *>(q_smem + (t * ROWS + r) * S::kQPitch + (2 * lane + 64 * i) * 2) = split2<T>(f0, f1);
          }
          if (lane == 0) s_qscale[r] = a.scale2 * pow2_of(e);
        }
      }
    }
    if (tid < ROWS) {
      int lo = 0, hi = 0;
      if (tid < g.rows) {
        row_range(a, w.q, (g.r0 + tid) / a.group, lo, hi);
        s_out[tid] = row_offset(a, w, tid, a.ld_out);
      }
      s_lo[tid] = lo;
      s_hi[tid] = hi;
      if (a.scores) s_row[tid] = row_index(a, w, tid) * c.max_length;
    }
    __syncthreads();

    const int n_tiles = w.n_tiles, inner_low = g.inner_low, inner_high = g.inner_high, g_rows = g.rows;
    const bool more = s_more != 0;
    int pos0 = w.q.begin + (w.u0 * KG + kg) * kTile, now = 0;  // of the tile at hand; the stage that is next to be used up
    uint32_t odd = 0;  // rows that came out non-finite
    if constexpr (S::kWide) {
      constexpr int kShare = 32 / kTile;  // lanes that share a key
      const int key = lane % kTile, share = lane / kTile, half = lane >> 4, dim = lane & 15;
      float m[RT], l[RT];
      float4 o[RT][kQuads];
#pragma unroll
      for (int r = 0; r < RT; r++) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int i = 0; i < kQuads; i++) o[r][i] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      for (int t = 0; t < n_tiles; t++, pos0 += unit) {
        // ---- scores: a lane takes one key, or every other quad of its row
        cp_async_wait<D - 2>();
        __syncwarp();
        ring.fill((D & 1) != 0, 2 * t + D - 1 < 2 * n_tiles);
        const uint32_t ok = s_ok[kg][now];
        const float4 *kt = reinterpret_cast<const float4 *>(ring_smem + now * S::kTileBytes + key * S::kPitch);
        now = now + 1 == D ? 0 : now + 1;
        float sc[RT];
#pragma unroll
        for (int r = 0; r < RT; r++) sc[r] = 0.f;
#pragma unroll 8
        for (int d = share; d < hs / 4; d += kShare) {
          const float4 kv = kt[d];
#pragma unroll
          for (int r = 0; r < RT; r++) {
            const float4 qv = reinterpret_cast<const float4 *>(q_smem)[r * (HSP / 4) + d];
            sc[r] = fmaf(qv.x, kv.x, sc[r]);
            sc[r] = fmaf(qv.y, kv.y, sc[r]);
            sc[r] = fmaf(qv.z, kv.z, sc[r]);
            sc[r] = fmaf(qv.w, kv.w, sc[r]);
          }
        }
        const bool whole = ok == 0xffffffffu && pos0 >= inner_low && pos0 + kTile <= inner_high;
        float f[RT];
        bool moved = false;
#pragma unroll
        for (int r = 0; r < RT; r++) {
          if (kShare == 2) sc[r] += __shfl_xor_sync(0xffffffffu, sc[r], 16);
          sc[r] *= a.scale2;
          if (!whole && !((ok >> key & 1u) && pos0 + key >= s_lo[r] && pos0 + key < s_hi[r])) sc[r] = -INFINITY;
          if (a.scores && share == 0 && r < g_rows && pos0 + key >= s_lo[r] && pos0 + key < s_hi[r])
            a.scores[s_row[r] + pos0 + key] = sc[r];
          float top = sc[r];
#pragma unroll
          for (int o2 = kTile / 2; o2 > 0; o2 >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o2));
          top = fmaxf(top, m[r]);
          f[r] = m[r] == top ? 1.f : exp2_of(m[r] - top);
          moved |= m[r] != top;
          const float p = sc[r] == -INFINITY ? 0.f : exp2_of(sc[r] - top);
          m[r] = top;
          l[r] = l[r] * f[r] + p;
          if (share == 0) p_smem[r * kTile + key] = p;
        }
        if (moved) {
#pragma unroll
          for (int r = 0; r < RT; r++)
#pragma unroll
            for (int i = 0; i < kQuads; i++) {
              o[r][i].x *= f[r];
              o[r][i].y *= f[r];
              o[r][i].z *= f[r];
              o[r][i].w *= f[r];
            }
        }
        // ---- values: a lane takes four dimensions (times kQuads) of each key, or of every other one
        cp_async_wait<D - 2>();
        __syncwarp();
        ring.fill((D & 1) == 0, 2 * t + D < 2 * n_tiles);
        const unsigned char *vt = ring_smem + now * S::kTileBytes;
        now = now + 1 == D ? 0 : now + 1;
        const int dim4 = kHalves == 2 ? dim : lane;
#pragma unroll
        for (int j0 = 0; j0 < kTile; j0 += 4 * kHalves) {
          float4 vv[4][kQuads];  // what lies behind a row's end is not read back
#pragma unroll
          for (int jj = 0; jj < 4; jj++)
#pragma unroll
            for (int i = 0; i < kQuads; i++)
              vv[jj][i] = *reinterpret_cast<const float4 *>(vt + (j0 + (kHalves == 2 ? 4 * half : 0) + jj) * S::kPitch + (dim4 + 32 * i) * 16);
#pragma unroll
          for (int r = 0; r < RT; r++) {
            const float4 p = *reinterpret_cast<const float4 *>(p_smem + r * kTile + j0 + (kHalves == 2 ? 4 * half : 0));
            const float pj[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
            for (int jj = 0; jj < 4; jj++)
#pragma unroll
              for (int i = 0; i < kQuads; i++) {
                o[r][i].x = fmaf(pj[jj], vv[jj][i].x, o[r][i].x);
                o[r][i].y = fmaf(pj[jj], vv[jj][i].y, o[r][i].y);
                o[r][i].z = fmaf(pj[jj], vv[jj][i].z, o[r][i].z);
                o[r][i].w = fmaf(pj[jj], vv[jj][i].w, o[r][i].w);
              }
          }
        }
      }
      cp_async_wait<0>();
      __syncwarp();
      if (more && a.ahead) start(s_part[turn ^ 1]);
#pragma unroll
      for (int r = 0; r < RT; r++) {
#pragma unroll
        for (int o2 = kTile / 2; o2 > 0; o2 >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o2);
#pragma unroll
        for (int i = 0; i < kQuads; i++) {
          float4 &v = o[r][i];
          if (kHalves == 2) {
            v.x += __shfl_xor_sync(0xffffffffu, v.x, 16);
            v.y += __shfl_xor_sync(0xffffffffu, v.y, 16);
            v.z += __shfl_xor_sync(0xffffffffu, v.z, 16);
            v.w += __shfl_xor_sync(0xffffffffu, v.w, 16);
          }
          const int d = (kHalves == 2 ? dim : lane) + 32 * i;
          if (r < g_rows && 4 * d < hs) {
            if (!(fabsf(v.x) + fabsf(v.y) + fabsf(v.z) + fabsf(v.w) < INFINITY)) odd |= 1u << r;
            if (kHalves == 1 || half == 0) *reinterpret_cast<float4 *>(o_smem + r * hs + 4 * d) = v;
          }
        }
        if (r < g_rows && !(fabsf(l[r]) < INFINITY)) odd |= 1u << r;
        if (lane == 0) {
          s_m[kg][r] = m[r];
          s_l[kg][r] = l[r];
        }
      }
    } else {
      // The keys are the matrix instruction's 16 rows and the queries its 8 columns: scores come out with a lane holding two
      // queries of keys lane / 4 and lane / 4 + 8, and the probabilities, transposed inside the warp, are the second operand
      // of the values' product, whose rows are dimensions.
      constexpr int KS = HSP / 16, KB = kTile / 16;  // steps of 16 dimensions, blocks of 16 positions
      const int gr = lane >> 2, cc = lane & 3;
      const uint32_t ring0 = smem_addr(ring_smem);
      const uint32_t q0 = smem_addr(q_smem) + (8 * rw + (lane & 7)) * S::kQPitch + (lane >> 3) * 16;  // 32 dimensions of eight queries
      const uint32_t k0 = ((lane & 7) + (lane & 8)) * S::kPitch + (lane >> 4) * 16;                  // a K tile's fragment
      const uint32_t v0 = ((lane & 7) + ((lane >> 4) << 3)) * S::kPitch + (lane & 8) * 2;            // a V tile's
      const bool active = 8 * rw < g_rows;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
      const float qs[2] = {s_qscale[8 * rw + 2 * cc], s_qscale[8 * rw + 2 * cc + 1]};
      float o[KS][4];
#pragma unroll
      for (int i = 0; i < KS; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      for (int t = 0; t < n_tiles; t++, pos0 += unit) {
        cp_async_wait<D - 2>();
        meet();
        ring.fill((D & 1) != 0, 2 * t + D - 1 < 2 * n_tiles);
        uint32_t p[TERMS][KB][2];
        float f[2];
        if (active) {
          const uint32_t ok = s_ok[kg][now];
          const uint32_t kt = ring0 + now * S::kTileBytes + k0;
          float sc[TERMS][KB][4];
#pragma unroll
          for (int u = 0; u < TERMS; u++)
#pragma unroll
            for (int b = 0; b < KB; b++) sc[u][b][0] = sc[u][b][1] = sc[u][b][2] = sc[u][b][3] = 0.f;
#pragma unroll
          for (int i = 0; i < KS; i += 2) {
            if (16 * i < hs) {
              uint32_t ka[KB][2][4];
#pragma unroll
              for (int b = 0; b < KB; b++) {
                ldmatrix4(kt + b * 16 * S::kPitch + i * 32, ka[b][0]);
                ldmatrix4(kt + b * 16 * S::kPitch + (i + 1) * 32, ka[b][1]);
              }
#pragma unroll
              for (int u = 0; u < TERMS; u++) {
                uint32_t qb[4];
                ldmatrix4(q0 + u * ROWS * S::kQPitch + i * 32, qb);
#pragma unroll
                for (int b = 0; b < KB; b++) mma_16x8x16<T>(sc[u][b], ka[b][0], qb[0], qb[1]);
#pragma unroll
                for (int b = 0; b < KB; b++) mma_16x8x16<T>(sc[u][b], ka[b][1], qb[2], qb[3]);
              }
            }
          }
          const bool whole = ok == 0xffffffffu && pos0 >= inner_low && pos0 + kTile <= inner_high;
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const int r = 8 * rw + 2 * cc + e;
            float x[2 * KB], top = m[e];  // of this lane's positions gr + 8 y
#pragma unroll
            for (int y = 0; y < 2 * KB; y++) {
              x[y] = sc[TERMS - 1][y / 2][2 * (y & 1) + e];
#pragma unroll
              for (int u = TERMS - 2; u >= 0; u--) x[y] += sc[u][y / 2][2 * (y & 1) + e];
              x[y] *= qs[e];
            }
            if (!whole) {
              const int lo = s_lo[r] - pos0, hi = s_hi[r] - pos0;
#pragma unroll
              for (int y = 0; y < 2 * KB; y++) {
                const int j = gr + 8 * y;
                if (!((ok >> j & 1u) && j >= lo && j < hi)) x[y] = -INFINITY;
              }
            }
            if (a.scores && r < g_rows) {
              float *to = a.scores + s_row[r] + pos0 + gr;
              const int lo = s_lo[r] - pos0, hi = s_hi[r] - pos0;
#pragma unroll
              for (int y = 0; y < 2 * KB; y++)
                if (gr + 8 * y >= lo && gr + 8 * y < hi) to[8 * y] = x[y];
            }
#pragma unroll
            for (int y = 0; y < 2 * KB; y++) top = fmaxf(top, x[y]);
#pragma unroll
            for (int o2 = 4; o2 < 32; o2 <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o2));
            f[e] = m[e] == top ? 1.f : exp2_of(m[e] - top);
            m[e] = top;
            const float less = top - kLift;
            float sum = 0.f;
#pragma unroll
            for (int y = 0; y < 2 * KB; y++) {
              x[y] = x[y] == -INFINITY ? 0.f : exp2_of(x[y] - less);
              sum += x[y];
              sc[0][y / 2][2 * (y & 1) + e] = x[y];
            }
            l[e] = fmaf(l[e], f[e], sum);
          }
#pragma unroll
          for (int b = 0; b < KB; b++)
#pragma unroll
            for (int u = 0; u < TERMS; u++) {
              p[u][b][0] = transpose8x8(split2<T>(sc[0][b][0], sc[0][b][1]));
              p[u][b][1] = transpose8x8(split2<T>(sc[0][b][2], sc[0][b][3]));
            }
        }
        now = now + 1 == D ? 0 : now + 1;
        cp_async_wait<D - 2>();
        meet();
        ring.fill((D & 1) == 0, 2 * t + D < 2 * n_tiles);
        if (active) {
          const uint32_t vt = ring0 + now * S::kTileBytes + v0;
#pragma unroll
          for (int i = 0; i < KS; i += 2)
            if (16 * i < hs) {
              uint32_t va[2][KB][4];
#pragma unroll
              for (int b = 0; b < KB; b++) {
                ldmatrix4_trans(vt + b * 16 * S::kPitch + i * 32, va[0][b]);
                ldmatrix4_trans(vt + b * 16 * S::kPitch + (i + 1) * 32, va[1][b]);
              }
              // a tile's values first, smallest terms ahead, then the running sums: the instruction cuts its sum off, which a
              // long row of additions to one accumulator would show
              float d[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
              for (int u = TERMS - 1; u >= 0; u--)
#pragma unroll
                for (int b = 0; b < KB; b++)
#pragma unroll
                  for (int y = 0; y < 2; y++) mma_16x8x16<T>(d[y], va[y][b], p[u][b][0], p[u][b][1]);
#pragma unroll
              for (int y = 0; y < 2; y++) {
                o[i + y][0] = fmaf(o[i + y][0], f[0], d[y][0]);
                o[i + y][1] = fmaf(o[i + y][1], f[1], d[y][1]);
                o[i + y][2] = fmaf(o[i + y][2], f[0], d[y][2]);
                o[i + y][3] = fmaf(o[i + y][3], f[1], d[y][3]);
              }
            }
        }
        now = now + 1 == D ? 0 : now + 1;
      }
      cp_async_wait<0>();
      meet();
      if (more && a.ahead) start(s_part[turn ^ 1]);
      const float down = kLift != 0.f ? 1.f / 16384.f : 1.f;
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int r = 8 * rw + 2 * cc + e;
#pragma unroll
        for (int o2 = 4; o2 < 32; o2 <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], o2);
        if (gr == 0) {
          s_m[kg][r] = m[e];
          s_l[kg][r] = l[e] * down;
        }
        if (r < g_rows) {
          bool finite = fabsf(l[e]) < INFINITY;
#pragma unroll
          for (int i = 0; i < KS; i++)
#pragma unroll
            for (int y = 0; y < 2; y++) {
              const float v = o[i][2 * y + e] * down;
              const int d = 16 * i + gr + 8 * y;
              if (d < hs) {
                finite = finite && fabsf(v) < INFINITY;
                o_smem[r * hs + d] = v;
              }
            }
          if (!finite) odd |= 1u << r;
        }
      }
    }
    odd = __reduce_or_sync(0xffffffffu, odd);
    if (odd != 0) paged_rows_apart<T, kTile, HSP / 32>(a, w, kg, KG, odd, lane, o_smem, s_m[kg], s_l[kg], nullptr);
    __syncthreads();

    // ---- the key groups' results, and the group's if other CTAs have a part of it
    const int first_cta = paged_first_cta(a, w, per), last_cta = (int)((w.end - 1) / per), parts = last_cta - first_cta + 1;
    const int quads = hs / 4, items = g_rows * quads;
    const int slot_floats = paged_slot(ROWS, hs);
    float *slot = a.partial + (2ll * blockIdx.x + ((int)blockIdx.x == first_cta ? 1 : 0)) * slot_floats;
    for (int i = tid; i < items; i += threads) {
      const int r = g_rows == 1 ? 0 : i / quads, d = i - r * quads;
      float top = s_m[0][r], sum = 0.f;
      for (int y = 1; y < KG; y++) top = fmaxf(top, s_m[y][r]);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int y = 0; y < KG; y++) {
        if (s_m[y][r] == -INFINITY && s_l[y][r] == 0.f) continue;
        const float f = exp2f(s_m[y][r] - top);
        const float4 o = reinterpret_cast<const float4 *>(rings + y * S::kRing + o_at)[i];
        sum += f * s_l[y][r];
        v.x += f * o.x;
        v.y += f * o.y;
        v.z += f * o.z;
        v.w += f * o.w;
      }
      if (parts == 1) {
        if (sum != 0.f) {
          const float inv = 1.f / sum;
          v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        }
        reinterpret_cast<float4 *>(a.out + s_out[r])[d] = v;
        if (a.stats && d == 0) a.stats[row_index(a, w, r)] = top + log2f(sum);
      } else {
        __stcg(reinterpret_cast<float4 *>(slot) + i, v);
        if (d == 0) {
          __stcg(slot + ROWS * hs + r, top);
          __stcg(slot + ROWS * hs + ROWS + r, sum);
        }
      }
    }
    if (parts > 1) {  // the factors take the place of the first key group's results, or of all rings once they are done with
      paged_join(a, w, first_cta, parts, ROWS, tid, threads, [] { __syncthreads(); }, s_red, s_red_sum,
                 reinterpret_cast<float *>(more ? rings + o_at : rings), (more ? S::kTileBytes : KG * S::kRing) / 8, s_out, &s_last);
    }
    __syncthreads();
    if (!more) break;
    if (padded) clear(reinterpret_cast<unsigned char *>(o_smem), a.ahead ? S::kTileBytes : S::kRing);
    if (!a.ahead) start(s_part[turn ^ 1]);
  }
}

// weights[s][j] += sum over the sequence's rows and heads, in their order, of 2^(score - log2 of the sum). A thread has a position;
// the scores of eight heads are asked for together: the kernel is a few dependent round trips to L2, about 9 us for 32 users of
// 12 heads over up to 4097 positions (4.5 MB of scores), where one head at a time took 13.
__global__ void __launch_bounds__(256)
paged_weights_kernel(const __grid_constant__ PagedAttention a, float *__restrict__ weights, long long ld) {
  pdl_launch_dependents();
  pdl_wait();
  const PagedView &c = a.c;
  const int s = blockIdx.y;
  const unsigned int skip = __ldcg(a.skip);
  int first, n, L;
  launch_rows(a, s, first, n, L);
  if (n == 0 || skip != 0) return;
  for (int j = blockIdx.x * 256 + threadIdx.x; j < L; j += gridDim.x * 256) {
    float w = 0.f;
    const float old = weights[s * ld + j];
    for (int t = 0; t < n; t++) {
      const int end = L - n + t + 1, begin = a.window > 0 ? max(0, end - a.window) : 0;
      if (j < begin || j >= end) continue;
      const long long row = (long long)(first - a.row0 + t) * a.n_head;
      for (int h0 = 0; h0 < a.n_head; h0 += 8) {
        float sc[8], lse[8];
#pragma unroll
        for (int u = 0; u < 8; u++) {
          const bool in = h0 + u < a.n_head;
          sc[u] = in ? __ldcg(a.scores + (row + h0 + u) * c.max_length + j) : -INFINITY;
          lse[u] = in ? __ldcg(a.stats + row + h0 + u) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < 8; u++) w += sc[u] != -INFINITY ? exp2_of(sc[u] - lse[u]) : 0.f;
      }
    }
    weights[s * ld + j] = old + w;
  }
}

}  // namespace wgpt
