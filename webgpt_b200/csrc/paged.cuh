// A paged key-value cache: writing new rows, attention of new tokens over it, and its eviction.
#pragma once
#include <cuda_bf16.h>

#include <type_traits>

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

// ------------------------------------------------------------------------------------------ attention
__device__ __forceinline__ float paged_value(const float *p) { return __ldcg(p); }
__device__ __forceinline__ float paged_value(const __half *p) { return __half2float(__ldcg(p)); }
__device__ __forceinline__ float paged_value(const __nv_bfloat16 *p) { return __bfloat162float(__ldcg(p)); }

//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(c s_ij - m_i),  s_ij = q_i . k_j,  c = scale / ln 2,  m_i = max_j c s_ij
// in one pass over the keys, with the running maximum and sum in f32 (sums and values are multiplied by 2^(old - new maximum)
// when it moves).
//
// What bounds it is the cache's bytes: a row of K and V is read once for all the query rows that share it (the heads of its
// group, times the new tokens), at most ROWS of them, a row tile. All (sequence, head of the cache, row tile) groups lie
// behind one another as units of four tiles of positions; every CTA takes as many units as any other, whatever the lengths are, so a CTA
// may hold the end of one group, whole ones, and the beginning of another. A group that is shared is joined by the CTA that
// finishes last, in the order of the positions.
//
// Inside a CTA four warps take a tile of positions each of a unit and never meet until the group ends: each has a ring of tiles in
// shared memory that cp.async fills, K and V tiles in turn, its own running maximum and its own sums.
constexpr int kPagedWarps = 4, kPagedThreads = 32 * kPagedWarps;

struct PagedAttention {
  PagedView c;
  NewRows r;
  int n_head, group, window;
  float scale2;  // scale / ln 2
  const float *q;
  float *out;
  long long ld_q, ld_out;
  int least;             // fewest units a CTA takes
  float *partial;        // [2 * CTAs][paged_slot(ROWS, hs)]
  unsigned int *join;    // a counter per CTA, zero on entry and left zero
  float *scores, *stats; // [n_rows * n_head][max_length] and [n_rows * n_head], in units of log 2, or NULL
};

// A sequence's share of the work.
struct PagedSeq {
  int first, n, L, begin;  // rows, length, position of the first unit
  int tiles, units;        // row tiles, units of each
};

template <int ROWS, int UNIT>
__device__ __forceinline__ PagedSeq paged_seq(const PagedAttention &a, int s) {
  PagedSeq q;
  new_rows(a.c, a.r, s, q.first, q.n);
  q.L = paged_length(a.c, s);
  const int lowest = a.window > 0 ? max(0, q.L - q.n + 1 - a.window) : 0;
  q.begin = min(lowest, q.L) / UNIT * UNIT;
  q.tiles = (q.n * a.group + ROWS - 1) / ROWS;
  q.units = max(1, (q.L - q.begin + UNIT - 1) / UNIT);  // one even if there is nothing to see: the rows are set to zero
  return q;
}

// What a part of a group leaves for the others: the rows' values, maxima and sums.
__host__ __device__ constexpr int paged_slot(int rows, int hs) { return rows * hs + (2 * rows + 3) / 4 * 4; }

// The row tile that a CTA works on.
struct PagedGroup {
  int s, kvh, r0, rows;    // sequence, head of the cache, first row of the tile (token * group + head in the group), rows
  int lowest, highest;     // positions that some row sees: [lowest, highest)
  int inner_low, inner_high;  // positions that every row sees
};

__device__ __forceinline__ void row_range(const PagedAttention &a, const PagedSeq &q, int token, int &lo, int &hi) {
  hi = max(0, q.L - q.n + token + 1);
  lo = a.window > 0 ? max(0, hi - a.window) : 0;
}

__device__ __forceinline__ long long row_offset(const PagedAttention &a, const PagedSeq &q, const PagedGroup &g, int r, long long ld) {
  const int token = (g.r0 + r) / a.group, head = g.kvh * a.group + (g.r0 + r) % a.group;
  return (long long)(q.first + token) * ld + (long long)head * a.c.hs;
}
__device__ __forceinline__ long long row_index(const PagedAttention &a, const PagedSeq &q, const PagedGroup &g, int r) {
  const int token = (g.r0 + r) / a.group, head = g.kvh * a.group + (g.r0 + r) % a.group;
  return (long long)(q.first + token) * a.n_head + head;
}

// Copies 16 bytes, or writes zeros where there is nothing to copy.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t to, const void *from, bool there) {
  const int bytes = there ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What the kernel of a type, a (padded) head size and a number of rows takes of shared memory.
template <typename T, int HSP, int RT>
struct PagedShape {
  static constexpr bool kWide = sizeof(T) == 4;  // f32: products on the CUDA cores, RT rows; else on the tensor cores, 8 RT rows
  static constexpr int kRows = kWide ? RT : 8 * RT;
  static constexpr int kTerms = kWide ? 1 : std::is_same<T, __half>::value ? 2 : 3;  // values that a query or probability is split into
  static constexpr int kPitch = HSP * (int)sizeof(T) + 16;  // of a row in shared memory: 16-byte pieces of 8 rows meet all banks
  static constexpr int kTile = HSP * (int)sizeof(T) <= 256 ? 32 : 16;  // positions of a warp's tile
  static constexpr int kUnit = kPagedWarps * kTile;
  static constexpr int kTileBytes = kTile * kPitch;
  static constexpr int kQPitch = kWide ? HSP * 4 : HSP * 2 + 16;
  static constexpr int kQBytes = kRows * kTerms * kQPitch;
  static constexpr int kPBytes = kWide ? kPagedWarps * kRows * kTile * 4 : 0;  // probabilities of a tile
  // tiles of a ring, of K and V in turn: two CTAs or more share an SM, where a row is small enough
  static constexpr int kStages = 3;
  static constexpr int kRing = kStages * kTileBytes;
  static constexpr int kSmem = kQBytes + kPBytes + kPagedWarps * kRing;
  static_assert(kRing >= kRows * HSP * 4, "a warp's values go where its ring was");
};

// Rows of a tile that a warp saw something non-finite in (an infinity or NaN in V, in a key, in q, also where a row's mask
// leaves it out: zero times infinity): the same again one position at a time, each row from what it sees alone. Leaves the row's
// maximum, sum and values as the fast path does.
template <typename T, int TILE>
__device__ __noinline__ void paged_rows_apart(const PagedAttention &a, const PagedSeq &q, const PagedGroup &g, int u0, int u1,
                                              int warp, int lane, float *o_out, float *m_out, float *l_out) {
  const PagedView &c = a.c;
  for (int r = 0; r < g.rows; r++) {
    int lo, hi;
    row_range(a, q, (g.r0 + r) / a.group, lo, hi);
    const float *x = a.q + row_offset(a, q, g, r, a.ld_q);
    float qv[8], o[8], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      qv[i] = lane + 32 * i < c.hs ? __ldcg(x + lane + 32 * i) : 0.f;
      o[i] = 0.f;
    }
    for (int u = u0; u < u1; u++) {
      const int base = q.begin + (u * kPagedWarps + warp) * TILE;
      for (int j = max(base, lo); j < min(base + TILE, hi); j++) {
        const long long at = paged_offset(c, g.s, j);
        float sc = -INFINITY;
        if (at >= 0) {
          const T *k = static_cast<const T *>(c.k) + at + g.kvh * c.head_stride, *v = static_cast<const T *>(c.v) + at + g.kvh * c.head_stride;
          float d = 0.f;
#pragma unroll
          for (int i = 0; i < 8; i++)
            if (lane + 32 * i < c.hs) d += qv[i] * paged_value(k + lane + 32 * i);
          sc = warp_sum(d) * a.scale2;
          if (sc != -INFINITY) {
            const float nm = fmaxf(m, sc), f = exp2f(m - nm), p = exp2f(sc - nm);
            l = l * f + p;
#pragma unroll
            for (int i = 0; i < 8; i++)
              if (lane + 32 * i < c.hs) o[i] = o[i] * f + p * paged_value(v + lane + 32 * i);
            m = nm;
          }
        }
        if (a.scores && lane == 0) a.scores[row_index(a, q, g, r) * c.max_length + j] = sc;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (lane + 32 * i < c.hs) o_out[r * c.hs + lane + 32 * i] = o[i];
    if (lane == 0) {
      m_out[r] = m;
      l_out[r] = l;
    }
  }
}

// A warp's view of its ring: fills tiles of K and of V in turn.
template <typename T, int HSP, int RT>
struct PagedRing {
  using S = PagedShape<T, HSP, RT>;
  static constexpr int kTile = S::kTile;
  static constexpr int kPerRow = HSP * (int)sizeof(T) / 16;          // 16-byte pieces of a row
  static constexpr int kLanes = kPerRow < 32 ? kPerRow : 32;         // lanes that share a row
  static constexpr int kAtOnce = 32 / kLanes, kWidth = kPerRow / kLanes;
  const PagedView &c;
  const T *k, *v;      // this head's rows of page 0
  const uint32_t *table;
  uint32_t base;       // shared-memory address of the ring
  uint32_t *ok;        // [kStages] which of a tile's positions are there
  int lowest, highest, pos, lane, next = 0;
  uint32_t page, slot; // of this lane's position of the next tile to fill
  long long at;        // where this lane's position of the tile at hand begins, or -1
  bool blocks;         // whether 16 positions from a multiple of 16 on always share a page
  bool plain;          // the tile at hand: all of its positions are there, and in blocks

  __device__ __forceinline__ PagedRing(const PagedView &c_, int s, int kvh, uint32_t base_, uint32_t *ok_, int lane_)
      : c(c_), k(static_cast<const T *>(c_.k) + kvh * c_.head_stride), v(static_cast<const T *>(c_.v) + kvh * c_.head_stride),
        table(c_.table + (size_t)s * c_.table_stride), base(base_), ok(ok_), lane(lane_) {
    blocks = c.page_size % 16 == 0;
  }

  __device__ __forceinline__ void look_up() {  // the page of this lane's position, asked for a tile ahead
    page = 0xFFFFFFFFu;
    slot = 0;
    if (pos >= lowest && pos < highest) {
      const uint32_t index = c.page_shift >= 0 ? (uint32_t)pos >> c.page_shift : (uint32_t)pos / c.page_size;
      slot = (uint32_t)pos - index * c.page_size;
      page = __ldcg(table + index);
    }
  }
  __device__ __forceinline__ void begin(int first, int lowest_, int highest_) {
    lowest = lowest_;
    highest = highest_;
    pos = first + (lane & (kTile - 1));
    look_up();
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
        plain = blocks && there == 0xffffffffu;
        if (lane == 0) ok[stage] = there;
        pos += S::kUnit;
        look_up();
      }
      const T *from = keys ? k : v;
      const uint32_t to = base + stage * S::kTileBytes + lane / kLanes * S::kPitch + lane % kLanes * 16;
      if (plain) {  // one address per 16 positions, the others at a fixed distance
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
#pragma unroll 4
        for (int i = 0; i < kTile / kAtOnce; i++) {
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

template <typename T, int HSP, int RT>
__global__ void __launch_bounds__(kPagedThreads)
paged_attention_kernel(const __grid_constant__ PagedAttention a) {
  using S = PagedShape<T, HSP, RT>;
  constexpr int ROWS = S::kRows, TERMS = S::kTerms, D = S::kStages, kTile = S::kTile;
  // f32: a lane holds four dimensions of kQuads pieces of a row; where 16 lanes hold a row, the halves of the warp take even and odd keys
  constexpr int kQuads = HSP <= 128 ? 1 : HSP / 128, kHalves = HSP <= 64 ? 2 : 1;
  constexpr float kLift = std::is_same<T, __half>::value ? 14.f : 0.f;  // probabilities are held times 2^14, in the middle of a half's range
  extern __shared__ __align__(16) unsigned char paged_smem[];
  __shared__ float s_m[kPagedWarps][ROWS], s_l[kPagedWarps][ROWS], s_qscale[ROWS];
  __shared__ int s_lo[ROWS], s_hi[ROWS];
  __shared__ long long s_row[ROWS];
  __shared__ uint32_t s_ok[kPagedWarps][D];
  __shared__ uint32_t s_sum[kPagedWarps], s_excl;
  __shared__ int s_seq, s_last;
  __shared__ PagedSeq s_q;
  const PagedView &c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hs = c.hs;
  unsigned char *q_smem = paged_smem, *ring_smem = paged_smem + S::kQBytes + S::kPBytes + warp * S::kRing;
  float *p_smem = reinterpret_cast<float *>(paged_smem + S::kQBytes) + warp * ROWS * kTile;
  pdl_launch_dependents();
  // where 32 does not divide the head size, what lies behind a row takes part in products: zeros, times zeros of the query's
  const bool padded = !S::kWide && (hs & 31) != 0;
  auto clear_ring = [&]() {
    for (int i = lane; i < S::kRing / 16; i += 32) reinterpret_cast<uint4 *>(ring_smem)[i] = make_uint4(0, 0, 0, 0);
    __syncwarp();
  };
  if (padded) clear_ring();
  pdl_wait();

  // ---- this CTA's units
  PagedSeq q;
  auto weight_of = [&](int s) -> uint32_t {
    if (s >= c.n_seq) return 0;
    q = paged_seq<ROWS, S::kUnit>(a, s);
    return (uint32_t)q.tiles * (uint32_t)q.units * (uint32_t)c.n_kv;
  };
  auto scan = [&](uint32_t mine, uint32_t &all) {  // sum over the threads before this one, and over all
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    __syncthreads();
    if (lane == 31) s_sum[warp] = upto;
    __syncthreads();
    all = 0;
    for (int w = 0; w < kPagedWarps; w++) {
      if (w < warp) upto += s_sum[w];
      all += s_sum[w];
    }
    return upto - mine;
  };
  uint32_t total = 0, mine = 0, before = 0;
  for (int s0 = 0; s0 < c.n_seq; s0 += kPagedThreads) {
    uint32_t all;
    mine = weight_of(s0 + tid);
    before = total + scan(mine, all);
    total += all;
  }
  const uint32_t per = max((uint32_t)a.least, (total + gridDim.x - 1) / gridDim.x);
  const uint32_t x0 = blockIdx.x * per, x1 = min(total, x0 + per);  // the caller sees to it that neither passes 2^31
  if (x0 >= x1) return;
  if (c.n_seq <= kPagedThreads) {
    if (before <= x0 && x0 < before + mine) {
      s_seq = tid;
      s_excl = before;
      s_q = q;
    }
  } else {
    uint32_t sum = 0;
    for (int s0 = 0; s0 < c.n_seq && sum <= x0; s0 += kPagedThreads) {
      uint32_t all;
      mine = weight_of(s0 + tid);
      before = sum + scan(mine, all);
      if (before <= x0 && x0 < before + mine) {
        s_seq = s0 + tid;
        s_excl = before;
        s_q = q;
      }
      sum += all;
    }
  }
  __syncthreads();
  int s = s_seq;
  uint32_t seq_begin = s_excl, x = x0;
  q = s_q;

  while (x < x1) {
    while (x >= seq_begin + (uint32_t)q.tiles * (uint32_t)q.units * (uint32_t)c.n_kv) {
      seq_begin += (uint32_t)q.tiles * (uint32_t)q.units * (uint32_t)c.n_kv;
      q = paged_seq<ROWS, S::kUnit>(a, ++s);
    }
    const uint32_t gi = (x - seq_begin) / (uint32_t)q.units, g_begin = seq_begin + gi * q.units, g_end = g_begin + q.units;
    PagedGroup g;
    g.s = s;
    g.kvh = (int)(gi / (uint32_t)q.tiles);
    g.r0 = (int)(gi - (uint32_t)g.kvh * (uint32_t)q.tiles) * ROWS;
    g.rows = min(ROWS, q.n * a.group - g.r0);
    {
      int lo, hi;
      row_range(a, q, g.r0 / a.group, lo, hi);
      g.lowest = lo;
      g.inner_high = hi;
      row_range(a, q, (g.r0 + g.rows - 1) / a.group, lo, hi);
      g.inner_low = lo;
      g.highest = hi;
    }
    // units [u0, u1) of the group are this CTA's; those that no row of the tile sees are left out
    int u0 = (int)(x - g_begin), u1 = (int)(min(x1, g_end) - g_begin);
    x = min(x1, g_end);
    u0 = max(u0, (g.lowest - q.begin) / S::kUnit);
    u1 = min(u1, (g.highest - q.begin + S::kUnit - 1) / S::kUnit);
    const int n_tiles = max(0, u1 - u0);

    PagedRing<T, HSP, RT> ring(c, s, g.kvh, smem_addr(ring_smem), s_ok[warp], lane);
    if (n_tiles > 0) ring.begin(q.begin + (u0 * kPagedWarps + warp) * kTile, g.lowest, g.highest);
#pragma unroll
    for (int h = 0; h < D - 1; h++) ring.fill((h & 1) == 0, h < 2 * n_tiles);
    int now = 0;  // the stage that is next to be used up

    // ---- the queries
    if constexpr (S::kWide) {
      float4 *q4 = reinterpret_cast<float4 *>(q_smem);
      for (int i = tid; i < ROWS * (HSP / 4); i += kPagedThreads) {
        const int r = i / (HSP / 4), d = i % (HSP / 4);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < g.rows && 4 * d < hs) v = __ldcg(reinterpret_cast<const float4 *>(a.q + row_offset(a, q, g, r, a.ld_q)) + d);
        q4[i] = v;
      }
    } else {
      for (int r = warp; r < ROWS; r += kPagedWarps) {
        float v[HSP / 32], top = 0.f;
        const float *row = r < g.rows ? a.q + row_offset(a, q, g, r, a.ld_q) : nullptr;
#pragma unroll
        for (int i = 0; i < HSP / 64; i++) {
          const int d = 2 * lane + 64 * i;
          const float2 f = row && d < hs ? __ldcg(reinterpret_cast<const float2 *>(row + d)) : make_float2(0.f, 0.f);
          v[2 * i] = f.x;
          v[2 * i + 1] = f.y;
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
        int e = 0;
        if constexpr (TERMS == 2) {  // a power of two that brings the row's largest value near 2^13
          top = warp_max(top);
          e = top > 0.f && top < INFINITY ? ilogbf(top) - 13 : 0;
        }
#pragma unroll
        for (int i = 0; i < HSP / 64; i++) {
          float f0 = scalbnf(v[2 * i], -e), f1 = scalbnf(v[2 * i + 1], -e);
#pragma unroll
          for (int t = 0; t < TERMS; t++)
            *reinterpret_cast<uint32_t *>(q_smem + (t * ROWS + r) * S::kQPitch + (2 * lane + 64 * i) * 2) = split2<T>(f0, f1);
        }
        if (lane == 0) s_qscale[r] = scalbnf(a.scale2, e);
      }
    }
    if (tid < ROWS) {
      int lo = 0, hi = 0;
      if (tid < g.rows) row_range(a, q, (g.r0 + tid) / a.group, lo, hi);
      s_lo[tid] = lo;
      s_hi[tid] = hi;
      s_row[tid] = row_index(a, q, g, tid) * c.max_length;
    }
    __syncthreads();

    bool finite = true;
    float *o_smem = reinterpret_cast<float *>(ring_smem);
    if constexpr (S::kWide) {
      constexpr int kShare = 32 / kTile;  // lanes that share a key
      const int key = lane % kTile, share = lane / kTile, half = lane >> 4, dim = lane & 15;
      float m[ROWS], l[ROWS];
      float4 o[ROWS][kQuads];
#pragma unroll
      for (int r = 0; r < ROWS; r++) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int w = 0; w < kQuads; w++) o[r][w] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      for (int t = 0; t < n_tiles; t++) {
        const int pos0 = q.begin + ((u0 + t) * kPagedWarps + warp) * kTile;
        // ---- scores: a lane takes one key, or every other quad of its row
        cp_async_wait<D - 2>();
        __syncwarp();
        ring.fill((D & 1) != 0, 2 * t + D - 1 < 2 * n_tiles);
        const uint32_t ok = s_ok[warp][now];
        const float4 *kt = reinterpret_cast<const float4 *>(ring_smem + now * S::kTileBytes + key * S::kPitch);
        now = now + 1 == D ? 0 : now + 1;
        float sc[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; r++) sc[r] = 0.f;
#pragma unroll 8
        for (int d = share; d < hs / 4; d += kShare) {
          const float4 kv = kt[d];
#pragma unroll
          for (int r = 0; r < ROWS; r++) {
            const float4 qv = reinterpret_cast<const float4 *>(q_smem)[r * (HSP / 4) + d];
            sc[r] = fmaf(qv.x, kv.x, sc[r]);
            sc[r] = fmaf(qv.y, kv.y, sc[r]);
            sc[r] = fmaf(qv.z, kv.z, sc[r]);
            sc[r] = fmaf(qv.w, kv.w, sc[r]);
          }
        }
        const bool whole = ok == 0xffffffffu && pos0 >= g.inner_low && pos0 + kTile <= g.inner_high;
        float f[ROWS];
        bool moved = false;
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
          if (kShare == 2) sc[r] += __shfl_xor_sync(0xffffffffu, sc[r], 16);
          sc[r] *= a.scale2;
          if (!whole && !((ok >> key & 1u) && pos0 + key >= s_lo[r] && pos0 + key < s_hi[r])) sc[r] = -INFINITY;
          if (a.scores && share == 0 && r < g.rows && pos0 + key >= s_lo[r] && pos0 + key < s_hi[r])
            a.scores[s_row[r] + pos0 + key] = sc[r];
          float top = sc[r];
#pragma unroll
          for (int w = kTile / 2; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
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
          for (int r = 0; r < ROWS; r++)
#pragma unroll
            for (int w = 0; w < kQuads; w++) {
              o[r][w].x *= f[r];
              o[r][w].y *= f[r];
              o[r][w].z *= f[r];
              o[r][w].w *= f[r];
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
          float4 vv[4][kQuads];
#pragma unroll
          for (int jj = 0; jj < 4; jj++)
#pragma unroll
            for (int w = 0; w < kQuads; w++) {
              const int j = j0 + (kHalves == 2 ? 4 * half : 0) + jj;
              vv[jj][w] = 4 * (dim4 + 32 * w) < hs ? *reinterpret_cast<const float4 *>(vt + j * S::kPitch + (dim4 + 32 * w) * 16)
                                                   : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
          for (int r = 0; r < ROWS; r++) {
            const float4 p = *reinterpret_cast<const float4 *>(p_smem + r * kTile + j0 + (kHalves == 2 ? 4 * half : 0));
            const float pj[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
            for (int jj = 0; jj < 4; jj++)
#pragma unroll
              for (int w = 0; w < kQuads; w++) {
                o[r][w].x = fmaf(pj[jj], vv[jj][w].x, o[r][w].x);
                o[r][w].y = fmaf(pj[jj], vv[jj][w].y, o[r][w].y);
                o[r][w].z = fmaf(pj[jj], vv[jj][w].z, o[r][w].z);
                o[r][w].w = fmaf(pj[jj], vv[jj][w].w, o[r][w].w);
              }
          }
        }
      }
      cp_async_wait<0>();
      __syncwarp();
#pragma unroll
      for (int r = 0; r < ROWS; r++) {
#pragma unroll
        for (int w = kTile / 2; w > 0; w >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], w);
#pragma unroll
        for (int w = 0; w < kQuads; w++) {
          float4 &v = o[r][w];
          if (kHalves == 2) {
            v.x += __shfl_xor_sync(0xffffffffu, v.x, 16);
            v.y += __shfl_xor_sync(0xffffffffu, v.y, 16);
            v.z += __shfl_xor_sync(0xffffffffu, v.z, 16);
            v.w += __shfl_xor_sync(0xffffffffu, v.w, 16);
          }
          const int d = (kHalves == 2 ? dim : lane) + 32 * w;
          finite = finite && fabsf(v.x) + fabsf(v.y) + fabsf(v.z) + fabsf(v.w) < INFINITY;
          if (r < g.rows && 4 * d < hs && (kHalves == 1 || half == 0)) *reinterpret_cast<float4 *>(o_smem + r * hs + 4 * d) = v;
        }
        finite = finite && fabsf(l[r]) < INFINITY;
        if (lane == 0) {
          s_m[warp][r] = m[r];
          s_l[warp][r] = l[r];
        }
      }
    } else {
      // The keys are the matrix instruction's 16 rows and the queries its 8 columns: scores come out with a lane holding two
      // queries of keys lane / 4 and lane / 4 + 8, and the probabilities, transposed inside the warp, are the second operand
      // of the values' product, whose rows are dimensions.
      constexpr int KS = HSP / 16, KB = kTile / 16;  // steps of 16 dimensions, blocks of 16 positions
      const int gr = lane >> 2, cc = lane & 3;
      const uint32_t ring0 = smem_addr(ring_smem), q0 = smem_addr(q_smem);
      const int k_row = (lane & 7) + (lane & 8), k_col = (lane >> 4) * 8;             // a lane's row and piece of a K tile's fragment
      const int v_row = (lane & 7) + ((lane >> 4) << 3), v_col = lane & 8;            // of a V tile's
      const int q_row = lane & 7, q_col = (lane >> 3) * 8;                            // of 32 dimensions of eight queries
      float m[RT][2], l[RT][2], qs[RT][2];
      float o[KS][RT][4];
#pragma unroll
      for (int n = 0; n < RT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          m[n][e] = -INFINITY;
          l[n][e] = 0.f;
          qs[n][e] = s_qscale[8 * n + 2 * cc + e];
        }
#pragma unroll
      for (int i = 0; i < KS; i++)
#pragma unroll
        for (int n = 0; n < RT; n++) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
      for (int t = 0; t < n_tiles; t++) {
        const int pos0 = q.begin + ((u0 + t) * kPagedWarps + warp) * kTile;
        cp_async_wait<D - 2>();
        __syncwarp();
        ring.fill((D & 1) != 0, 2 * t + D - 1 < 2 * n_tiles);
        const uint32_t ok = s_ok[warp][now];
        const uint32_t kt = ring0 + now * S::kTileBytes + k_row * S::kPitch + k_col * 2;
        now = now + 1 == D ? 0 : now + 1;
        float sc[TERMS][KB][RT][4];
#pragma unroll
        for (int u = 0; u < TERMS; u++)
#pragma unroll
          for (int b = 0; b < KB; b++)
#pragma unroll
            for (int n = 0; n < RT; n++) sc[u][b][n][0] = sc[u][b][n][1] = sc[u][b][n][2] = sc[u][b][n][3] = 0.f;
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
            for (int u = 0; u < TERMS; u++)
#pragma unroll
              for (int n = 0; n < RT; n++) {
                uint32_t qb[4];
                ldmatrix4(q0 + (u * ROWS + 8 * n + q_row) * S::kQPitch + (i * 16 + q_col) * 2, qb);
#pragma unroll
                for (int b = 0; b < KB; b++) mma_16x8x16<T>(sc[u][b][n], ka[b][0], qb[0], qb[1]);
#pragma unroll
                for (int b = 0; b < KB; b++) mma_16x8x16<T>(sc[u][b][n], ka[b][1], qb[2], qb[3]);
              }
          }
        }
        const bool whole = ok == 0xffffffffu && pos0 >= g.inner_low && pos0 + kTile <= g.inner_high;
        uint32_t p[TERMS][KB][RT][2];
        float f[RT][2];
#pragma unroll
        for (int n = 0; n < RT; n++) {
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const int r = 8 * n + 2 * cc + e;
            float x[2 * KB], top = m[n][e];  // of this lane's positions gr + 8 y
#pragma unroll
            for (int y = 0; y < 2 * KB; y++) {
              x[y] = sc[TERMS - 1][y / 2][n][2 * (y & 1) + e];
#pragma unroll
              for (int u = TERMS - 2; u >= 0; u--) x[y] += sc[u][y / 2][n][2 * (y & 1) + e];
              x[y] *= qs[n][e];
            }
            if (!whole) {
              const int lo = s_lo[r] - pos0, hi = s_hi[r] - pos0;
#pragma unroll
              for (int y = 0; y < 2 * KB; y++) {
                const int j = gr + 8 * y;
                if (!((ok >> j & 1u) && j >= lo && j < hi)) x[y] = -INFINITY;
              }
            }
            if (a.scores && r < g.rows) {
              float *to = a.scores + s_row[r] + pos0 + gr;
              const int lo = s_lo[r] - pos0, hi = s_hi[r] - pos0;
#pragma unroll
              for (int y = 0; y < 2 * KB; y++)
                if (gr + 8 * y >= lo && gr + 8 * y < hi) to[8 * y] = x[y];
            }
#pragma unroll
            for (int y = 0; y < 2 * KB; y++) top = fmaxf(top, x[y]);
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            f[n][e] = m[n][e] == top ? 1.f : exp2_of(m[n][e] - top);
            m[n][e] = top;
            const float less = top - kLift;
            float sum = 0.f;
#pragma unroll
            for (int y = 0; y < 2 * KB; y++) {
              x[y] = x[y] == -INFINITY ? 0.f : exp2_of(x[y] - less);
              sum += x[y];
              sc[0][y / 2][n][2 * (y & 1) + e] = x[y];
            }
            l[n][e] = fmaf(l[n][e], f[n][e], sum);
          }
#pragma unroll
          for (int b = 0; b < KB; b++)
#pragma unroll
            for (int u = 0; u < TERMS; u++) {
              p[u][b][n][0] = transpose8x8(split2<T>(sc[0][b][n][0], sc[0][b][n][1]));
              p[u][b][n][1] = transpose8x8(split2<T>(sc[0][b][n][2], sc[0][b][n][3]));
            }
        }
        cp_async_wait<D - 2>();
        __syncwarp();
        ring.fill((D & 1) == 0, 2 * t + D < 2 * n_tiles);
        const uint32_t vt = ring0 + now * S::kTileBytes + v_row * S::kPitch + v_col * 2;
        now = now + 1 == D ? 0 : now + 1;
#pragma unroll
        for (int i = 0; i < KS; i++)
          if (16 * i < hs) {
            uint32_t va[KB][4];
#pragma unroll
            for (int b = 0; b < KB; b++) ldmatrix4_trans(vt + b * 16 * S::kPitch + i * 32, va[b]);
#pragma unroll
            for (int n = 0; n < RT; n++) {
              // a tile's values first, smallest terms ahead, then the running sums: the instruction cuts its sum off, which a
              // long row of additions to one accumulator would show
              float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int u = TERMS - 1; u >= 0; u--)
#pragma unroll
                for (int b = 0; b < KB; b++) mma_16x8x16<T>(d, va[b], p[u][b][n][0], p[u][b][n][1]);
              o[i][n][0] = fmaf(o[i][n][0], f[n][0], d[0]);
              o[i][n][1] = fmaf(o[i][n][1], f[n][1], d[1]);
              o[i][n][2] = fmaf(o[i][n][2], f[n][0], d[2]);
              o[i][n][3] = fmaf(o[i][n][3], f[n][1], d[3]);
            }
          }
      }
      cp_async_wait<0>();
      __syncwarp();
      const float down = kLift != 0.f ? 1.f / 16384.f : 1.f;
#pragma unroll
      for (int n = 0; n < RT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int r = 8 * n + 2 * cc + e;
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], w);
          finite = finite && fabsf(l[n][e]) < INFINITY;
          if (gr == 0) {
            s_m[warp][r] = m[n][e];
            s_l[warp][r] = l[n][e] * down;
          }
#pragma unroll
          for (int i = 0; i < KS; i++)
#pragma unroll
            for (int y = 0; y < 2; y++) {
              const float v = o[i][n][2 * y + e] * down;
              const int d = 16 * i + gr + 8 * y;
              finite = finite && fabsf(v) < INFINITY;
              if (r < g.rows && d < hs) o_smem[r * hs + d] = v;
            }
        }
    }
    if (!__all_sync(0xffffffffu, finite)) {
      __syncwarp();
      paged_rows_apart<T, S::kTile>(a, q, g, u0, u1, warp, lane, o_smem, s_m[warp], s_l[warp]);
    }
    __syncthreads();

    // ---- the four warps' results, and the group's if other CTAs have a part of it
    const int first_cta = (int)(g_begin / per), last_cta = (int)((g_end - 1) / per), parts = last_cta - first_cta + 1;
    const int quads = hs / 4, items = g.rows * quads;
    const int slot_floats = paged_slot(ROWS, hs);
    float *slot = a.partial + (2ll * blockIdx.x + ((int)blockIdx.x == first_cta ? 1 : 0)) * slot_floats;
    for (int i = tid; i < items; i += kPagedThreads) {
      const int r = i / quads, d = i % quads;
      float top = s_m[0][r], sum = 0.f;
#pragma unroll
      for (int w = 1; w < kPagedWarps; w++) top = fmaxf(top, s_m[w][r]);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kPagedWarps; w++) {
        if (s_m[w][r] == -INFINITY && s_l[w][r] == 0.f) continue;
        const float f = exp2f(s_m[w][r] - top);
        const float4 o = reinterpret_cast<const float4 *>(paged_smem + S::kQBytes + S::kPBytes + w * S::kRing)[i];
        sum += f * s_l[w][r];
        v.x += f * o.x;
        v.y += f * o.y;
        v.z += f * o.z;
        v.w += f * o.w;
      }
      if (parts == 1) {
        const float inv = sum != 0.f ? 1.f / sum : 0.f;
        if (sum != 0.f) v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        reinterpret_cast<float4 *>(a.out + row_offset(a, q, g, r, a.ld_out))[d] = v;
        if (a.stats && d == 0) a.stats[row_index(a, q, g, r)] = top + log2f(sum);
      } else {
        __stcg(reinterpret_cast<float4 *>(slot) + i, v);
        if (d == 0) {
          __stcg(slot + ROWS * hs + r, top);
          __stcg(slot + ROWS * hs + ROWS + r, sum);
        }
      }
    }
    if (parts > 1) {
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const unsigned int done = atomicAdd(a.join + first_cta, 1u);
        s_last = done == (unsigned)parts - 1;
        if (s_last) a.join[first_cta] = 0;
      }
      __syncthreads();
      if (s_last) {
        __threadfence();
        // where a row tile has few values, several threads share a quad and take every so many parts
        float4 *red = reinterpret_cast<float4 *>(paged_smem);
        float *red_sum = reinterpret_cast<float *>(red + kPagedThreads);
        auto part_of = [&](int k) { return a.partial + (2ll * (first_cta + k) + (k == 0 ? 1 : 0)) * slot_floats; };
        const int share = items >= kPagedThreads ? 1 : kPagedThreads / items;
        for (int i0 = 0; i0 < items; i0 += kPagedThreads) {
          const int i = share > 1 ? tid % items : i0 + tid, sh = share > 1 ? tid / items : 0;
          const bool live = i < items && sh < share;
          const int r = live ? i / quads : 0;
          float top = -INFINITY, sum = 0.f;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (live) {
#pragma unroll 8
            for (int k = 0; k < parts; k++) top = fmaxf(top, __ldcg(part_of(k) + ROWS * hs + r));
#pragma unroll 8
            for (int k = sh; k < parts; k += share) {
              const float *part = part_of(k);
              const float m = __ldcg(part + ROWS * hs + r), l = __ldcg(part + ROWS * hs + ROWS + r);
              const float4 o = __ldcg(reinterpret_cast<const float4 *>(part) + i);
              const float f = m == -INFINITY && l == 0.f ? 0.f : exp2f(m - top);
              sum += f * l;
              v.x += f * o.x;
              v.y += f * o.y;
              v.z += f * o.z;
              v.w += f * o.w;
            }
          }
          if (share > 1) {
            red[tid] = v;
            red_sum[tid] = sum;
            __syncthreads();
            if (tid < items)
              for (int w = 1; w < share; w++) {
                const float4 o = red[w * items + tid];
                v.x += o.x;
                v.y += o.y;
                v.z += o.z;
                v.w += o.w;
                sum += red_sum[w * items + tid];
              }
          }
          if (live && sh == 0) {
            if (sum != 0.f) {
              const float inv = 1.f / sum;
              v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
            }
            reinterpret_cast<float4 *>(a.out + row_offset(a, q, g, r, a.ld_out))[i % quads] = v;
            if (a.stats && i % quads == 0) a.stats[row_index(a, q, g, r)] = top + log2f(sum);
          }
        }
      }
    }
    __syncthreads();
    if (padded && x < x1) clear_ring();  // the results lay there
  }
}

// weights[s][j] += sum over the sequence's rows and heads, in their order, of 2^(score - log2 of the sum).
__global__ void __launch_bounds__(256)
paged_weights_kernel(PagedAttention a, float *__restrict__ weights, long long ld) {
  pdl_launch_dependents();
  pdl_wait();
  const PagedView &c = a.c;
  const int s = blockIdx.y;
  int first, n;
  new_rows(c, a.r, s, first, n);
  const int L = paged_length(c, s);
  for (int j = blockIdx.x * 256 + threadIdx.x; j < L; j += gridDim.x * 256) {
    float w = 0.f;
    for (int t = 0; t < n; t++) {
      const int end = L - n + t + 1, begin = a.window > 0 ? max(0, end - a.window) : 0;
      if (j < begin || j >= end) continue;
      for (int h = 0; h < a.n_head; h++) {
        const long long rh = (long long)(first + t) * a.n_head + h;
        const float sc = __ldcg(a.scores + rh * c.max_length + j);
        if (sc != -INFINITY) w += exp2f(sc - __ldcg(a.stats + rh));
      }
    }
    weights[s * ld + j] += w;
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
