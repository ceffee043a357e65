// The operators that serve sequences of different lengths: the paged key-value cache (append, attention, eviction) and the
// verification of drafted tokens, behind the C ABI of include/webgpt_b200.h.
#include <algorithm>
#include <atomic>

#include "host.cuh"
#include "paged.cuh"
#include "paged_attention.cuh"
#include "paged_tc.cuh"
#include "verify.cuh"

using namespace wgpt;

// ------------------------------------------------------------------------------------------ checks
static int type_bytes(int type) { return type == WGPT_TYPE_F32 ? 4 : 2; }

static int32_t check_cache(wgpt_device *dev, const wgpt_paged_cache *c, PagedView *out) {
  REQUIRE(c && c->k && c->v && c->table && c->lengths, WGPT_ERR_ARG, "null pointer in the cache");
  REQUIRE(c->type >= WGPT_TYPE_F32 && c->type <= WGPT_TYPE_BF16, WGPT_ERR_ARG, "unknown cache type %d", c->type);
  REQUIRE(c->n_pages >= 1 && c->page_size >= 1 && c->n_kv_head >= 1 && c->n_seq >= 1 && c->table_stride >= 1 &&
              c->max_length >= 1,
          WGPT_ERR_SHAPE, "empty cache: %d pages of %d, %d heads, %d sequences of up to %d positions, %d pages a table row",
          c->n_pages, c->page_size, c->n_kv_head, c->n_seq, c->max_length, c->table_stride);
  // positions are counted in 32 bits, with room for the tiles that are asked for ahead
  REQUIRE(c->n_seq <= 65535 && c->max_length <= 1 << 30, WGPT_ERR_SHAPE, "%d sequences of up to %d positions: at most 65535 of 2^30",
          c->n_seq, c->max_length);
  REQUIRE(c->head_size >= 8 && c->head_size <= 256 && c->head_size % 8 == 0, WGPT_ERR_SHAPE,
          "head_size %d is not a multiple of 8 up to 256", c->head_size);
  REQUIRE((int64_t)c->table_stride * c->page_size >= c->max_length, WGPT_ERR_SHAPE,
          "%d pages of %d positions a sequence hold fewer than max_length %d", c->table_stride, c->page_size, c->max_length);
  const int per16 = 16 / type_bytes(c->type);
  REQUIRE(c->page_stride >= 0 && c->position_stride >= 0 && c->head_stride >= 0, WGPT_ERR_SHAPE, "a stride is negative");
  REQUIRE(aligned16(c->k) && aligned16(c->v) && c->page_stride % per16 == 0 && c->position_stride % per16 == 0 &&
              c->head_stride % per16 == 0,
          WGPT_ERR_ALIGN, "pools must be 16-byte aligned and their strides multiples of 16 bytes");
  int shift = 0;
  while (shift < 31 && (1 << shift) < c->page_size) shift++;
  if ((1u << shift) != (uint32_t)c->page_size) shift = -1;
  *out = PagedView{c->k,          c->v,         c->table,     c->lengths, c->page_stride,  c->position_stride,
                   c->head_stride, (uint32_t)c->n_pages, (uint32_t)c->page_size, shift, c->n_kv_head, c->head_size, c->n_seq,
                   c->table_stride, c->max_length, dev->d_err};
  return WGPT_OK;
}

static int32_t check_rows(const wgpt_paged_cache *c, int32_t n_rows, const int32_t *starts, NewRows *out) {
  REQUIRE(n_rows >= 1, WGPT_ERR_SHAPE, "no rows");
  REQUIRE(starts || n_rows % c->n_seq == 0, WGPT_ERR_SHAPE, "%d rows do not divide among %d sequences", n_rows, c->n_seq);
  *out = NewRows{starts, n_rows, n_rows / c->n_seq};
  return WGPT_OK;
}

static int32_t check_matrix(const void *p, int64_t ld, int64_t cols, const char *what) {
  REQUIRE(p != nullptr, WGPT_ERR_ARG, "%s is null", what);
  REQUIRE(ld >= cols, WGPT_ERR_SHAPE, "rows of %s are %lld values, fewer than %lld", what, (long long)ld, (long long)cols);
  REQUIRE(aligned16(p) && ld % 4 == 0, WGPT_ERR_ALIGN, "%s must be 16-byte aligned, its rows a multiple of 4 values", what);
  return WGPT_OK;
}

// ------------------------------------------------------------------------------------------ cache
WGPT_EXPORT int32_t wgpt_paged_append(wgpt_device *dev, const wgpt_paged_cache *cache, int32_t n_rows,
                                      const int32_t *starts, const float *k, const float *v, int64_t ld) {
  TRY(use(dev));
  PagedView c;
  NewRows r;
  TRY(check_cache(dev, cache, &c));
  TRY(check_rows(cache, n_rows, starts, &r));
  TRY(check_matrix(k, ld, (int64_t)c.n_kv * c.hs, "k"));
  TRY(check_matrix(v, ld, (int64_t)c.n_kv * c.hs, "v"));
  const int grid = (n_rows + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
  if (cache->type == WGPT_TYPE_F32)
    LAUNCH_PDL(dev, paged_append_kernel<float>, grid, kAppendThreads, 0, c, r, k, v, (long long)ld);
  else if (cache->type == WGPT_TYPE_F16)
    LAUNCH_PDL(dev, paged_append_kernel<__half>, grid, kAppendThreads, 0, c, r, k, v, (long long)ld);
  else
    LAUNCH_PDL(dev, paged_append_kernel<__nv_bfloat16>, grid, kAppendThreads, 0, c, r, k, v, (long long)ld);
  return WGPT_OK;
}

// What an attention kernel of this grid and unit takes of the workspace.
static int32_t paged_workspace(wgpt_device *dev, PagedAttention &a, int grid, int unit) {
  // units and rows are counted in 32 bits
  REQUIRE((int64_t)a.r.n_rows * a.group < (int64_t)1 << 30 &&
              ((int64_t)a.r.n_rows * a.group / a.rows + a.c.n_seq) * (a.c.max_length / unit + 2 + a.extra) <
                  (((int64_t)1 << 32) - ((int64_t)1 << 20)) / a.c.n_kv,
          WGPT_ERR_SHAPE, "%d rows over up to %d positions of %d heads: split the call", a.r.n_rows, a.c.max_length, a.c.n_kv);
  const size_t rows = a.stats ? (size_t)(a.row1 - a.row0) * a.n_head : 0, scores = rows * (size_t)a.c.max_length;
  const size_t partial = (size_t)2 * grid * paged_slot(a.rows, a.c.hs);
  TRY(scratch_reserve(dev, (partial + 1 + rows + scores) * 4));
  a.partial = static_cast<float *>(dev->scratch);
  a.skip = nullptr;
  if (a.stats) {
    a.skip = reinterpret_cast<unsigned int *>(a.partial + partial);
    a.stats = a.partial + partial + 1;
    a.scores = a.stats + rows;
  }
  a.join = dev->d_join;
  return WGPT_OK;
}

template <typename T, int HSP, int RT, int STAGES>
static int32_t launch_paged_attention(wgpt_device *dev, PagedAttention &a) {
  using S = PagedShape<T, HSP, RT, STAGES>;
  const auto kernel = paged_attention_kernel<T, HSP, RT, STAGES>;
  const int threads = 32 * a.key_groups * a.row_warps, smem = S::smem(a.key_groups, a.rows), unit = a.key_groups * S::kTile;
  // CTAs that an SM holds, asked once per shape and GPU
  static std::atomic<int> known[64][5];
  REQUIRE(dev->ordinal < 64, WGPT_ERR_UNSUPPORTED, "device ordinal %d not supported", dev->ordinal);
  int per_sm = known[dev->ordinal][a.row_warps].load();
  if (per_sm == 0) {
    CK(allow_smem(dev, kernel, true));
    CK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem));
    REQUIRE(per_sm >= 1, WGPT_ERR_UNSUPPORTED, "the attention kernel does not fit an SM");
    known[dev->ordinal][a.row_warps].store(per_sm);
  }
  const int grid = std::min(per_sm * dev->sm_count, kJoinCounters);
  REQUIRE(S::fits(a.rows, a.c.hs), WGPT_ERR_UNSUPPORTED, "%d rows of %d do not fit the ring", a.rows, a.c.hs);
  a.extra = 2;  // 128 users of 500 f16 positions, 8 heads of 128: 60 us, 66 with none; 8 users of 8192: 45 and 47; 1 to 4 are alike
  TRY(paged_workspace(dev, a, grid, unit));
  a.ahead = S::ahead(a.rows, a.c.hs);
  a.least = 2;
  LAUNCH_PDL(dev, kernel, grid, threads, smem, a);
  return WGPT_OK;
}

template <typename T, int HB, int N>
static int32_t launch_paged_tc(wgpt_device *dev, PagedAttention &a) {
  using S = TcShape<T, HB, N>;
  a.rows = N;
  a.extra = 8;  // 8 users, 5 tokens each, f16, 8 heads of 128: 8192 positions 52 us, 58 with none, 56 with 4; 500 positions 19, 28, 18
  TRY(paged_workspace(dev, a, std::min(dev->sm_count, kJoinCounters), kTcKeys));
  a.least = 1;
  CK(allow_smem(dev, paged_attention_tc_kernel<T, HB, N>, true));
  LAUNCH_PDL(dev, (paged_attention_tc_kernel<T, HB, N>), std::min(dev->sm_count, kJoinCounters), S::kThreads, S::kSmem, a);
  return WGPT_OK;
}

// Whether no CTA can get more than a few units: such calls are a chain of latencies, and the form with all of them in flight,
// one CTA an SM, is shorter than that with more CTAs an SM and fewer tiles in each one's rings. One sequence with a new token:
// 12 heads of 64 in f32, 200 positions, 7.3 us against 8.7; 8 heads of 128 in f16, 4000 positions, 18.1 us against 19.6.
static bool paged_few(const wgpt_device *dev, const PagedAttention &a, int unit) {
  return ((int64_t)a.c.max_length / unit + 1) * a.c.n_seq * a.c.n_kv <= 4 * (int64_t)dev->sm_count;
}

// How many of the rows that share a head of the cache a CTA takes at once: what a sequence has of them on average. More row
// tiles read the cache again, fewer rows leave room for more keys in flight. 16-bit types, head sizes up to 128: up to eight rows
// are one tile of mma.sync, more go to tcgen05 (a rule on rows alone: long sequences with eight rows are better there, as the first of these
// figures shows, the others are not). Measured with both, f16, 4 heads of the cache, one new token, tcgen05 first: head size
// 128, 8 users of 8192 positions, 8 rows 27.4 / 30.8 us, 12 rows 28.3 / 41.7; 64 users of 1000, 35.4 / 33.1 and 36.4 / 50.9; head
// size 64, 24.2 / 21.0 and 23.7 / 26.7, 32.2 / 24.6 and 32.1 / 31.0. 12 rows in tiles of 16 and of 32: 28.4 / 30.9 and 32.0 / 34.8.
// f32, 8 users of 8192, 4 heads of 64, 2 rows in tiles of two and of four: 27.2 / 31.4, 4 rows in tiles of four and of eight: 31.5 / 41.7.
// Tiles of a ring: as many as leave room for another CTA on the SM. f32, head size 64, one row (16 users of 25 heads), two and three:
// 29.7 / 30.7; f16, head size 128, 8 users of 8 heads, 8192 positions, two and three: 43.6 / 59.7, where only one CTA is left.
template <typename T, int HSP>
static int32_t launch_paged_rows(wgpt_device *dev, PagedAttention &a, long long rows) {
  if constexpr (sizeof(T) == 4) {
    a.key_groups = 4;
    a.row_warps = 1;
    a.rows = rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : 8;
    if (rows <= 1) {
      if constexpr (HSP == 64)
        if (paged_few(dev, a, 128)) return launch_paged_attention<T, HSP, 1, 4>(dev, a);
      return launch_paged_attention<T, HSP, 1, HSP == 64 ? 2 : 3>(dev, a);
    }
    if (rows <= 2) return launch_paged_attention<T, HSP, 2, 3>(dev, a);
    if (rows <= 4) return launch_paged_attention<T, HSP, 4, 3>(dev, a);
    return launch_paged_attention<T, HSP, 8, 3>(dev, a);
  } else {
    if constexpr (HSP <= 128) {
      if (rows > 8)
        return rows <= 16 ? launch_paged_tc<T, HSP / 64, 16>(dev, a) : launch_paged_tc<T, HSP / 64, 32>(dev, a);
    }
    // up to eight rows, or head sizes above 128: a key group of one warp for every eight rows, up to 24
    const long long eights = HSP <= 128 ? 1 : (rows + 7) / 8, tiles = (eights + 2) / 3;
    a.row_warps = (int)((eights + tiles - 1) / tiles);
    a.key_groups = a.row_warps == 1 ? 4 : 2;
    a.rows = 8 * a.row_warps;
    if constexpr (HSP == 128)
      if (paged_few(dev, a, 128)) return launch_paged_attention<T, HSP, 1, 4>(dev, a);
    return launch_paged_attention<T, HSP, 1, HSP == 128 ? 2 : 3>(dev, a);
  }
}

template <typename T>
static int32_t launch_paged_type(wgpt_device *dev, PagedAttention &a) {
  long long tokens = ((long long)a.r.n_rows + a.c.n_seq - 1) / a.c.n_seq;
  if (a.r.starts && tokens > 1) tokens += (tokens + 1) / 2;  // some have more than the average
  const long long rows = tokens * a.group;
  if (a.c.hs <= 64) return launch_paged_rows<T, 64>(dev, a, rows);
  if (a.c.hs <= 128) return launch_paged_rows<T, 128>(dev, a, rows);
  return launch_paged_rows<T, 256>(dev, a, rows);
}

WGPT_EXPORT int32_t wgpt_paged_attention(wgpt_device *dev, const wgpt_paged_cache *cache, int32_t n_rows,
                                         const int32_t *starts, int32_t n_head, float scale, int32_t window,
                                         const float *q, int64_t ld_q, float *out, int64_t ld_out, float *weights,
                                         int64_t ld_weights) {
  TRY(use(dev));
  PagedAttention a;
  TRY(check_cache(dev, cache, &a.c));
  TRY(check_rows(cache, n_rows, starts, &a.r));
  REQUIRE(n_head >= 1 && n_head % cache->n_kv_head == 0, WGPT_ERR_SHAPE, "%d heads do not divide among %d of the cache",
          n_head, cache->n_kv_head);
  REQUIRE(window >= 0, WGPT_ERR_SHAPE, "window %d is negative", window);
  const int64_t E = (int64_t)n_head * cache->head_size;
  TRY(check_matrix(q, ld_q, E, "q"));
  TRY(check_matrix(out, ld_out, E, "out"));
  REQUIRE(!weights || ld_weights >= cache->max_length, WGPT_ERR_SHAPE, "rows of weights are %lld values, fewer than max_length %d",
          (long long)ld_weights, cache->max_length);
  a.n_head = n_head;
  a.group = n_head / cache->n_kv_head;
  a.window = window < cache->max_length ? window : 0;  // one that no sequence fills is none; differences of it stay in 32 bits
  a.scale2 = scale * 1.44269504088896f;
  a.q = q;
  a.out = out;
  a.ld_q = ld_q;
  a.ld_out = ld_out;
  // Scores are kept for the kernel that adds them up: as many rows at a time as take no more than this of the workspace, or one
  const size_t per_row = (size_t)n_head * cache->max_length * sizeof(float), most = (size_t)1 << 30;
  const int64_t slice = weights ? std::max<int64_t>(1, (int64_t)(most / per_row)) : n_rows;
  for (int64_t row = 0; row < n_rows; row += slice) {
    a.row0 = (int)row;
    a.row1 = (int)std::min<int64_t>(n_rows, row + slice);
    a.scores = nullptr;
    a.stats = weights;  // that there are any; their place is found with the rest of the workspace
    if (cache->type == WGPT_TYPE_F32)
      TRY(launch_paged_type<float>(dev, a));
    else if (cache->type == WGPT_TYPE_F16)
      TRY(launch_paged_type<__half>(dev, a));
    else
      TRY(launch_paged_type<__nv_bfloat16>(dev, a));
    if (weights) {
      const int blocks = std::min((cache->max_length + 255) / 256, std::max(1, 8 * dev->sm_count / cache->n_seq));
      LAUNCH_PDL(dev, paged_weights_kernel, dim3(blocks, cache->n_seq), dim3(256), 0, a, weights, (long long)ld_weights);
    }
  }
  return WGPT_OK;
}

WGPT_EXPORT int32_t wgpt_paged_evict(wgpt_device *dev, const wgpt_paged_cache *from, const wgpt_paged_cache *to,
                                     int32_t keep, int32_t recent, const float *weights, int64_t ld_weights,
                                     float *weights_to, int64_t ld_weights_to, int32_t *kept) {
  TRY(use(dev));
  PagedEvict e;
  TRY(check_cache(dev, from, &e.from));
  TRY(check_cache(dev, to, &e.to));
  REQUIRE(weights && kept, WGPT_ERR_ARG, "null pointer");
  REQUIRE(from->type == to->type && from->n_kv_head == to->n_kv_head && from->head_size == to->head_size &&
              from->n_seq == to->n_seq,
          WGPT_ERR_SHAPE, "the two caches differ in type, heads or sequences");
  REQUIRE(keep >= 1 && recent >= 0 && recent <= keep, WGPT_ERR_SHAPE, "keep %d and recent %d: 0 <= recent <= keep, keep >= 1",
          keep, recent);
  REQUIRE(to->max_length >= std::min(keep, from->max_length), WGPT_ERR_SHAPE, "%d positions do not hold the %d that stay",
          to->max_length, std::min(keep, from->max_length));
  REQUIRE(ld_weights >= from->max_length && (!weights_to || ld_weights_to >= keep), WGPT_ERR_SHAPE,
          "rows of weights are shorter than their sequences");
  REQUIRE(from->table != to->table, WGPT_ERR_ARG, "the two caches have one table: nothing is moved in place");
  const float *weights_end = weights + (from->n_seq - 1) * ld_weights + from->max_length;
  REQUIRE(!weights_to || weights_to >= weights_end || weights_to + (from->n_seq - 1) * ld_weights_to + keep <= weights, WGPT_ERR_ARG,
          "weights_to overlaps weights");
  e.keep = keep;
  e.recent = recent;
  e.weights = weights;
  e.weights_to = weights_to;
  e.kept = kept;
  e.ld = ld_weights;
  e.ld_to = ld_weights_to;
  // Up to a few positions a thread one CTA is done before a cluster has met. 4 sequences, a quarter goes, one CTA and eight: 1024 positions
  // 12.0 / 17.2 us, 4096 17.0 / 20.6, 8192 22.4 / 24.2, 16384 36.3 / 34.0, 32768 80 / 60.
  const int cluster = from->max_length > 8 * kEvictThreads ? kEvictCluster : 1;
  CK(launch_ex_x(dev->pdl, cluster, dev->stream, paged_select_kernel, dim3(cluster * from->n_seq), dim3(kEvictThreads), 0, e));
  dev->launches++;
  const int most = std::min(keep, from->max_length);
  const int blocks = std::min((most + 7) / 8, std::max(1, 8 * dev->sm_count / from->n_seq));
  LAUNCH_PDL(dev, paged_gather_kernel, dim3(blocks, from->n_seq), dim3(256), 0, e, type_bytes(from->type));
  return WGPT_OK;
}

// ------------------------------------------------------------------------------------------ drafts
WGPT_EXPORT int32_t wgpt_verify_drafts(wgpt_device *dev, int32_t n_seq, int32_t n_draft, int32_t V, const float *target,
                                       int64_t ld_target, const float *draft, int64_t ld_draft, const uint32_t *draft_ids,
                                       const int32_t *n_drafted, int32_t top_k, double temperature,
                                       const double *uniforms, uint32_t *ids_out, int32_t *n_accepted) {
  TRY(use(dev));
  REQUIRE(target && uniforms && ids_out && n_accepted && (draft_ids || n_draft == 0), WGPT_ERR_ARG, "null pointer");
  REQUIRE(n_seq >= 1 && n_seq <= 65535 && V >= 1 && V <= 1 << 30, WGPT_ERR_SHAPE, "%d sequences with %d logits a row", n_seq, V);
  REQUIRE(n_draft >= 0 && n_draft <= WGPT_MAX_DRAFT, WGPT_ERR_SHAPE, "n_draft %d outside 0..%d", n_draft, WGPT_MAX_DRAFT);
  REQUIRE(top_k >= 0 && top_k <= WGPT_MAX_TOP_K && top_k <= V, WGPT_ERR_SHAPE, "top_k %d outside 0..%d", top_k,
          std::min<int>(WGPT_MAX_TOP_K, V));
  REQUIRE(temperature > 0.0, WGPT_ERR_ARG, "temperature must be positive");
  REQUIRE(ld_target >= V && (!draft || n_draft == 0 || ld_draft >= V), WGPT_ERR_SHAPE, "rows of logits are shorter than %d", V);
  Verify a;
  a.n_seq = n_seq;
  a.n_draft = n_draft;
  a.V = V;
  a.top_k = top_k;
  a.chunks = (V + kVerifyChunk - 1) / kVerifyChunk;
  a.target = target;
  a.draft = n_draft ? draft : nullptr;
  a.ld_target = ld_target;
  a.ld_draft = ld_draft;
  a.draft_ids = draft_ids;
  a.n_drafted = n_drafted;
  a.temperature = std::min(temperature, 1e37);  // its reciprocal is no zero in f32, so that -infinity stays what it is; beyond it all is flat
  a.uniforms = uniforms;
  a.ids_out = ids_out;
  a.n_accepted = n_accepted;
  a.err = dev->d_err;
  const int rows = a.draft ? 2 * n_draft + 1 : n_draft + 1;
  const size_t places = (size_t)n_seq * (2 * n_draft + 1);
  if (top_k > 0) {
    TRY(scratch_reserve(dev, places * (16 + (size_t)top_k * 8)));
    a.list_sum = static_cast<double2 *>(dev->scratch);
    a.list_value = reinterpret_cast<float *>(a.list_sum + places);
    a.list_id = reinterpret_cast<int *>(a.list_value + places * top_k);
    const int cap = std::max(kListCap, top_k * ((V + kListThreads - 1) / kListThreads));
    REQUIRE(cap * sizeof(unsigned long long) <= size_t(200) << 10, WGPT_ERR_SHAPE,
            "top_k %d with a vocabulary of %d needs %zu bytes of shared memory for the candidate list", top_k, V,
            cap * sizeof(unsigned long long));
    CK(allow_smem(dev, verify_list_kernel));
    LAUNCH_PDL(dev, verify_list_kernel, dim3(rows, n_seq), dim3(kListThreads), cap * sizeof(unsigned long long), a, cap);
    LAUNCH_PDL(dev, verify_draw_list_kernel, n_seq, 128, 0, a);
    return WGPT_OK;
  }
  TRY(scratch_reserve(dev, places * a.chunks * sizeof(float2)));
  a.partial = static_cast<float2 *>(dev->scratch);
  const int warps = kVerifyThreads / 32;
  LAUNCH_PDL(dev, verify_sums_kernel, dim3((a.chunks + warps - 1) / warps, rows, n_seq), dim3(kVerifyThreads), 0, a);
  // As many CTAs a sequence as are resident at once, two an SM: 64 sequences of 4 drafts over 50257 ids take 43.5 us with four CTAs each,
  // some 10 more with eight (two waves) or two. As long as one wave of clusters of eight has a CTA an SM (14 sequences; the SMs next to
  // one another do not always make another cluster), a CTA may take all the registers: four logits of each row at once against two, and
  // two CTAs an SM: 1 sequence 15.0 / 15.6 us, 8 19.4 / 21.3, 14 21.8 / 24.8, 16 28.9 / 25.1.
  int C = kDrawCluster;
  while (C > 1 && C * n_seq > 2 * dev->sm_count) C /= 2;
  const dim3 grid(C * n_seq), block(kDrawThreads);
  if (C == kDrawCluster && 5 * C * n_seq <= 4 * dev->sm_count)
    CK(launch_ex_x(dev->pdl, C, dev->stream, verify_draw_kernel<4, 1>, grid, block, 0, a));
  else
    CK(launch_ex_x(dev->pdl, C, dev->stream, verify_draw_kernel<2, 2>, grid, block, 0, a));
  dev->launches++;
  return WGPT_OK;
}
