// Decode of rows whose leading keys lie in the same pages (a system prompt, a document, samples of one prompt): the
// shared keys attended once for all rows, each row's own keys by itself, joined by log-sum-exp.
//
// A query that sees keys 0 .. L - 1, the first P of them shared, has o = sum_j e^(s_j) v_j / sum_j e^(s_j). Cut into
// ranges of keys with partial outputs o_i and log-sum-exps l_i it is sum_i e^(l_i - M) o_i / sum_i e^(l_i - M) for any
// M, so the shared ranges can be walked with every row's queries together: their keys are read rows times less often
// than by lv_paged_attention (math of TorchAttention.decode, lean_vllm/attention/torch_backend.py:93-103, row by row).
//
// Two launches: the items, which are the prefix's (query tiles x kv heads x pieces of its keys) and the rows' own
// (rows x kv heads x splits of their keys), and the merge of their fp32 partials. Everything is sized by the host from
// shapes and bounds; the rows' lengths are read on the device, so a call can be captured.
//
// What bounds it: the prefix's items MFMA once some 100 query rows share a kv head, the rows' own and small batches HBM.
// The two kinds run in one launch, the prefix's first, on a grid that gives them one of the two workgroups that a CU holds
// and the rows' own the other, so that one kind's MFMA work runs under the other's loads. Measured, 32/8 heads, d128, bf16
// (prefix keys, rows, own keys a row; us):
//                                         one launch      prefix, own and merge launches   lv_paged_attention
//   32,768, 200 rows, 64-2048             227             303                              2380
//   8192, 64 rows, 16-1024                42.6            60.8                             244
//   2048, 128 rows, 64-1024, 16 a page    61.1            80.4                             149
//   65,536, 256 rows, 16-64               283             312                              5786
//   16,384, 16 rows, 64-512               24.9            38.6                             123
// What is left at 200 rows: the prefix alone takes 134 us on whole CUs and 179 on one workgroup of each, the own keys
// alone 161 (4 to 9 pieces of the prefix 231 / 240 / 252 / 264 / - / 281 us; raised wave priority of either kind 232
// and 269; partials stored past the caches 231; a last tile's empty waves that skip the products 232).
#include "few_item.h"

namespace lv {

constexpr int kSharedRound = 512;      // workgroups that run at once (two per CU)
constexpr int kSharedPieceKeys = 256;  // least keys of a piece of the prefix
constexpr int kMaxOwnSplits = 32;
constexpr int kMaxSharedPieces = 256;
// 64-key tiles of prompt items that the GPU takes in a microsecond with two workgroups on each CU (245; 190 with one);
// a workgroup's time for a tile beside own items (1.3 alone on its CU); the rate at which own keys stream, and what
// their items take besides. 32/8 heads of 128 and 64/8 of 64.
constexpr double kTilesPerUs = 245, kTileUs = 2.0, kOwnBytesPerUs = 6.0e6, kOwnStartUs = 10;

struct SharedParams : AttnParams {
  int32_t shared, queries, tokens;  // keys of the prefix; queries per row; all queries
  int32_t tile_rows, tiles;         // (query, head) rows of a prefix tile, tiles per kv head
  int32_t per_piece;                // keys per piece (p.pieces of them)
  int32_t splits, own_least;        // most splits of a row's own keys, and the least keys that one is cut for
};

// A row's own part: its keys from `start` on, in `n` splits of `per` (none where the row has no keys). A row that does
// not see the whole prefix (its first query sees fewer keys) is attended by itself from key 0 on.
struct OwnSpan {
  int start, per, n;
};
__device__ __forceinline__ OwnSpan own_span(const SharedParams& p, int len) {
  OwnSpan s;
  s.start = len - p.queries + 1 >= p.shared ? p.shared : 0;
  const int keys = len - s.start;
  const int want = min(p.splits, (keys + p.own_least - 1) / p.own_least);
  s.per = want > 1 ? ((keys + want - 1) / want + 63) / 64 * 64 : max(keys, 1);
  s.n = keys > 0 ? (keys + s.per - 1) / s.per : 0;
  return s;
}

// Partials lie by slot: piece i of token t's prefix in slot i tokens + t, its row's own split j in slot
// (pieces + j) tokens + t.

// How a kernel computes its items. Few<ROWS>: few-query items (few_item.h) of at most 16, 32 or 64 (query, head) rows,
// of the prefix or of a row's own keys. Tile<TP>: prompt items (attn_common.h), 128 rows of the prefix against 64-key
// tiles that the workgroup's waves share; TP: pages per 64-key tile, as there.
template <int ROWS, int HP = 1>
struct Few {
  static constexpr int kRows = ROWS;
  template <int D>
  static constexpr int bytes() { return kWaves * kFewStages * kFewStage; }
  template <typename T, int D>
  static __device__ __forceinline__ void attend(const SharedParams& p, int kvh, char* smem, const FewPart& part) {
    constexpr bool two = ROWS == 64 && D == 128;  // as few_query.hip's launches
    constexpr FewSets sets = HP == 2 ? kTwoHeads : two ? kTwoBlocks : kOneSet;
    few_item<T, D, (two ? 2 : ROWS / 16), sets, true>(p, 0, 0, 0, kvh, smem, part);
  }
  template <typename T, int D>
  static __device__ __forceinline__ void prefix(const SharedParams& p, int kvh, int piece, int tile, char* smem) {
    FewPart part;
    part.table = p.tables;
    part.lk = p.shared;
    part.lq = p.tokens;
    part.tok = 0;
    part.kbeg = piece * p.per_piece;
    part.kend = min(p.shared, part.kbeg + p.per_piece);
    part.row0 = tile * p.tile_rows;
    part.row_end = min(p.tokens * p.group, part.row0 + p.tile_rows);
    part.slot0 = piece * p.tokens;
    part.causal = false;
    attend<T, D>(p, kvh, smem, part);
  }
};
template <int TP>
struct Tile {
  static constexpr int kRows = kPrefillRows;
  template <int D>
  static constexpr int bytes() { return 2 * PromptSmem<D, D, (TP > 1)>::kBytes; }
  template <typename T, int D>
  static __device__ __forceinline__ void prefix(const SharedParams& p, int kvh, int piece, int tile, char* smem) {
    PromptPart part;
    part.lk = p.shared;
    part.lq = p.tokens;
    part.tile0 = piece * (p.per_piece / kPrefillKeys);
    part.tiles = (min(p.per_piece, p.shared - piece * p.per_piece) + kPrefillKeys - 1) / kPrefillKeys;
    part.slot0 = piece * p.tokens;
    prefill_item<T, D, D, true, false, 2, 4, false, TP, false, true>(p, 0, tile, kvh, smem, 0, 0, part);
  }
};
// Workgroups [0, prefix_wgs) take the prefix's items, the rest the rows' own.
template <typename T, int D, typename PREFIX, int OWN_ROWS, int HP>
__global__ __launch_bounds__(256, 2) void shared_items_kernel(SharedParams p, int32_t prefix_wgs) {
  constexpr int kBytes = std::max(PREFIX::template bytes<D>(), Few<OWN_ROWS, HP>::template bytes<D>());
  __shared__ __attribute__((aligned(16))) char smem[kBytes];
  int b = blockIdx.x;
  if (b < prefix_wgs) {
    const int kvh = b % p.hkv, i = b / p.hkv;
    const int piece = i / p.tiles, tile = i - piece * p.tiles;
    PREFIX::template prefix<T, D>(p, kvh, piece, tile, smem);
    return;
  }
  b -= prefix_wgs;
  const int ny = p.hkv / HP, kvh = b % ny * HP, i = b / ny;
  const int split = i / p.rows, row = i - split * p.rows;
  const int len = sload(p.lens_k + row);
  const OwnSpan s = own_span(p, len);
  if (split >= s.n) return;
  FewPart part;
  part.table = p.tables + (int64_t)row * p.t_stride;
  part.lk = len;
  part.lq = p.queries;
  part.tok = row * p.queries;
  part.kbeg = s.start + split * s.per;
  part.kend = min(len, part.kbeg + s.per);
  part.row0 = 0;
  part.row_end = p.queries * p.group;
  part.slot0 = (p.pieces + split) * p.tokens + part.tok;
  part.causal = true;
  Few<OWN_ROWS, HP>::template attend<T, D>(p, kvh, smem, part);
}

// The merge of one (token, head)'s partials: D / 4 threads a partial, G partials at a time and BATCH such rounds' loads
// in flight, the G threads of each four dims joined through LDS. A workgroup holds 256 / (D / 4) / G of them: few
// partials each would leave most of a workgroup idle, and thousands of workgroups are three microseconds of launching
// (6400 of 6 partials 11.2 -> 6.6 us, 256 rows on 1K shared tokens 67 -> 61.6 in all).
constexpr int kMergeBatch = 8;
template <typename T, int D, int G, int BATCH>
__global__ __launch_bounds__(256) void shared_merge_kernel(SharedParams p) {
  using E = Elem<T>;
  constexpr int LPR = D / 4, PER = 256 / LPR / G;
  __shared__ __attribute__((aligned(16))) float part[G > 1 ? PER * G : 1][D + 4];
  const int slot = threadIdx.x / LPR, g = PER > 1 ? slot % G : slot, d0 = threadIdx.x % LPR * 4;
  const int row = PER > 1 ? blockIdx.x * PER + slot / G : blockIdx.x;  // of the tokens x heads
  const bool live = PER == 1 || row < p.tokens * p.hq;
  const int tok = live ? row / p.hq : 0, head = live ? row - tok * p.hq : 0;
  const OwnSpan s = own_span(p, p.lens_k[tok / p.queries]);
  const int shared = s.start > 0 ? p.pieces : 0;  // the partials: so many of the prefix, then s.n
  const int count = live ? shared + s.n : 0;
  float m = -INFINITY, den = 0.f;
  f32x4 o = {0, 0, 0, 0};
  for (int e0 = g; e0 < count; e0 += G * BATCH) {
    float ls[BATCH];
    f32x4 x[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int e = e0 + i * G;
      ls[i] = -INFINITY;
      x[i] = f32x4{0, 0, 0, 0};
      if (e < count) {
        const int64_t at = ((int64_t)(e < shared ? e : p.pieces + e - shared) * p.tokens + tok) * p.hq + head;
        ls[i] = p.part_lse[at];
        x[i] = *reinterpret_cast<const f32x4*>(p.part_o + at * D + d0);
      }
    }
    float bm = m;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) bm = fmaxf(bm, ls[i]);
    const float base = merge_base(bm), alpha = fast_exp2(m - base);
    den *= alpha;
    o *= alpha;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const float w = fast_exp2(ls[i] - base);
      den += w;
      o += w * x[i];
    }
    m = bm;
  }
  if constexpr (G > 1) {
    *reinterpret_cast<f32x4*>(&part[slot][d0]) = o;
    if (d0 == 0) part[slot][D] = m, part[slot][D + 1] = den;
    __syncthreads();
    if (g > 0) return;
    float bm = -INFINITY;
#pragma unroll
    for (int i = 0; i < G; ++i) bm = fmaxf(bm, part[slot + i][D]);
    const float base = merge_base(bm);
    den = 0.f;
    o = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const float w = fast_exp2(part[slot + i][D] - base);
      den += w * part[slot + i][D + 1];
      o += w * *reinterpret_cast<const f32x4*>(&part[slot + i][d0]);
    }
  }
  if (!live) return;
  o *= inv_sum(den);
  *reinterpret_cast<u32x2*>(p.out + (int64_t)tok * p.o_st + (int64_t)head * p.o_sh + d0 * 2) =
      u32x2{E::pack(o[0], o[1]), E::pack(o[2], o[3])};
}

template <typename T, int D, int G, int BATCH>
static void launch_merge(const SharedParams& p, hipStream_t stream) {
  constexpr int per = 256 / (D / 4) / G;
  const int64_t rows = (int64_t)p.tokens * p.hq;
  hipLaunchKernelGGL((shared_merge_kernel<T, D, G, BATCH>), dim3((uint32_t)((rows + per - 1) / per)), dim3(256), 0, stream, p);
}

// What the host decides from the shapes.
struct SharedPlan {
  int32_t tile_pages;  // pages per 64-key tile of prompt items (0: few-query items)
  int32_t tile_rows, tiles, pieces, per_piece, splits, own_least, own_heads;
  size_t o_bytes, bytes;  // partial outputs, then their log-sum-exps
};

// (query, head) rows of a few-query item, by how many there are.
static int few_rows(int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

static SharedPlan shared_plan(int32_t rows, int32_t queries, int32_t hq, int32_t hkv, int32_t d, int32_t block_size,
                              int32_t shared, int32_t max_k, int64_t own_keys) {
  SharedPlan s{};
  const int group = hq / hkv;
  const int64_t tokens = (int64_t)rows * queries, query_rows = tokens * group;
  // Prompt items hold 128 rows; below, few-query items, which read no more than they need. 33 to 64 rows, few / prompt
  // items, prefixes of 2K, 16K, 64K: d128 17.9 / 15.0, 31.2 / 25.9, 74.5 / 67.8 us; d64 12.8 / -, 18.7 / 17.8, 36.5 /
  // 35.9. 17 to 32 rows at d128 13.0 / 13.9, 23.4 / 23.3, 55.3 / 63.2. On pages that 64-key tiles do not fit,
  // few-query items of 64 rows whatever their number.
  if (query_rows > (d == 64 ? 64 : 32))
    s.tile_pages = block_size % 64 == 0 ? 1 : block_size == 32 ? 2 : block_size == 16 ? 4 : 0;
  s.tile_rows = s.tile_pages > 0 ? kPrefillRows / group * group : few_rows(query_rows);
  s.tiles = (int32_t)((query_rows + s.tile_rows - 1) / s.tile_rows);
  // Unknown: half the bound; for the prefix's pieces, which a bound far off would make too few, at most 1024 a row.
  const int64_t row_keys = own_keys > 0 ? own_keys / rows : (max_k - shared) / 2;
  if (own_keys <= 0) own_keys = (int64_t)rows * std::min<int64_t>(row_keys + 1, 1024);
  const double own_us = (double)own_keys * hkv * d * 4 / kOwnBytesPerUs;
  s.per_piece = kPrefillKeys;
  if (shared > 0) {
    // Pieces: one workgroup of the prefix per CU beside the own keys (few-query items always: their prefix streams
    // too, 64K keys for 2 rows 50.6 us against 52.5 with two), or two where the own keys are worth less than what half
    // the workgroups lose (256 rows on 64K tokens 349 -> 288). And no more than make a piece end within the own keys'
    // time: each costs its partials' way through memory (128 rows on 2K tokens, 1 / 2 / 4 / 8 pieces 78 / 65 / 68 / 74
    // us; 256 on 1K, 1 / 2 / 4 / 8 68 / 74 / 78 / 85; 64 rows on 8K, 8 / 16 / 32 43 / 47 / 59).
    const int64_t units = (int64_t)s.tiles * hkv, key_tiles = (shared + kPrefillKeys - 1) / kPrefillKeys;
    const bool beside = s.tile_pages == 0 || own_us > 0.3 * (double)(units * key_tiles) / kTilesPerUs;
    int64_t want = (beside ? kSharedRound / 2 : kSharedRound) / units;
    if (s.tile_pages > 0 && beside)
      want = std::min(want, (int64_t)std::ceil((double)key_tiles * kTileUs / (own_us + kOwnStartUs)));
    want = std::max<int64_t>(1, std::min<int64_t>({want, kMaxSharedPieces, shared / kSharedPieceKeys}));
    s.per_piece = (int32_t)(((shared + want - 1) / want + 63) / 64 * 64);
    s.pieces = (shared + s.per_piece - 1) / s.per_piece;
  }
  // Own keys: kv heads in pairs (512 adjacent bytes of a token) where those still make a workgroup for every second
  // CU: 32 rows on 8K tokens 39.3 -> 33.1 us, 4 rows of 8 kv heads 9.6 -> 11.4. Split to one round of the workgroups
  // that the prefix leaves (64 rows on 8K: one split 49, two 43), or in two where there is more than a round (128 rows
  // alone: one split 63.5, two 59.4, four 59.6), finer where rows are long. A split holds at least 384 keys where
  // workgroups are many (256 rows on 1K 68.5 -> 67), 256 where they are few (4 rows 10.5 -> 9.7).
  s.own_heads = hkv % 2 == 0 && (int64_t)rows * hkv >= kSharedRound / 2 && queries * group <= 16 ? 2 : 1;
  const int64_t units = (int64_t)rows * hkv / s.own_heads;
  const int64_t beside = std::max<int64_t>(kSharedRound - (int64_t)s.pieces * s.tiles * hkv, kSharedRound / 2);
  int64_t splits = units < beside ? (beside + units / 2) / units : 2;
  splits = std::max(splits, std::min<int64_t>((4 * kSharedRound + units - 1) / units, row_keys / 1024));
  s.own_least = 2 * units <= beside ? 256 : 384;
  // A row that does not see the prefix walks all its keys, so the bound is on those, not on the keys behind it.
  s.splits = (int32_t)std::max<int64_t>(
      1, std::min<int64_t>({splits, kMaxOwnSplits, ((int64_t)max_k + s.own_least - 1) / s.own_least}));
  const int64_t partials = ((int64_t)s.pieces + s.splits) * tokens * hq;
  s.o_bytes = (size_t)partials * d * sizeof(float);
  s.bytes = s.o_bytes + (size_t)partials * sizeof(float);
  return s;
}

template <typename T, int D, typename PREFIX>
static void launch_items(const SharedParams& p, int own_heads, hipStream_t stream) {
  const int rows = p.queries * p.group, prefix = p.pieces * p.tiles * p.hkv;
  auto* kernel = own_heads == 2 ? &shared_items_kernel<T, D, PREFIX, 16, 2> : &shared_items_kernel<T, D, PREFIX, 16, 1>;
  // A prefix of few-query items has at least as many rows as one of its rows' own.
  if constexpr (PREFIX::kRows >= 32)
    if (rows > 16) kernel = &shared_items_kernel<T, D, PREFIX, 32, 1>;
  if constexpr (PREFIX::kRows >= 64)
    if (rows > 32) kernel = &shared_items_kernel<T, D, PREFIX, 64, 1>;
  hipLaunchKernelGGL(kernel, dim3(prefix + p.splits * p.rows * (p.hkv / own_heads)), dim3(256), 0, stream, p, prefix);
}

template <typename T, int D>
static int launch_shared(const SharedParams& p, const SharedPlan& s, hipStream_t stream) {
  if (s.tile_pages == 1) launch_items<T, D, Tile<1>>(p, s.own_heads, stream);
  else if (s.tile_pages == 2) launch_items<T, D, Tile<2>>(p, s.own_heads, stream);
  else if (s.tile_pages == 4) launch_items<T, D, Tile<4>>(p, s.own_heads, stream);
  else if (p.tile_rows == 16) launch_items<T, D, Few<16>>(p, s.own_heads, stream);
  else if (p.tile_rows == 32) launch_items<T, D, Few<32>>(p, s.own_heads, stream);
  else launch_items<T, D, Few<64>>(p, s.own_heads, stream);
  LV_LAUNCH_CHECK("shared_items_kernel");
  // One batch of loads a thread where there are that many threads; all of a workgroup's where there are few rows.
  const int most = p.pieces + p.splits;
  if (most > 2 * kMergeBatch || (int64_t)p.tokens * p.hq < kSharedRound) launch_merge<T, D, 256 / (D / 4), 4>(p, stream);
  else if (most > kMergeBatch) launch_merge<T, D, 2, kMergeBatch>(p, stream);
  else launch_merge<T, D, 1, kMergeBatch>(p, stream);
  LV_LAUNCH_CHECK("shared_merge_kernel");
  return LV_OK;
}

static int check_shared(int32_t rows, int32_t queries, int32_t hq, int32_t hkv, int32_t d, int32_t block_size,
                        int32_t shared, int32_t max_k) {
  LV_REQUIRE(rows >= 0 && queries > 0, "shared_prefix_decode: bad sizes rows=%d queries=%d", rows, queries);
  LV_REQUIRE(hq > 0 && hkv > 0 && hq % hkv == 0, "shared_prefix_decode: %d query heads do not group over %d key heads",
             hq, hkv);
  LV_REQUIRE(d == 64 || d == 128, "shared_prefix_decode: head_dim %d is not 64 or 128", d);
  LV_REQUIRE((int64_t)queries * (hq / hkv) <= kFewMaxRows,
             "shared_prefix_decode: %d queries of %d heads a key head; at most %d together", queries, hq / hkv,
             kFewMaxRows);
  LV_REQUIRE(block_size > 0 && block_size % 16 == 0, "shared_prefix_decode: page size %d is not a multiple of 16",
             block_size);
  LV_REQUIRE(max_k >= 0 && max_k <= (1 << 30), "shared_prefix_decode: max_seqlen_k %d is negative or above 2^30 keys",
             max_k);
  LV_REQUIRE(shared >= 0 && shared <= max_k && shared % block_size == 0,
             "shared_prefix_decode: %d shared keys are not whole pages of %d within max_seqlen_k %d", shared, block_size,
             max_k);
  const int64_t tokens = (int64_t)rows * queries;
  LV_REQUIRE(fits_one_launch(tokens * hq, 256) && fits_one_launch((int64_t)rows * hkv * kMaxOwnSplits, 256) &&
                 tokens * hq * (kMaxOwnSplits + kMaxSharedPieces) < (int64_t)1 << 31,
             "shared_prefix_decode: %lld queries of %d heads are more than one launch holds", (long long)tokens, hq);
  return LV_OK;
}

}  // namespace lv

using namespace lv;

extern "C" size_t lv_shared_prefix_workspace_bytes(int32_t num_rows, int32_t queries_per_row, int32_t num_heads,
                                                   int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                                   int32_t shared_len, int32_t max_seqlen_k, int64_t own_keys) {
  if (num_rows <= 0 || check_shared(num_rows, queries_per_row, num_heads, num_kv_heads, head_dim, block_size,
                                    shared_len, max_seqlen_k) != LV_OK)
    return 0;
  return shared_plan(num_rows, queries_per_row, num_heads, num_kv_heads, head_dim, block_size, shared_len,
                     max_seqlen_k, own_keys)
      .bytes;
}

extern "C" int lv_shared_prefix_decode(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_cache,
                                       const void* v_cache, int64_t cache_stride_block, int64_t cache_stride_token,
                                       int64_t cache_stride_head, int32_t block_size, const int32_t* block_tables,
                                       int64_t table_stride, const int32_t* context_lens, int32_t num_rows,
                                       int32_t queries_per_row, int32_t num_heads, int32_t num_kv_heads,
                                       int32_t head_dim, float scale, int32_t shared_len, int32_t max_seqlen_k,
                                       int64_t own_keys, void* out, int64_t out_stride_t, int64_t out_stride_h,
                                       void* workspace, size_t workspace_bytes, int32_t dtype, void* stream) {
  LV_REQUIRE(dtype == LV_DTYPE_BF16 || dtype == LV_DTYPE_F16, "shared_prefix_decode: dtype %d is not bf16 or fp16",
             dtype);
  const int rc = check_shared(num_rows, queries_per_row, num_heads, num_kv_heads, head_dim, block_size, shared_len,
                              max_seqlen_k);
  if (rc != LV_OK || num_rows == 0) return rc;
  LV_REQUIRE(q && k_cache && v_cache && out && context_lens && (block_tables || max_seqlen_k == 0),
             "shared_prefix_decode: null tensor pointer");
  LV_REQUIRE(aligned(q, 16) && aligned(out, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) &&
                 (q_stride_t * 2) % 16 == 0 && (q_stride_h * 2) % 16 == 0 && (out_stride_t * 2) % 16 == 0 &&
                 (out_stride_h * 2) % 16 == 0 && (cache_stride_block * 2) % 16 == 0 &&
                 (cache_stride_token * 2) % 16 == 0 && (cache_stride_head * 2) % 16 == 0,
             "shared_prefix_decode: tensors and their strides must be 16-byte aligned");
  LV_REQUIRE(cache_stride_token >= 0 && (int64_t)kPrefillKeys * cache_stride_token * 2 < (int64_t)1 << 30,
             "shared_prefix_decode: cache token stride %lld is negative or too large", (long long)cache_stride_token);
  LV_REQUIRE(scale > 0.f, "shared_prefix_decode: the softmax scale must be positive, got %g", (double)scale);
  const SharedPlan s =
      shared_plan(num_rows, queries_per_row, num_heads, num_kv_heads, head_dim, block_size, shared_len, max_seqlen_k,
                  own_keys);
  LV_REQUIRE(workspace && workspace_bytes >= s.bytes, "shared_prefix_decode: workspace of %zu bytes given, %zu needed",
             workspace_bytes, s.bytes);
  LV_REQUIRE(aligned(workspace, 256), "shared_prefix_decode: workspace must be 256-byte aligned");
  SharedParams p{};
  p.q = (const char*)q;
  p.q_st = q_stride_t * 2;
  p.q_sh = q_stride_h * 2;
  p.k_cache = (const char*)k_cache;
  p.v_cache = (const char*)v_cache;
  p.c_sb = cache_stride_block * 2;
  p.c_st = p.v_st = cache_stride_token * 2;
  p.c_sh = p.v_sh = cache_stride_head * 2;
  p.paged = true;
  p.bs = FastDiv::make(block_size);
  p.tables = block_tables;
  p.t_stride = table_stride;
  p.lens_k = context_lens;
  p.rows = num_rows;
  p.hq = num_heads;
  p.hkv = num_kv_heads;
  p.group = num_heads / num_kv_heads;
  p.qgroups = 1;
  p.scale_log2 = scale * kLog2e;
  p.out = (char*)out;
  p.o_st = out_stride_t * 2;
  p.o_sh = out_stride_h * 2;
  p.part_o = (float*)workspace;
  p.part_lse = (float*)((char*)workspace + s.o_bytes);
  p.pieces = s.pieces;
  p.shared = shared_len;
  p.queries = queries_per_row;
  p.tokens = num_rows * queries_per_row;
  p.tile_rows = s.tile_rows;
  p.tiles = s.tiles;
  p.per_piece = s.per_piece;
  p.splits = s.splits;
  p.own_least = s.own_least;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == LV_DTYPE_BF16)
    return head_dim == 64 ? launch_shared<BF16, 64>(p, s, st) : launch_shared<BF16, 128>(p, s, st);
  return head_dim == 64 ? launch_shared<F16, 64>(p, s, st) : launch_shared<F16, 128>(p, s, st);
}
