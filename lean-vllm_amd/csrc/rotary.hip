// Rotary positions on queries and keys, after an RMS norm of each head where the model has one, and the same on the
// way into the paged cache: what lies between a layer's projection and store_kvcache + attention
// (lean_vllm/attention/abstract.py:107-116 takes the keys as they leave this).
//
// With x one head row of D elements, r its rotary width, c and s the table's cosines and sines of the token's position:
//   x <- x * rsqrt(mean(x^2) + eps) * w                                  (where a weight is given)
//   (y_a, y_b) = (x_a c_i - x_b s_i, x_b c_i + x_a s_i)  for every pair i < r / 2,
//   (a, b) = (i, i + r / 2) or, interleaved, (2 i, 2 i + 1); dims >= r are left as they are.
// All of it in fp32, rounded once. Bound by HBM: every element is read and written once, some 3 (normed: 7) flops each.
#include "lv_common.h"

namespace lv {

struct RotaryParams {
  const char *q, *k, *v;  // head rows [T, H, D]; byte strides
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
  char *q_out, *k_out;  // k_out and v_cache: the caches, where the keys go by slot
  int64_t qo_st, qo_sh, ko_st, ko_sh;
  char* v_cache;
  int64_t c_sb;       // cache page stride; ko_st, ko_sh are its token and head strides
  const int32_t* slots;  // null: no cache
  FastDiv bs;
  const int64_t* positions;
  const float* table;  // [max_position, r]: r / 2 cosines, then r / 2 sines
  int64_t max_position;
  const char *q_weight, *k_weight;  // null: not normed
  float eps;
  int32_t tokens, hq, hkv, dim, rot, interleaved;
};

// A token's table row. A padding row of a captured step has a negative position: it rotates as position 0. One past the
// table has no row: its head rows come out as NaN (amp), so that an overrun does not pass for a result.
__device__ __forceinline__ const float* table_row(const RotaryParams& p, int64_t pos, float& amp) {
  amp = pos < p.max_position ? 1.f : __builtin_nanf("");
  return p.table + (pos < 0 || pos >= p.max_position ? 0 : pos) * p.rot;
}

// The head rows of a token: q's, then k's, then (into a cache) v's. Row h's source and destination; dst is null where
// nothing is stored.
struct HeadRow {
  const char* src;
  char* dst;
  const char* weight;
  bool turned;  // not a value
};
__device__ __forceinline__ HeadRow head_row(const RotaryParams& p, int64_t t, int h) {
  if (h < p.hq) return HeadRow{p.q + t * p.q_st + h * p.q_sh, p.q_out + t * p.qo_st + h * p.qo_sh, p.q_weight, true};
  h -= p.hq;
  const bool value = h >= p.hkv;
  if (value) h -= p.hkv;
  const char* src = value ? p.v + t * p.v_st + h * p.v_sh : p.k + t * p.k_st + h * p.k_sh;
  char* dst;
  if (p.slots) {
    const int slot = p.slots[t];
    const int page = (int)p.bs.div((uint32_t)max(slot, 0));
    dst = slot < 0 ? nullptr
                   : (value ? p.v_cache : p.k_out) + (int64_t)page * p.c_sb +
                         (int64_t)(slot - page * (int)p.bs.d) * p.ko_st + h * p.ko_sh;
  } else {
    dst = p.k_out + t * p.ko_st + h * p.ko_sh;
  }
  return HeadRow{src, dst, value ? nullptr : p.k_weight, !value};
}

template <typename T>
__device__ __forceinline__ float load1(const char* row, int d) {
  return Elem<T>::lo(*reinterpret_cast<const uint16_t*>(row + 2 * (int64_t)d));
}
template <typename T>
__device__ __forceinline__ void store1(char* row, int d, float x) {
  *reinterpret_cast<uint16_t*>(row + 2 * (int64_t)d) = (uint16_t)Elem<T>::pack(x, 0.f);
}

// Any width, stride and alignment: one wave per head row, an element pair per lane. Each element is read and written by
// one lane, so the outputs may be the inputs.
template <typename T>
__global__ __launch_bounds__(256) void rotary_any_kernel(RotaryParams p, int32_t head_rows) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= (int64_t)p.tokens * head_rows) return;
  const int64_t t = row / head_rows;
  const HeadRow r = head_row(p, t, (int)(row - t * head_rows));
  if (!r.dst) return;
  if (!r.turned) {
    for (int d = lane; d < p.dim; d += 64)
      *reinterpret_cast<uint16_t*>(r.dst + 2 * d) = *reinterpret_cast<const uint16_t*>(r.src + 2 * d);
    return;
  }
  float scale = 1.f;
  if (r.weight) {
    float sum = 0.f;
    for (int d = lane; d < p.dim; d += 64) {
      const float x = load1<T>(r.src, d);
      sum = fmaf(x, x, sum);
    }
    scale = rsqrtf(wave_sum(sum) / (float)p.dim + p.eps);
  }
  auto normed = [&](int d) {
    const float x = load1<T>(r.src, d);
    return r.weight ? x * scale * load1<T>(r.weight, d) : x;
  };
  float amp;
  const int half = p.rot / 2;
  const float* row_table = table_row(p, p.positions[t], amp);
  for (int i = lane; i < half; i += 64) {
    const int da = p.interleaved ? 2 * i : i, db = p.interleaved ? 2 * i + 1 : i + half;
    const float a = normed(da), b = normed(db), c = row_table[i] * amp, s = row_table[half + i] * amp;
    store1<T>(r.dst, da, a * c - b * s);
    store1<T>(r.dst, db, b * c + a * s);
  }
  for (int d = p.rot + lane; d < p.dim; d += 64) store1<T>(r.dst, d, normed(d));
}

template <typename T>
static int launch_rotary(const RotaryParams& p, hipStream_t stream) {
  const int32_t head_rows = p.hq + p.hkv * (p.slots ? 2 : 1);
  const int64_t wgs = ((int64_t)p.tokens * head_rows + 3) / 4;
  LV_REQUIRE(fits_one_launch(wgs, 256), "rotary: %d tokens of %d head rows need a grid larger than one launch holds",
             p.tokens, head_rows);
  hipLaunchKernelGGL(rotary_any_kernel<T>, dim3((uint32_t)wgs), dim3(256), 0, stream, p, head_rows);
  LV_LAUNCH_CHECK("rotary_any_kernel");
  return LV_OK;
}

// What both entry points require of the heads and the table.
static int check_rotary(const char* what, const RotaryParams& p, int64_t max_position, int32_t dtype) {
  LV_REQUIRE(dtype == LV_DTYPE_BF16 || dtype == LV_DTYPE_F16, "%s: dtype %d is not bf16 or fp16", what, dtype);
  LV_REQUIRE(p.tokens >= 0 && p.hq >= 0 && p.hkv >= 0 && p.hq + (int64_t)p.hkv > 0 && p.hq < (1 << 20) &&
                 p.hkv < (1 << 20),
             "%s: bad sizes T=%d Hq=%d Hkv=%d", what, p.tokens, p.hq, p.hkv);
  LV_REQUIRE(p.dim >= 2 && p.rot >= 2 && p.rot <= p.dim && p.rot % 2 == 0,
             "%s: the rotary width %d must be even and at most the head width %d", what, p.rot, p.dim);
  LV_REQUIRE(max_position > 0, "%s: a table of %lld positions", what, (long long)max_position);
  LV_REQUIRE(!(p.q_weight || p.k_weight) || p.eps >= 0.f, "%s: the norm's eps must not be negative, got %g", what,
             (double)p.eps);
  return LV_OK;
}

}  // namespace lv

using namespace lv;

extern "C" int lv_rotary(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k, int64_t k_stride_t,
                         int64_t k_stride_h, const int64_t* positions, const float* table, int64_t max_position,
                         int32_t rotary_dim, int32_t interleaved, const void* q_weight, const void* k_weight,
                         float eps, int32_t num_tokens, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                         void* q_out, int64_t q_out_stride_t, int64_t q_out_stride_h, void* k_out,
                         int64_t k_out_stride_t, int64_t k_out_stride_h, int32_t dtype, void* stream) {
  RotaryParams p{};
  p.q = (const char*)q, p.q_st = q_stride_t * 2, p.q_sh = q_stride_h * 2;
  p.k = (const char*)k, p.k_st = k_stride_t * 2, p.k_sh = k_stride_h * 2;
  p.q_out = (char*)q_out, p.qo_st = q_out_stride_t * 2, p.qo_sh = q_out_stride_h * 2;
  p.k_out = (char*)k_out, p.ko_st = k_out_stride_t * 2, p.ko_sh = k_out_stride_h * 2;
  p.bs = FastDiv::make(1);
  p.positions = positions, p.table = table, p.max_position = max_position;
  p.q_weight = (const char*)q_weight, p.k_weight = (const char*)k_weight, p.eps = eps;
  p.tokens = num_tokens, p.hq = num_heads, p.hkv = num_kv_heads, p.dim = head_dim, p.rot = rotary_dim;
  p.interleaved = interleaved != 0;
  const int rc = check_rotary("rotary", p, max_position, dtype);
  if (rc != LV_OK || num_tokens == 0) return rc;
  LV_REQUIRE(positions && table && (num_heads == 0 || (q && q_out)) && (num_kv_heads == 0 || (k && k_out)),
             "rotary: null pointer");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return dtype == LV_DTYPE_BF16 ? launch_rotary<BF16>(p, st) : launch_rotary<F16>(p, st);
}

extern "C" int lv_append_kvcache(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k,
                                 int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t,
                                 int64_t v_stride_h, const int64_t* positions, const float* table,
                                 int64_t max_position, int32_t rotary_dim, int32_t interleaved, const void* q_weight,
                                 const void* k_weight, float eps, int32_t num_tokens, int32_t num_heads,
                                 int32_t num_kv_heads, int32_t head_dim, void* q_out, int64_t q_out_stride_t,
                                 int64_t q_out_stride_h, void* k_cache, void* v_cache, int64_t cache_stride_block,
                                 int64_t cache_stride_token, int64_t cache_stride_head, int32_t block_size,
                                 const int32_t* slot_mapping, int32_t dtype, void* stream) {
  LV_REQUIRE(block_size > 0, "append_kvcache: block_size must be positive, got %d", block_size);
  RotaryParams p{};
  p.q = (const char*)q, p.q_st = q_stride_t * 2, p.q_sh = q_stride_h * 2;
  p.k = (const char*)k, p.k_st = k_stride_t * 2, p.k_sh = k_stride_h * 2;
  p.v = (const char*)v, p.v_st = v_stride_t * 2, p.v_sh = v_stride_h * 2;
  p.q_out = (char*)q_out, p.qo_st = q_out_stride_t * 2, p.qo_sh = q_out_stride_h * 2;
  p.k_out = (char*)k_cache, p.v_cache = (char*)v_cache;
  p.c_sb = cache_stride_block * 2, p.ko_st = cache_stride_token * 2, p.ko_sh = cache_stride_head * 2;
  p.slots = slot_mapping, p.bs = FastDiv::make(block_size);
  p.positions = positions, p.table = table, p.max_position = max_position;
  p.q_weight = (const char*)q_weight, p.k_weight = (const char*)k_weight, p.eps = eps;
  p.tokens = num_tokens, p.hq = num_heads, p.hkv = num_kv_heads, p.dim = head_dim, p.rot = rotary_dim;
  p.interleaved = interleaved != 0;
  const int rc = check_rotary("append_kvcache", p, max_position, dtype);
  if (rc != LV_OK) return rc;
  LV_REQUIRE(num_kv_heads > 0, "append_kvcache: no key heads");
  if (num_tokens == 0) return LV_OK;
  LV_REQUIRE(positions && table && (num_heads == 0 || (q && q_out)) && k && v && k_cache && v_cache && slot_mapping,
             "append_kvcache: null pointer");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return dtype == LV_DTYPE_BF16 ? launch_rotary<BF16>(p, st) : launch_rotary<F16>(p, st);
}
