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

// Rows of whole 16-byte chunks: LPH lanes a head row, each two chunks that hold both elements of every pair in them
// (half layout: chunks c and c + r / 16; interleaved, and behind the rotary width: c and the one as many further on as
// there are such lanes, so that neighbouring lanes' chunks lie side by side: two adjacent chunks a lane took 43.3 us
// where these take 37.3, 8192 tokens interleaved), so a row is read once, turned in registers and written once. A wave
// takes kRounds rounds of 64 / LPH head rows of one token, their loads all issued before the first is used, and the
// table's 8 cosines and 8 sines a lane once for all rounds.
//
// Measured on 32/8 heads of 128, bf16, normed, into the cache: 8192 tokens 36.7 us, 5.60 TB/s (a 1 GiB copy: 5.25);
// normed only, 16384 tokens 60.3 us, 5.71 TB/s; 1 to 100 tokens 4 us, a launch and three dependent loads (position,
// table row, and under them the head rows). One, two, three and four rounds a wave: 8192 tokens 44.6 / 40.7 / 44.6 /
// 42.1 us.
//
// STREAM: loads and stores past the caches. A step's q, k and v come from the projection before and go to the attention
// after, so a call that fits the 256 MB Infinity Cache leaves its outputs there; one that does not only evicts. A
// projection's write, the append and a read of its outputs, cached / streamed: 12.6 MB 18.6 / 19.3 us, 100 MB 58.8 /
// 60.9, 201 MB 122.1 / 113.2, 402 MB 233 / 220 (the append alone 40.7 / 36.7 at 201 MB). The line is drawn at 128 MB.
constexpr int kRounds = 2;
constexpr int64_t kStreamBytes = 128ll << 20;
template <typename T, int LPH, bool INTERLEAVED, bool STREAM>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryParams p, int32_t head_rows) {
  using E = Elem<T>;
  constexpr int NR = kRounds;
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= p.tokens) return;
  const int64_t pos = p.positions[t];
  const int lanes = p.dim / 16;  // lanes that hold a row
  const bool holds = lane % LPH < lanes;
  const int sub = holds ? lane % LPH : 0;
  const int paired = INTERLEAVED ? 0 : p.rot / 16;  // lanes of the half layout's pairs of chunks
  const int chunk_a = sub < paired ? sub : sub + paired, chunk_b = sub < paired ? sub + paired : sub + lanes;
  const bool turns_a = 8 * chunk_a < p.rot, turns_b = 8 * chunk_b < p.rot;
  const int ca = 16 * chunk_a, cb = 16 * chunk_b;  // bytes
  HeadRow row[NR];
  u32x4 xa[NR], xb[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int h = ((int)blockIdx.y * NR + r) * (64 / LPH) + lane / LPH;
    row[r] = head_row(p, t, min(h, head_rows - 1));
    if (h >= head_rows || !holds) row[r].dst = nullptr;
    xa[r] = STREAM ? ld16_stream(row[r].src + ca) : ld16(row[r].src + ca);
    xb[r] = STREAM ? ld16_stream(row[r].src + cb) : ld16(row[r].src + cb);
  }
  float amp;
  const float* cosines = table_row(p, pos, amp);
  // Half layout: the lane's eight pairs; interleaved: four in each chunk.
  const int pa = turns_a ? (INTERLEAVED ? 4 * chunk_a : 8 * chunk_a) : 0;
  const int pb = turns_b ? (INTERLEAVED ? 4 * chunk_b : 8 * chunk_a + 4) : 0;
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c[i] = cosines[pa + i], c[4 + i] = cosines[pb + i];
    s[i] = cosines[p.rot / 2 + pa + i], s[4 + i] = cosines[p.rot / 2 + pb + i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] *= amp;
    s[i] *= amp;
  }
  const bool any_norm = p.q_weight || p.k_weight;
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    float a[8], b[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[2 * i] = E::lo(xa[r][i]), a[2 * i + 1] = E::hi(xa[r][i]);
      b[2 * i] = E::lo(xb[r][i]), b[2 * i + 1] = E::hi(xb[r][i]);
    }
    if (any_norm) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(a[i], a[i], fmaf(b[i], b[i], sum));
      sum = holds ? sum : 0.f;
      sum = group_sum<LPH>(sum);
      if (row[r].weight) {
        const float scale = rsqrtf(sum / (float)p.dim + p.eps);
        const u32x4 wa = ld16(row[r].weight + ca), wb = ld16(row[r].weight + cb);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[2 * i] *= scale * E::lo(wa[i]), a[2 * i + 1] *= scale * E::hi(wa[i]);
          b[2 * i] *= scale * E::lo(wb[i]), b[2 * i + 1] *= scale * E::hi(wb[i]);
        }
      }
    }
    u32x4 ya, yb;
    if (!row[r].turned || (!turns_a && !row[r].weight)) {  // values, and dims that neither turn nor are normed: the bits
      ya = xa[r];
      yb = xb[r];
    } else {
      if constexpr (INTERLEAVED) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a0 = a[2 * i], b0 = b[2 * i];
          if (turns_a) {
            a[2 * i] = a0 * c[i] - a[2 * i + 1] * s[i];
            a[2 * i + 1] = a[2 * i + 1] * c[i] + a0 * s[i];
          }
          if (turns_b) {
            b[2 * i] = b0 * c[4 + i] - b[2 * i + 1] * s[4 + i];
            b[2 * i + 1] = b[2 * i + 1] * c[4 + i] + b0 * s[4 + i];
          }
        }
      } else if (turns_a) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float a0 = a[i];
          a[i] = a0 * c[i] - b[i] * s[i];
          b[i] = b[i] * c[i] + a0 * s[i];
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ya[i] = E::pack(a[2 * i], a[2 * i + 1]);
        yb[i] = E::pack(b[2 * i], b[2 * i + 1]);
      }
    }
    if (row[r].dst) {
      if (STREAM) {
        __builtin_nontemporal_store(ya, reinterpret_cast<u32x4*>(row[r].dst + ca));
        __builtin_nontemporal_store(yb, reinterpret_cast<u32x4*>(row[r].dst + cb));
      } else {
        st16(row[r].dst + ca, ya);
        st16(row[r].dst + cb, yb);
      }
    }
  }
}

// The same rows with a rotary width that is no multiple of 16 (interleaved: 8), so that a pair's elements lie in other
// lanes (quarters of 80- and 96-wide heads: 20 and 24): a lane holds two adjacent chunks and takes its elements'
// partners, and the table's row, from the LDS. 8192 tokens, 32/8 heads of 80 of which 20 turn, normed, us: 45; the table
// read from memory by each lane 52; the partners too 79; rotary_any_kernel 140.
template <typename T, int LPH>
__global__ __launch_bounds__(256) void rotary_ragged_kernel(RotaryParams p, int32_t head_rows) {
  using E = Elem<T>;
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= p.tokens) return;
  const bool holds = lane % LPH < p.dim / 16;
  const int d0 = holds ? lane % LPH * 16 : 0, half = p.rot / 2;
  const int h = (int)blockIdx.y * (64 / LPH) + lane / LPH;
  HeadRow row = head_row(p, t, min(h, head_rows - 1));
  if (h >= head_rows || !holds) row.dst = nullptr;
  u32x4 x[2] = {ld16(row.src + 2 * d0), ld16(row.src + 2 * d0 + 16)};
  // The token's table row, once for the wave's head rows (p.rot <= p.dim <= 256).
  __shared__ float turns[4][256];
  float* turn = turns[threadIdx.x >> 6];
  float amp;
  const float* row_table = table_row(p, p.positions[t], amp);
  for (int i = lane; i < p.rot; i += 64) turn[i] = row_table[i] * amp;
  float e[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[2 * i] = E::lo(x[i / 4][i % 4]), e[2 * i + 1] = E::hi(x[i / 4][i % 4]);
  if (p.q_weight || p.k_weight) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum = fmaf(e[i], e[i], sum);
    sum = group_sum<LPH>(holds ? sum : 0.f);
    if (row.weight) {
      const float scale = rsqrtf(sum / (float)p.dim + p.eps);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const u32x4 w = ld16(row.weight + 2 * d0 + 16 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[8 * c + 2 * i] *= scale * E::lo(w[i]);
          e[8 * c + 2 * i + 1] *= scale * E::hi(w[i]);
        }
      }
    }
  }
  // 17 floats a lane, so that neighbours' i-th elements lie in different banks. A wave reads what it wrote.
  __shared__ float held[4][64 * 17];
  float* mine = held[threadIdx.x >> 6] + 17 * (lane - lane % LPH);
#pragma unroll
  for (int i = 0; i < 16; ++i) mine[17 * (lane % LPH) + i] = e[i];
  __builtin_amdgcn_wave_barrier();
  if (row.turned && d0 < p.rot) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int d = min(d0 + i, p.rot - 1);
      const bool second = p.interleaved ? d & 1 : d >= half;
      const int pair = p.interleaved ? d / 2 : second ? d - half : d;
      const int other = p.interleaved ? d ^ 1 : second ? pair : d + half;
      const float y = mine[other + other / 16];
      const float c = turn[pair], s = turn[half + pair];
      if (d0 + i < p.rot) e[i] = second ? e[i] * c + y * s : e[i] * c - y * s;
    }
  }
  if (row.turned && (row.weight || d0 < p.rot)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i / 4][i % 4] = E::pack(e[2 * i], e[2 * i + 1]);
  }
  if (row.dst) {
    st16(row.dst + 2 * d0, x[0]);
    st16(row.dst + 2 * d0 + 16, x[1]);
  }
}

template <typename T, int LPH>
static void launch_chunks(const RotaryParams& p, int32_t head_rows, hipStream_t stream) {
  const int32_t rounds = (head_rows + 64 / LPH - 1) / (64 / LPH);
  const uint32_t x = (uint32_t)((p.tokens + 3) / 4);
  if (p.rot % (p.interleaved ? 8 : 16) != 0) {
    hipLaunchKernelGGL((rotary_ragged_kernel<T, LPH>), dim3(x, rounds), dim3(256), 0, stream, p, head_rows);
    return;
  }
  const bool stream_past = (int64_t)p.tokens * head_rows * p.dim * 4 > kStreamBytes;
  auto* const kernel = p.interleaved ? (stream_past ? &rotary_kernel<T, LPH, true, true>
                                                    : &rotary_kernel<T, LPH, true, false>)
                                     : (stream_past ? &rotary_kernel<T, LPH, false, true>
                                                    : &rotary_kernel<T, LPH, false, false>);
  hipLaunchKernelGGL(kernel, dim3(x, (rounds + kRounds - 1) / kRounds), dim3(256), 0, stream, p, head_rows);
}

template <typename T>
static int launch_rotary(const RotaryParams& p, hipStream_t stream) {
  const int32_t head_rows = p.hq + p.hkv * (p.slots ? 2 : 1);
  const int64_t wgs = ((int64_t)p.tokens * head_rows + 3) / 4;
  LV_REQUIRE(fits_one_launch(wgs, 256), "rotary: %d tokens of %d head rows need a grid larger than one launch holds",
             p.tokens, head_rows);
  // Whole 16-byte chunks everywhere (the table's and the weights' alignment does not matter to the ragged kernel).
  bool chunks = p.dim % 16 == 0 && p.dim <= 256 && aligned(p.q, 16) && aligned(p.k, 16) && aligned(p.v, 16) &&
                aligned(p.q_out, 16) && aligned(p.k_out, 16) && aligned(p.v_cache, 16) && aligned(p.q_weight, 16) &&
                aligned(p.k_weight, 16);
  for (int64_t st : {p.q_st, p.q_sh, p.k_st, p.k_sh, p.v_st, p.v_sh, p.qo_st, p.qo_sh, p.ko_st, p.ko_sh, p.c_sb})
    chunks = chunks && st % 16 == 0;
  if (!chunks)
    hipLaunchKernelGGL(rotary_any_kernel<T>, dim3((uint32_t)wgs), dim3(256), 0, stream, p, head_rows);
  else if (p.dim <= 64) launch_chunks<T, 4>(p, head_rows, stream);
  else if (p.dim <= 128) launch_chunks<T, 8>(p, head_rows, stream);
  else launch_chunks<T, 16>(p, head_rows, stream);
  LV_LAUNCH_CHECK("rotary kernel");
  return LV_OK;
}

// What both entry points require of the heads and the table.
static int check_rotary(const char* what, const RotaryParams& p, int64_t max_position, int32_t dtype) {
  LV_REQUIRE(dtype == LV_DTYPE_BF16 || dtype == LV_DTYPE_F16, "%s: dtype %d is not bf16 or fp16", what, dtype);
  LV_REQUIRE(p.tokens >= 0 && p.hq >= 0 && p.hkv >= 0 && p.hq + (int64_t)p.hkv > 0 && p.hq <= (1 << 14) &&
                 p.hkv <= (1 << 14),
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
