// Writing, linking and reading a pool held in 8 bits, on gfx950 (MI355X).
//
// One layer's keys (and values) are codes c[slot][head][d] of e4m3 and bytes
// x[block][head] of e8m0, block = slot / B: a value is c * 2^(x - 127).  The scales
// are powers of two: codes times scale are exact in bf16 (x from 3 to 246) and fp32 (x up
// to 246; beyond, the largest are infinite), and a scale that grows costs the rows under
// it nothing but the bits that fall below e4m3's least number (2^-9 of the scale).
//
// Rows y (computed before any rounding to 8 bits) that a call writes to block b:
//   need = the least byte with max |y| <= 448 * 2^(need - 127), y finite
//   x'   = need where the call writes all of b's rows, else max(x, need)
//   c(written) = e4m3(y * 2^(127 - x')), to nearest even; inf and NaN become NaN
//   c(others)  = e4m3(c * 2^(x - x')) where x' > x
//
// append: y = a new token's key, normed and rotated, and its value.
// link:   y = the value of another row of the pool, a key turned by the angle from
//         its old to its new position: cos = c' c + s' s, sin = s' c - c' s with rows
//         (c, s) of the table at the old and (c', s') at the new position.
//
// A call's rows of one block are neighbours in the call (a run; padding between them
// does not count), so that one wave, or the waves of one workgroup for blocks over 16
// rows, holds them all, one head of the keys or values: their maximum is known before
// the first code is written, and every row is read once.  Keys are turned in 64 bits: a code changes by up to 1/8 of
// itself where a value lies at the border of two, which 32 bits meet some hundred
// times in a call of 32,768 tokens.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>

#include "legolink_kv.h"
#include "ll_internal.h"
#include "quantized_device.h"

namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kWave = 64;
constexpr int kThreads = 256;
constexpr int kMaxDim = 256;
constexpr int kMaxBlock = 128;
constexpr int kMostWindow = 64;
constexpr int kHeldSteps = 2;  // of 64 / kGroup rows, in a wave's registers

int fail(int code, const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  const int rc = ll_record_error(code, fmt, ap);
  va_end(ap);
  return rc;
}

struct Rows {
  const uint16_t *base;
  long long token, head;
};

// One of the pool's two halves.
struct Half {
  uint8_t *codes;  // [slots][heads][dim]
  uint8_t *scales;  // [blocks][heads]
};

struct PoolParams {
  Half key, value;
  const void *slots;  // where the rows go
  unsigned long long *skipped;
  long long num_tokens, num_slots;
  int block_shift, hkv, dim;
  int slots64;
  int window;       // tokens whose runs a workgroup looks for
  int pair_groups;  // workgroups for the heads' keys and values of a window
  unsigned run_groups;  // workgroups of all windows; those of the queries come behind them
  // The table and the keys' positions in it.
  const void *table, *positions, *old_positions;  // (old: of a link)
  long long table_rows, table_stride;
  int table_dtype, rotary, neox, positions64;
  bool table_chunks;  // rows of whole 16-byte chunks
  // append
  Rows query, new_key, new_value;
  uint16_t *query_output;
  long long query_output_token, query_output_head;
  const void *query_weight, *key_weight;
  int weight_dtype, hq, query_steps;
  double eps;
  // link
  const void *sources;
  const uint8_t *masked;
  long long prefix;
};

struct Bf16 {
  __device__ static f32x2 unpack(uint32_t pair) {
    return f32x2{__uint_as_float(pair << 16), __uint_as_float(pair & 0xffff0000u)};
  }
  __device__ static uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
  }
  __device__ static uint32_t decode(uint32_t codes, float scale, bool high) {
    return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true)
                                             : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false));
  }
};
struct F16 {
  __device__ static f32x2 unpack(uint32_t pair) {
    return __builtin_convertvector(__builtin_bit_cast(f16x2, pair), f32x2);
  }
  __device__ static uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, f16x2));
  }
  __device__ static uint32_t decode(uint32_t codes, float scale, bool high) {
    return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, true)
                                             : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, false));
  }
};

__device__ inline long long index_at(const void *values, int is64, long long i) {
  return is64 ? static_cast<const int64_t *>(values)[i] : static_cast<const int32_t *>(values)[i];
}

__device__ inline float value_at(const void *values, int dtype, long long i) {
  if (dtype == LL_DTYPE_FLOAT32) return static_cast<const float *>(values)[i];
  const uint32_t bits = static_cast<const uint16_t *>(values)[i];
  return dtype == LL_DTYPE_BFLOAT16 ? Bf16::unpack(bits)[0] : F16::unpack(bits)[0];
}

// Eight neighbouring values of a table or weight.
__device__ inline void values8(const void *values, int dtype, bool chunks, long long i, float *out) {
  if (!chunks) {
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = value_at(values, dtype, i + j);
  } else if (dtype == LL_DTYPE_FLOAT32) {
    const f32x4 *v = reinterpret_cast<const f32x4 *>(static_cast<const float *>(values) + i);
    const f32x4 lo = v[0], hi = v[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      out[j] = lo[j];
      out[4 + j] = hi[j];
    }
  } else {
    const u32x4 bits = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(values) + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x2 two = dtype == LL_DTYPE_BFLOAT16 ? Bf16::unpack(bits[j]) : F16::unpack(bits[j]);
      out[2 * j] = two[0];
      out[2 * j + 1] = two[1];
    }
  }
}

// A double as a float whose last bit says whether something was lost, so that a
// rounding of it to fewer bits falls where that of the double falls.
__device__ inline float to_odd(double x) {
  unsigned long long bits = __builtin_bit_cast(unsigned long long, x);
  const unsigned long long lost = bits & 0x1fffffffull;
  bits = (bits & ~0x1fffffffull) | (lost != 0 ? 0x20000000ull : 0ull);
  return static_cast<float>(__builtin_bit_cast(double, bits));
}

// A lane's two chunks of a row: its rotary pairs' halves (neox), or neighbours.
struct Lane {
  int i, first, second;
  bool active, rotates;
};
template <int kGroup>
__device__ inline Lane lane_of(const PoolParams &p) {
  Lane l;
  l.i = static_cast<int>(threadIdx.x) % kGroup;
  l.active = l.i < p.dim / 16;
  const int rotary_lanes = p.rotary / 16;
  l.rotates = l.i < rotary_lanes;
  l.first = l.rotates && p.neox ? 8 * l.i : 16 * l.i;
  l.second = l.rotates && p.neox ? 8 * (l.i + rotary_lanes) : 16 * l.i + 8;
  return l;
}

template <typename E>
__device__ inline void load_row(const uint16_t *row, const Lane &l, float *a, float *b) {
  const u32x4 x = *reinterpret_cast<const u32x4 *>(row + l.first), y = *reinterpret_cast<const u32x4 *>(row + l.second);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const f32x2 u = E::unpack(x[j]), v = E::unpack(y[j]);
    a[2 * j] = u[0];
    a[2 * j + 1] = u[1];
    b[2 * j] = v[0];
    b[2 * j + 1] = v[1];
  }
}

__device__ inline bool in_table(const PoolParams &p, long long position) {
  return position >= 0 && position < p.table_rows;
}

// Eight codes as values under a scale, exactly, and values as codes under one.
__device__ inline void decode8(u32x2 codes, float scale, float *out) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const f32x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[j], scale, false);
    const f32x2 hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[j], scale, true);
    out[4 * j] = lo[0];
    out[4 * j + 1] = lo[1];
    out[4 * j + 2] = hi[0];
    out[4 * j + 3] = hi[1];
  }
}
__device__ inline u32x2 encode8(const float *values, float scale) {
  typedef short i16x2 __attribute__((ext_vector_type(2)));
  u32x2 codes;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    i16x2 word = i16x2{0, 0};
    word = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(word, values[4 * j], values[4 * j + 1], scale, false);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(word, values[4 * j + 2], values[4 * j + 3], scale, true);
    codes[j] = __builtin_bit_cast(uint32_t, word);
  }
  return codes;
}

// What a workgroup knows of a token: where it goes (-1: nowhere), where it comes from
// (of a link; -1: it is not written), its position (-1: it is not turned), and a link's
// position before that or an append's place in the call.
struct Token {
  int slot, from, position, origin;
};

// A pair's cosine and sine.
struct Angle {
  double cos, sin;
};

// Four neighbouring values of the table.
__device__ inline void values4(const PoolParams &p, long long i, float *out) {
  if (p.table_chunks && p.table_dtype == LL_DTYPE_FLOAT32) {
    const f32x4 v = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(p.table) + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = v[j];
  } else if (p.table_chunks) {  // (rows of whole 16-byte chunks: four values are at 8 bytes)
    const u32x2 bits = *reinterpret_cast<const u32x2 *>(static_cast<const uint16_t *>(p.table) + i);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f32x2 two = p.table_dtype == LL_DTYPE_BFLOAT16 ? Bf16::unpack(bits[j]) : F16::unpack(bits[j]);
      out[2 * j] = two[0];
      out[2 * j + 1] = two[1];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = value_at(p.table, p.table_dtype, i + j);
  }
}

// The rows of append: a step's new tokens.
template <typename E>
struct NewTokens {
  struct Raw {
    u32x4 x, y;
  };
  static constexpr bool kNorms = true;

  __device__ static Token token(const PoolParams &p, long long t, bool *bad) {
    Token k{-1, -1, -1, -1};
    const long long slot = index_at(p.slots, p.slots64, t), position = index_at(p.positions, p.positions64, t);
    if (slot >= 0 && slot < p.num_slots) k.slot = static_cast<int>(slot);
    k.origin = static_cast<int>(t);
    if (in_table(p, position)) {
      k.position = static_cast<int>(position);
      k.from = k.slot;
    }
    *bad = false;  // (counted with the queries)
    return k;
  }
  __device__ static Raw fetch(const PoolParams &p, const Half &, bool is_key, int head, const Token &k, const Lane &l) {
    const Rows &in = is_key ? p.new_key : p.new_value;
    const uint16_t *row = in.base + k.origin * in.token + head * in.head;
    return Raw{*reinterpret_cast<const u32x4 *>(row + l.first), *reinterpret_cast<const u32x4 *>(row + l.second)};
  }
  __device__ static void unpack(const Raw &raw, float *a, float *b) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x2 u = E::unpack(raw.x[j]), v = E::unpack(raw.y[j]);
      a[2 * j] = u[0];
      a[2 * j + 1] = u[1];
      b[2 * j] = v[0];
      b[2 * j + 1] = v[1];
    }
  }
  // Pairs i to i + 3 of a token.
  __device__ static void angles(const PoolParams &p, const Token &k, int i, Angle *out) {
    float c[4], s[4];
    const long long at = k.position * p.table_stride + i;
    values4(p, at, c);
    values4(p, at + p.rotary / 2, s);
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = Angle{c[j], s[j]};
  }
};

// The rows of a link: the pool's own.
struct CachedRows {
  struct Raw {
    u32x2 x, y;
    float scale;
  };
  static constexpr bool kNorms = false;

  __device__ static Token token(const PoolParams &p, long long t, bool *bad) {
    Token k{-1, -1, -1, -1};
    const long long slot = index_at(p.slots, p.slots64, t), source = index_at(p.sources, p.slots64, t);
    const long long position = index_at(p.positions, p.positions64, t);
    const long long old_position = index_at(p.old_positions, p.positions64, t);
    const bool masked = p.masked != nullptr && p.masked[t] != 0;
    const bool turned = t >= p.prefix;
    const bool there = source >= 0 && source < p.num_slots &&
                       (!turned || (in_table(p, position) && in_table(p, old_position)));
    if (slot >= 0 && slot < p.num_slots) k.slot = static_cast<int>(slot);
    if (there && !masked && k.slot >= 0) {
      k.from = static_cast<int>(source);
      if (turned) {
        k.position = static_cast<int>(position);
        k.origin = static_cast<int>(old_position);
      }
    }
    *bad = !masked && (slot >= p.num_slots || (slot >= 0 && !there));
    return k;
  }
  __device__ static Raw fetch(const PoolParams &p, const Half &half, bool, int head, const Token &k, const Lane &l) {
    const uint8_t *codes = half.codes + (static_cast<long long>(k.from) * p.hkv + head) * p.dim;
    return Raw{*reinterpret_cast<const u32x2 *>(codes + l.first), *reinterpret_cast<const u32x2 *>(codes + l.second),
               scale_of(half.scales[static_cast<long long>(k.from >> p.block_shift) * p.hkv + head])};
  }
  __device__ static void unpack(const Raw &raw, float *a, float *b) {
    decode8(raw.x, raw.scale, a);
    decode8(raw.y, raw.scale, b);
  }
  __device__ static void angles(const PoolParams &p, const Token &k, int i, Angle *out) {
    float c[4], s[4], from_c[4], from_s[4];
    const long long to = k.position * p.table_stride + i, from = k.origin * p.table_stride + i;
    values4(p, to, c);
    values4(p, to + p.rotary / 2, s);
    values4(p, from, from_c);
    values4(p, from + p.rotary / 2, from_s);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      out[j].cos = static_cast<double>(c[j]) * from_c[j] + static_cast<double>(s[j]) * from_s[j];
      out[j].sin = static_cast<double>(s[j]) * from_c[j] - static_cast<double>(c[j]) * from_s[j];
    }
  }
};

__device__ inline float finite_size(float x) {
  const float size = fabsf(x);
  return size < INFINITY ? size : 0.f;  // (and of NaN)
}

// The queries of append: kGroup lanes a head, 64 / kGroup heads of one token a wave.
template <typename E, int kGroup>
__device__ inline void turn_queries(const PoolParams &p, unsigned unit) {
  constexpr int kHeads = kWave / kGroup;
  const int lane = threadIdx.x % kWave;
  const long long t = unit / static_cast<unsigned>(p.query_steps);
  const int step = static_cast<int>(unit % static_cast<unsigned>(p.query_steps));
  if (t >= p.num_tokens) return;
  const Lane l = lane_of<kGroup>(p);
  const int head = step * kHeads + lane / kGroup;
  const bool active = l.active && head < p.hq;
  float a[8], b[8], c[8], s[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = b[j] = 0.f;
  if (active) load_row<E>(p.query.base + t * p.query.token + head * p.query.head, l, a, b);
  const long long position = index_at(p.positions, p.positions64, t);
  const bool turned = in_table(p, position);
  if (step == 0 && lane == 0 && p.skipped != nullptr && (!turned || index_at(p.slots, p.slots64, t) >= p.num_slots))
    atomicAdd(p.skipped, 1ull);
  if (!turned) return;
  if (active && l.rotates) {
    const long long at = position * p.table_stride + 8 * l.i;
    values8(p.table, p.table_dtype, p.table_chunks, at, c);
    values8(p.table, p.table_dtype, p.table_chunks, at + p.rotary / 2, s);
  }
  if (p.query_weight != nullptr) {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += a[j] * a[j] + b[j] * b[j];
#pragma unroll
    for (int lanes_apart = 1; lanes_apart < kGroup; lanes_apart *= 2) sum += __shfl_xor(sum, lanes_apart);
    if (active) {
      const float scale = rsqrtf(sum / static_cast<float>(p.dim) + static_cast<float>(p.eps));
      float w[8];
      values8(p.query_weight, p.weight_dtype, true, l.first, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = a[j] * scale * w[j];
      values8(p.query_weight, p.weight_dtype, true, l.second, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) b[j] = b[j] * scale * w[j];
    }
  }
  if (!active) return;
  if (l.rotates && p.neox) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float lo = a[j], hi = b[j];
      a[j] = lo * c[j] - hi * s[j];
      b[j] = hi * c[j] + lo * s[j];
    }
  } else if (l.rotates) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a0 = a[2 * j], a1 = a[2 * j + 1], b0 = b[2 * j], b1 = b[2 * j + 1];
      a[2 * j] = a0 * c[j] - a1 * s[j];
      a[2 * j + 1] = a1 * c[j] + a0 * s[j];
      b[2 * j] = b0 * c[4 + j] - b1 * s[4 + j];
      b[2 * j + 1] = b1 * c[4 + j] + b0 * s[4 + j];
    }
  }
  u32x4 out_a, out_b;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    out_a[j] = E::pack(a[2 * j], a[2 * j + 1]);
    out_b[j] = E::pack(b[2 * j], b[2 * j + 1]);
  }
  uint16_t *dst = p.query_output + t * p.query_output_token + head * p.query_output_head;
  *reinterpret_cast<u32x4 *>(dst + l.first) = out_a;
  *reinterpret_cast<u32x4 *>(dst + l.second) = out_b;
}

template <typename E, int kGroup>
__global__ void __launch_bounds__(kThreads) quantized_query_kernel(const PoolParams p) {
  turn_queries<E, kGroup>(p, blockIdx.x * (kThreads / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave));
}

// Bits of rows: of up to 32 (kWords 0), 64 or 128.
template <int kWords>
struct RowBits {
  unsigned long long low, high;  // (members, not an array: the compiler would index it in memory)

  __device__ void set(int word, unsigned long long bits) {
    if (word == 0) low = bits;
    else high = bits;
  }
  __device__ static unsigned long long up_to(int bit) { return (2ull << bit) - 1; }
  __device__ bool at(int row) const {
    const unsigned shifted_low = static_cast<unsigned>(low >> (row % kWave)) & 1u;
    if (kWords == 1) return shifted_low != 0;
    const unsigned shifted_high = static_cast<unsigned>(high >> (row % kWave)) & 1u;
    return (row >= kWave ? shifted_high : shifted_low) != 0;
  }
  // The last one up to `row` (0: none).
  __device__ int last_to(int row) const {
    const unsigned long long in_low = kWords > 1 && row >= kWave ? low : low & up_to(row % kWave);
    const unsigned long long in_high = kWords > 1 && row >= kWave ? high & up_to(row % kWave) : 0ull;
    if (in_high != 0) return 2 * kWave - 1 - __builtin_clzll(in_high);
    return in_low == 0 ? 0 : kWave - 1 - __builtin_clzll(in_low);
  }
  // The first one from `row` on (64 kWords: none).
  __device__ int first_from(int row) const {
    const unsigned long long in_low = row >= kWave ? 0ull : low & (~0ull << row);
    if (in_low != 0) return __builtin_ctzll(in_low);
    if (kWords == 1) return kWave;
    const unsigned long long in_high = row >= 2 * kWave ? 0ull : row <= kWave ? high : high & (~0ull << (row - kWave));
    return in_high == 0 ? 2 * kWave : kWave + __builtin_ctzll(in_high);
  }
  // How many of [begin, end).
  __device__ int count(int begin, int end) const {
    return (begin >= end) ? 0 : below(end) - below(begin);
  }
  __device__ int below(int end) const {
    int sum = __builtin_popcountll(end >= kWave ? low : low & ((1ull << end) - 1));
    if (kWords > 1 && end > kWave) sum += __builtin_popcountll(end >= 2 * kWave ? high : high & ((1ull << (end - kWave)) - 1));
    return sum;
  }
};

template <>
struct RowBits<0> {
  uint32_t word;

  __device__ void set(int, unsigned long long bits) { word = static_cast<uint32_t>(bits); }
  __device__ bool at(int row) const { return ((word >> row) & 1u) != 0; }
  __device__ int last_to(int row) const {
    const uint32_t low = word & ((2u << row) - 1u);
    return low == 0 ? 0 : 31 - __builtin_clz(low);
  }
  __device__ int first_from(int row) const {
    const uint32_t low = row >= 32 ? 0u : word & (~0u << row);
    return low == 0 ? 32 : __builtin_ctz(low);
  }
  __device__ int count(int begin, int end) const {
    if (begin >= end) return 0;
    return __builtin_popcount((word >> begin) & (~0u >> (32 - (end - begin))));
  }
};

// Waves a SIMD that the registers leave room for: what reads most latency away for few
// spilled registers (32,768 tokens linked in blocks of 16: 39 us with four, 44 with
// three; 8,192 in blocks of 128 29 and 36, but 8,192 appended with norms 75 and 63).
template <typename Source>
constexpr int least_waves(int parts) {
  return parts <= 2 || (parts == 8 && !Source::kNorms) ? 4 : parts <= 8 ? 3 : 1;
}

// The tokens that have a slot, moved together over the padding between them: tokens[1]
// on are then the window's, behind them the others up to the end of the last one's run
// (as far as a workgroup holds), tokens[0] the last one in front of the window.  Padding
// may be of any length, so the call is searched both ways, kLooks tokens a lane at a time
// (64 single tokens padded to 2,048 at their end: 11.4 us, 3 of them for this; in 64
// places one gap in the middle costs 1.4).  Of one wave; returns how many of the window's
// there are (at least one).
template <typename Source, int kRunRows>
__device__ inline int pack_tokens(const PoolParams &p, long long t0, Token *tokens) {
  constexpr int kLooks = 8;
  const int lane = threadIdx.x % kWave;
  // The first of kLooks * 64 tokens from `at` on (or back) that has a slot; that many: none.
  auto first_of = [&](long long at, int step) {
    auto place = [&](int i) { return at + step * (i * kWave + lane); };
    auto exists = [&](int i) { return place(i) >= 0 && place(i) < p.num_tokens; };
    long long slot[kLooks];  // (of one type a branch: all loads in flight)
    if (p.slots64 != 0) {
#pragma unroll
      for (int i = 0; i < kLooks; ++i) slot[i] = index_at(p.slots, 1, exists(i) ? place(i) : 0);
    } else {
#pragma unroll
      for (int i = 0; i < kLooks; ++i) slot[i] = index_at(p.slots, 0, exists(i) ? place(i) : 0);
    }
    int first = kLooks * kWave;
#pragma unroll
    for (int i = kLooks - 1; i >= 0; --i) {
      const unsigned long long there = __builtin_amdgcn_ballot_w64(exists(i) && slot[i] >= 0 && slot[i] < p.num_slots);
      if (there != 0) first = i * kWave + __builtin_ctzll(there);
    }
    return first;
  };
  // Those of `taken` to the places behind `to` (never past their own).
  auto move = [&](const Token &k, unsigned long long taken, int to, int last) {
    const int place = to + 1 + __builtin_popcountll(taken & ((1ull << lane) - 1));
    if (((taken >> lane) & 1ull) != 0 && place <= last) tokens[place] = k;
  };
  const Token own = tokens[1 + min(lane, p.window - 1)];
  const unsigned long long of_window = __builtin_amdgcn_ballot_w64(lane < p.window && own.slot >= 0);
  const int count = __builtin_popcountll(of_window), last = count + kRunRows;
  if (tokens[0].slot < 0) {
    for (long long at = t0 - 1; at >= 0; at -= kLooks * kWave) {
      const int first = first_of(at, -1);
      if (first == kLooks * kWave) continue;
      if (lane == 0) tokens[0].slot = static_cast<int>(index_at(p.slots, p.slots64, at - first));
      break;
    }
  }
  move(own, of_window, 0, count);
  const int block = __builtin_amdgcn_readlane(own.slot, kWave - 1 - __builtin_clzll(of_window)) >> p.block_shift;
  int held = count;
  bool ended = false;  // the run; its end is the first token of another block
  auto take = [&](const Token &k, bool exists) {
    unsigned long long taken = __builtin_amdgcn_ballot_w64(exists && k.slot >= 0);
    const unsigned long long others = __builtin_amdgcn_ballot_w64(exists && k.slot >= 0 && k.slot >> p.block_shift != block);
    if (others != 0) taken &= others ^ (others - 1);  // (up to the first one)
    move(k, taken, held, last);
    held = min(held + static_cast<int>(__builtin_popcountll(taken)), last);
    ended = others != 0 || held == last;
  };
  for (int i = p.window + 1; !ended && i <= p.window + kRunRows; i += kWave)
    take(tokens[min(i + lane, p.window + kRunRows)], i + lane <= p.window + kRunRows);
  for (long long t = t0 + p.window + kRunRows + 1; !ended && t < p.num_tokens;) {
    const int first = first_of(t, 1);
    t += first;
    if (first == kLooks * kWave) continue;
    Token k{-1, -1, -1, -1};
    bool bad;
    if (t + lane < p.num_tokens) k = Source::token(p, t + lane, &bad);
    take(k, t + lane < p.num_tokens);
    t += kWave;
  }
  for (int i = held + 1 + lane; i <= last; i += kWave) tokens[i] = Token{-1, -1, -1, -1};
  return count;
}

// Writes runs of rows.  A pair is one head's keys or values; kParts waves of a
// workgroup hold up to kRunRows rows of it at a time, two steps of 64 / kGroup rows
// each: as many of the window's runs as fit whole (one of a prompt's blocks, or many
// single tokens').
//
// A call is bound by memory, or for few rows by the chain slot -> row and angle -> code.
// So what there is to know of the window's tokens is read at once, each row's loads do
// not wait for its angles, and the rows' angles are made once for the workgroup's heads
// and kept in LDS (a link's are four table rows' worth of products; every head by
// itself would read 1 KB of table for 256 bytes of codes).  LDS has the angles of
// lane i's pair j as element 9 R row + R j + i, R = rotary lanes of a row, so that 16
// lanes' 16-byte reads meet every bank once.
//
// 4 heads of 128 in blocks of 16: 32,768 tokens linked 37 us (100 MB with the table's
// rows, 2.7 TB/s: the vector units are busy for more than half of it, the rest is what
// four waves a SIMD leave of the latencies), 1,024 6.8 us; 16,384 tokens' keys and
// values appended 33 us, 64 single tokens 6.2 us.
template <typename Source, typename E, int kGroup, int kParts, bool kQueries>
__global__ void __launch_bounds__(kParts > 4 ? kParts * kWave : kThreads, least_waves<Source>(kParts))
    quantized_write_kernel(const PoolParams p) {
  constexpr int kWaves = kParts > 4 ? kParts : kThreads / kWave;
  constexpr int kPairs = kWaves / kParts;  // of a workgroup
  constexpr int kRows = kWave / kGroup;    // of a step
  constexpr int kSteps = kHeldSteps;
  constexpr int kHeldRows = kSteps * kRows;  // of a wave
  constexpr int kRunRows = kParts * kHeldRows;
  constexpr int kWords = (kRunRows + kWave - 1) / kWave;
  static_assert(kRunRows <= kMaxBlock, "RowBits holds two words, and no block has more rows");
  constexpr bool kShares = kPairs > 1;
  constexpr int kTokens = 1 + kMostWindow + kRunRows;  // the one before the window, the window, a run from its last on
  typedef RowBits<kRunRows <= 32 ? 0 : kWords> Bits;
  __shared__ unsigned most_of[kPairs][kRunRows];  // of a run, at its first row: a float's bits
  __shared__ Token tokens[kTokens];
  __shared__ int packed;
  __shared__ Angle shared_angles[kShares ? kRunRows * 9 * kGroup : 1];
  __shared__ float key_weights[Source::kNorms ? 16 * kGroup : 1];
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int lane = threadIdx.x % kWave;
  const unsigned group = blockIdx.x;
  if constexpr (kQueries) {
    // (The runs, which take longer, come first.)
    if (group >= p.run_groups) {
      turn_queries<E, kGroup>(p, (group - p.run_groups) * kWaves + wave);
      return;
    }
  }
  const unsigned window = group / static_cast<unsigned>(p.pair_groups);
  const int pair_group = static_cast<int>(group % static_cast<unsigned>(p.pair_groups));
  const long long t0 = static_cast<long long>(window) * p.window - 1;  // of tokens[0]
  const int own_pair = wave / kParts;  // of the workgroup's
  const int pair = pair_group * kPairs + own_pair;
  const int part = wave % kParts;
  const bool has_pair = pair < 2 * p.hkv;
  const bool is_key = pair < p.hkv;
  const int head = is_key ? pair : pair - p.hkv;
  const Half half = is_key ? p.key : p.value;
  const int block_rows = 1 << p.block_shift;
  const Lane l = lane_of<kGroup>(p);

  for (int i = threadIdx.x; i < 1 + p.window + kRunRows; i += kWaves * kWave) {
    Token k{-1, -1, -1, -1};
    bool bad = false;
    if (t0 + i >= 0 && t0 + i < p.num_tokens) k = Source::token(p, t0 + i, &bad);
    tokens[i] = k;
    if (bad && i >= 1 && i <= p.window && pair_group == 0 && p.skipped != nullptr) atomicAdd(p.skipped, 1ull);
  }
  if constexpr (Source::kNorms)
    for (int i = threadIdx.x; i < p.dim; i += kWaves * kWave)
      key_weights[i] = p.key_weight != nullptr ? value_at(p.key_weight, p.weight_dtype, i) : 1.f;
  __syncthreads();
  int own_tokens = p.window;
  {
    const int exist = static_cast<int>(min(p.num_tokens - t0, static_cast<long long>(1 + p.window + kRunRows)));
    const int begin = t0 < 0 ? 1 : 0;
    int least = 0;  // (every wave reads all of them, at once)
#pragma unroll
    for (int i = 0; i < kTokens; i += kWave) least = min(least, tokens[max(begin, min(i + lane, exist - 1))].slot);
    if (__builtin_amdgcn_ballot_w64(least < 0) != 0) {
      // It matters where a token may follow that belongs to the runs that begin here:
      // not behind the first one of another block than the window's last, or at the end.
      const int last_block = tokens[p.window].slot >> p.block_shift;
      unsigned long long owns = 0;
      int first_gap = kTokens, run_end = kTokens, last_there = -1;
#pragma unroll
      for (int i = 0; i < kTokens; i += kWave) {
        const int at = i + lane, slot = tokens[min(at, exist - 1)].slot;
        const bool in = at >= begin && at < exist;
        const unsigned long long gaps = __builtin_amdgcn_ballot_w64(in && slot < 0);
        const unsigned long long there = __builtin_amdgcn_ballot_w64(in && slot >= 0);
        const unsigned long long others =
            __builtin_amdgcn_ballot_w64(in && slot >= 0 && at > p.window && slot >> p.block_shift != last_block);
        owns |= __builtin_amdgcn_ballot_w64(in && slot >= 0 && at >= 1 && at <= p.window);
        if (first_gap == kTokens && gaps != 0) first_gap = i + __builtin_ctzll(gaps);
        if (run_end == kTokens && others != 0) run_end = i + __builtin_ctzll(others);
        if (there != 0) last_there = i + kWave - 1 - __builtin_clzll(there);
      }
      if (owns == 0) return;
      if (first_gap < run_end && (last_there > first_gap || t0 + exist < p.num_tokens)) {
        __syncthreads();
        if (wave == 0) {
          const int count = pack_tokens<Source, kRunRows>(p, t0, tokens);
          if (lane == 0) packed = count;
        }
        __syncthreads();
        own_tokens = __builtin_amdgcn_readfirstlane(packed);
      }
    }
  }
  auto block_of = [&](int i) { return tokens[i].slot < 0 ? -1 : tokens[i].slot >> p.block_shift; };
  // A run begins where the block changes.  Bit l: token 1 + l of those here.
  unsigned long long begins;
  {
    const int block = block_of(1 + min(lane, own_tokens - 1));
    begins = __builtin_amdgcn_ballot_w64(lane < own_tokens && block >= 0 && block != block_of(min(lane, own_tokens - 1)));
  }
  while (begins != 0) {
    const int first = 1 + __builtin_ctzll(begins);  // token of row 0
    // The rows from there on: those of a block, those that begin a run, those written.
    Bits member, begin, written, bounds;  // (bounds: those that belong to no run before them)
    int stop = kRunRows;  // behind the last run that begins in the window
    bool ends = true;     // row kRunRows, too, is of another run
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      const int row = min(w * kWave + lane, kRunRows - 1);
      const bool exists = w * kWave + lane < kRunRows;
      const int block = block_of(first + row);
      const bool starts = block >= 0 && (row == 0 || block != block_of(first + row - 1));
      member.set(w, __builtin_amdgcn_ballot_w64(exists && block >= 0));
      begin.set(w, __builtin_amdgcn_ballot_w64(exists && starts));
      written.set(w, __builtin_amdgcn_ballot_w64(exists && tokens[first + row].from >= 0));
      bounds.set(w, __builtin_amdgcn_ballot_w64(exists && (starts || block < 0)));
      const unsigned long long out =
          __builtin_amdgcn_ballot_w64(exists && first + row > own_tokens && (starts || block < 0));
      if (stop == kRunRows && out != 0) stop = w * kWave + __builtin_ctzll(out);
    }
    {
      const int next = block_of(first + kRunRows), last = block_of(first + kRunRows - 1);
      ends = next < 0 || next != last;
    }
    // (A run that goes on past the last row is left to the next turn, unless it is the
    // only one: blocks have no more than kRunRows rows.)
    if (stop == kRunRows && !ends) {
      const int last = begin.last_to(kRunRows - 1);
      if (last > 0) stop = last;
    }
    begins = first - 1 + stop >= kWave ? 0ull : begins & (~0ull << (first - 1 + stop));
    auto end_of = [&](int row) { return min(bounds.first_from(row + 1), stop); };  // of the run of a row

    // Lane r: row r's run and its scale.
    unsigned old[kWords];
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      const int row = w * kWave + lane;
      old[w] = 0u;
      if (has_pair && row < stop && member.at(row))
        old[w] = half.scales[static_cast<long long>(block_of(first + row)) * p.hkv + head];
    }
    if (part == 0)
      for (int row = lane; row < kRunRows; row += kWave) most_of[own_pair][row] = 0u;

    auto held_of = [&](int step) { return part * kHeldRows + step * kRows + lane / kGroup; };
    auto token_of = [&](int step) { return first + held_of(step); };
    bool has[kSteps];
    typename Source::Raw raw[kSteps];
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
      has[step] = has_pair && l.active && held_of(step) < stop && written.at(held_of(step));
      raw[step] = typename Source::Raw{};
      if (has[step]) raw[step] = Source::fetch(p, half, is_key, head, tokens[token_of(step)], l);
    }
    const int lanes = p.rotary / 16;
    if constexpr (kShares) {
      if (pair_group * kPairs < p.hkv) {  // (keys among its pairs)
        const int quads = 2 * lanes;      // of four pairs, a row's
        for (int i = threadIdx.x; i < stop * quads; i += kWaves * kWave) {
          const int row = i / quads, quad = i - row * quads;
          if (!written.at(row) || tokens[first + row].position < 0) continue;
          Angle four[4];
          Source::angles(p, tokens[first + row], 4 * quad, four);
#pragma unroll
          for (int j = 0; j < 4; ++j) shared_angles[(9 * row + 4 * (quad % 2) + j) * lanes + quad / 2] = four[j];
        }
      }
    }
    __syncthreads();
    float a[kSteps][8], b[kSteps][8];
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
      if (__builtin_amdgcn_ballot_w64(has[step]) == 0) continue;
      Source::unpack(raw[step], a[step], b[step]);
      if (is_key) {
        const bool normed = Source::kNorms && p.key_weight != nullptr;
        double scale = 1.0;
        if (normed) {
          double sum = 0.0;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            sum += static_cast<double>(a[step][j]) * a[step][j];
            sum += static_cast<double>(b[step][j]) * b[step][j];
          }
#pragma unroll
          for (int apart = 1; apart < kGroup; apart *= 2) sum += __shfl_xor(sum, apart);
          scale = 1.0 / sqrt(sum / static_cast<double>(p.dim) + p.eps);
        }
        const Token &k = tokens[token_of(step)];
        const bool turns = has[step] && l.rotates && k.position >= 0;
        Angle made[kShares ? 1 : 8];
        const Angle *from = shared_angles + 9 * held_of(step) * lanes + l.i;
        if constexpr (!kShares) {
          if (turns) {
            Source::angles(p, k, 8 * l.i, made);
            Source::angles(p, k, 8 * l.i + 4, made + 4);
          }
        }
        // A pair of dims, at these places of the row: normed, turned and rounded.
        auto pair_of = [&](int j, float &one, float &two, int at, int other, bool turned) {
          double x = one, y = two;
          if (Source::kNorms) {  // (weights of 1 under a scale of 1 without a norm)
            x = x * scale * key_weights[at];
            y = y * scale * key_weights[other];
          }
          if (turned) {
            const Angle angle = kShares ? from[j * lanes] : made[kShares ? 0 : j];
            const double lo = x, hi = y;
            x = lo * angle.cos - hi * angle.sin;
            y = hi * angle.cos + lo * angle.sin;
          }
          one = to_odd(x);
          two = to_odd(y);
          if (j % 2 == 1) __builtin_amdgcn_sched_barrier(0);  // (few doubles at a time)
        };
        if (turns && p.neox != 0) {
#pragma unroll
          for (int j = 0; j < 8; ++j) pair_of(j, a[step][j], b[step][j], l.first + j, l.second + j, true);
        } else if (turns || normed) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int at = 2 * j;
            if (turns) {
              pair_of(j, a[step][at], a[step][at + 1], l.first + at, l.first + at + 1, true);
              pair_of(4 + j, b[step][at], b[step][at + 1], l.second + at, l.second + at + 1, true);
            } else {
              pair_of(j, a[step][at], a[step][at + 1], l.first + at, l.first + at + 1, false);
              pair_of(4 + j, b[step][at], b[step][at + 1], l.second + at, l.second + at + 1, false);
            }
          }
        }
      }
      float most = 0.f;
      if (has[step]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) most = fmaxf(fmaxf(most, fabsf(a[step][j])), fabsf(b[step][j]));  // (NaN left out)
        if (!(most < INFINITY)) {  // (rare: infinities left out, too)
          most = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) most = fmaxf(most, fmaxf(finite_size(a[step][j]), finite_size(b[step][j])));
        }
      }
#pragma unroll
      for (int apart = 1; apart < kGroup; apart *= 2) most = fmaxf(most, __shfl_xor(most, apart));
      if (has[step] && l.i == 0)
        atomicMax(&most_of[own_pair][begin.last_to(held_of(step))], __float_as_uint(most));
    }
#pragma unroll
    for (int w = 0; w < kWords; ++w) asm volatile("" : "+v"(old[w]));  // read before another wave may write it
    if constexpr (kParts > 1) __syncthreads();
    unsigned byte[kWords];
    Bits grown;
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      const int row = min(w * kWave + lane, kRunRows - 1);
      const bool exists = has_pair && w * kWave + lane < stop && member.at(row);
      const int from = begin.last_to(row);
      const int count = exists ? written.count(from, end_of(row)) : 0;
      const unsigned need = byte_for(__uint_as_float(most_of[own_pair][from]));
      byte[w] = count == 0 ? old[w] : count == block_rows ? need : max(old[w], need);
      if (exists && part == 0 && row == from && byte[w] != old[w])
        half.scales[static_cast<long long>(block_of(first + row)) * p.hkv + head] = static_cast<uint8_t>(byte[w]);
      grown.set(w, __builtin_amdgcn_ballot_w64(exists && row == from && count < block_rows && byte[w] > old[w]));
    }
    auto of_row = [&](const unsigned *values, int row) {  // lane r's value
      unsigned value = static_cast<unsigned>(__shfl(static_cast<int>(values[0]), row % kWave));
      if (kWords > 1) {
        const unsigned high = static_cast<unsigned>(__shfl(static_cast<int>(values[kWords - 1]), row % kWave));
        value = row >= kWave ? high : value;
      }
      return value;
    };
    auto codes_at = [&](int slot) { return half.codes + (static_cast<long long>(slot) * p.hkv + head) * p.dim; };
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
      const float scale = scale_of(of_row(byte, held_of(step)));
      if (!has[step]) continue;
      uint8_t *dst = codes_at(tokens[token_of(step)].slot);
      *reinterpret_cast<u32x2 *>(dst + l.first) = encode8(a[step], scale);
      *reinterpret_cast<u32x2 *>(dst + l.second) = encode8(b[step], scale);
    }
    // The other rows of blocks whose scale has grown.
    for (int run = grown.first_from(0); run < kRunRows; run = grown.first_from(run + 1)) {
      const int run_end = end_of(run), block = block_of(first + run);
      unsigned long long offsets[kWords];  // that are written
#pragma unroll
      for (int w = 0; w < kWords; ++w) offsets[w] = 0;
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        const int row = w * kWave + lane;
        const bool own = row >= run && row < run_end && written.at(min(row, kRunRows - 1));
        const int offset = own ? tokens[first + min(row, kRunRows - 1)].slot & (block_rows - 1) : 0;
#pragma unroll
        for (int v = 0; v < kWords; ++v) {
          unsigned long long bits = own && offset / kWave == v ? 1ull << (offset % kWave) : 0ull;
#pragma unroll
          for (int apart = 1; apart < kWave; apart *= 2) bits |= __shfl_xor(bits, apart);
          offsets[v] |= bits;
        }
      }
      Bits taken;
#pragma unroll
      for (int w = 0; w < kWords; ++w) taken.set(w, offsets[w]);
      const unsigned rise = of_row(byte, run) - of_row(old, run);
      const float ratio = rise < 127u ? __uint_as_float((127u - rise) << 23) : 0.f;
      u32x2 others[kSteps][2];
      auto is_other = [&](int step) {
        const int offset = held_of(step);
        return offset < block_rows && l.active && !taken.at(min(offset, kRunRows - 1));
      };
      auto other_at = [&](int step) { return codes_at((block << p.block_shift) + held_of(step)); };
#pragma unroll
      for (int step = 0; step < kSteps; ++step)
        if (is_other(step)) {
          others[step][0] = *reinterpret_cast<const u32x2 *>(other_at(step) + l.first);
          others[step][1] = *reinterpret_cast<const u32x2 *>(other_at(step) + l.second);
        }
#pragma unroll
      for (int step = 0; step < kSteps; ++step)
        if (is_other(step)) {
          float values[8];
          decode8(others[step][0], ratio, values);
          *reinterpret_cast<u32x2 *>(other_at(step) + l.first) = encode8(values, 1.f);
          decode8(others[step][1], ratio, values);
          *reinterpret_cast<u32x2 *>(other_at(step) + l.second) = encode8(values, 1.f);
        }
    }
    if (begins != 0) __syncthreads();  // (the next rows take most_of and the angles)
  }
}

// Rows of the pool in 16 or 32 bits: a lane takes chunks of eight codes, several in
// flight, of the workgroup's tokens.  40,960 rows of 4 heads of 128 in bf16: 20 us,
// 6.2 TB/s read and written (codes from the memory-side cache); 701 rows 3.9 us.
struct LoadParams {
  const uint8_t *key, *value, *key_scales, *value_scales;
  void *key_output, *value_output;  // [tokens][heads][dim]
  const void *slots;                // NULL: the pool's own order
  long long num_slots, num_rows;
  int slots64, block_shift, hkv, dim_chunks, row_chunks, dtype;
  int group_rows;  // of a workgroup
};
constexpr int kLoadChunks = 4;

__global__ void __launch_bounds__(kThreads) quantized_load_kernel(const LoadParams p) {
  const bool is_key = blockIdx.y == 0;
  const uint8_t *codes = is_key ? p.key : p.value, *scales = is_key ? p.key_scales : p.value_scales;
  const long long t0 = static_cast<long long>(blockIdx.x) * p.group_rows;
  const unsigned row_chunks = static_cast<unsigned>(p.row_chunks);
  const unsigned total = static_cast<unsigned>(min(static_cast<long long>(p.group_rows), p.num_rows - t0)) * row_chunks;
  const long long first = t0 * p.row_chunks;  // of the outputs' chunks
  void *output = is_key ? p.key_output : p.value_output;
  for (unsigned begin = threadIdx.x; begin < total; begin += kThreads * kLoadChunks) {
    u32x2 bits[kLoadChunks];
    unsigned byte[kLoadChunks];
#pragma unroll
    for (int k = 0; k < kLoadChunks; ++k) {
      const unsigned c = begin + k * kThreads;
      bits[k] = u32x2{0u, 0u};
      byte[k] = 0;
      if (c >= total) continue;
      const unsigned row = c / row_chunks, within = c - row * row_chunks;
      const long long slot = p.slots == nullptr ? t0 + row : index_at(p.slots, p.slots64, t0 + row);
      if (slot < 0 || slot >= p.num_slots) continue;  // a row of zeros
      bits[k] = *reinterpret_cast<const u32x2 *>(codes + (slot * p.row_chunks + within) * 8);
      byte[k] = scales[(slot >> p.block_shift) * p.hkv + within / static_cast<unsigned>(p.dim_chunks)];
    }
#pragma unroll
    for (int k = 0; k < kLoadChunks; ++k) {
      const unsigned c = begin + k * kThreads;
      if (c >= total) continue;
      const float scale = scale_of(byte[k]);
      if (p.dtype == LL_DTYPE_FLOAT32) {
        float values[8];
        decode8(bits[k], scale, values);
        f32x4 *dst = reinterpret_cast<f32x4 *>(output) + 2 * (first + c);
        dst[0] = f32x4{values[0], values[1], values[2], values[3]};
        dst[1] = f32x4{values[4], values[5], values[6], values[7]};
      } else {
        u32x4 out;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            out[2 * j + h] = p.dtype == LL_DTYPE_BFLOAT16 ? Bf16::decode(bits[k][j], scale, h != 0)
                                                          : F16::decode(bits[k][j], scale, h != 0);
        reinterpret_cast<u32x4 *>(output)[first + c] = out;
      }
    }
  }
}

bool aligned(const void *p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
bool float_code(int64_t dtype) {
  return dtype == LL_DTYPE_FLOAT16 || dtype == LL_DTYPE_BFLOAT16 || dtype == LL_DTYPE_FLOAT32;
}
bool index_code(int64_t dtype) { return dtype == LL_DTYPE_INT32 || dtype == LL_DTYPE_INT64; }

int check_pool(const ll_quantized_pool *pool) {
  if (pool->scale_block < 1 || pool->scale_block > kMaxBlock || (pool->scale_block & (pool->scale_block - 1)) != 0)
    return fail(LL_ERR_INVALID_ARGUMENT, "scale_block must be a power of two, at most %d", kMaxBlock);
  if (pool->num_slots < 0 || pool->num_slots > 0x7fffffff || pool->num_slots % pool->scale_block != 0)
    return fail(LL_ERR_INVALID_ARGUMENT, "num_slots must be whole blocks, below 2^31");
  if (pool->num_kv_heads < 1 || pool->num_kv_heads > 65535)
    return fail(LL_ERR_KV_HEAD_LAYOUT_MISMATCH, "num_kv_heads must be in [1, 65535]");
  if (pool->head_dim < 16 || pool->head_dim > kMaxDim || pool->head_dim % 16 != 0)
    return fail(LL_ERR_HEAD_DIMENSION_OUT_OF_RANGE, "head_dim must be a multiple of 16, at most %d", kMaxDim);
  if (pool->num_slots > 0 && (pool->key_buffer == nullptr || pool->value_buffer == nullptr ||
                              pool->key_scales == nullptr || pool->value_scales == nullptr))
    return fail(LL_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
  if (!aligned(pool->key_buffer, 16) || !aligned(pool->value_buffer, 16))
    return fail(LL_ERR_INVALID_ARGUMENT, "the pool's buffers must be 16-byte aligned");
  return LL_OK;
}

int check_table(int64_t dtype, int64_t rows, int64_t cols, int64_t stride, int64_t rotary, int64_t dim) {
  if (rotary < 2 || rotary % 2 != 0) return fail(LL_ERR_EVEN_ROTARY_DIM_REQUIRED, "rotary_dim must be positive and even");
  if (rotary > dim) return fail(LL_ERR_ROTARY_DIM_EXCEEDS_HEAD_DIM, "rotary_dim exceeds head_dim");
  if (rotary % 16 != 0) return fail(LL_ERR_INVALID_ARGUMENT, "rotary_dim must be a multiple of 16");
  if (!float_code(dtype)) return fail(LL_ERR_UNSUPPORTED_COS_SIN_DTYPE, "cos/sin dtype");
  if (rows < 0 || rows > 0x7fffffff || cols < rotary || stride < 0)
    return fail(LL_ERR_UNSUPPORTED_COS_SIN_CACHE, "the cos/sin table needs rotary_dim columns");
  return LL_OK;
}

bool whole_chunks(const void *base, int64_t token, int64_t head) {
  return aligned(base, 16) && token % 8 == 0 && head % 8 == 0;
}

void fill_pool(const ll_quantized_pool &pool, PoolParams *p) {
  p->key = Half{static_cast<uint8_t *>(pool.key_buffer), static_cast<uint8_t *>(pool.key_scales)};
  p->value = Half{static_cast<uint8_t *>(pool.value_buffer), static_cast<uint8_t *>(pool.value_scales)};
  p->num_slots = pool.num_slots;
  p->hkv = static_cast<int>(pool.num_kv_heads);
  p->dim = static_cast<int>(pool.head_dim);
  p->block_shift = 0;
  while ((1ll << p->block_shift) < pool.scale_block) ++p->block_shift;
}

void fill_table(const void *table, int64_t dtype, int64_t rows, int64_t stride, int64_t rotary, bool neox,
                PoolParams *p) {
  p->table = table;
  p->table_dtype = static_cast<int>(dtype);
  p->table_rows = rows;
  p->table_stride = stride;
  p->rotary = static_cast<int>(rotary);
  p->neox = neox ? 1 : 0;
  p->table_chunks = aligned(table, 16) && stride * (dtype == LL_DTYPE_FLOAT32 ? 4 : 2) % 16 == 0;
}

template <typename Source, typename E, int kGroup, int kParts, bool kQueries>
int launch_write(PoolParams &p, hipStream_t s) {
  constexpr int kWaves = kParts > 4 ? kParts : kThreads / kWave;
  constexpr int kPairs = kWaves / kParts;
  p.pair_groups = (2 * p.hkv + kPairs - 1) / kPairs;
  // A window's runs share a workgroup's turns.  It is as wide as a block (a prompt's
  // runs then begin in one window each), or less where that makes fewer waves than one
  // a SIMD (1,024 tokens linked: 7.0 us, and 10.7 with four waves a SIMD).
  const long long waves = p.num_tokens * 2 * p.hkv * kParts;
  const int widest = std::min(kMostWindow, std::max(16, 1 << p.block_shift));
  p.window = 1;
  while (p.window < widest && waves / p.window > 256 * 4) p.window *= 2;
  const long long run_groups = (p.num_tokens + p.window - 1) / p.window * p.pair_groups;
  p.run_groups = static_cast<unsigned>(std::min(run_groups, 0xffffffffll));
  const long long query_waves = p.num_tokens * p.query_steps;
  // The queries of a small call go with its runs in one launch.  Those of a large one
  // are bound by memory, and go by themselves: the runs' registers leave room for three
  // or four waves a SIMD.  28/4 heads of 128, blocks of 16: 4,096 tokens (16,384 waves
  // of queries) 23 us together and 32 apart, 8,192 44 and 48, 16,384 95 and 85; blocks
  // of 64: 4,096 tokens 20 and 25, 8,192 49 and 46.
  const bool together = kQueries && query_waves <= (kParts <= 2 ? 32768 : 16384);
  const long long groups = run_groups + (together ? (query_waves + kWaves - 1) / kWaves : 0);
  if (groups * (kWaves * kWave) > 0xffffffffll || query_waves * kWave > 0xffffff00ll)
    return fail(LL_ERR_INVALID_ARGUMENT, "too many rows for one launch");  // (fewer than 2^32 threads)
  const dim3 grid(static_cast<unsigned>(groups));
  if (together) {
    quantized_write_kernel<Source, E, kGroup, kParts, kQueries><<<grid, kWaves * kWave, 0, s>>>(p);
  } else {
    if (kQueries)
      quantized_query_kernel<E, kGroup>
          <<<static_cast<unsigned>((query_waves + kThreads / kWave - 1) / (kThreads / kWave)), kThreads, 0, s>>>(p);
    quantized_write_kernel<Source, E, kGroup, kParts, false><<<grid, kWaves * kWave, 0, s>>>(p);
  }
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(LL_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(err));
  return LL_OK;
}

// As few waves of a pair as hold a block's rows.
template <typename Source, typename E, int kGroup, bool kQueries, int kParts = 1>
int launch_by_block(PoolParams &p, hipStream_t s) {
  constexpr int kHeld = kParts * kHeldSteps * kWave / kGroup;
  if constexpr (kHeld >= kMaxBlock) {
    return launch_write<Source, E, kGroup, kParts, kQueries>(p, s);
  } else {
    if (1 << p.block_shift <= kHeld) return launch_write<Source, E, kGroup, kParts, kQueries>(p, s);
    return launch_by_block<Source, E, kGroup, kQueries, 2 * kParts>(p, s);
  }
}

template <typename Source, typename E, bool kQueries>
int launch_by_dim(PoolParams &p, hipStream_t s) {
  if (p.dim <= 64) return launch_by_block<Source, E, 4, kQueries>(p, s);
  if (p.dim <= 128) return launch_by_block<Source, E, 8, kQueries>(p, s);
  return launch_by_block<Source, E, 16, kQueries>(p, s);
}

}  // namespace

extern "C" {

int64_t ll_quantized_append_args_size(void) { return static_cast<int64_t>(sizeof(ll_quantized_append_args)); }
int64_t ll_quantized_link_args_size(void) { return static_cast<int64_t>(sizeof(ll_quantized_link_args)); }
int64_t ll_quantized_load_args_size(void) { return static_cast<int64_t>(sizeof(ll_quantized_load_args)); }

int ll_quantized_append(const ll_quantized_append_args *a, ll_stream_t stream) {
  if (a == nullptr) return fail(LL_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->struct_size != static_cast<int64_t>(sizeof(*a)))
    return fail(LL_ERR_INVALID_ARGUMENT, "struct_size %lld, expected %lld", static_cast<long long>(a->struct_size),
                static_cast<long long>(sizeof(*a)));
  int rc = check_pool(&a->pool);
  if (rc != LL_OK) return rc;
  if (a->num_tokens < 0 || a->num_tokens > 0x7fffffff)
    return fail(LL_ERR_INVALID_ARGUMENT, "num_tokens must be in [0, 2^31)");
  if (a->num_q_heads < 1 || a->num_q_heads > 65535)
    return fail(LL_ERR_KV_HEAD_LAYOUT_MISMATCH, "num_q_heads must be in [1, 65535]");
  if (a->dtype != LL_DTYPE_FLOAT16 && a->dtype != LL_DTYPE_BFLOAT16)
    return fail(LL_ERR_FP16_OR_BF16_REQUIRED, "dtype must be fp16 or bf16");
  rc = check_table(a->cos_sin_dtype, a->cos_sin_rows, a->cos_sin_cols, a->cos_sin_stride_row, a->rotary_dim,
                   a->pool.head_dim);
  if (rc != LL_OK) return rc;
  if (!index_code(a->positions_dtype) || !index_code(a->destination_slots_dtype))
    return fail(LL_ERR_INTEGER_TOKEN_MAPS_REQUIRED, "positions and slots must be int32 or int64");
  const bool normed = a->query_norm_weight != nullptr || a->key_norm_weight != nullptr;
  if (normed && !float_code(a->norm_weight_dtype))
    return fail(LL_ERR_INVALID_ARGUMENT, "norm weights must be fp16, bf16 or fp32");
  if (normed && !(a->norm_eps >= 0.0)) return fail(LL_ERR_INVALID_ARGUMENT, "norm_eps must not be negative");
  if (a->num_tokens == 0) return LL_OK;
  if (a->query == nullptr || a->query_output == nullptr || a->key == nullptr || a->value == nullptr ||
      a->positions == nullptr || a->cos_sin_cache == nullptr || a->destination_slots == nullptr)
    return fail(LL_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
  if (!whole_chunks(a->query, a->query_token_stride, a->query_head_stride) ||
      !whole_chunks(a->query_output, a->query_output_token_stride, a->query_output_head_stride) ||
      !whole_chunks(a->key, a->key_token_stride, a->key_head_stride) ||
      !whole_chunks(a->value, a->value_token_stride, a->value_head_stride) || !aligned(a->query_norm_weight, 16) ||
      !aligned(a->key_norm_weight, 16))
    return fail(LL_ERR_INVALID_ARGUMENT, "rows and norm weights must begin at multiples of 16 bytes");
  PoolParams p;
  memset(&p, 0, sizeof(p));
  fill_pool(a->pool, &p);
  fill_table(a->cos_sin_cache, a->cos_sin_dtype, a->cos_sin_rows, a->cos_sin_stride_row, a->rotary_dim,
             a->is_neox_style != 0, &p);
  p.slots = a->destination_slots;
  p.slots64 = a->destination_slots_dtype == LL_DTYPE_INT64 ? 1 : 0;
  p.positions = a->positions;
  p.positions64 = a->positions_dtype == LL_DTYPE_INT64 ? 1 : 0;
  p.skipped = reinterpret_cast<unsigned long long *>(a->skipped_rows);
  p.num_tokens = a->num_tokens;
  p.query = Rows{static_cast<const uint16_t *>(a->query), a->query_token_stride, a->query_head_stride};
  p.new_key = Rows{static_cast<const uint16_t *>(a->key), a->key_token_stride, a->key_head_stride};
  p.new_value = Rows{static_cast<const uint16_t *>(a->value), a->value_token_stride, a->value_head_stride};
  p.query_output = static_cast<uint16_t *>(a->query_output);
  p.query_output_token = a->query_output_token_stride;
  p.query_output_head = a->query_output_head_stride;
  p.query_weight = a->query_norm_weight;
  p.key_weight = a->key_norm_weight;
  p.weight_dtype = static_cast<int>(a->norm_weight_dtype);
  p.eps = a->norm_eps;
  p.hq = static_cast<int>(a->num_q_heads);
  const int query_heads = kWave / (p.dim <= 64 ? 4 : p.dim <= 128 ? 8 : 16);  // of a wave
  p.query_steps = (p.hq + query_heads - 1) / query_heads;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return a->dtype == LL_DTYPE_FLOAT16 ? launch_by_dim<NewTokens<F16>, F16, true>(p, s)
                                      : launch_by_dim<NewTokens<Bf16>, Bf16, true>(p, s);
}

int ll_quantized_link(const ll_quantized_link_args *a, ll_stream_t stream) {
  if (a == nullptr) return fail(LL_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->struct_size != static_cast<int64_t>(sizeof(*a)))
    return fail(LL_ERR_INVALID_ARGUMENT, "struct_size %lld, expected %lld", static_cast<long long>(a->struct_size),
                static_cast<long long>(sizeof(*a)));
  int rc = check_pool(&a->pool);
  if (rc != LL_OK) return rc;
  if (a->num_tokens < 0 || a->num_tokens > 0x7fffffff)
    return fail(LL_ERR_INVALID_ARGUMENT, "num_tokens must be in [0, 2^31)");
  rc = check_table(a->cos_sin_dtype, a->cos_sin_rows, a->cos_sin_cols, a->cos_sin_stride_row, a->rotary_dim,
                   a->pool.head_dim);
  if (rc != LL_OK) return rc;
  if (!index_code(a->slots_dtype) || !index_code(a->positions_dtype))
    return fail(LL_ERR_INTEGER_TOKEN_MAPS_REQUIRED, "slots and positions must be int32 or int64");
  if (a->prefix_token_count < 0 || a->prefix_token_count > a->num_tokens)
    return fail(LL_ERR_INVALID_ARGUMENT, "prefix_token_count must be in [0, num_tokens]");
  if (a->num_tokens == 0) return LL_OK;
  if (a->source_slots == nullptr || a->destination_slots == nullptr || a->local_positions == nullptr ||
      a->global_positions == nullptr || a->cos_sin_cache == nullptr)
    return fail(LL_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
  PoolParams p;
  memset(&p, 0, sizeof(p));
  fill_pool(a->pool, &p);
  fill_table(a->cos_sin_cache, a->cos_sin_dtype, a->cos_sin_rows, a->cos_sin_stride_row, a->rotary_dim,
             a->is_neox_style != 0, &p);
  p.slots = a->destination_slots;
  p.sources = a->source_slots;
  p.slots64 = a->slots_dtype == LL_DTYPE_INT64 ? 1 : 0;
  p.positions = a->global_positions;
  p.old_positions = a->local_positions;
  p.positions64 = a->positions_dtype == LL_DTYPE_INT64 ? 1 : 0;
  p.skipped = reinterpret_cast<unsigned long long *>(a->skipped_rows);
  p.num_tokens = a->num_tokens;
  p.masked = static_cast<const uint8_t *>(a->repair_mask);
  p.prefix = a->prefix_token_count;
  return launch_by_dim<CachedRows, Bf16, false>(p, reinterpret_cast<hipStream_t>(stream));
}

int ll_quantized_load(const ll_quantized_load_args *a, ll_stream_t stream) {
  if (a == nullptr) return fail(LL_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->struct_size != static_cast<int64_t>(sizeof(*a)))
    return fail(LL_ERR_INVALID_ARGUMENT, "struct_size %lld, expected %lld", static_cast<long long>(a->struct_size),
                static_cast<long long>(sizeof(*a)));
  const int rc = check_pool(&a->pool);
  if (rc != LL_OK) return rc;
  if (a->num_rows < 0 || a->num_rows > 0x7fffffff)
    return fail(LL_ERR_INVALID_ARGUMENT, "num_rows must be in [0, 2^31)");
  if (!float_code(a->dtype)) return fail(LL_ERR_INVALID_ARGUMENT, "dtype must be fp16, bf16 or fp32");
  if (a->slots != nullptr && !index_code(a->slots_dtype))
    return fail(LL_ERR_INTEGER_TOKEN_MAPS_REQUIRED, "slots must be int32 or int64");
  if (a->num_rows == 0) return LL_OK;
  if (a->key_output == nullptr || a->value_output == nullptr)
    return fail(LL_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
  if (!aligned(a->key_output, 16) || !aligned(a->value_output, 16))
    return fail(LL_ERR_INVALID_ARGUMENT, "the outputs must be 16-byte aligned");
  PoolParams pool;
  memset(&pool, 0, sizeof(pool));
  fill_pool(a->pool, &pool);
  LoadParams p;
  memset(&p, 0, sizeof(p));
  p.key = pool.key.codes;
  p.value = pool.value.codes;
  p.key_scales = pool.key.scales;
  p.value_scales = pool.value.scales;
  p.key_output = a->key_output;
  p.value_output = a->value_output;
  p.slots = a->slots;
  p.slots64 = a->slots_dtype == LL_DTYPE_INT64 ? 1 : 0;
  p.num_slots = pool.num_slots;
  p.block_shift = pool.block_shift;
  p.hkv = pool.hkv;
  p.dim_chunks = pool.dim / 8;
  p.row_chunks = pool.hkv * p.dim_chunks;
  p.num_rows = a->num_rows;
  p.group_rows = std::max(1, kThreads * kLoadChunks / p.row_chunks);
  p.dtype = static_cast<int>(a->dtype);
  const long long groups = (p.num_rows + p.group_rows - 1) / p.group_rows;
  if (groups * 2 * kThreads > 0xffffffffll)
    return fail(LL_ERR_INVALID_ARGUMENT, "too many rows for one launch");
  quantized_load_kernel<<<dim3(static_cast<unsigned>(groups), 2), kThreads, 0,
                          reinterpret_cast<hipStream_t>(stream)>>>(p);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(LL_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(err));
  return LL_OK;
}

}  // extern "C"
