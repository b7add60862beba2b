// Norms of queries and keys for each head with their position rotation, in
// place of a model's separate norm, rotation and cache-write passes, on gfx950
// (MI355X); with a pool, the keys and values go to their slots on the way.
//
// For a row x of D values (one token's one head), in fp32:
//   y = x * rsqrt(mean(x^2) + eps) * w          (with a norm weight w)
//   (y_i, y_j) -> (y_i c - y_j s, y_j c + y_i s)  for the rotary pairs
// with c, s = row `position` of the cos/sin table; pairs are (i, i + R / 2)
// (neox) or (2 i, 2 i + 1) of the first R = rotary_dim values, the rest pass
// through, and the result is rounded once.
//
// Every call is bound by memory (about 2 flops per byte) or, for the few rows
// of a decode step, by the chain position -> table row -> result.  So a lane
// holds both chunks of its rotary pairs (16 values: no exchange between lanes
// but the norm's sum), a row's loads do not wait for the position, and a wave
// holds whole heads of one token: 8 heads of 128 values at a time.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <string.h>

#include "legolink_kv.h"
#include "ll_internal.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kWave = 64;
constexpr int kThreads = 256;
constexpr int kMaxDim = 256;

int fail(int code, const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  const int rc = ll_record_error(code, fmt, ap);
  va_end(ap);
  return rc;
}

// A strided set of rows: element t, h, d at base[t * token + h * head + d].
struct Rows {
  uint16_t *base;
  long long token, head;
};

struct RotaryParams {
  Rows query, query_output, key, key_output, value;
  uint16_t *key_buffer, *value_buffer;
  const void *positions, *slots, *table, *query_weight, *key_weight;
  unsigned long long *skipped;
  long long num_tokens, num_slots, table_rows, table_stride;
  float eps;
  int hq, hkv, dim, value_dim, rotary;
  int positions64, slots64, table_dtype, weight_dtype, neox;
  int turn_steps, steps;  // vector kernel: waves per token, those of its queries and keys first
};

struct Bf16 {
  __device__ static f32x2 unpack(uint32_t pair) {  // exact
    return f32x2{__uint_as_float(pair << 16), __uint_as_float(pair & 0xffff0000u)};
  }
  __device__ static uint32_t pack(float lo, float hi) {  // round to nearest even
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
  }
};

struct F16 {
  __device__ static f32x2 unpack(uint32_t pair) {
    return __builtin_convertvector(__builtin_bit_cast(f16x2, pair), f32x2);
  }
  __device__ static uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, f16x2));
  }
};

__device__ inline long long index_at(const void *values, int is64, long long i) {
  return is64 ? static_cast<const int64_t *>(values)[i] : static_cast<const int32_t *>(values)[i];
}

// One value of a table or weight of any of the three float types.
__device__ inline float value_at(const void *values, int dtype, long long i) {
  if (dtype == LL_DTYPE_FLOAT32) return static_cast<const float *>(values)[i];
  const uint32_t bits = static_cast<const uint16_t *>(values)[i];
  return dtype == LL_DTYPE_BFLOAT16 ? Bf16::unpack(bits)[0] : F16::unpack(bits)[0];
}

template <typename E>
__device__ inline void unpack8(u32x4 bits, float *out) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x2 two = E::unpack(bits[i]);
    out[2 * i] = two[0];
    out[2 * i + 1] = two[1];
  }
}

// Eight neighbouring values of any of the three types, 16-byte aligned.
__device__ inline void values8(const void *values, int dtype, long long i, float *out) {
  if (dtype == LL_DTYPE_FLOAT32) {
    const f32x4 *v = reinterpret_cast<const f32x4 *>(static_cast<const float *>(values) + i);
    const f32x4 lo = v[0], hi = v[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      out[j] = lo[j];
      out[4 + j] = hi[j];
    }
    return;
  }
  const u32x4 bits = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(values) + i);
  if (dtype == LL_DTYPE_BFLOAT16) unpack8<Bf16>(bits, out);
  else unpack8<F16>(bits, out);
}

__device__ inline u32x4 load_chunk(const uint16_t *p) { return *reinterpret_cast<const u32x4 *>(p); }
__device__ inline void store_chunk(uint16_t *p, u32x4 bits) { *reinterpret_cast<u32x4 *>(p) = bits; }

// What a token's waves do: nothing where its position is outside the table;
// its keys and values are written where its slot is a row of the pool.  The
// token's first wave counts a position outside the table and a slot past the
// pool (a negative slot is padding).
struct Token {
  long long position, slot;
  bool turned, written;
};

__device__ inline Token token_at(const RotaryParams &p, long long t, bool first) {
  Token r;
  r.position = index_at(p.positions, p.positions64, t);
  r.slot = p.slots != nullptr ? index_at(p.slots, p.slots64, t) : -1;
  r.turned = r.position >= 0 && r.position < p.table_rows;
  r.written = r.turned && r.slot >= 0 && r.slot < p.num_slots;
  if (first && p.skipped != nullptr && (!r.turned || r.slot >= p.num_slots) && threadIdx.x % kWave == 0)
    atomicAdd(p.skipped, 1ull);
  return r;
}

// Head dims of whole 16-value lanes, rotary dims likewise, everything 16-byte
// aligned.  A wave is one step of one token: kGroup lanes a head (the next
// power of two of D / 16, so that the norm's sum is kGroup's xor shuffles;
// lanes past D / 16 idle), 64 / kGroup heads a step, queries first, then keys;
// the steps behind them copy the values, 128 chunks of 8 at a time.  8,192 tokens
// of 64 + 8 normed heads of 128: 64.6 us, 4.7 TB/s read and written (a copy of as
// many bytes 62 us); one token 3.1 us, the latency of its position, the table row
// behind it and the stores.
template <typename E, int kGroup>
__global__ void __launch_bounds__(kThreads) head_rotary_vec_kernel(const RotaryParams p) {
  constexpr int kHeads = kWave / kGroup;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int lane = threadIdx.x % kWave;
  const unsigned unit = blockIdx.x * (kThreads / kWave) + wave;  // (a launch holds fewer than 2^26)
  const long long t = unit / static_cast<unsigned>(p.steps);
  const int step = static_cast<int>(unit % static_cast<unsigned>(p.steps));
  if (t >= p.num_tokens) return;

  if (step >= p.turn_steps) {
    const int row_chunks = p.value_dim / 8;
    const int chunks = p.hkv * row_chunks;
    const int c = (step - p.turn_steps) * 2 * kWave + lane;
    u32x4 bits[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int chunk = min(c + j * kWave, chunks - 1);  // past the end: the last again, dropped
      const int head = chunk / row_chunks;
      bits[j] = load_chunk(p.value.base + t * p.value.token + head * p.value.head + (chunk - head * row_chunks) * 8);
    }
    const Token token = token_at(p, t, false);
    if (!token.written) return;
    uint16_t *dst = p.value_buffer + token.slot * p.hkv * p.value_dim;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (c + j * kWave < chunks) store_chunk(dst + static_cast<long long>(c + j * kWave) * 8, bits[j]);
    return;
  }

  const int row = step * kHeads + lane / kGroup;
  const int i = lane % kGroup;
  const int rotary_lanes = p.rotary / 16;
  const bool rotates = i < rotary_lanes;
  const bool active = row < p.hq + p.hkv && i < p.dim / 16;
  const bool is_key = row >= p.hq;
  const int head = is_key ? row - p.hq : row;
  // The lane's two chunks: its pairs' halves (neox), or neighbours.
  const int first = rotates && p.neox ? 8 * i : 16 * i;
  const int second = rotates && p.neox ? 8 * (i + rotary_lanes) : 16 * i + 8;
  u32x4 bits_a = u32x4{0u, 0u, 0u, 0u}, bits_b = bits_a;
  if (active) {
    const Rows &in = is_key ? p.key : p.query;
    const uint16_t *src = in.base + t * in.token + head * in.head;
    bits_a = load_chunk(src + first);
    bits_b = load_chunk(src + second);
  }
  const Token token = token_at(p, t, step == 0);
  if (!token.turned) return;
  float c[8], s[8];
  if (active && rotates) {
    const long long at = token.position * p.table_stride + 8 * i;
    values8(p.table, p.table_dtype, at, c);
    values8(p.table, p.table_dtype, at + p.rotary / 2, s);
  }
  float a[8], b[8];
  unpack8<E>(bits_a, a);
  unpack8<E>(bits_b, b);
  if (p.query_weight != nullptr || p.key_weight != nullptr) {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += a[j] * a[j] + b[j] * b[j];
#pragma unroll
    for (int step_lanes = 1; step_lanes < kGroup; step_lanes *= 2) sum += __shfl_xor(sum, step_lanes);
    const void *weight = is_key ? p.key_weight : p.query_weight;
    if (active && weight != nullptr) {
      const float scale = rsqrtf(sum / static_cast<float>(p.dim) + p.eps);
      float w[8];
      values8(weight, p.weight_dtype, first, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = a[j] * scale * w[j];
      values8(weight, p.weight_dtype, second, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) b[j] = b[j] * scale * w[j];
    }
  }
  if (!active) return;
  if (rotates && p.neox) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float lo = a[j], hi = b[j];
      a[j] = lo * c[j] - hi * s[j];
      b[j] = hi * c[j] + lo * s[j];
    }
  } else if (rotates) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a0 = a[2 * j], a1 = a[2 * j + 1], b0 = b[2 * j], b1 = b[2 * j + 1];
      a[2 * j] = a0 * c[j] - a1 * s[j];
      a[2 * j + 1] = a1 * c[j] + a0 * s[j];
      b[2 * j] = b0 * c[4 + j] - b1 * s[4 + j];
      b[2 * j + 1] = b1 * c[4 + j] + b0 * s[4 + j];
    }
  }
  uint16_t *dst;
  if (!is_key) {
    dst = p.query_output.base + t * p.query_output.token + head * p.query_output.head;
  } else if (p.slots == nullptr) {
    dst = p.key_output.base + t * p.key_output.token + head * p.key_output.head;
  } else {
    if (!token.written) return;
    dst = p.key_buffer + (token.slot * p.hkv + head) * p.dim;
  }
  u32x4 out_a, out_b;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    out_a[j] = E::pack(a[2 * j], a[2 * j + 1]);
    out_b[j] = E::pack(b[2 * j], b[2 * j + 1]);
  }
  store_chunk(dst + first, out_a);
  store_chunk(dst + second, out_b);
}

// Every other shape: a wave is one row of one token (queries, keys, then
// values), a lane every 64th of its rotary pairs and of the values behind them.
// All of a row's loads come before its stores, so that it may be rotated in
// place, and those of the row do not wait for the position.  Bound by its 2-byte
// loads and stores: the rows above, one value off their alignment, take 285 us
// (1.1 TB/s; 393 with a lane per value, each loading its partner too), 8,192 tokens
// of 72 heads of 40 and of 200 values 177 and 358 us (0.5 and 1.3 TB/s).
template <typename E>
__global__ void __launch_bounds__(kThreads) head_rotary_element_kernel(const RotaryParams p) {
  constexpr int kPer = kMaxDim / kWave;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int lane = threadIdx.x % kWave;
  const unsigned unit = blockIdx.x * (kThreads / kWave) + wave;
  const long long t = unit / static_cast<unsigned>(p.steps);
  const int row = static_cast<int>(unit % static_cast<unsigned>(p.steps));
  if (t >= p.num_tokens) return;
  if (row >= p.turn_steps) {
    const int head = row - p.turn_steps;
    const uint16_t *src = p.value.base + t * p.value.token + head * p.value.head;
    uint16_t values[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      if (lane + k * kWave < p.value_dim) values[k] = src[lane + k * kWave];
    const Token token = token_at(p, t, false);
    if (!token.written) return;
    uint16_t *dst = p.value_buffer + (token.slot * p.hkv + head) * p.value_dim;
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      if (lane + k * kWave < p.value_dim) dst[lane + k * kWave] = values[k];
    return;
  }
  const bool is_key = row >= p.hq;
  const int head = is_key ? row - p.hq : row;
  const Rows &in = is_key ? p.key : p.query;
  const uint16_t *src = in.base + t * in.token + head * in.head;
  const void *weight = is_key ? p.key_weight : p.query_weight;
  // Item i below `half` is the pair (first, second), the others a value each.
  const int half = p.rotary / 2;
  const int items = half + p.dim - p.rotary;
  auto first_of = [&](int i) { return i >= half ? i + half : p.neox ? i : 2 * i; };
  auto second_of = [&](int i) { return p.neox ? i + half : 2 * i + 1; };
  float x[kPer], y[kPer];
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int i = lane + k * kWave;
    x[k] = y[k] = 0.f;
    if (k * kWave >= items) continue;  // (of no lane)
    if (i < items) x[k] = E::unpack(src[first_of(i)])[0];
    if (i < half) y[k] = E::unpack(src[second_of(i)])[0];
  }
  const Token token = token_at(p, t, row == 0);
  if (!token.turned) return;
  if (weight != nullptr) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) sum += x[k] * x[k] + y[k] * y[k];
#pragma unroll
    for (int step_lanes = 1; step_lanes < kWave; step_lanes *= 2) sum += __shfl_xor(sum, step_lanes);
    const float scale = rsqrtf(sum / static_cast<float>(p.dim) + p.eps);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      if (k * kWave >= items) continue;
      const int i = lane + k * kWave;
      if (i < items) x[k] = x[k] * scale * value_at(weight, p.weight_dtype, first_of(i));
      if (i < half) y[k] = y[k] * scale * value_at(weight, p.weight_dtype, second_of(i));
    }
  }
  uint16_t *dst;
  if (!is_key) {
    dst = p.query_output.base + t * p.query_output.token + head * p.query_output.head;
  } else if (p.slots == nullptr) {
    dst = p.key_output.base + t * p.key_output.token + head * p.key_output.head;
  } else {
    if (!token.written) return;
    dst = p.key_buffer + (token.slot * p.hkv + head) * p.dim;
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (k * kWave >= items) continue;
    const int i = lane + k * kWave;
    if (i < half) {
      const float c = value_at(p.table, p.table_dtype, token.position * p.table_stride + i);
      const float s = value_at(p.table, p.table_dtype, token.position * p.table_stride + half + i);
      dst[first_of(i)] = static_cast<uint16_t>(E::pack(x[k] * c - y[k] * s, 0.f));
      dst[second_of(i)] = static_cast<uint16_t>(E::pack(y[k] * c + x[k] * s, 0.f));
    } else if (i < items) {
      dst[first_of(i)] = static_cast<uint16_t>(E::pack(x[k], 0.f));
    }
  }
}

bool aligned(const void *p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

bool float_code(int64_t dtype) {
  return dtype == LL_DTYPE_FLOAT16 || dtype == LL_DTYPE_BFLOAT16 || dtype == LL_DTYPE_FLOAT32;
}
bool index_code(int64_t dtype) { return dtype == LL_DTYPE_INT32 || dtype == LL_DTYPE_INT64; }

int check_args(const ll_head_rotary_args *a) {
  if (a == nullptr) return fail(LL_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->struct_size != static_cast<int64_t>(sizeof(ll_head_rotary_args)))
    return fail(LL_ERR_INVALID_ARGUMENT, "struct_size %lld, expected %lld", static_cast<long long>(a->struct_size),
                static_cast<long long>(sizeof(ll_head_rotary_args)));
  if (a->num_tokens < 0 || a->num_tokens > 0x7fffffff)
    return fail(LL_ERR_INVALID_ARGUMENT, "num_tokens must be in [0, 2^31)");
  if (a->num_q_heads < 1 || a->num_kv_heads < 1 || a->num_q_heads > 65535 || a->num_kv_heads > 65535)
    return fail(LL_ERR_KV_HEAD_LAYOUT_MISMATCH, "head counts must be in [1, 65535]");
  if (a->dtype != LL_DTYPE_FLOAT16 && a->dtype != LL_DTYPE_BFLOAT16)
    return fail(LL_ERR_FP16_OR_BF16_REQUIRED, "dtype must be fp16 or bf16");
  if (a->head_dim < 1 || a->head_dim > kMaxDim)
    return fail(LL_ERR_HEAD_DIMENSION_OUT_OF_RANGE, "head_dim must be in [1, %d]", kMaxDim);
  if (a->rotary_dim < 2 || a->rotary_dim % 2 != 0)
    return fail(LL_ERR_EVEN_ROTARY_DIM_REQUIRED, "rotary_dim must be positive and even");
  if (a->rotary_dim > a->head_dim)
    return fail(LL_ERR_ROTARY_DIM_EXCEEDS_HEAD_DIM, "rotary_dim exceeds head_dim");
  if (!float_code(a->cos_sin_dtype)) return fail(LL_ERR_UNSUPPORTED_COS_SIN_DTYPE, "cos/sin dtype");
  if (a->cos_sin_rows < 0 || a->cos_sin_cols < a->rotary_dim || a->cos_sin_stride_row < 0)
    return fail(LL_ERR_UNSUPPORTED_COS_SIN_CACHE, "the cos/sin table needs rotary_dim columns");
  if (!index_code(a->positions_dtype)) return fail(LL_ERR_INTEGER_TOKEN_MAPS_REQUIRED, "positions dtype");
  if ((a->query_norm_weight != nullptr || a->key_norm_weight != nullptr) && !float_code(a->norm_weight_dtype))
    return fail(LL_ERR_INVALID_ARGUMENT, "norm weights must be fp16, bf16 or fp32");
  if ((a->query_norm_weight != nullptr || a->key_norm_weight != nullptr) && !(a->norm_eps >= 0.0))
    return fail(LL_ERR_INVALID_ARGUMENT, "norm_eps must not be negative");
  if (a->destination_slots != nullptr) {
    if (a->value_head_dim < 1 || a->value_head_dim > kMaxDim)
      return fail(LL_ERR_HEAD_DIMENSION_OUT_OF_RANGE, "value_head_dim must be in [1, %d]", kMaxDim);
    if (a->num_slots < 0) return fail(LL_ERR_INVALID_ARGUMENT, "num_slots is negative");
    if (!index_code(a->destination_slots_dtype))
      return fail(LL_ERR_INTEGER_TOKEN_MAPS_REQUIRED, "destination slots dtype");
  }
  if (a->num_tokens == 0) return LL_OK;
  if (a->query == nullptr || a->query_output == nullptr || a->key == nullptr || a->positions == nullptr ||
      a->cos_sin_cache == nullptr)
    return fail(LL_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
  if (a->destination_slots == nullptr ? a->key_output == nullptr || a->key_buffer != nullptr
                                      : a->key_output != nullptr || a->value == nullptr)
    return fail(LL_ERR_INVALID_ARGUMENT, "keys go to key_output, or with destination_slots and values to a pool");
  if (a->destination_slots != nullptr && a->num_slots > 0 && (a->key_buffer == nullptr || a->value_buffer == nullptr))
    return fail(LL_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
  return LL_OK;
}

Rows rows_of(const void *base, int64_t token, int64_t head) {
  return Rows{static_cast<uint16_t *>(const_cast<void *>(base)), token, head};
}

// Rows that the vector kernel takes: 16-byte chunks.
bool whole_chunks(const Rows &rows) { return aligned(rows.base, 16) && rows.token % 8 == 0 && rows.head % 8 == 0; }

template <typename E>
void launch_vec(const RotaryParams &p, unsigned grid, hipStream_t s) {
  if (p.dim <= 16) head_rotary_vec_kernel<E, 1><<<grid, kThreads, 0, s>>>(p);
  else if (p.dim <= 32) head_rotary_vec_kernel<E, 2><<<grid, kThreads, 0, s>>>(p);
  else if (p.dim <= 64) head_rotary_vec_kernel<E, 4><<<grid, kThreads, 0, s>>>(p);
  else if (p.dim <= 128) head_rotary_vec_kernel<E, 8><<<grid, kThreads, 0, s>>>(p);
  else head_rotary_vec_kernel<E, 16><<<grid, kThreads, 0, s>>>(p);
}

}  // namespace

extern "C" {

int64_t ll_head_rotary_args_size(void) { return static_cast<int64_t>(sizeof(ll_head_rotary_args)); }

int ll_head_rotary(const ll_head_rotary_args *a, ll_stream_t stream) {
  const int rc = check_args(a);
  if (rc != LL_OK || a->num_tokens == 0) return rc;
  const bool appends = a->destination_slots != nullptr;
  RotaryParams p;
  memset(&p, 0, sizeof(p));
  p.query = rows_of(a->query, a->query_token_stride, a->query_head_stride);
  p.query_output = rows_of(a->query_output, a->query_output_token_stride, a->query_output_head_stride);
  p.key = rows_of(a->key, a->key_token_stride, a->key_head_stride);
  p.positions = a->positions;
  p.table = a->cos_sin_cache;
  p.query_weight = a->query_norm_weight;
  p.key_weight = a->key_norm_weight;
  p.skipped = reinterpret_cast<unsigned long long *>(a->skipped_rows);
  p.num_tokens = a->num_tokens;
  p.table_rows = a->cos_sin_rows;
  p.table_stride = a->cos_sin_stride_row;
  p.eps = static_cast<float>(a->norm_eps);
  p.hq = static_cast<int>(a->num_q_heads);
  p.hkv = static_cast<int>(a->num_kv_heads);
  p.dim = static_cast<int>(a->head_dim);
  p.rotary = static_cast<int>(a->rotary_dim);
  p.positions64 = a->positions_dtype == LL_DTYPE_INT64 ? 1 : 0;
  p.table_dtype = static_cast<int>(a->cos_sin_dtype);
  p.weight_dtype = static_cast<int>(a->norm_weight_dtype);
  p.neox = a->is_neox_style != 0 ? 1 : 0;
  const long long table_bytes = a->cos_sin_dtype == LL_DTYPE_FLOAT32 ? 4 : 2;
  bool vector = p.dim % 16 == 0 && p.rotary % 16 == 0 && whole_chunks(p.query) && whole_chunks(p.query_output) &&
                whole_chunks(p.key) && aligned(p.table, 16) && p.table_stride * table_bytes % 16 == 0 &&
                aligned(p.query_weight, 16) && aligned(p.key_weight, 16);
  if (appends) {
    p.value = rows_of(a->value, a->value_token_stride, a->value_head_stride);
    p.key_buffer = static_cast<uint16_t *>(a->key_buffer);
    p.value_buffer = static_cast<uint16_t *>(a->value_buffer);
    p.slots = a->destination_slots;
    p.slots64 = a->destination_slots_dtype == LL_DTYPE_INT64 ? 1 : 0;
    p.num_slots = a->num_slots;
    p.value_dim = static_cast<int>(a->value_head_dim);
    vector = vector && p.value_dim % 8 == 0 && whole_chunks(p.value) && aligned(p.key_buffer, 16) &&
             aligned(p.value_buffer, 16);
  } else {
    p.key_output = rows_of(a->key_output, a->key_output_token_stride, a->key_output_head_stride);
    vector = vector && whole_chunks(p.key_output);
  }
  if (vector) {
    int group = 1;
    while (group * 16 < p.dim) group *= 2;
    const int heads = kWave / group;
    p.turn_steps = (p.hq + p.hkv + heads - 1) / heads;
    p.steps = p.turn_steps + (appends ? (p.hkv * (p.value_dim / 8) + 2 * kWave - 1) / (2 * kWave) : 0);
  } else {
    p.turn_steps = p.hq + p.hkv;
    p.steps = p.turn_steps + (appends ? p.hkv : 0);
  }
  const long long blocks = (p.num_tokens * p.steps + kThreads / kWave - 1) / (kThreads / kWave);
  if (blocks > 0xffffffll)  // a launch holds fewer than 2^32 threads
    return fail(LL_ERR_INVALID_ARGUMENT, "too many rows for one launch");
  const unsigned grid = static_cast<unsigned>(blocks);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool f16 = a->dtype == LL_DTYPE_FLOAT16;
  if (vector) {
    if (f16) launch_vec<F16>(p, grid, s);
    else launch_vec<Bf16>(p, grid, s);
  } else {
    if (f16) head_rotary_element_kernel<F16><<<grid, kThreads, 0, s>>>(p);
    else head_rotary_element_kernel<Bf16><<<grid, kThreads, 0, s>>>(p);
  }
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(LL_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(err));
  return LL_OK;
}

}  // extern "C"
