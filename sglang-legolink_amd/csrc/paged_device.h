// What the library's paged attention kernels share, whatever type their pool holds:
// how a call's work is cut into units and found, the join of split requests, the
// checks of a call's block and its launch shape.
//
// Request r has n query rows (its last n tokens) and L keys in the pool; query
// i stands at position p = L - n + i and sees the keys j <= p.  G query heads
// share a KV head.  For one KV head the (query, head) pairs of a request are
// the columns of one matrix, token-major: column c is query c / G, head c % G.
// So single tokens fill G columns of an MFMA and chunks fill every one.
//
//   tile   = `columns` neighbouring columns of one request
//   chunk  = `chunk_keys` neighbouring keys
//   unit   = (request, tile, chunk); workgroup = (unit, KV head)
//
// The lengths are on the device, and no host plan or synchronisation comes
// before a call: every workgroup reads the requests' lengths, derives the chunk
// length that cuts the whole call's work into about `target` units, and finds
// its own unit by a prefix sum.  A tile of one chunk writes its output; the
// others leave partial results (fp32) that a second launch joins.
#ifndef PAGED_DEVICE_H
#define PAGED_DEVICE_H

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>

#include "attention_device.h"
#include "legolink_kv.h"
#include "ll_internal.h"
#include "paged_units.h"

namespace {

constexpr int kWave = 64;
constexpr int kPageTile = 64;  // chunk lengths are multiples of this many keys
constexpr float kSlack = 8.f;  // log2 headroom of the lazily updated softmax maximum

int fail(int code, const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  const int rc = ll_record_error(code, fmt, ap);
  va_end(ap);
  return rc;
}

struct PagedParams {
  const uint16_t *q;
  uint16_t *out;
  const uint16_t *k, *v;
  const int *pages;
  const void *kv_lengths, *query_starts;  // query_starts NULL: one query each
  float *ws;
  int *plan;  // of many requests (NULL: every workgroup makes its own)
  long long q_token, q_head, pages_stride;
  unsigned long long page_magic;
  double inv_target;
  double long_work, inv_long_target;  // of calls of so much work (in key tiles times column tiles) and more
  unsigned row_bytes;  // of one slot's K (or V) row: hkv * D values
  int page_shift, page_size, num_pages, max_keys;
  int num_queries, num_requests, hq, hkv, group;
  int lengths64, starts64;
  int min_chunk;  // key tiles
  int max_partials;
  float scale_log2;
};

struct Request {
  int q_start, q_len, kv_len;
};

__device__ inline long long index_at(const void *values, int is64, int i) {
  return is64 ? static_cast<const int64_t *>(values)[i] : static_cast<const int32_t *>(values)[i];
}

// Request r's sizes, held within the call's queries and page table.
__device__ inline Request request_at(const PagedParams &p, int r) {
  Request x;
  if (p.query_starts == nullptr) {
    x.q_start = r;
    x.q_len = 1;
  } else {
    const long long all = p.num_queries;
    const long long begin = min(max(index_at(p.query_starts, p.starts64, r), 0ll), all);
    const long long end = min(max(index_at(p.query_starts, p.starts64, r + 1), begin), all);
    x.q_start = static_cast<int>(begin);
    x.q_len = static_cast<int>(end - begin);
  }
  x.kv_len = static_cast<int>(min(max(index_at(p.kv_lengths, p.lengths64, r), 0ll), static_cast<long long>(p.max_keys)));
  return x;
}

// The bytes of slot's row from `base` on (one 32 x 32 + 64-bit multiply-add).
__device__ inline const unsigned char *row_at(const PagedParams &p, const unsigned char *base, int slot) {
  return base + static_cast<unsigned long long>(static_cast<unsigned>(slot)) * p.row_bytes;
}

// Lanes below, added within rows of 16 and then across them by DPP moves (a lane
// without a source adds 0).
template <int kControl, int kRows>
__device__ inline int moved(int value) {
  return __builtin_amdgcn_update_dpp(0, value, kControl, kRows, 0xf, false);
}
__device__ inline int inclusive_scan(int value) {
  value += moved<0x111, 0xf>(value);  // row_shr 1, 2, 4, 8
  value += moved<0x112, 0xf>(value);
  value += moved<0x114, 0xf>(value);
  value += moved<0x118, 0xf>(value);
  value += moved<0x142, 0xa>(value);  // row_bcast 15: rows 1 and 3
  value += moved<0x143, 0xc>(value);  // row_bcast 31: rows 2 and 3
  return value;
}
template <int kControl, int kRows>
__device__ inline double moved(double value) {
  return __hiloint2double(moved<kControl, kRows>(__double2hiint(value)), moved<kControl, kRows>(__double2loint(value)));
}
__device__ inline double sum_of_wave(double value) {
  value += moved<0x111, 0xf>(value);
  value += moved<0x112, 0xf>(value);
  value += moved<0x114, 0xf>(value);
  value += moved<0x118, 0xf>(value);
  value += moved<0x142, 0xa>(value);
  value += moved<0x143, 0xc>(value);
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(value), kWave - 1),
                          __builtin_amdgcn_readlane(__double2loint(value), kWave - 1));
}

// What a workgroup has to do: the tile and its request, the chunk of a unit,
// the tile's first unit and its count of chunks.
struct Work {
  Request request;
  int index;  // of the request; -1: none
  int tile, chunk, chunk_keys;
  int chunks;                        // of the tile
  int first_partial, partial_step;   // its chunk c leaves partial first_partial + c partial_step
  int key_end;             // keys that some column of the tile sees
};

// The request's columns (num_queries * G stays below 2^31).
__device__ inline int tiles_of(const PagedParams &p, int q_len, int columns) {
  return (q_len * p.group + columns - 1) >> (31 - __builtin_clz(columns));  // (a power of two)
}

__device__ inline int key_tiles_of(const Request &x) { return (x.kv_len + kPageTile - 1) / kPageTile; }

// A chunk's key tiles, of a call with this work (in key tiles times column tiles).
__device__ inline int chunk_of(const PagedParams &p, double work) {
  // (2^25 key tiles are more than any length; readfirstlane: uniform to the compiler too)
  const double inv_target = work >= p.long_work ? p.inv_long_target : p.inv_target;
  return __builtin_amdgcn_readfirstlane(
      max(p.min_chunk, static_cast<int>(min(ceil(work * inv_target - 1e-6), 33554432.0))));
}

// Many requests: chunk_of, and what lies up to the end of every 64 of them, once for
// the call (one workgroup), so that the others need not scan them all.
// plan[0] is the chunk; plan[1 + 3 b ..] units, partial results and tiles of the
// requests up to 64 (b + 1).
constexpr int kPlanThreads = 1024;
__host__ __device__ inline long long plan_ints(long long requests) { return 1 + 3 * ((requests + kWave - 1) / kWave); }

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PagedParams p, int columns) {
  constexpr int kWaves = kPlanThreads / kWave;
  __shared__ double work_of[kWaves];
  __shared__ int sums[2][kWaves][3];
  const int lane = threadIdx.x % kWave;
  const int wave = threadIdx.x / kWave;
  double work = 0.0;  // (exact below 2^53, in any order)
  for (int r = threadIdx.x; r < p.num_requests; r += kPlanThreads) {
    const Request x = request_at(p, r);
    work += static_cast<double>(tiles_of(p, x.q_len, columns)) * key_tiles_of(x);
  }
  work = sum_of_wave(work);
  if (lane == 0) work_of[wave] = work;
  __syncthreads();
  work = 0.0;
  for (int v = 0; v < kWaves; ++v) work += work_of[v];
  const int chunk = chunk_of(p, work);
  if (threadIdx.x == 0) p.plan[0] = chunk;
  int before[3] = {0, 0, 0};
  for (int r0 = 0, turn = 0; r0 < p.num_requests; r0 += kPlanThreads, turn ^= 1) {
    const int r = r0 + static_cast<int>(threadIdx.x);
    Request x = Request{0, 0, 0};
    if (r < p.num_requests) x = request_at(p, r);
    const int tiles = tiles_of(p, x.q_len, columns);
    const int chunks = parts_of(key_tiles_of(x), chunk);
    const int of_wave[3] = {inclusive_scan(tiles * chunks), inclusive_scan(chunks > 1 ? tiles * chunks : 0),
                            inclusive_scan(tiles)};
    if (lane == kWave - 1)
      for (int i = 0; i < 3; ++i) sums[turn][wave][i] = of_wave[i];
    __syncthreads();  // (the other turn's sums may still be read behind it)
    int up_to[3] = {before[0], before[1], before[2]};
    for (int v = 0; v < kWaves; ++v)
      for (int i = 0; i < 3; ++i) {
        before[i] += sums[turn][v][i];
        if (v == wave) up_to[i] = before[i];
      }
    if (lane == 0 && r < p.num_requests)
      for (int i = 0; i < 3; ++i) p.plan[1 + 3 * (r / kWave) + i] = up_to[i];
  }
}

// Unit `index` of the call (kOfTiles: tile `index`).  Every wave finds it for
// itself: two passes over the requests, 64 at a time, the first for the call's
// work in key tiles times column tiles (or, with a plan, over its entries, and one
// of 64 requests).  With L = max(min_chunk, work / target)
// key tiles a chunk, the units number at most work / L + tiles <= target +
// tiles, which the launch holds.  Those of requests of more than one chunk, which
// may leave partial results, number below 2 work / L <= 2 target + 2: a request of
// k > L key tiles has fewer than k / L + 1 < 2 k / L chunks.
//
// The units of 64 requests at a time come in order of falling length, as far as it
// is known before the columns' positions: the chunks of full length, then the
// requests' last chunks, the longest first (kByLength), or by the quarter of a full
// chunk that they fill (kByQuarter, whose cost does not grow with the requests).
// Workgroups start in that order, so the short units fill the last round.  Six
// chunks of 5 to 701 queries, 14/2 heads of 64, over 300 to 9,000 keys: 80 us by
// length, 84 by quarter, 98 request by request; 64 and 128 uneven requests of
// single tokens, 64/8 heads of 128: 390 and 212 us by quarter, 389 and 242 by
// length, 406 and 224 request by request.
enum class Order { kTiles, kByLength, kByQuarter };  // (kTiles: tiles, request by request)

template <Order kOrder>
__device__ inline Work find_work(const PagedParams &p, int columns, int index) {
  constexpr bool kOfTiles = kOrder == Order::kTiles;
  const int lane = threadIdx.x % kWave;
  Request mine = Request{0, 0, 0};
  Work w;
  w.index = -1;
  int chunk, first = 0, stop = p.num_requests;  // the requests to look at
  int units_before = 0, tiles_before = 0, partials_before = 0;
  if (p.plan == nullptr) {
    double work = 0.0;  // (exact below 2^53)
    for (int r0 = 0; r0 < p.num_requests; r0 += kWave) {
      Request x = Request{0, 0, 0};
      if (r0 + lane < p.num_requests) x = request_at(p, r0 + lane);
      if (r0 == 0) mine = x;
      work += static_cast<double>(tiles_of(p, x.q_len, columns)) * key_tiles_of(x);
    }
    chunk = chunk_of(p, sum_of_wave(work));
  } else {
    chunk = __builtin_amdgcn_readfirstlane(p.plan[0]);
    const int *ends = p.plan + 1;
    const int blocks = (p.num_requests + kWave - 1) / kWave;
    int block = 0;
    for (; block < blocks; block += kWave) {
      const bool reaches = block + lane < blocks && ends[3 * (block + lane) + (kOfTiles ? 2 : 0)] > index;
      const unsigned long long past = __builtin_amdgcn_ballot_w64(reaches);
      if (past != 0) {
        block += __builtin_ctzll(past);
        break;
      }
    }
    if (block >= blocks) return w;
    first = block * kWave;
    stop = min(stop, first + kWave);
    if (block > 0) {
      units_before = __builtin_amdgcn_readfirstlane(ends[3 * block - 3]);
      partials_before = __builtin_amdgcn_readfirstlane(ends[3 * block - 2]);
      tiles_before = __builtin_amdgcn_readfirstlane(ends[3 * block - 1]);
    }
    if (first + lane < stop) mine = request_at(p, first + lane);
  }

  w.chunk_keys = min(chunk, kOneChunk) * kPageTile;
  for (int r0 = first; r0 < stop; r0 += kWave) {
    Request x = mine;
    if (r0 > first) {
      x = Request{0, 0, 0};
      if (r0 + lane < p.num_requests) x = request_at(p, r0 + lane);
    }
    const int tiles = tiles_of(p, x.q_len, columns);
    const int key_tiles = key_tiles_of(x);
    const int chunks = parts_of(key_tiles, chunk);
    const int units_to = inclusive_scan(tiles * chunks);
    const int partials_to = inclusive_scan(chunks > 1 ? tiles * chunks : 0);
    const int tiles_to = kOfTiles ? inclusive_scan(tiles) : 0;
    const bool listed = r0 + lane < p.num_requests;
    // The request whose units hold `index`, the index within them.
    int within;
    bool is_last = false;  // a last chunk
    bool holds;
    if constexpr (kOfTiles) {
      within = index - tiles_before - tiles_to + tiles;
      holds = within >= 0 && within < tiles;
    } else {
      const int full_to = inclusive_scan(tiles * (chunks - 1));
      const int full = __builtin_amdgcn_readlane(full_to, kWave - 1);
      is_last = index - units_before >= full;
      if (!is_last) {
        within = index - units_before - full_to + tiles * (chunks - 1);
        holds = within >= 0 && within < tiles * (chunks - 1);
      } else {
        const int length = key_tiles - (chunks - 1) * chunk;
        int before = 0;  // tiles of last chunks in front of the lane's
        if constexpr (kOrder == Order::kByLength) {
          for (int j = 0; j < min(kWave, p.num_requests - r0); ++j) {
            const int other = __builtin_amdgcn_readlane(length, j);
            const int count = __builtin_amdgcn_readlane(tiles, j);
            before += other > length || (other == length && j < lane) ? count : 0;
          }
        } else {
          const int quarter = min(3, 4 * (chunk - length) / chunk);  // 0: the longest
          int of_former = 0;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int to = inclusive_scan(quarter == q ? tiles : 0);
            if (quarter == q) before = of_former + to - tiles;
            of_former += __builtin_amdgcn_readlane(to, kWave - 1);
          }
        }
        within = index - units_before - full - before;
        holds = within >= 0 && within < tiles;
      }
    }
    const unsigned long long past = __builtin_amdgcn_ballot_w64(listed && holds);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      w.index = r0 + at;
      w.request.q_start = __builtin_amdgcn_readlane(x.q_start, at);
      w.request.q_len = __builtin_amdgcn_readlane(x.q_len, at);
      w.request.kv_len = __builtin_amdgcn_readlane(x.kv_len, at);
      const int own_tiles = __builtin_amdgcn_readlane(tiles, at);  // at least 1
      const int own_chunks = __builtin_amdgcn_readlane(chunks, at);
      const int own_within = __builtin_amdgcn_readlane(within, at);
      // A request's units: chunk 0 of every tile, the last tile (which sees the most
      // keys) first, and so on.  The units that run together then read the same keys.
      int nth = own_within;
      w.chunk = 0;
      if constexpr (!kOfTiles) {
        if (is_last) {
          w.chunk = own_chunks - 1;
        } else {
          w.chunk = own_within / own_tiles;
          nth = own_within - w.chunk * own_tiles;
        }
      }
      w.tile = own_tiles - 1 - nth;
      w.first_partial = partials_before + __builtin_amdgcn_readlane(partials_to, at) - own_tiles * own_chunks + nth;
      w.partial_step = own_tiles;
      // The tile's last query and its position bound the keys.
      const int last_query = min(w.request.q_len - 1, ((w.tile + 1) * columns - 1) / p.group);
      w.key_end = max(0, w.request.kv_len - w.request.q_len + last_query + 1);
      w.chunks = parts_of(w.key_end, w.chunk_keys);
      break;
    }
    units_before += __builtin_amdgcn_readlane(units_to, kWave - 1);
    partials_before += __builtin_amdgcn_readlane(partials_to, kWave - 1);
    if constexpr (kOfTiles) tiles_before += __builtin_amdgcn_readlane(tiles_to, kWave - 1);
  }
  return w;
}

// A partial result of one KV head: `columns` rows of D floats (the sum of the
// weighted values, unnormalised), then (maximum of the scores before their scale,
// sum) pairs.
template <int D>
__device__ inline float *partial_of(const PagedParams &p, int columns, int partial, int head) {
  return p.ws + (static_cast<long long>(partial) * p.hkv + head) * columns * (D + 2);
}
__device__ inline bool partials_fit(const PagedParams &p, const Work &w) {  // (always, by the bound above)
  return w.first_partial >= 0 &&
         w.first_partial + static_cast<long long>(w.chunks - 1) * w.partial_step < p.max_partials;
}

__device__ inline uint16_t *output_row(const PagedParams &p, const Work &w, int head, int column, int dim) {
  const int token = column / p.group;
  const int h = head * p.group + (column - token * p.group);
  return p.out + ((static_cast<long long>(w.request.q_start) + token) * p.hq + h) * dim;
}

// Infinities and NaN among a tile's values.  A column that does not see a row
// weighs it 0, and 0 * inf is NaN; so in the tiles that some columns see in part,
// the values that are not finite are taken out of LDS before the product, and
// added to the columns that do see their rows afterwards (inf or NaN, whatever the
// weight).
template <typename E>
__device__ inline bool nonfinite(uint32_t value) { return (value & E::kExponent) == E::kExponent; }
template <typename E>
__device__ inline bool any_nonfinite(u32x4 bits) {
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) any = any || nonfinite<E>(bits[i]) || nonfinite<E>(bits[i] >> 16);
  return any;
}
template <typename E>
__device__ inline u32x4 finite_only(u32x4 bits) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (nonfinite<E>(bits[i])) bits[i] &= 0xffff0000u;
    if (nonfinite<E>(bits[i] >> 16)) bits[i] &= 0xffffu;
  }
  return bits;
}
template <typename E>
__device__ inline f32x4 nonfinite_only(u32x2 bits) {  // four values, the finite ones 0
  f32x4 out;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t value = bits[i / 2] >> (16 * (i % 2));
    out[i] = nonfinite<E>(value) ? E::unpack(bits[i / 2])[i % 2] : 0.f;
  }
  return out;
}

// Weights are 2^kWeightShift times what they are of the maximum, and so are their
// sums: they go to the value product in the KV type, where fp16 ends at 2^-25.  With
// the shift, a weight counts down to 2^-32 of the maximum, so that those lost beside
// one large key weigh less than 2^-15 over 131,072 keys (unshifted, 2^-8 and eight
// times the output's rounding); the largest, at kSlack above the maximum, is 2^15.
// (bf16 has fp32's range.)
//
// The exponent of a score s under the maximum m is s * scale - m * scale, one fma,
// whose second term is rounded: by up to 2^-5 below this limit, which is the same
// factor for every weight of the row, but by more than the weights' range holds where
// it is far beyond.  A wave with such a row subtracts first: (s - m) * scale.
constexpr float kLarge = 1048576.f;
__device__ inline bool is_large(float bias) { return fabsf(bias) >= kLarge; }

template <typename E>
__device__ inline float weight_bias(float m, float scale_log2) {
  return __builtin_fmaf(-m, scale_log2, E::kWeightShift);
}

// The weight, under the maximum `top` of several, of a result with the maximum `own`
// (of scores without their scale).
__device__ inline float joined_weight(float own, float top, float scale_log2) {
  return own == -INFINITY && top == -INFINITY ? 1.f : exp2f((own - top) * scale_log2);  // (sums of nothing seen are 0)
}

// Column statistics across the four lane groups of a 16-column MFMA.
__device__ inline float max_of_groups(float x) {
  unsigned a = __builtin_bit_cast(unsigned, x), b = a;
  permlane16_swap(a, b);
  x = max_f32(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
  a = b = __builtin_bit_cast(unsigned, x);
  permlane32_swap(a, b);
  return max_f32(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ inline float sum_of_groups(float x) {
  unsigned a = __builtin_bit_cast(unsigned, x), b = a;
  permlane16_swap(a, b);
  x = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
  a = b = __builtin_bit_cast(unsigned, x);
  permlane32_swap(a, b);
  return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}

template <int n>
__device__ inline void wait_vm() {
  __builtin_amdgcn_s_waitcnt(0xF70 | (n & 15) | ((n >> 4) << 14));
}

// Joins the partial results of tiles of more than one chunk.  A lane holds four
// values of a column, so a wave 256 / D columns; a workgroup of four waves 16
// columns or, with kSplit waves (few tiles of many chunks each, whose latency adds
// up), the columns of one wave, the waves taking turns at their chunks.  A batch's
// loads are in flight together.
template <int D, int kSplit>
struct Combine {
  static constexpr int kPerWave = 256 / D;
  static constexpr int kColumns = kSplit == 1 ? 16 : kPerWave;  // of a workgroup
  static constexpr int kTurns = kSplit == 1 ? kColumns / (4 * kPerWave) : 1;
  static constexpr int kBatch = kSplit == 1 ? 4 : 8;
  static constexpr int kThreads = kSplit == 1 ? 256 : kSplit * kWave;
};

template <int D, typename E, int kSplit>
__global__ void __launch_bounds__((Combine<D, kSplit>::kThreads)) paged_combine_kernel(const PagedParams p, int columns) {
  typedef Combine<D, kSplit> C;
  const int groups = columns / C::kColumns;
  const int tile_head = blockIdx.x / groups;
  const int head = tile_head % p.hkv;
  const Work w = find_work<Order::kTiles>(p, columns, tile_head / p.hkv);
  if (w.index < 0 || w.chunks <= 1 || !partials_fit(p, w)) return;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int quad = lane % (D / 4);
#pragma unroll
  for (int turn = 0; turn < C::kTurns; ++turn) {
    const int c = (blockIdx.x % groups) * C::kColumns + (kSplit == 1 ? (turn * 4 + wave) * C::kPerWave : 0) +
                  lane / (D / 4);
    const int column = w.tile * columns + c;
    const bool exists = column / p.group < w.request.q_len;
    if (kSplit == 1 && __builtin_amdgcn_ballot_w64(exists) == 0) return;  // (columns behind are none either)
    float top = -INFINITY, sum = 0.f;
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s0 = kSplit == 1 ? 0 : wave; s0 < w.chunks; s0 += kSplit * C::kBatch) {
      float tops[C::kBatch], sums[C::kBatch];
      f32x4 rows[C::kBatch];
#pragma unroll
      for (int i = 0; i < C::kBatch; ++i) {
        // Past the last chunk: the last again, dropped.  (Columns that do not exist
        // are within the partial, and dropped too.)
        const int chunk = min(s0 + i * kSplit, w.chunks - 1);
        const float *part = partial_of<D>(p, columns, w.first_partial + chunk * w.partial_step, head);
        tops[i] = part[columns * D + 2 * c];
        sums[i] = part[columns * D + 2 * c + 1];
        rows[i] = *reinterpret_cast<const f32x4 *>(part + c * D + 4 * quad);
      }
      float high = top;
#pragma unroll
      for (int i = 0; i < C::kBatch; ++i)
        if (s0 + i * kSplit < w.chunks) high = fmaxf(high, tops[i]);
      const float old = joined_weight(top, high, p.scale_log2);
      sum *= old;
      acc *= old;
      top = high;
#pragma unroll
      for (int i = 0; i < C::kBatch; ++i)
        if (s0 + i * kSplit < w.chunks) {
          const float weight = joined_weight(tops[i], top, p.scale_log2);
          sum += weight * sums[i];
          acc += weight * rows[i];
        }
    }
    if constexpr (kSplit > 1) {
      __shared__ float tops[kSplit][kWave], sums[kSplit][kWave];
      __shared__ f32x4 parts[kSplit][kWave];
      tops[wave][lane] = top;
      sums[wave][lane] = sum;
      parts[wave][lane] = acc;
      __syncthreads();
      if (wave > 0) return;
#pragma unroll
      for (int v = 1; v < kSplit; ++v) top = fmaxf(top, tops[v][lane]);
      sum = 0.f;
      acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < kSplit; ++v) {
        const float weight = joined_weight(tops[v][lane], top, p.scale_log2);
        sum += weight * sums[v][lane];
        acc += weight * parts[v][lane];
      }
    }
    if (!exists) continue;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    u32x2 packed;
    packed[0] = E::pack(acc[0] * inv, acc[1] * inv);
    packed[1] = E::pack(acc[2] * inv, acc[3] * inv);
    *reinterpret_cast<u32x2 *>(output_row(p, w, head, column, D) + 4 * quad) = packed;
  }
}

// How a call is launched: known from sizes that the host has.
// More requests than this have a plan made before the call's kernels (single tokens
// over 800 to 1,200 keys, 28/4 heads of 128: 128 requests 62 us with a plan, 61
// without; 256 117 and 128; 1,024 428 and 571; 2,048 837 and 1,507).
constexpr long long kPlanned = 128;

struct Launch {
  int columns;
  long long max_tiles, max_units;
  int max_partials, target, long_target, min_chunk;
  double long_work;  // from here on the units are long_target (at least target), below it target
  bool wide, splits;
  long long ws_floats, plan_at;  // of the workspace; where the plan begins in it (ws_floats: none)
};

constexpr int kComputeUnits = 256;  // MI355X

// `together`: KV heads that a workgroup of the narrow kernel takes.  `codes`: a pool of
// 8 bits.
Launch plan_launch(const ll_paged_attention_args *a, int together = 1, bool codes = false) {
  Launch x;
  const long long group = a->num_q_heads / a->num_kv_heads;
  const long long queries = a->num_queries, requests = a->num_requests;
  // By the average request's columns, since the host knows no more: up to 16 on the
  // narrow kernel, more on the wide one.  Of equal requests over 4,000 keys, heads of
  // 128: 16 of 32 columns (64/8 heads) 59 us wide, 68 narrow; 32 of 20 (8/8) 123 and
  // 139; 16 of 21 (28/4) 36 and 55.  (One request alone may be faster on the narrow
  // one: 32 columns over 32,768 keys of one head 22 and 17 us, 56 over 2,048 15 and
  // 14.)  Where the requests differ the average may fit none: 127 single tokens over
  // 2,000 keys and a chunk of 128 over 8,000 (28/4 heads, 14 columns on average) take
  // 204 us, in two calls 113 and 41; 63 single tokens and a chunk of 2,048 take 310,
  // in two calls 108 and 212.
  const long long average = queries == 0 ? 1 : (queries + requests - 1) / requests;
  const long long wanted = average * group;
  x.wide = wanted > 16;
  x.columns = x.wide ? (a->head_dim == 256 ? 128 : 256) : 16;
  x.max_tiles = a->query_starts == nullptr ? requests * ((group + x.columns - 1) / x.columns)
                                           : queries * group / x.columns + requests;
  x.min_chunk = 2;
  // A workgroup fills a compute unit (by its LDS: rings and slot list), so `places`
  // units of every KV head run at once.  Chunks: as many units as places, the longest first, leave
  // the least over.  Single tokens: where the tiles are few, as many units as run
  // at once; where they are many, two rounds, whose second the short ones fill (64
  // and 128 uneven requests: 390 and 212 us; one round 404 and 214, four 391 and 218).
  const int heads = static_cast<int>(a->num_kv_heads) / (x.wide ? 1 : together);
  const int places = std::max(1, kComputeUnits / heads);
  const long long max_keys = a->page_table_columns * a->page_size;
  x.target = x.wide                           ? places
             : 2 * x.max_tiles <= places ? places - static_cast<int>(x.max_tiles) + 1
                                         : 2 * places;
  // Up to half as many tiles as places, one round cuts requests of one length into long
  // chunks and rests; two cut evenly, but pay a second start, which the longer rows and
  // the more tiles make good.  Codes, one round and two, 8 KV heads of 128 (64 places):
  // 20 requests over 8,000 keys 78 and 82 us, 32,768 291 and 282; 24 over 6,000 67 and
  // 71, 8,000 102 and 94, 32,768 358 and 317; 28 over 4,000 55 and 59, 6,000 94 and 84;
  // 31 over 4,000 59 and 58, 5,000 90 and 72; 32 over 2,000 36 and 40, 5,000 94 and 75,
  // 32,768 518 and 424.  10 KV heads (51 places): 13 over 8,000 52 and 72, 22 over 4,000
  // 53 and 58, 6,000 90 and 82.  8 of 256 (32 places): 10 over 16,000 152 and 140, 12 over
  // 3,000 41 and 48, 16 59 and 48 (12 over 4,000 49 and 54: two come early).  So from (places / tiles)^2 times 1,000 keys of 128 on,
  // in the mean of what the call turns out to have, and from a quarter of the places (the
  // cut of 22 and 26 of 64 places suits neither: 312 and 330, 394 and 409 over 32,768).
  // A single tile is cut evenly either way.  (Rows of 16 bits keep one round: unmeasured.)
  const double long_values = 1000.0 * 128 * places * places / static_cast<double>(x.max_tiles);  // of the call's rows
  const bool may_be_long = codes && !x.wide && x.max_tiles > 1 && 2 * x.max_tiles <= places &&
                           4 * x.max_tiles > places &&
                           static_cast<double>(max_keys * a->head_dim * x.max_tiles) >= long_values;
  x.long_work = may_be_long ? long_values / static_cast<double>(kPageTile * a->head_dim) : INFINITY;
  x.long_target = may_be_long ? 2 * places : x.target;
  x.splits = max_keys > x.min_chunk * kPageTile;
  x.max_units = x.max_tiles + (x.splits ? x.long_target + 1 : 0);
  x.max_partials = x.splits ? 2 * x.long_target + 2 : 0;
  x.plan_at = x.max_partials * a->num_kv_heads * x.columns * (a->head_dim + 2);
  x.ws_floats = x.plan_at + (requests > kPlanned ? plan_ints(requests) : 0);
  return x;
}

bool aligned(const void *p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
bool index_code(int64_t dtype) { return dtype == LL_DTYPE_INT32 || dtype == LL_DTYPE_INT64; }

int check_args(const ll_paged_attention_args *a) {
  if (a == nullptr) return fail(LL_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->struct_size != static_cast<int64_t>(sizeof(ll_paged_attention_args)))
    return fail(LL_ERR_INVALID_ARGUMENT, "struct_size %lld, expected %lld", static_cast<long long>(a->struct_size),
                static_cast<long long>(sizeof(ll_paged_attention_args)));
  if (a->num_q_heads < 1 || a->num_kv_heads < 1 || a->num_q_heads > 65535 || a->num_q_heads % a->num_kv_heads != 0)
    return fail(LL_ERR_KV_HEAD_LAYOUT_MISMATCH, "num_q_heads must be a multiple of num_kv_heads, at most 65535");
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256)
    return fail(LL_ERR_HEAD_DIMENSION_OUT_OF_RANGE, "head_dim must be 64, 128 or 256");
  if (a->kv_dtype != LL_DTYPE_FLOAT16 && a->kv_dtype != LL_DTYPE_BFLOAT16)
    return fail(LL_ERR_FP16_OR_BF16_REQUIRED, "kv_dtype must be fp16 or bf16");
  // (In fp32 the scale and kSlack over it are normal numbers: with a scale of 0 the
  // score of a hidden key, -inf, would weigh exp2(-inf * 0).)
  if (!(a->softmax_scale >= 1e-37) || !(a->softmax_scale < 1e30))
    return fail(LL_ERR_INVALID_ARGUMENT, "softmax_scale must be in [1e-37, 1e30)");
  const long long group = a->num_q_heads / a->num_kv_heads;
  if (a->num_queries < 0 || a->num_requests < 0 || a->num_requests > 0x3fffffff ||
      a->num_queries > 0x3fffffff / group)
    return fail(LL_ERR_INVALID_ARGUMENT, "num_queries and num_requests must not be negative and stay below 2^30 "
                "(queries times query heads per KV head)");
  if (a->query_starts == nullptr && a->num_queries != a->num_requests)
    return fail(LL_ERR_INVALID_ARGUMENT, "without query_starts every request has one query");
  if (a->query_starts != nullptr && !index_code(a->query_starts_dtype))
    return fail(LL_ERR_INTEGER_TOKEN_MAPS_REQUIRED, "query_starts dtype");
  if (!index_code(a->kv_lengths_dtype)) return fail(LL_ERR_INTEGER_TOKEN_MAPS_REQUIRED, "kv_lengths dtype");
  if (a->page_size < 1 || a->page_size > 0x3fffffff || a->page_table_columns < 0 ||
      a->page_table_columns > 0x3fffffff / a->page_size)
    return fail(LL_ERR_INVALID_ARGUMENT, "page_size must be positive and a table row hold fewer than 2^30 keys");
  if (a->page_table_stride < 0) return fail(LL_ERR_INVALID_ARGUMENT, "page_table_stride is negative");
  if (a->num_slots < 0 || a->num_slots > 0x7fffffff)
    return fail(LL_ERR_INVALID_ARGUMENT, "num_slots must be in [0, 2^31)");
  if (a->query_token_stride % 8 != 0 || a->query_head_stride % 8 != 0)
    return fail(LL_ERR_INVALID_ARGUMENT, "query strides must be multiples of 8 values");
  if (a->num_queries == 0 || a->num_requests == 0) return LL_OK;
  if (a->query == nullptr || a->output == nullptr || a->kv_lengths == nullptr)
    return fail(LL_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
  if (a->num_slots > 0 && (a->key_buffer == nullptr || a->value_buffer == nullptr))
    return fail(LL_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
  if (a->page_table_columns > 0 && a->page_table == nullptr)
    return fail(LL_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
  if (!aligned(a->query, 16) || !aligned(a->output, 16) || !aligned(a->key_buffer, 16) ||
      !aligned(a->value_buffer, 16))
    return fail(LL_ERR_INVALID_ARGUMENT, "query, output and KV buffers must be 16-byte aligned");
  const Launch x = plan_launch(a);
  // A launch holds fewer than 2^32 threads: at most 512 a unit and KV head, 16 a
  // column.
  if (x.max_units * a->num_kv_heads > 0x7fffffll ||
      x.max_tiles * a->num_kv_heads * x.columns > 0xfffffffll)
    return fail(LL_ERR_INVALID_ARGUMENT, "too many queries for one launch");
  return LL_OK;
}

// The launches in front of and behind a call's kernel.
void launch_plan(const PagedParams &p, const Launch &x, hipStream_t s) {
  if (p.plan != nullptr) paged_plan_kernel<<<1, kPlanThreads, 0, s>>>(p, x.columns);
}

template <int D, typename E>
int launch_join(const PagedParams &p, const Launch &x, hipStream_t s) {
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(LL_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(err));
  if (!x.splits) return LL_OK;
  const unsigned tile_heads = static_cast<unsigned>(x.max_tiles) * static_cast<unsigned>(p.hkv);
  const unsigned columns = static_cast<unsigned>(x.columns);
  // Few tiles of many chunks: a column's chunks on several waves, eight where there
  // may be more than 32 (64 chunks: 6.0 us on eight, 7.2 on four; 16 chunks: 4.9 and
  // 4.4).  Elsewhere a wave for all chunks of its columns: workgroups that mostly
  // find no column cost more than they save (16 requests on tiles of 256 columns).
  // Between the two, by the chunks a tile may have (behind 32,768 keys: 64 tokens of
  // 16/2 heads of 256, 25 chunks a tile, 64 us split and 84 not; 128 of 28/4 heads of
  // 128, 16 chunks, 92 and 83).
  const unsigned split_groups = tile_heads * (columns / Combine<D, 4>::kColumns);
  if (x.target < (split_groups > 4 * kComputeUnits ? 24 : 8) * x.max_tiles)
    paged_combine_kernel<D, E, 1><<<tile_heads * (columns / Combine<D, 1>::kColumns), 256, 0, s>>>(p, x.columns);
  else if (p.max_keys <= 32 * x.min_chunk * kPageTile)
    paged_combine_kernel<D, E, 4><<<split_groups, 4 * kWave, 0, s>>>(p, x.columns);
  else
    paged_combine_kernel<D, E, 8><<<split_groups, 8 * kWave, 0, s>>>(p, x.columns);
  err = hipGetLastError();
  if (err != hipSuccess) return fail(LL_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(err));
  return LL_OK;
}

// The kernels' parameters of a call that check_args took (but for the pool's buffers).
int fill_params(const ll_paged_attention_args *a, const Launch &x, PagedParams *filled) {
  if (x.ws_floats > 0 && (a->workspace == nullptr || a->workspace_bytes < x.ws_floats * 4 || !aligned(a->workspace, 16)))
    return fail(LL_ERR_INVALID_ARGUMENT, "the call needs a 16-byte aligned workspace of %lld bytes",
                static_cast<long long>(x.ws_floats * 4));
  PagedParams &p = *filled;
  p.q = static_cast<const uint16_t *>(a->query);
  p.out = static_cast<uint16_t *>(a->output);
  p.pages = static_cast<const int *>(a->page_table);
  p.kv_lengths = a->kv_lengths;
  p.query_starts = a->query_starts;
  p.ws = static_cast<float *>(a->workspace);
  if (x.ws_floats > x.plan_at) p.plan = reinterpret_cast<int *>(p.ws + x.plan_at);
  p.q_token = a->query_token_stride;
  p.q_head = a->query_head_stride;
  p.pages_stride = a->page_table_stride;
  // key / page_size = key * magic >> shift for every key below 2^31: magic
  // exceeds 2^shift / page_size by at most 1, and 2^(shift - 31) >= page_size.
  int bits = 0;
  while ((1ll << bits) < a->page_size) ++bits;
  p.page_shift = 31 + bits;
  p.page_magic = (1ull << p.page_shift) / static_cast<unsigned long long>(a->page_size) + 1;
  p.page_size = static_cast<int>(a->page_size);
  p.num_pages = static_cast<int>(a->num_slots / a->page_size);
  p.max_keys = static_cast<int>(a->page_table_columns * a->page_size);
  p.num_queries = static_cast<int>(a->num_queries);
  p.num_requests = static_cast<int>(a->num_requests);
  p.hq = static_cast<int>(a->num_q_heads);
  p.hkv = static_cast<int>(a->num_kv_heads);
  p.group = p.hq / p.hkv;
  p.lengths64 = a->kv_lengths_dtype == LL_DTYPE_INT64 ? 1 : 0;
  p.starts64 = a->query_starts_dtype == LL_DTYPE_INT64 ? 1 : 0;
  p.min_chunk = x.splits ? x.min_chunk : kOneChunk;
  p.inv_target = 1.0 / x.target;
  p.long_work = x.long_work;
  p.inv_long_target = 1.0 / x.long_target;
  p.max_partials = x.max_partials;
  p.scale_log2 = static_cast<float>(a->softmax_scale * 1.4426950408889634);  // log2(e)
  return LL_OK;
}

}  // namespace

#endif  // PAGED_DEVICE_H
