// Attention of each request's new tokens over its pages of the KV pool, on
// gfx950 (MI355X).
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
//
// Per 32 or 64 keys, with S^T = K Q^T and O^T += V^T P^T on MFMAs: K and V rows
// are gathered by slot straight into LDS; the softmax runs in fp32 with exp2
// and a maximum that is only raised where a score passes it by 8 (in log2);
// the probabilities go from the S^T accumulators to the value product rounded
// to the KV type, V^T through transposed LDS reads.  That rounding is the price of
// the matrix unit, which takes both operands of one 16-bit type: a second product
// with what the rounding leaves would be half as many MFMAs again (and 0 times an
// infinity a NaN).  The sums are of the rounded weights, so a constant comes back as
// it is; of random values the results are 1.1 to 1.4 times as far from 64 bits as a
// single rounding of the output (bf16 0.0018-0.0024 of their norm against 0.0017,
// fp16 0.00029 against 0.00021).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <type_traits>

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
  return __builtin_amdgcn_readfirstlane(
      max(p.min_chunk, static_cast<int>(min(ceil(work * p.inv_target - 1e-6), 33554432.0))));
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

// Up to 16 columns: single tokens, bound by reading the keys and values once.  The
// waves of a workgroup take turns at its 32-key subtiles, each through an LDS ring
// of its own (no barriers: a wave waits for its own gathers alone), and join their
// results at the end.  131,072 keys of 4 heads of 128: 47.5 us, 5.65 TB/s (a read-only
// pass reaches 6.0); 64 uneven requests, 2.13 GB: 391 us, 5.5 TB/s; 2,048 keys
// 7.7 us, the latencies of the lengths, the pages, the rows and the join.
// v_mfma_f32_16x16x32, lane layouts: A and B lane l element e -> row / column
// l % 16, k = 8 (l / 16) + e; accumulator register r -> row 4 (l / 16) + r, column
// l % 16.  The value product's k order is the scores' register order: k = 8 g + e
// is token 4 g + e (e < 4) or 16 + 4 g + e - 4.
// LDS rows are token-major with their 16-byte chunks swizzled by token, so that
// the 16 lanes of a K read (16 tokens, one chunk) and the 32 lanes of a
// transposed V read (8 tokens x 32 bytes) each cover the 64 banks once.
template <int D>
struct Narrow {
  static constexpr int kKeys = 32;
  static constexpr int kWaves = D == 256 ? 2 : 4;
  static constexpr int kStages = D == 64 ? 4 : 2;  // 128 KB of rings
  static constexpr int kThreads = kWaves * kWave;
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kHalf = kKeys * kRowBytes;  // a subtile's K or V rows
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kChunksPerRow = D / 8;
  static constexpr int kGathers = kHalf / (16 * kWave);  // of K and of V, per subtile
  static constexpr int kList = 4096;                     // slots held at a time
  __device__ static int k_swizzle(int t) { return D >= 128 ? t % 16 : (t / 2) % 8; }
  __device__ static int v_swizzle(int t) { return D >= 128 ? 2 * (t % 8) : 2 * ((t / 2) % 4); }
};

template <int D, typename E>
__global__ void __launch_bounds__(Narrow<D>::kThreads) paged_narrow_kernel(const PagedParams p) {
  typedef Narrow<D> N;
  typedef typename E::frag frag;
  constexpr int kColumns = 16;
  constexpr int kKSteps = D / 32;
  constexpr int kBlocks = D / 16;
  constexpr int kPitch = D + 4;  // floats of a joined row: 16 lanes' 16-byte writes meet 64 banks
  static_assert(N::kWaves * 16 * kPitch * 4 <= N::kWaves * N::kRing, "a tile's results fit the rings");
  __shared__ __attribute__((aligned(16))) unsigned char rings[N::kWaves * N::kRing];
  __shared__ int slot_list[N::kList];
  __shared__ float stats[N::kWaves][kColumns][2];

  const int head = blockIdx.x % p.hkv;
  const int unit = blockIdx.x / p.hkv;
  const Work w = find_work<Order::kByQuarter>(p, kColumns, unit);
  if (w.index < 0 || w.chunk >= w.chunks || (w.chunks > 1 && !partials_fit(p, w))) return;
  const int key_begin = w.chunk * w.chunk_keys;  // below the tile's key_end, or 0
  int key_end = key_begin + min(w.chunk_keys, w.key_end - key_begin);
  if (p.num_pages == 0) key_end = key_begin;  // no row that may be read

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int lane = tid % kWave;
  const int g = lane / 16;
  const int col = lane % 16;
  unsigned char *ring = rings + wave * N::kRing;

  // The lane's column and its query.
  const int column = w.tile * kColumns + col;
  const int token = column / p.group;
  const bool exists = token < w.request.q_len;
  const int pos = exists ? w.request.kv_len - w.request.q_len + token : -1;
  // Keys below it are visible to every column (to the first one, that is).
  const int seen_by_all = w.request.kv_len - w.request.q_len + (w.tile * kColumns) / p.group + 1;
  frag qf[kKSteps];
  {
    const int q_head = head * p.group + (column - token * p.group);
    const uint16_t *row =
        p.q + (static_cast<long long>(w.request.q_start) + token) * p.q_token + q_head * p.q_head + 8 * g;
#pragma unroll
    for (int ks = 0; ks < kKSteps; ++ks) {
      u32x4 bits = u32x4{0u, 0u, 0u, 0u};
      if (exists) bits = *reinterpret_cast<const u32x4 *>(row + 32 * ks);
      qf[ks] = __builtin_bit_cast(frag, bits);
    }
  }

  float m = -INFINITY, l = 0.f;
  bool large = false;  // of a column of the wave
  f32x4 o[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) o[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  const float scale_log2 = p.scale_log2;
  const float slack = kSlack / scale_log2;

  // The lane's share of a gather: its 16 bytes of instruction j hold chunk
  // (64 j + lane) of the subtile's rows in LDS order.
  const unsigned char *k_base = reinterpret_cast<const unsigned char *>(p.k + static_cast<long long>(head) * D);
  const unsigned char *v_base = reinterpret_cast<const unsigned char *>(p.v + static_cast<long long>(head) * D);
  auto gather = [&](int sub, int stage) {
    unsigned char *dst = ring + stage * N::kStage;
#pragma unroll
    for (int j = 0; j < N::kGathers; ++j) {
      const int at = j * kWave + lane;
      const int token = at / N::kChunksPerRow;
      const int place = at % N::kChunksPerRow;
      const int slot = max(slot_list[sub * N::kKeys + token], 0);
      dma_pair(row_at(p, k_base + 16 * (place ^ N::k_swizzle(token)), slot), dst + j * 16 * kWave,
               row_at(p, v_base + 16 * (place ^ N::v_swizzle(token)), slot), dst + N::kHalf + j * 16 * kWave);
    }
  };
  // Offsets of the lane's fragments within a stage.
  int k_off[kKSteps];
#pragma unroll
  for (int ks = 0; ks < kKSteps; ++ks) k_off[ks] = col * N::kRowBytes + (((4 * ks + g) ^ N::k_swizzle(col)) * 16);
  const int v_token = 4 * g + col / 4;
  int v_off[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
    v_off[b] = N::kHalf + v_token * N::kRowBytes + (((2 * b + (col % 4) / 2) ^ N::v_swizzle(v_token)) * 16) + 8 * (col % 2);
  const unsigned ring_lds =
      static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char *)ring));

  const int *pages = p.pages + static_cast<long long>(w.index) * p.pages_stride;
  for (int list_begin = key_begin; list_begin < key_end; list_begin += N::kList) {
    const int listed = min(key_end - list_begin, N::kList);
    const int subs = (listed + N::kKeys - 1) / N::kKeys;
    __syncthreads();  // every wave is past the former list
    for (int i = tid; i < subs * N::kKeys; i += N::kThreads) {
      const unsigned key = static_cast<unsigned>(list_begin + min(i, listed - 1));
      const unsigned page = static_cast<unsigned>((key * p.page_magic) >> p.page_shift);
      const int entry = pages[page];
      const bool valid = i < listed && static_cast<unsigned>(entry) < static_cast<unsigned>(p.num_pages);
      slot_list[i] = valid ? entry * p.page_size + static_cast<int>(key - page * p.page_size) : -1;
    }
    // The compiler does not count the gathers: nothing that it waits for in the
    // loop below may be left in flight.
    wait_vm<0>();
    __syncthreads();

#pragma unroll
    for (int s = 0; s < N::kStages; ++s)
      if (wave + s * N::kWaves < subs) gather(wave + s * N::kWaves, s);
    int stage = 0;
    for (int sub = wave; sub < subs; sub += N::kWaves) {
      const int key0 = list_begin + sub * N::kKeys;
      const int own_slot = slot_list[sub * N::kKeys + lane % N::kKeys];
      const unsigned valid =
          static_cast<unsigned>(__builtin_amdgcn_ballot_w64(own_slot >= 0));  // both halves hold the same keys
      // This stage's gathers are complete when at most the later stages' are outstanding.
      const int later = min(N::kStages - 1, (subs - 1 - sub) / N::kWaves);
      if (N::kStages == 4 && later == 3) wait_vm<3 * 2 * N::kGathers % 64>();
      else if (N::kStages == 4 && later == 2) wait_vm<2 * 2 * N::kGathers % 64>();
      else if (later >= 1) wait_vm<2 * N::kGathers>();
      else wait_vm<0>();
      asm volatile("" ::: "memory");
      unsigned char *rows = ring + stage * N::kStage;
      const bool whole = valid == 0xffffffffu && key0 + N::kKeys <= seen_by_all;
      if (valid != 0xffffffffu) {
        // Rows that no column sees may hold anything: zeros in their place.
        for (int c = lane; c < N::kKeys * N::kChunksPerRow; c += kWave)
          if (((valid >> (c / N::kChunksPerRow)) & 1u) == 0)
            *reinterpret_cast<u32x4 *>(rows + N::kHalf + c * 16) = u32x4{0u, 0u, 0u, 0u};
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
        asm volatile("" ::: "memory");
      }
      unsigned odd = 0;  // rows whose values are not all finite, where some columns do not see the subtile whole
      if (key0 + N::kKeys > seen_by_all && seen_by_all < w.key_end) {
        for (int c = lane; c < N::kKeys * N::kChunksPerRow; c += kWave) {
          u32x4 *chunk = reinterpret_cast<u32x4 *>(rows + N::kHalf + c * 16);
          if (any_nonfinite<E>(*chunk)) {
            odd |= 1u << (c / N::kChunksPerRow);
            *chunk = finite_only<E>(*chunk);
          }
        }
        if (__builtin_amdgcn_ballot_w64(odd != 0) != 0) {
#pragma unroll
          for (int step = 1; step < kWave; step *= 2) odd |= __shfl_xor(odd, step);
        }
        odd = __builtin_amdgcn_readfirstlane(odd);
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
        asm volatile("" ::: "memory");
      }

      f32x4 s[2];
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) s[rb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < kKSteps; ++ks)
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
          const frag kf = *reinterpret_cast<const frag *>(rows + k_off[ks] + rb * 16 * N::kRowBytes);
          s[rb] = E::mfma16(kf, qf[ks], s[rb]);
        }
      if (!whole) {
#pragma unroll
        for (int rb = 0; rb < 2; ++rb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int rel = 16 * rb + 4 * g + r;
            const bool visible = ((valid >> rel) & 1u) != 0 && key0 + rel <= pos;
            s[rb][r] = visible ? s[rb][r] : -INFINITY;
          }
      }
      float top = -INFINITY;
#pragma unroll
      for (int rb = 0; rb < 2; ++rb)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, s[rb][r]);
      top = max_of_groups(top);
      const bool raise = top > m + slack;
      const float m_new = raise ? top : m;
      const float bias = m_new == -INFINITY ? 0.f : weight_bias<E>(m_new, scale_log2);  // nothing seen yet: all weights 0
      if (__builtin_amdgcn_ballot_w64(raise) != 0) {
        const float alpha = raise ? __builtin_amdgcn_exp2f((m - m_new) * scale_log2) : 1.f;
        l *= alpha;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) o[b] *= alpha;
        large = __builtin_amdgcn_ballot_w64(is_large(bias)) != 0;
      }
      m = m_new;
      const float top_seen = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int rb = 0; rb < 2; ++rb)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          s[rb][r] = __builtin_amdgcn_exp2f(large ? __builtin_fmaf(s[rb][r] - top_seen, scale_log2, E::kWeightShift)
                                                  : __builtin_fmaf(s[rb][r], scale_log2, bias));
      u32x4 weights;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        weights[j] = E::pack(s[j / 2][2 * (j % 2)], s[j / 2][2 * (j % 2) + 1]);
        l = E::dot2_ones(weights[j], l);  // the weights that the value product sees
      }
      const frag pb = __builtin_bit_cast(frag, weights);
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const unsigned at = ring_lds + stage * N::kStage + v_off[b];
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_i16x4 *>(static_cast<uintptr_t>(at)));
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            reinterpret_cast<lds_i16x4 *>(static_cast<uintptr_t>(at + 16 * N::kRowBytes)));
        u32x4 va;
        va[0] = __builtin_bit_cast(u32x2, lo)[0];
        va[1] = __builtin_bit_cast(u32x2, lo)[1];
        va[2] = __builtin_bit_cast(u32x2, hi)[0];
        va[3] = __builtin_bit_cast(u32x2, hi)[1];
        o[b] = E::mfma16(__builtin_bit_cast(frag, va), pb, o[b]);
      }
      while (odd != 0) {
        const int rel = __builtin_ctz(odd);
        odd &= odd - 1;
        const unsigned char *row = row_at(p, v_base, slot_list[sub * N::kKeys + rel]) + 8 * g;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          const f32x4 x = nonfinite_only<E>(*reinterpret_cast<const u32x2 *>(row + 32 * b));
          if (key0 + rel <= pos) o[b] += x;
          __builtin_amdgcn_sched_barrier(0);  // (rare: few registers rather than loads in flight)
        }
      }
      // The stage's reads are done: the gather kStages turns ahead takes it.
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (sub + N::kStages * N::kWaves < subs) gather(sub + N::kStages * N::kWaves, stage);
      stage = stage + 1 == N::kStages ? 0 : stage + 1;
    }
  }

  // The waves' results joined.
  const bool direct = w.chunks == 1;
  float *partial = direct ? nullptr : partial_of<D>(p, kColumns, w.first_partial + w.chunk * w.partial_step, head);
  float *joined = reinterpret_cast<float *>(rings);
  __syncthreads();  // the rings are read
  const float total = sum_of_groups(l);
  if (g == 0) {
    stats[wave][col][0] = m;
    stats[wave][col][1] = total;
  }
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
    *reinterpret_cast<f32x4 *>(joined + (wave * 16 + col) * kPitch + 16 * b + 4 * g) = o[b];
  __syncthreads();
  for (int i = tid; i < 16 * (D / 4); i += N::kThreads) {
    const int c = i / (D / 4);
    const int quad = i % (D / 4);
    if ((w.tile * kColumns + c) / p.group >= w.request.q_len) continue;
    float top = stats[0][c][0];
#pragma unroll
    for (int v = 1; v < N::kWaves; ++v) top = fmaxf(top, stats[v][c][0]);
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < N::kWaves; ++v) {
      const float weight = joined_weight(stats[v][c][0], top, scale_log2);
      sum += weight * stats[v][c][1];
      acc += weight * *reinterpret_cast<const f32x4 *>(joined + (v * 16 + c) * kPitch + 4 * quad);
    }
    if (direct) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing is zero
      u32x2 packed;
      packed[0] = E::pack(acc[0] * inv, acc[1] * inv);
      packed[1] = E::pack(acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<u32x2 *>(output_row(p, w, head, w.tile * kColumns + c, D) + 4 * quad) = packed;
    } else {
      *reinterpret_cast<f32x4 *>(partial + c * D + 4 * quad) = acc;
      if (quad == 0) {
        partial[kColumns * D + 2 * c] = top;
        partial[kColumns * D + 2 * c + 1] = sum;
      }
    }
  }
}

// Many columns: chunks, bound by the matrix products.  Eight waves of 32 columns
// each (four at head dim 256, whose registers do not leave room for a second wave
// per SIMD) share every gathered tile of 64 keys.  2,048 queries behind 4,096 to
// 32,768 keys take, per tile of 64 keys (from the difference of two lengths), 1.82 us
// at head dim 128, the matrix unit's rate in a library product of 8192^3 (1.17
// PFLOP/s), 1.91 at 256 (1.13 PFLOP/s) and 1.23 at 64 (0.87 PFLOP/s; the products
// alone would be 0.92, and what the rest is has not been found); 27 to 39 us a call do
// not grow with the keys (starts of the units, their unevenness, the join).  28/4 heads
// of 128 over 32,768 keys: 812 us.  v_mfma_f32_32x32x16, lane layouts: A and B lane l
// element e -> row / column l % 32, k = 8 (l / 32) + e; accumulator register r -> row
// 8 (r / 4) + 4 (l / 32) + r % 4, column l % 32.  The value product's k order is the
// scores' register order.
//
// A tile is two phases, the products (the values of tile t - 1, the scores of
// tile t) and the softmax, about as long as each other: the products keep the
// matrix unit busy for 1,024 cycles at head dim 128, the softmax the vector unit
// for about 900.  With two waves per SIMD in step, both would want the same
// unit; so the second half of the waves runs one phase behind the first (one
// barrier more in front), and a SIMD's waves alternate.
//
// LDS: K and V rings of kStages tiles, rows token-major with their 16-byte chunks
// swizzled by token as in the narrow kernel (for 32 lanes of 4 tokens x 64 bytes
// a transposed read).  Iteration t is the softmax of tile t, then the products:
// the values of tile t, the scores of tile t + 1.  Before its first barrier a
// wave waits for its share of V tile t and K tile t + 1; behind it, it issues its
// share of K tile t + kLead and V tile t + kLead - 1.  Their stages held K tile t -
// 1 and V tile t - 2 (four stages; the waves one phase behind have left them too),
// or K tile t and V tile t - 1 (two stages, all waves in step).
template <int D>
struct Wide {
  static constexpr int kKeys = 64;
  static constexpr int kWaves = D == 256 ? 4 : 8;
  static constexpr int kStages = D == 256 ? 2 : 4;
  static constexpr int kLead = D == 256 ? 2 : 3;  // tiles that K gathers run ahead
  static constexpr int kThreads = kWaves * kWave;
  static constexpr int kColumns = 32 * kWaves;
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kStage = kKeys * kRowBytes;
  static constexpr int kChunksPerRow = D / 8;
  static constexpr int kGathers = kStage / (16 * kWave) / kWaves;  // a wave's, of K and of V, per tile
  static constexpr int kList = 7168;                               // slots held at a time
  __host__ __device__ static constexpr int k_swizzle(int t) { return D >= 128 ? t % 16 : (t / 2) % 8; }
  __host__ __device__ static constexpr int v_swizzle(int t) { return D >= 128 ? 4 * (t % 4) : 4 * ((t / 2) % 2); }
};

template <int D, typename E>
__global__ void __launch_bounds__(Wide<D>::kThreads) paged_wide_kernel(const PagedParams p) {
  typedef Wide<D> W;
  typedef typename E::frag frag;
  constexpr int kKSteps = D / 16;
  constexpr int kBlocks = D / 32;
  constexpr int kLead = W::kLead;
  __shared__ __attribute__((aligned(16))) unsigned char k_ring[W::kStages * W::kStage];
  __shared__ __attribute__((aligned(16))) unsigned char v_ring[W::kStages * W::kStage];
  __shared__ int slot_list[W::kList];
  __shared__ unsigned long long tile_valid[W::kList / W::kKeys];
  __shared__ unsigned odd_rows[W::kList / 32];  // a bit per key: values that are not all finite

  const int head = blockIdx.x % p.hkv;
  const int unit = blockIdx.x / p.hkv;
  const Work w = find_work<Order::kByLength>(p, W::kColumns, unit);
  if (w.index < 0 || w.chunk >= w.chunks || (w.chunks > 1 && !partials_fit(p, w))) return;
  const int key_begin = w.chunk * w.chunk_keys;  // below the tile's key_end, or 0
  int key_end = key_begin + min(w.chunk_keys, w.key_end - key_begin);
  if (p.num_pages == 0) key_end = key_begin;  // no row that may be read

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int lane = tid % kWave;
  const int h = lane / 32;
  const int col = lane % 32;

  // The lane's column.
  const int column = w.tile * W::kColumns + 32 * wave + col;
  const int token = column / p.group;
  const bool exists = token < w.request.q_len;
  const int first_pos = w.request.kv_len - w.request.q_len;  // of the request's query 0
  const int pos = exists ? first_pos + token : -1;
  // Of the wave's columns: keys that all of them see, keys that any of them sees.
  const int wave_first = (w.tile * W::kColumns + 32 * wave) / p.group;
  const int wave_last = min(w.request.q_len - 1, (w.tile * W::kColumns + 32 * wave + 31) / p.group);
  const bool wave_computes = wave_first < w.request.q_len;
  // Keys from here on are not seen by every column of the workgroup (none, where all stand at one position).
  const int tile_first_seen = first_pos + (w.tile * W::kColumns) / p.group + 1;
  const int seen_in_part = tile_first_seen < w.key_end ? tile_first_seen : 0x7fffffff;
  const int seen_by_all = first_pos + wave_first + 1;
  const int wave_stop = wave_computes ? min(key_end, first_pos + wave_last + 1) : key_begin;

  frag qf[kKSteps];
  {
    const int q_head = head * p.group + (column - token * p.group);
    const uint16_t *row =
        p.q + (static_cast<long long>(w.request.q_start) + token) * p.q_token + q_head * p.q_head + 8 * h;
#pragma unroll
    for (int ks = 0; ks < kKSteps; ++ks) {
      u32x4 bits = u32x4{0u, 0u, 0u, 0u};
      if (exists) bits = *reinterpret_cast<const u32x4 *>(row + 16 * ks);
      qf[ks] = __builtin_bit_cast(frag, bits);
    }
  }

  float m = -INFINITY;
  bool large = false;  // of a column of the wave
  float l4[4] = {0.f, 0.f, 0.f, 0.f};  // the weights' sum, in four chains: a dot product waits for the one before
  f32x16 o[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[b][r] = 0.f;
  const float scale_log2 = p.scale_log2;
  const float slack = kSlack / scale_log2;

  // The wave's share of a tile's gathers: instruction j fills the 64 16-byte
  // chunks from 64 (kGathers wave + j) on.  Its rows are kRows j further than
  // instruction 0's, which changes their swizzles by an xor (tokens of a wave begin
  // at a multiple of kGathers kRows).
  const unsigned char *k_base = reinterpret_cast<const unsigned char *>(p.k + static_cast<long long>(head) * D);
  const unsigned char *v_base = reinterpret_cast<const unsigned char *>(p.v + static_cast<long long>(head) * D);
  constexpr int kRows = kWave / W::kChunksPerRow;
  const int g_token = W::kGathers * wave * kRows + lane / W::kChunksPerRow;
  unsigned g_k = 16 * ((lane % W::kChunksPerRow) ^ W::k_swizzle(g_token));  // the lane's bytes of a row
  unsigned g_v = 16 * ((lane % W::kChunksPerRow) ^ W::v_swizzle(g_token));
  const int share = W::kGathers * wave * kWave * 16;  // the wave's first byte of a stage
  auto slot_of = [&](int tile, int j) __attribute__((always_inline)) {
    return slot_list[tile * W::kKeys + g_token + j * kRows];
  };
  // Gather j of a tile, in three steps that can go between MFMAs: the row's address,
  // the lane's part of it, the load.
  const unsigned k_lds = lds_offset(k_ring) + share, v_lds = lds_offset(v_ring) + share;
  const unsigned char *gather_from;
  auto gather_step = [&](int step, auto values_tag, int slot, int stage, int j) __attribute__((always_inline)) {
    constexpr bool values = decltype(values_tag)::value;
    unsigned &g = values ? g_v : g_k;
    if (step == 0) gather_from = row_at(p, values ? v_base : k_base, slot);
    if (step == 1) {
      asm volatile("" : "+v"(g));  // (made per use: fewer registers over the loop)
      gather_from += g ^ (16u * (values ? W::v_swizzle(j * kRows) : W::k_swizzle(j * kRows)));
    }
    if (step == 2) dma_row(gather_from, (values ? v_lds : k_lds) + stage * W::kStage + j * kWave * 16);
    else asm volatile("" : "+v"(gather_from));  // (made here)
  };
  auto gather_k = [&](int slot, int stage, int j) __attribute__((always_inline)) {
#pragma unroll
    for (int step = 0; step < 3; ++step) gather_step(step, std::false_type{}, slot, stage, j);
  };
  auto gather_v = [&](int slot, int stage, int j) __attribute__((always_inline)) {
#pragma unroll
    for (int step = 0; step < 3; ++step) gather_step(step, std::true_type{}, slot, stage, j);
  };

  // Offsets of the lane's fragments within a stage.
  // Step ks of the scores reads chunk 2 ks + h, at (2 ks + h) ^ swizzle = (h ^
  // swizzle) ^ 2 ks: an xor of the offset's bits 5 on with ks.
  static_assert(W::kRowBytes >= 2 * 16 * kKSteps, "ks stays within the row's bits");
  const int k_off = col * W::kRowBytes + ((h ^ W::k_swizzle(col)) * 16);
  const int li = lane % 16;
  const int v_token = 4 * h + li / 4;
  unsigned v_off[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const int chunk = 4 * b + 2 * ((lane / 16) % 2) + (li % 4) / 2;
    v_off[b] = lds_offset(v_ring) + v_token * W::kRowBytes + (chunk ^ W::v_swizzle(v_token)) * 16 + 8 * (li % 2);
    asm volatile("" : "+v"(v_off[b]));
  }

  f32x16 s[2];
  frag pb[4];

  // The products: the values of the tile that pb weighs (stage v_stage) onto O^T,
  // the scores of the next (stage k_stage) into s.  A wave's instructions issue in
  // order and an MFMA takes 32 cycles, so everything else goes between them, a
  // little behind each: fragments are read one batch ahead of the MFMAs that take
  // them (of the values two transposed reads a dim block of a 16-key step, keys 16
  // step + 4 h .. + 3 and, 8 further, the second read; of the scores a chunk of
  // each 32-key block's rows for each of two 16-dim steps), and beside(i) is called
  // behind MFMA i.
  constexpr int kMfmas = 4 * kBlocks + 2 * kKSteps;
  static_assert(kMfmas % (2 * W::kGathers) == 0 && kMfmas / (2 * W::kGathers) >= 3, "a place for every step of a gather");
  auto products = [&](int v_stage, int k_stage, auto values_tag, auto beside) __attribute__((always_inline)) {
    auto fence = [] { __builtin_amdgcn_sched_barrier(0); };  // the order below, kept
    constexpr bool values = decltype(values_tag)::value;  // else scores alone
    constexpr int kBatches = kKSteps / 2;
    const unsigned char *rows = k_ring + k_stage * W::kStage;
    int k_at = k_off;
    asm volatile("" : "+v"(k_at));  // the steps' offsets made per tile: eight registers fewer over the loop
    u32x4 vf[2][kBlocks];
    frag kf[2][4];
    auto load_v = [&](int step, int b) __attribute__((always_inline)) {
      const unsigned at = v_off[b] + v_stage * W::kStage + 16 * step * W::kRowBytes;
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_i16x4 *>(static_cast<uintptr_t>(at)));
      const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          reinterpret_cast<lds_i16x4 *>(static_cast<uintptr_t>(at + 8 * W::kRowBytes)));
      vf[step % 2][b][0] = __builtin_bit_cast(u32x2, lo)[0];
      vf[step % 2][b][1] = __builtin_bit_cast(u32x2, lo)[1];
      vf[step % 2][b][2] = __builtin_bit_cast(u32x2, hi)[0];
      vf[step % 2][b][3] = __builtin_bit_cast(u32x2, hi)[1];
    };
    auto load_k = [&](int batch, int i) __attribute__((always_inline)) {
      kf[batch % 2][i] = *reinterpret_cast<const frag *>(rows + (k_at ^ (32 * (2 * batch + i / 2))) + (i % 2) * 32 * W::kRowBytes);
    };
    if constexpr (values) {
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) load_v(0, b);
      fence();
#pragma unroll
      for (int step = 0; step < 4; ++step)
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          o[b] = E::mfma32(__builtin_bit_cast(frag, vf[step % 2][b]), pb[step], o[b]);
          if (step + 1 < 4) {
            load_v(step + 1, b);
          } else {
#pragma unroll
            for (int i = 4 * b / kBlocks; i < 4 * (b + 1) / kBlocks; ++i) load_k(0, i);
          }
          beside(kBlocks * step + b);
          fence();
        }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) load_k(0, i);
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
#pragma unroll
    for (int batch = 0; batch < kBatches; ++batch)
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // (dims 16 (2 batch + i / 2) on of block i % 2)
        s[i % 2] = E::mfma32(kf[batch % 2][i], qf[2 * batch + i / 2], s[i % 2]);
        if (batch + 1 < kBatches) load_k(batch + 1, i);
        beside(4 * kBlocks + 4 * batch + i);
        fence();
      }
  };
  // The weights of the scores in s, into pb; the sums so far rescaled where the maximum rises.
  auto weigh_tile = [&](int key0, unsigned long long valid) __attribute__((always_inline)) {
    const bool whole = valid == ~0ull && key0 + W::kKeys <= seen_by_all;
    if (!whole) {
      // Register r of block kb: key 32 kb + 8 (r / 4) + 4 h + r % 4.
      const int limit = pos - key0 - 4 * h;
      const unsigned long long lane_valid = valid >> (4 * h);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int rel = 32 * kb + 8 * (r / 4) + r % 4;
          const bool visible = rel <= limit && ((lane_valid >> rel) & 1ull) != 0;
          s[kb][r] = visible ? s[kb][r] : -INFINITY;
        }
    }
    float top = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[kb][r]);
    {
      unsigned a = __builtin_bit_cast(unsigned, top), b = a;
      permlane32_swap(a, b);
      top = max_f32(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
    }
    const bool raise = top > m + slack;
    const float m_new = raise ? top : m;
    const float bias = m_new == -INFINITY ? 0.f : weight_bias<E>(m_new, scale_log2);  // nothing seen yet: all weights 0
    if (__builtin_amdgcn_ballot_w64(raise) != 0) {
      const float alpha = raise ? __builtin_amdgcn_exp2f((m - m_new) * scale_log2) : 1.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) l4[i] *= alpha;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) o[b] *= alpha;
      large = __builtin_amdgcn_ballot_w64(is_large(bias)) != 0;
    }
    m = m_new;
    if (!large) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[kb][r] = __builtin_fmaf(s[kb][r], scale_log2, bias);
    } else {
      const float top_seen = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[kb][r] = __builtin_fmaf(s[kb][r] - top_seen, scale_log2, E::kWeightShift);
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kb][r] = __builtin_amdgcn_exp2f(s[kb][r]);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        u32x4 bits;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          bits[j] = E::pack(s[kb][8 * st + 2 * j], s[kb][8 * st + 2 * j + 1]);
          l4[j] = E::dot2_ones(bits[j], l4[j]);  // the weights that the value product sees
        }
        pb[2 * kb + st] = __builtin_bit_cast(frag, bits);
      }
  };

  const int *pages = p.pages + static_cast<long long>(w.index) * p.pages_stride;
  const bool behind = W::kWaves == 8 && wave >= W::kWaves / 2;  // one phase behind the others
  for (int list_begin = key_begin; list_begin < key_end; list_begin += W::kList) {
    const int listed = min(key_end - list_begin, W::kList);
    const int tiles = (listed + W::kKeys - 1) / W::kKeys;
    __syncthreads();  // every wave is past the former list and its tiles
    for (int i = tid; i < tiles * W::kKeys; i += W::kThreads) {
      const unsigned key = static_cast<unsigned>(list_begin + min(i, listed - 1));
      const unsigned page = static_cast<unsigned>((key * p.page_magic) >> p.page_shift);
      const int entry = pages[page];
      const bool valid = i < listed && static_cast<unsigned>(entry) < static_cast<unsigned>(p.num_pages);
      // (A key without a row: slot 0, which the tile's bits keep out.)
      slot_list[i] = valid ? entry * p.page_size + static_cast<int>(key - page * p.page_size) : 0;
      const unsigned long long bits = __builtin_amdgcn_ballot_w64(valid);  // whole tiles: the loop strides by waves
      if (lane == 0) tile_valid[i / W::kKeys] = bits;
    }
    for (int i = tid; i < 2 * tiles; i += W::kThreads) odd_rows[i] = 0;
    // The compiler does not count the gathers: nothing that it waits for in the
    // loop below may be left in flight.
    wait_vm<0>();
    __syncthreads();

    // K tiles 0 .. kLead - 1 and V tiles 0 .. kLead - 2.  (Past the last tile the
    // last is gathered again, into stages that no products take: every iteration
    // issues the same count, without branches.)
    const int last = tiles - 1;
#pragma unroll
    for (int t = 0; t < kLead; ++t) {
      int slots[W::kGathers];
#pragma unroll
      for (int j = 0; j < W::kGathers; ++j) slots[j] = slot_of(min(t, last), j);
#pragma unroll
      for (int j = 0; j < W::kGathers; ++j) gather_k(slots[j], t % W::kStages, j);
      if (t + 1 < kLead) {
#pragma unroll
        for (int j = 0; j < W::kGathers; ++j) gather_v(slots[j], t, j);
      }
    }
    // K tile 0 is there once the rest, issued after it, is all that is outstanding
    // (kLead - 1 tiles of each).
    wait_vm<2 * W::kGathers * (kLead - 1)>();
    workgroup_barrier();
    if (behind) workgroup_barrier();
    if (list_begin < wave_stop) products(0, 0, std::false_type{}, [](int) {});
    // Bits of keys with a row, the same in every lane.
    auto uniform = [](unsigned long long bits) __attribute__((always_inline)) {
      // readfirstlane returns int: each half goes through unsigned.
      const unsigned lo = static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<unsigned>(bits))));
      const unsigned hi = static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<unsigned>(bits >> 32))));
      return (static_cast<unsigned long long>(hi) << 32) | lo;
    };
    // The wave's share of V tile t, gathered, as the products may take it.
    auto settle_values = [&](int t, int stage, unsigned long long valid) __attribute__((always_inline)) {
      unsigned char *own = v_ring + stage * W::kStage + share + lane * 16;
      if (valid != ~0ull) {
        // Rows that no column sees may hold anything: zeros in their place.
#pragma unroll
        for (int j = 0; j < W::kGathers; ++j)
          if (((valid >> (g_token + j * kRows)) & 1ull) == 0)
            *reinterpret_cast<u32x4 *>(own + j * kWave * 16) = u32x4{0u, 0u, 0u, 0u};
      }
      if (list_begin + (t + 1) * W::kKeys > seen_in_part) {
#pragma unroll 1
        for (int j = 0; j < W::kGathers; ++j) {
          u32x4 *chunk = reinterpret_cast<u32x4 *>(own + j * kWave * 16);
          if (any_nonfinite<E>(*chunk)) {
            *chunk = finite_only<E>(*chunk);
            const int row = g_token + j * kRows;
            atomicOr(&odd_rows[2 * t + row / 32], 1u << (row % 32));
          }
        }
      }
    };
    // Eight waves, one half a phase behind the other.  What a tile needs from the
    // slot list is read during the softmax before it: between the products and the
    // barrier behind them a wave only waits.
    int k_slots[W::kGathers], v_slots[W::kGathers];
    unsigned long long valid = uniform(tile_valid[0]);
    auto iteration = [&](const int t, auto stage_tag) __attribute__((always_inline)) {
      constexpr int stage = decltype(stage_tag)::value;  // t % kStages
      const int key0 = list_begin + t * W::kKeys;
      const bool computes = key0 < wave_stop;
      // The share of K tile t + 1 and V tile t: all but what the last kLead - 2
      // iterations issued.
      wait_vm<2 * W::kGathers * (kLead - 2)>();
      settle_values(t, stage, valid);
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the wave's reads and writes of the stages are done
      __builtin_amdgcn_sched_barrier(0);
      workgroup_barrier();
#pragma unroll
      for (int j = 0; j < W::kGathers; ++j) {
        k_slots[j] = slot_of(min(t + kLead, last), j);
        v_slots[j] = slot_of(min(t + kLead - 1, last), j);
      }
      const unsigned long long next_bits = tile_valid[min(t + 1, last)];
      if (computes) weigh_tile(key0, valid);
      valid = uniform(next_bits);
      __builtin_amdgcn_sched_barrier(0);
      workgroup_barrier();
      auto gather = [&](int step, int i) __attribute__((always_inline)) {
        if (i % 2 == 0) gather_step(step, std::false_type{}, k_slots[i / 2], (stage + kLead) % W::kStages, i / 2);
        else gather_step(step, std::true_type{}, v_slots[i / 2], (stage + kLead - 1) % W::kStages, i / 2);
      };
      constexpr int kApart = kMfmas / (2 * W::kGathers);  // MFMAs from one gather to the next
      __builtin_amdgcn_s_setprio(1);
      // (Behind the wave's last tile the scores are of an old stage, and not used.)
      if (computes) {
        products(stage, (stage + 1) % W::kStages, std::true_type{}, [&](int i) __attribute__((always_inline)) {
          if (i % kApart < 3) gather(i % kApart, i / kApart);
        });
      } else {
#pragma unroll
        for (int i = 0; i < 6 * W::kGathers; ++i) gather(i % 3, i / 3);
      }
      __builtin_amdgcn_s_setprio(0);
    };
    // Four waves, alone on their SIMDs: one barrier a tile, and the gathers of K
    // tile t + 2 and V tile t + 1 between the batches of its products, so that none
    // waits behind the others' requests.
    auto iteration_alone = [&](const int t, auto stage_tag) __attribute__((always_inline)) {
      constexpr int stage = decltype(stage_tag)::value;  // t % kStages
      const int key0 = list_begin + t * W::kKeys;
      const bool computes = key0 < wave_stop;
      const unsigned long long tile_keys = uniform(tile_valid[t]);
      if (computes) weigh_tile(key0, tile_keys);
      wait_vm<0>();  // the share of K tile t + 1 and V tile t
      settle_values(t, stage, tile_keys);
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
      __builtin_amdgcn_sched_barrier(0);
      workgroup_barrier();
      // The gathers, V and K in turn; their slots are read two gathers ahead.
      int slots[2];
      auto read_slot = [&](int i) __attribute__((always_inline)) {
        if (i < 2 * W::kGathers) slots[i % 2] = slot_of(min(t + 1 + i % 2, last), i / 2);
      };
      auto gather = [&](int step, int i) __attribute__((always_inline)) {
        if (i % 2 == 0) gather_step(step, std::true_type{}, slots[0], (stage + 1) % W::kStages, i / 2);
        else gather_step(step, std::false_type{}, slots[1], stage, i / 2);
        if (step == 0) read_slot(i + 2);
      };
      constexpr int kApart = kMfmas / (2 * W::kGathers);  // MFMAs from one gather to the next
      read_slot(0);
      read_slot(1);
      if (computes) {
        products(stage, (stage + 1) % W::kStages, std::true_type{}, [&](int i) __attribute__((always_inline)) {
          if (i % kApart < 3) gather(i % kApart, i / kApart);
        });
      } else {
#pragma unroll
        for (int i = 0; i < 6 * W::kGathers; ++i) gather(i % 3, i / 3);
      }
    };
    if constexpr (W::kWaves == 8) {
      for (int t = 0; t < tiles; t += 4) {
        iteration(t, std::integral_constant<int, 0>{});
        if (t + 1 < tiles) iteration(t + 1, std::integral_constant<int, 1>{});
        if (t + 2 < tiles) iteration(t + 2, std::integral_constant<int, 2>{});
        if (t + 3 < tiles) iteration(t + 3, std::integral_constant<int, 3>{});
      }
      if (!behind) workgroup_barrier();
    } else {
      for (int t = 0; t < tiles; t += 2) {
        iteration_alone(t, std::integral_constant<int, 0>{});
        if (t + 1 < tiles) iteration_alone(t + 1, std::integral_constant<int, 1>{});
      }
    }
    wait_vm<0>();  // the last gathers, before their stages are taken again (or the workgroup ends)
    if (list_begin + listed > seen_in_part) {
      for (int base = 0; base < 2 * tiles; base += kWave) {
        const unsigned word = base + lane < 2 * tiles ? odd_rows[base + lane] : 0u;
        unsigned long long words = __builtin_amdgcn_ballot_w64(word != 0);
        while (words != 0) {
          const int at = __builtin_ctzll(words);
          words &= words - 1;
          for (unsigned bits = __builtin_amdgcn_readlane(word, at); bits != 0; bits &= bits - 1) {
            const int key = (base + at) * 32 + __builtin_ctz(bits);  // of the list
            const unsigned char *row = row_at(p, v_base, slot_list[key]) + 8 * h;
            if (list_begin + key > pos) continue;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
              for (int rr = 0; rr < 4; ++rr) {
                const f32x4 x = nonfinite_only<E>(*reinterpret_cast<const u32x2 *>(row + 64 * b + 16 * rr));
#pragma unroll
                for (int e = 0; e < 4; ++e) o[b][4 * rr + e] += x[e];
                __builtin_amdgcn_sched_barrier(0);  // (rare: few registers rather than loads in flight)
              }
          }
        }
      }
    }
  }

  float l = (l4[0] + l4[1]) + (l4[2] + l4[3]);
  {  // the column's other half (lane l ^ 32) summed the other keys
    unsigned a = __builtin_bit_cast(unsigned, l), b = a;
    permlane32_swap(a, b);
    l = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
  }
  if (!exists) return;
  // Register r of block b: dim 32 b + 8 (r / 4) + 4 h + r % 4.
  if (w.chunks == 1) {
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing is zero
    uint16_t *dst = output_row(p, w, head, column, D) + 4 * h;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int rr = 0; rr < 4; ++rr) {
        u32x2 packed;
        packed[0] = E::pack(o[b][4 * rr] * inv, o[b][4 * rr + 1] * inv);
        packed[1] = E::pack(o[b][4 * rr + 2] * inv, o[b][4 * rr + 3] * inv);
        *reinterpret_cast<u32x2 *>(dst + 32 * b + 8 * rr) = packed;
      }
    return;
  }
  float *partial = partial_of<D>(p, W::kColumns, w.first_partial + w.chunk * w.partial_step, head);
  const int c = 32 * wave + col;
  if (h == 0) {
    partial[W::kColumns * D + 2 * c] = m;
    partial[W::kColumns * D + 2 * c + 1] = l;
  }
  float *dst = partial + c * D + 4 * h;
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int rr = 0; rr < 4; ++rr) {
      f32x4 row;
#pragma unroll
      for (int e = 0; e < 4; ++e) row[e] = o[b][4 * rr + e];
      *reinterpret_cast<f32x4 *>(dst + 32 * b + 8 * rr) = row;
    }
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
  int max_partials, target, min_chunk;
  bool wide, splits;
  long long ws_floats, plan_at;  // of the workspace; where the plan begins in it (ws_floats: none)
};

constexpr int kComputeUnits = 256;  // MI355X

Launch plan_launch(const ll_paged_attention_args *a) {
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
  const int places = std::max(1, kComputeUnits / static_cast<int>(a->num_kv_heads));
  x.target = x.wide                           ? places
             : 2 * x.max_tiles <= places ? places - static_cast<int>(x.max_tiles) + 1
                                         : 2 * places;
  const long long max_keys = a->page_table_columns * a->page_size;
  x.splits = max_keys > x.min_chunk * kPageTile;
  x.max_units = x.max_tiles + (x.splits ? x.target + 1 : 0);
  x.max_partials = x.splits ? 2 * x.target + 2 : 0;
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

template <int D, typename E>
int launch_all(const PagedParams &p, const Launch &x, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>(x.max_units) * static_cast<unsigned>(p.hkv);
  if (p.plan != nullptr) paged_plan_kernel<<<1, kPlanThreads, 0, s>>>(p, x.columns);
  if (x.wide) paged_wide_kernel<D, E><<<grid, Wide<D>::kThreads, 0, s>>>(p);
  else paged_narrow_kernel<D, E><<<grid, Narrow<D>::kThreads, 0, s>>>(p);
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

}  // namespace

extern "C" {

int64_t ll_paged_attention_args_size(void) { return static_cast<int64_t>(sizeof(ll_paged_attention_args)); }

int64_t ll_paged_attention_workspace_bytes(const ll_paged_attention_args *a) {
  const int rc = check_args(a);
  if (rc != LL_OK) return rc;
  if (a->num_queries == 0 || a->num_requests == 0) return 0;
  return plan_launch(a).ws_floats * 4;
}

int ll_paged_attention(const ll_paged_attention_args *a, ll_stream_t stream) {
  const int rc = check_args(a);
  if (rc != LL_OK || a->num_queries == 0 || a->num_requests == 0) return rc;
  const Launch x = plan_launch(a);
  if (x.ws_floats > 0 && (a->workspace == nullptr || a->workspace_bytes < x.ws_floats * 4 || !aligned(a->workspace, 16)))
    return fail(LL_ERR_INVALID_ARGUMENT, "the call needs a 16-byte aligned workspace of %lld bytes",
                static_cast<long long>(x.ws_floats * 4));
  PagedParams p;
  memset(&p, 0, sizeof(p));
  p.q = static_cast<const uint16_t *>(a->query);
  p.out = static_cast<uint16_t *>(a->output);
  p.k = static_cast<const uint16_t *>(a->key_buffer);
  p.v = static_cast<const uint16_t *>(a->value_buffer);
  p.pages = static_cast<const int *>(a->page_table);
  p.kv_lengths = a->kv_lengths;
  p.query_starts = a->query_starts;
  p.ws = static_cast<float *>(a->workspace);
  if (x.ws_floats > x.plan_at) p.plan = reinterpret_cast<int *>(p.ws + x.plan_at);
  p.q_token = a->query_token_stride;
  p.q_head = a->query_head_stride;
  p.pages_stride = a->page_table_stride;
  p.row_bytes = static_cast<unsigned>(a->num_kv_heads * a->head_dim * 2);
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
  p.max_partials = x.max_partials;
  p.scale_log2 = static_cast<float>(a->softmax_scale * 1.4426950408889634);  // log2(e)
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool f16 = a->kv_dtype == LL_DTYPE_FLOAT16;
  if (a->head_dim == 64) return f16 ? launch_all<64, F16>(p, x, s) : launch_all<64, Bf16>(p, x, s);
  if (a->head_dim == 128) return f16 ? launch_all<128, F16>(p, x, s) : launch_all<128, Bf16>(p, x, s);
  return f16 ? launch_all<256, F16>(p, x, s) : launch_all<256, Bf16>(p, x, s);
}

}  // extern "C"
