// Attention of each request's new tokens over its pages of the KV pool, on
// gfx950 (MI355X): the kernels of a pool of fp16 or bf16.  How a call is cut into
// units (request, tile of columns, chunk of keys), one for a workgroup and KV head,
// and how split requests are joined is in paged_device.h.
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

#include <type_traits>

#include "attention_device.h"
#include "legolink_kv.h"
#include "paged_device.h"

namespace {

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

template <int D, typename E>
int launch_all(const PagedParams &p, const Launch &x, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>(x.max_units) * static_cast<unsigned>(p.hkv);
  launch_plan(p, x, s);
  if (x.wide) paged_wide_kernel<D, E><<<grid, Wide<D>::kThreads, 0, s>>>(p);
  else paged_narrow_kernel<D, E><<<grid, Narrow<D>::kThreads, 0, s>>>(p);
  return launch_join<D, E>(p, x, s);
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
  int rc = check_args(a);
  if (rc != LL_OK || a->num_queries == 0 || a->num_requests == 0) return rc;
  const Launch x = plan_launch(a);
  PagedParams p;
  memset(&p, 0, sizeof(p));
  rc = fill_params(a, x, &p);
  if (rc != LL_OK) return rc;
  p.k = static_cast<const uint16_t *>(a->key_buffer);
  p.v = static_cast<const uint16_t *>(a->value_buffer);
  p.row_bytes = static_cast<unsigned>(a->num_kv_heads * a->head_dim * 2);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool f16 = a->kv_dtype == LL_DTYPE_FLOAT16;
  if (a->head_dim == 64) return f16 ? launch_all<64, F16>(p, x, s) : launch_all<64, Bf16>(p, x, s);
  if (a->head_dim == 128) return f16 ? launch_all<128, F16>(p, x, s) : launch_all<128, Bf16>(p, x, s);
  return f16 ? launch_all<256, F16>(p, x, s) : launch_all<256, Bf16>(p, x, s);
}

}  // extern "C"
