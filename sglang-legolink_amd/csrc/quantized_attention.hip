// Attention of each request's new tokens over its pages of a pool held in 8 bits, on
// gfx950 (MI355X).  How a call is cut into units (request, tile of columns, chunk of
// keys), one for a workgroup and KV head (or a few of them), and how split requests are
// joined is in paged_device.h; the pool's format in quantized_device.h.
//
// Codes become the queries' type before the matrix unit: code * 2^(byte - 127) is
// exact in bf16 (bytes 3 to 246; in fp16 from 2^-21 up to 65504), one instruction for
// two values, so the products and the softmax are those of a pool in that type.  (An
// 8-bit product would need the queries and the weights in 4 significant bits, or two
// products of the halves of each: as many cycles as one in 16 bits.)  Pages are whole
// blocks of at least 16 tokens, so the keys come in groups of 16 neighbouring rows under one scale
// for the head: page, row and scale are looked up once for a group.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <string.h>

#include <type_traits>

#include "attention_device.h"
#include "legolink_kv.h"
#include "paged_device.h"
#include "quantized_device.h"

namespace {

constexpr int kGroupKeys = 16;  // neighbouring rows under one scale

struct QuantizedParams : PagedParams {
  const uint8_t *k8, *v8;
  const uint8_t *k_scales, *v_scales;
  int block_shift;
};

typedef __attribute__((ext_vector_type(2))) int i32x2;
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

// Two codes of a word's half as two values of the type.
template <typename E>
__device__ inline uint32_t decode2(uint32_t codes, float scale, bool high);
template <>
__device__ inline uint32_t decode2<Bf16>(uint32_t codes, float scale, bool high) {
  return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true)
                                           : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false));
}
template <>
__device__ inline uint32_t decode2<F16>(uint32_t codes, float scale, bool high) {
  return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, true)
                                           : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, false));
}
// Four codes.
template <typename E>
__device__ inline u32x2 decode4(uint32_t codes, float scale) {
  return u32x2{decode2<E>(codes, scale, false), decode2<E>(codes, scale, true)};
}

// The keys of a list, by groups: the group's first row (-1: of no page of the pool),
// and the scales of its keys and values for each of the workgroup's heads (bytes 0 and 1).
template <int kHeads>
struct Group {
  int slot;
  int scales[kHeads];
  __device__ void clear() {
    slot = -1;
#pragma unroll
    for (int h = 0; h < kHeads; ++h) scales[h] = 0x7f7f;
  }
};

template <int kHeads>
__device__ inline Group<kHeads> group_at(const QuantizedParams &p, const int *pages, int head, int key) {
  const unsigned first = static_cast<unsigned>(key);
  const unsigned page = static_cast<unsigned>((first * p.page_magic) >> p.page_shift);
  const int entry = pages[page];
  Group<kHeads> g;
  g.clear();
  if (static_cast<unsigned>(entry) < static_cast<unsigned>(p.num_pages)) {
    g.slot = entry * p.page_size + static_cast<int>(first - page * p.page_size);
    const long long at = static_cast<long long>(g.slot >> p.block_shift) * p.hkv + head;
#pragma unroll
    for (int h = 0; h < kHeads; ++h) g.scales[h] = p.k_scales[at + h] | p.v_scales[at + h] << 8;
  }
  return g;
}

__device__ inline float uniform_scale(unsigned byte) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, scale_of(byte))));
}

// Up to 16 columns: single tokens, bound by reading the codes once.  As for a 16-bit
// pool, the waves of a workgroup take turns at its 32-key subtiles, each through an
// LDS ring of its own, and join their results at the end.  LDS holds codes; a lane
// decodes its fragments.  v_mfma_f32_16x16x32, lane layouts: A and B lane l element e
// -> row / column l % 16, k = 8 (l / 16) + e; accumulator register r -> row 4 (l / 16)
// + r, column l % 16.  The scores' k order is free: of the 64 dims of two steps the
// lane takes 16 neighbouring ones, one 16-byte read.  The value product's k order is
// the scores' register order: k = 8 g + e is key 4 g + e (e < 4) or 16 + 4 g + e - 4,
// so that a lane's first four elements lie in one group of 16 keys and the others in
// the next.  A transposed read of 16 lanes takes 8 rows x 16 codes, lane l row l / 2,
// codes 8 (l % 2) on, and leaves lane l dim l of the 8 rows.
// LDS rows are token-major with their 16-byte chunks swizzled by token, so that the 16
// lanes of a K read (16 tokens, one chunk) and the 32 lanes of a transposed V read
// (tokens 8 i .. + 3 and 16 on of two groups, one chunk) cover the 64 banks once.
// 131,072 keys of 4 heads of 128: 25.4 us, 5.3 TB/s; 64 uneven requests, 1.06 GB, two heads
// a workgroup: 210 us, 5.1 TB/s (the vector units are busy a third of the time); 2,048
// keys 7.4 us, latencies as for a 16-bit pool.
template <int D>
struct Narrow8 {
  static constexpr int kKeys = 32;
  static constexpr int kWaves = D == 256 ? 4 : 8;
  static constexpr int kStages = D == 64 ? 4 : 2;
  static constexpr int kThreads = kWaves * kWave;
  static constexpr int kRowBytes = D;
  static constexpr int kHalf = kKeys * kRowBytes;  // a subtile's K or V rows
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kChunksPerRow = D / 16;
  static constexpr int kGathers = kHalf / (16 * kWave);  // of K and of V, per subtile
  static constexpr int kList = 4096;                     // keys held at a time
  __device__ static int k_swizzle(int t) { return D == 64 ? (t / 4) % 4 : D == 128 ? (t / 2) % 8 : t % 16; }
  __device__ static int v_swizzle(int t) {
    return D == 64 ? (t / 4) % 2 + 2 * ((t / 16) % 2) : D == 128 ? (t / 2) % 4 + 4 * ((t / 16) % 2)
                                                                 : t % 8 + 8 * ((t / 16) % 2);
  }
};

template <int D, typename E, int kHeads>
__global__ void __launch_bounds__(Narrow8<D>::kThreads) quantized_narrow_kernel(const QuantizedParams p) {
  typedef Narrow8<D> N;
  typedef typename E::frag frag;
  constexpr int kColumns = 16;
  constexpr int kPairs = D / 64;  // of the scores' steps
  constexpr int kBlocks = D / 16;
  constexpr int kTurns = N::kWaves / kHeads;  // waves of a head
  constexpr int kPitch = D + 4;  // floats of a joined row: 16 lanes' 16-byte writes meet 64 banks
  constexpr int kShared = N::kWaves * (N::kRing > 16 * kPitch * 4 ? N::kRing : 16 * kPitch * 4);
  __shared__ __attribute__((aligned(16))) unsigned char rings[kShared];
  __shared__ Group<kHeads> groups[N::kList / kGroupKeys];
  __shared__ float stats[N::kWaves][kColumns][2];

  const int first_head = static_cast<int>(blockIdx.x % static_cast<unsigned>(p.hkv / kHeads)) * kHeads;
  const int unit = static_cast<int>(blockIdx.x / static_cast<unsigned>(p.hkv / kHeads));
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
  const int own_head = wave / kTurns;  // of the workgroup's
  const int head = first_head + own_head;
  unsigned char *ring = rings + wave * N::kRing;

  // The lane's column and its query.
  const int column = w.tile * kColumns + col;
  const int token = column / p.group;
  const bool exists = token < w.request.q_len;
  const int pos = exists ? w.request.kv_len - w.request.q_len + token : -1;
  // Keys below it are visible to every column (to the first one, that is).
  const int seen_by_all = w.request.kv_len - w.request.q_len + (w.tile * kColumns) / p.group + 1;
  frag qf[2 * kPairs];
  {
    const int q_head = head * p.group + (column - token * p.group);
    const uint16_t *row =
        p.q + (static_cast<long long>(w.request.q_start) + token) * p.q_token + q_head * p.q_head + 16 * g;
#pragma unroll
    for (int i = 0; i < 2 * kPairs; ++i) {  // dims 64 (i / 2) + 16 g + 8 (i % 2) on
      u32x4 bits = u32x4{0u, 0u, 0u, 0u};
      if (exists) bits = *reinterpret_cast<const u32x4 *>(row + 64 * (i / 2) + 8 * (i % 2));
      qf[i] = __builtin_bit_cast(frag, bits);
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
  // (64 j + lane) of the subtile's rows in LDS order, so row (64 j + lane) /
  // kChunksPerRow of the two groups.
  const unsigned char *k_base = p.k8 + static_cast<long long>(head) * D;
  const unsigned char *v_base = p.v8 + static_cast<long long>(head) * D;
  auto gather = [&](int sub, int stage) {
    unsigned char *dst = ring + stage * N::kStage;
    const int slots[2] = {__builtin_amdgcn_readfirstlane(max(groups[2 * sub].slot, 0)),
                          __builtin_amdgcn_readfirstlane(max(groups[2 * sub + 1].slot, 0))};
#pragma unroll
    for (int j = 0; j < N::kGathers; ++j) {
      const int at = j * kWave + lane;
      const int row = at / N::kChunksPerRow;
      const int place = at % N::kChunksPerRow;
      const int slot = slots[row / kGroupKeys] + row % kGroupKeys;
      dma_pair(row_at(p, k_base + 16 * (place ^ N::k_swizzle(row)), slot), dst + j * 16 * kWave,
               row_at(p, v_base + 16 * (place ^ N::v_swizzle(row)), slot), dst + N::kHalf + j * 16 * kWave);
    }
  };
  // Offsets of the lane's fragments within a stage.
  int k_off[kPairs];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) k_off[i] = col * N::kRowBytes + (((4 * i + g) ^ N::k_swizzle(col)) * 16);
  const int v_row = col / 2;  // of the read's eight
  const int v_token = v_row < 4 ? 4 * g + v_row : 16 + 4 * g + v_row - 4;
  int v_off[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
    v_off[b] = N::kHalf + v_token * N::kRowBytes + ((b ^ N::v_swizzle(v_token)) * 16) + 8 * (col % 2);
  const unsigned ring_lds = lds_offset(ring);

  const int *pages = p.pages + static_cast<long long>(w.index) * p.pages_stride;
  for (int list_begin = key_begin; list_begin < key_end; list_begin += N::kList) {
    const int listed = min(key_end - list_begin, N::kList);
    const int subs = (listed + N::kKeys - 1) / N::kKeys;
    __syncthreads();  // every wave is past the former list
    for (int i = tid; i < 2 * subs; i += N::kThreads) {
      Group<kHeads> x;
      x.clear();
      if (i * kGroupKeys < listed) x = group_at<kHeads>(p, pages, first_head, list_begin + i * kGroupKeys);
      groups[i] = x;
    }
    // The compiler does not count the gathers: nothing that it waits for in the
    // loop below may be left in flight.
    wait_vm<0>();
    __syncthreads();

#pragma unroll
    for (int s = 0; s < N::kStages; ++s)
      if (wave % kTurns + s * kTurns < subs) gather(wave % kTurns + s * kTurns, s);
    int stage = 0;
    for (int sub = wave % kTurns; sub < subs; sub += kTurns) {
      const int key0 = list_begin + sub * N::kKeys;
      float k_scale[2], v_scale[2];
      unsigned valid = 0;  // keys that have a row and are not behind the list's last
      bool bad_scale[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int slot = __builtin_amdgcn_readfirstlane(groups[2 * sub + i].slot);
        const unsigned scales = static_cast<unsigned>(__builtin_amdgcn_readfirstlane(groups[2 * sub + i].scales[own_head]));
        k_scale[i] = uniform_scale(scales & 0xffu);
        v_scale[i] = uniform_scale(scales >> 8);
        bad_scale[i] = (scales >> 8) == 255u;
        const int rows = min(max(key_end - key0 - 16 * i, 0), 16);
        if (slot >= 0) valid |= ((1u << rows) - 1u) << (16 * i);
      }
      // This stage's gathers are complete when at most the later stages' are outstanding.
      const int later = min(N::kStages - 1, (subs - 1 - sub) / kTurns);
      if (N::kStages == 4 && later == 3) wait_vm<3 * 2 * N::kGathers % 64>();
      else if (N::kStages == 4 && later == 2) wait_vm<2 * 2 * N::kGathers % 64>();
      else if (later >= 1) wait_vm<2 * N::kGathers>();
      else wait_vm<0>();
      asm volatile("" ::: "memory");
      unsigned char *rows = ring + stage * N::kStage;
      const bool whole = valid == 0xffffffffu && key0 + N::kKeys <= seen_by_all;
      unsigned odd = 0;  // rows whose values are not all finite, where some columns do not see the subtile whole
      if (!whole) {
        // Rows that no column sees may hold anything: zeros in their place.  And in
        // rows that some columns see, what is not finite (codes, or with the scale).
        const bool in_part = key0 + N::kKeys > seen_by_all && seen_by_all < w.key_end;
        for (int c = lane; c < N::kKeys * N::kChunksPerRow; c += kWave) {
          const int row = c / N::kChunksPerRow;
          u32x4 *chunk = reinterpret_cast<u32x4 *>(rows + N::kHalf + c * 16);
          if (((valid >> row) & 1u) == 0) {
            *chunk = u32x4{0u, 0u, 0u, 0u};
          } else if (in_part) {
            u32x4 codes = *chunk;
            bool changed = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const u32x2 values = decode4<E>(codes[i], v_scale[row / 16]);
              uint32_t keep = 0xffffffffu;
              if (nonfinite<E>(values[0])) keep &= ~0xffu;
              if (nonfinite<E>(values[0] >> 16)) keep &= ~0xff00u;
              if (nonfinite<E>(values[1])) keep &= ~0xff0000u;
              if (nonfinite<E>(values[1] >> 16)) keep &= ~0xff000000u;
              changed = changed || keep != 0xffffffffu;
              codes[i] &= keep;
            }
            if (changed) {
              odd |= 1u << row;
              *chunk = codes;
            }
          }
        }
        if (in_part) {
          if (__builtin_amdgcn_ballot_w64(odd != 0) != 0) {
#pragma unroll
            for (int step = 1; step < kWave; step *= 2) odd |= __shfl_xor(odd, step);
          }
          odd = static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(odd)));
        }
        // (Codes of 0 are NaN under the scale of NaN: rows without visible ones get another.)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (bad_scale[i] && (in_part || ((valid >> (16 * i)) & 0xffffu) == 0)) v_scale[i] = 1.f;
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
        asm volatile("" ::: "memory");
      }

      f32x4 s[2];
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) s[rb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kPairs; ++i)
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
          const u32x4 codes = *reinterpret_cast<const u32x4 *>(rows + k_off[i] + rb * 16 * N::kRowBytes);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const u32x2 lo = decode4<E>(codes[2 * e], k_scale[rb]), hi = decode4<E>(codes[2 * e + 1], k_scale[rb]);
            s[rb] = E::mfma16(__builtin_bit_cast(frag, u32x4{lo[0], lo[1], hi[0], hi[1]}), qf[2 * i + e], s[rb]);
          }
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
        const i32x2 codes =
            __builtin_amdgcn_ds_read_tr8_b64_v2i32(reinterpret_cast<lds_i32x2 *>(static_cast<uintptr_t>(at)));
        const u32x2 lo = decode4<E>(static_cast<uint32_t>(codes[0]), v_scale[0]);
        const u32x2 hi = decode4<E>(static_cast<uint32_t>(codes[1]), v_scale[1]);
        o[b] = E::mfma16(__builtin_bit_cast(frag, u32x4{lo[0], lo[1], hi[0], hi[1]}), pb, o[b]);
      }
      while (odd != 0) {
        const int rel = __builtin_ctz(odd);
        odd &= odd - 1;
        const unsigned char *row = row_at(p, v_base, groups[2 * sub + rel / 16].slot + rel % 16) + 4 * g;
        const float scale = scale_of(static_cast<unsigned>(groups[2 * sub + rel / 16].scales[own_head]) >> 8);
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          const f32x4 x4 = nonfinite_only<E>(decode4<E>(*reinterpret_cast<const uint32_t *>(row + 16 * b), scale));
          if (key0 + rel <= pos) o[b] += x4;
          __builtin_amdgcn_sched_barrier(0);  // (rare: few registers rather than loads in flight)
        }
      }
      // The stage's reads are done: the gather kStages turns ahead takes it.
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (sub + N::kStages * kTurns < subs) gather(sub + N::kStages * kTurns, stage);
      stage = stage + 1 == N::kStages ? 0 : stage + 1;
    }
  }

  // The waves' results joined.
  const bool direct = w.chunks == 1;
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
  for (int i = tid; i < kHeads * 16 * (D / 4); i += N::kThreads) {
    const int of_head = i / (16 * (D / 4));
    const int first = of_head * kTurns;  // of the head's waves
    const int c = i / (D / 4) % 16;
    const int quad = i % (D / 4);
    if ((w.tile * kColumns + c) / p.group >= w.request.q_len) continue;
    float top = stats[first][c][0];
#pragma unroll
    for (int v = 1; v < kTurns; ++v) top = fmaxf(top, stats[first + v][c][0]);
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < kTurns; ++v) {
      const float weight = joined_weight(stats[first + v][c][0], top, scale_log2);
      sum += weight * stats[first + v][c][1];
      acc += weight * *reinterpret_cast<const f32x4 *>(joined + ((first + v) * 16 + c) * kPitch + 4 * quad);
    }
    if (direct) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing is zero
      u32x2 packed;
      packed[0] = E::pack(acc[0] * inv, acc[1] * inv);
      packed[1] = E::pack(acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<u32x2 *>(output_row(p, w, first_head + of_head, w.tile * kColumns + c, D) + 4 * quad) = packed;
    } else {
      float *partial =
          partial_of<D>(p, kColumns, w.first_partial + w.chunk * w.partial_step, first_head + of_head);
      *reinterpret_cast<f32x4 *>(partial + c * D + 4 * quad) = acc;
      if (quad == 0) {
        partial[kColumns * D + 2 * c] = top;
        partial[kColumns * D + 2 * c + 1] = sum;
      }
    }
  }
}

// Many columns: chunks, bound by the matrix products, whose tiles, phases and lane
// layouts are those of a 16-bit pool: eight waves of 32 columns each (four at head dim
// 256) share every tile of 64 keys, and half of them runs a phase behind the other, so
// that a SIMD's two waves take turns at the matrix unit (the products: the values of
// tile t, the scores of tile t + 1) and at the vector unit (the softmax).
//
// A tile is decoded once for the workgroup: a wave loads its share of codes, 8 or 16
// rows, into registers a whole tile ahead, and between the MFMAs of the products
// decodes it, in the MFMAs' shadow, and writes it to LDS.  So LDS holds two tiles of
// keys and two of values, in the queries' type.  2,048 queries of 28/4 heads of 128
// behind 30,720 keys: 841 us a call, 1.11 PFLOP/s (819 over a 16-bit pool, whose tiles
// need no decoding; a library product of 8192^3 1.15 PFLOP/s).
template <int D>
struct Wide8 {
  static constexpr int kKeys = 64;
  static constexpr int kWaves = D == 256 ? 4 : 8;
  static constexpr int kThreads = kWaves * kWave;
  static constexpr int kColumns = 32 * kWaves;
  static constexpr int kStages = 2;
  static constexpr int kRowBytes = 2 * D;  // in LDS
  static constexpr int kStage = kKeys * kRowBytes;
  static constexpr int kRows = kKeys / kWaves;              // of a wave's share
  static constexpr int kPiece = D == 64 ? 8 : 16;           // codes of a lane's load
  static constexpr int kChunks = kPiece / 8;                // 16-byte chunks that they become
  static constexpr int kPiecesPerRow = D / kPiece;
  static constexpr int kRowsApart = kWave / kPiecesPerRow;  // from a lane's piece to its next
  static constexpr int kPieces = kRows / kRowsApart;        // of a lane, of K and of V, per tile
  static constexpr int kList = 7168;                        // keys held at a time
  static_assert(kRows <= kGroupKeys && kGroupKeys % kRows == 0, "a share lies in one group");
  __host__ __device__ static constexpr int k_swizzle(int t) { return D >= 128 ? t % 16 : (t / 2) % 8; }
  // (Of values, the last bit for the writes: two neighbouring rows' even chunks meet no
  // bank twice.)
  __host__ __device__ static constexpr int v_swizzle(int t) { return D >= 128 ? 4 * (t % 4) + t % 2 : 4 * ((t / 2) % 2); }
};

typedef __attribute__((address_space(3))) u32x4 lds_u32x4;

template <int D, typename E>
__global__ void __launch_bounds__(Wide8<D>::kThreads) quantized_wide_kernel(const QuantizedParams p) {
  typedef Wide8<D> W;
  typedef typename E::frag frag;
  constexpr int kKSteps = D / 16;
  constexpr int kBlocks = D / 32;
  __shared__ __attribute__((aligned(512))) unsigned char k_ring[W::kStages * W::kStage];
  __shared__ __attribute__((aligned(512))) unsigned char v_ring[W::kStages * W::kStage];
  __shared__ Group<1> groups[W::kList / kGroupKeys];
  __shared__ int tile_groups[W::kList / W::kKeys];  // a bit for each of a tile's four groups: it has rows
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

  typedef uint32_t codes_t __attribute__((ext_vector_type(W::kPiece / 4)));
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

  // The wave's share of a tile, kRows rows of one group: piece j of a lane is its
  // codes from byte kPiece * piece of row piece_row + j * kRowsApart of the share on.
  // (Rows of 256 codes: 16 neighbouring lanes take half of each of two rows. A row's
  // every second chunk meets each of these banks twice; two rows' swizzles differ by one.)
  const unsigned char *k_base = p.k8 + static_cast<long long>(head) * D;
  const unsigned char *v_base = p.v8 + static_cast<long long>(head) * D;
  const int share_row = wave * W::kRows;  // of a tile
  const int piece_row = W::kPiecesPerRow == 16 ? lane / 32 * 2 + lane / 8 % 2 : lane / W::kPiecesPerRow;
  const int piece = W::kPiecesPerRow == 16 ? lane / 16 % 2 * 8 + lane % 8 : lane % W::kPiecesPerRow;
  const unsigned piece_from = static_cast<unsigned>(piece_row) * p.row_bytes + piece * W::kPiece;
  // Where a piece's values go in a stage: 16-byte chunks kChunks * piece on of row
  // share_row + piece_row + j * kRowsApart, swizzled (of j, by an xor).
  const int own_row = share_row + piece_row;
  const unsigned k_to = lds_offset(k_ring) + own_row * W::kRowBytes + ((W::kChunks * piece) ^ W::k_swizzle(own_row)) * 16;
  const unsigned v_to = lds_offset(v_ring) + own_row * W::kRowBytes + ((W::kChunks * piece) ^ W::v_swizzle(own_row)) * 16;
  codes_t k_codes[W::kPieces], v_codes[W::kPieces];
  float k_scale = 1.f, v_scale = 1.f;  // of the codes above
  auto group_of = [&](int tile) __attribute__((always_inline)) {
    const Group<1> x = groups[tile * (W::kKeys / kGroupKeys) + share_row / kGroupKeys];
    Group<1> u;
    u.slot = __builtin_amdgcn_readfirstlane(x.slot);
    u.scales[0] = __builtin_amdgcn_readfirstlane(x.scales[0]);
    return u;
  };
  auto load_piece = [&](auto values_tag, const Group<1> &x, int j) __attribute__((always_inline)) {
    constexpr bool values = decltype(values_tag)::value;
    const int slot = max(x.slot, 0) + share_row % kGroupKeys + j * W::kRowsApart;
    (values ? v_codes : k_codes)[j] =
        *reinterpret_cast<const codes_t *>(row_at(p, values ? v_base : k_base, slot) + piece_from);
    // (Behind the last piece of the tile before.)
    if (j == W::kPieces - 1) (values ? v_scale : k_scale) = scale_of((values ? x.scales[0] >> 8 : x.scales[0]) & 0xff);
  };
  // The words of a piece's values, two codes each.
  uint32_t words[W::kPiece / 2];
  auto decode_part = [&](auto values_tag, int j, int half) __attribute__((always_inline)) {
    constexpr bool values = decltype(values_tag)::value;
    const codes_t codes = (values ? v_codes : k_codes)[j];
#pragma unroll
    for (int i = half * W::kPiece / 8; i < (half + 1) * W::kPiece / 8; ++i) {
      const u32x2 four = decode4<E>(codes[i], values ? v_scale : k_scale);
      words[2 * i] = four[0];
      words[2 * i + 1] = four[1];
    }
  };
  // V piece j of tile t: rows that no column sees may hold anything, zeros in their
  // place; rows that some see give up what is not finite.
  auto settle_piece = [&](int list_begin, int listed, int t, int slot, int j) __attribute__((always_inline)) {
    const int key = t * W::kKeys + own_row + j * W::kRowsApart;  // of the list
    if (slot < 0 || key >= listed) {
#pragma unroll
      for (int i = 0; i < W::kPiece / 2; ++i) words[i] = 0u;
    } else if (list_begin + (t + 1) * W::kKeys > seen_in_part) {
      bool any = false;
#pragma unroll
      for (int i = 0; i < W::kPiece / 2; ++i) {
        const bool low = nonfinite<E>(words[i]), high = nonfinite<E>(words[i] >> 16);
        any = any || low || high;
        words[i] &= (low ? 0xffff0000u : 0xffffffffu) & (high ? 0xffffu : 0xffffffffu);
      }
      if (any) atomicOr(&odd_rows[key / 32], 1u << (key % 32));
    }
  };
  auto write_piece = [&](auto values_tag, int stage, int j) __attribute__((always_inline)) {
    constexpr bool values = decltype(values_tag)::value;
    const unsigned swizzle = 16u * (values ? W::v_swizzle(j * W::kRowsApart) : W::k_swizzle(j * W::kRowsApart));
    const unsigned at = ((values ? v_to : k_to) ^ swizzle) + stage * W::kStage + j * W::kRowsApart * W::kRowBytes;
#pragma unroll
    for (int c = 0; c < W::kChunks; ++c)
      *reinterpret_cast<lds_u32x4 *>(static_cast<uintptr_t>(at ^ (16u * c))) =
          u32x4{words[4 * c], words[4 * c + 1], words[4 * c + 2], words[4 * c + 3]};
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
  constexpr int kApart = kMfmas / (8 * W::kPieces);  // MFMAs from one step of the staging to the next
  static_assert(kMfmas % (8 * W::kPieces) == 0, "a place for every step of the staging");
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
  auto weigh_tile = [&](int key0, int with_rows) __attribute__((always_inline)) {
    const bool whole = with_rows == 15 && key0 + W::kKeys <= seen_by_all;
    if (!whole) {
      // Register r of block kb: key 32 kb + 8 (r / 4) + 4 h + r % 4, of group 2 kb + r / 8.
      const int limit = pos - key0 - 4 * h;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int rel = 32 * kb + 8 * (r / 4) + r % 4;
          const bool visible = rel <= limit && ((with_rows >> (2 * kb + r / 8)) & 1) != 0;
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
    for (int i = tid; i < tiles * (W::kKeys / kGroupKeys); i += W::kThreads) {
      Group<1> x;
      x.clear();
      if (i * kGroupKeys < listed) x = group_at<1>(p, pages, head, list_begin + i * kGroupKeys);
      groups[i] = x;
    }
    for (int i = tid; i < 2 * tiles; i += W::kThreads) odd_rows[i] = 0;
    __syncthreads();
    for (int i = tid; i < tiles; i += W::kThreads) {
      int bits = 0;
#pragma unroll
      for (int g = 0; g < 4; ++g) bits |= groups[4 * i + g].slot >= 0 ? 1 << g : 0;
      tile_groups[i] = bits;
    }

    // V tile 0 and K tiles 0 and 1 go to their stages, V tile 1 and K tile 2 to
    // registers.  (Past the last tile the last is taken again, into stages that no
    // products take.)
    const std::true_type of_values{};
    const std::false_type of_keys{};
    const int last = tiles - 1;
    int v_slot;  // of the V codes held
    auto load_tile = [&](auto values_tag, int t) __attribute__((always_inline)) {
      const Group<1> x = group_of(min(t, last));
      if (decltype(values_tag)::value) v_slot = x.slot;
#pragma unroll
      for (int j = 0; j < W::kPieces; ++j) load_piece(values_tag, x, j);
    };
    auto put_tile = [&](auto values_tag, int t, int stage) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < W::kPieces; ++j) {
        decode_part(values_tag, j, 0);
        decode_part(values_tag, j, 1);
        if (decltype(values_tag)::value) settle_piece(list_begin, listed, t, v_slot, j);
        write_piece(values_tag, stage, j);
      }
    };
    load_tile(of_values, 0);
    load_tile(of_keys, 0);
    put_tile(of_values, 0, 0);
    put_tile(of_keys, 0, 0);
    load_tile(of_keys, 1);
    put_tile(of_keys, 1, 1);
    load_tile(of_values, 1);
    load_tile(of_keys, 2);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    workgroup_barrier();
    if (behind) workgroup_barrier();
    if (list_begin < wave_stop) products(0, 0, std::false_type{}, [](int) {});
    // One step of the staging during the products of tile t (stage t % 2): V tile t + 1
    // and K tile t + 2, held in registers, to their stages, then V tile t + 2 and K
    // tile t + 3 from memory.  Their stages held V tile t - 1 and K tile t, which all
    // waves have left.
    Group<1> next_v, next_k;
    auto staging = [&](int step, int t, auto stage_tag) __attribute__((always_inline)) {
      constexpr int stage = decltype(stage_tag)::value;
      const int j = step / 4 % W::kPieces, what = step % 4;
      const bool values = step / 4 < W::kPieces;
      if (what < 2) {
        if (values) decode_part(of_values, j, what);
        else decode_part(of_keys, j, what);
      } else if (what == 2) {
        if (values) {
          const int to = t + 1;
          if (v_slot < 0 || to * W::kKeys + share_row + W::kRows > listed || list_begin + (to + 1) * W::kKeys > seen_in_part)
            settle_piece(list_begin, listed, to, v_slot, j);
          write_piece(of_values, stage ^ 1, j);
        } else {
          write_piece(of_keys, stage, j);
        }
      } else if (values) {
        load_piece(of_values, next_v, j);
        if (j == W::kPieces - 1) v_slot = next_v.slot;
      } else {
        load_piece(of_keys, next_k, j);
      }
    };
    int with_rows = __builtin_amdgcn_readfirstlane(tile_groups[0]);
    // Eight waves, one half a phase behind the other.  Four waves (kWaves 4) are alone on their
    // SIMDs: one barrier a tile.
    auto iteration = [&](const int t, auto stage_tag) __attribute__((always_inline)) {
      constexpr int stage = decltype(stage_tag)::value;  // t % 2
      const int key0 = list_begin + t * W::kKeys;
      const bool computes = key0 < wave_stop;
      auto look_up = [&]() __attribute__((always_inline)) {
        next_v = group_of(min(t + 2, last));
        next_k = group_of(min(t + 3, last));
      };
      if constexpr (W::kWaves == 4) {
        look_up();
        if (computes) weigh_tile(key0, with_rows);
      }
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the wave's reads and writes of the stages are done
      __builtin_amdgcn_sched_barrier(0);
      workgroup_barrier();
      const int next_rows = tile_groups[min(t + 1, last)];
      if constexpr (W::kWaves == 8) {
        look_up();
        if (computes) weigh_tile(key0, with_rows);
      }
      with_rows = __builtin_amdgcn_readfirstlane(next_rows);
      if constexpr (W::kWaves == 8) {
        __builtin_amdgcn_sched_barrier(0);
        workgroup_barrier();
        __builtin_amdgcn_s_setprio(1);
      }
      // (Behind the wave's last tile the scores are of an old stage, and not used.)
      if (computes) {
        products(stage, stage ^ 1, std::true_type{}, [&](int i) __attribute__((always_inline)) {
          if (i % kApart == 0) staging(i / kApart, t, stage_tag);
        });
      } else {
#pragma unroll
        for (int i = 0; i < 8 * W::kPieces; ++i) staging(i, t, stage_tag);
      }
      if constexpr (W::kWaves == 8) __builtin_amdgcn_s_setprio(0);
    };
    for (int t = 0; t < tiles; t += 2) {
      iteration(t, std::integral_constant<int, 0>{});
      if (t + 1 < tiles) iteration(t + 1, std::integral_constant<int, 1>{});
    }
    if (W::kWaves == 8 && !behind) workgroup_barrier();
    // (odd_rows of the last tile are written in the products of the one before.)
    if (list_begin + listed > seen_in_part) {
      for (int base = 0; base < 2 * tiles; base += kWave) {
        const unsigned word = base + lane < 2 * tiles ? odd_rows[base + lane] : 0u;
        unsigned long long words = __builtin_amdgcn_ballot_w64(word != 0);
        while (words != 0) {
          const int at = __builtin_ctzll(words);
          words &= words - 1;
          for (unsigned bits = __builtin_amdgcn_readlane(word, at); bits != 0; bits &= bits - 1) {
            const int key = (base + at) * 32 + __builtin_ctz(bits);  // of the list
            const Group<1> x = groups[key / kGroupKeys];
            const unsigned char *row = row_at(p, v_base, x.slot + key % kGroupKeys) + 4 * h;
            const float scale = scale_of(x.scales[0] >> 8);
            if (list_begin + key > pos) continue;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
              for (int rr = 0; rr < 4; ++rr) {
                const f32x4 four =
                    nonfinite_only<E>(decode4<E>(*reinterpret_cast<const uint32_t *>(row + 32 * b + 8 * rr), scale));
#pragma unroll
                for (int e = 0; e < 4; ++e) o[b][4 * rr + e] += four[e];
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

// KV heads that a workgroup of the narrow kernel takes together: what they read of a
// row is one piece of 256 bytes where the heads' count allows it.
// Heads of 128, one at a time and two: 32 requests over 32,768 keys of 4 KV heads
// 290 and 215 us, 16 requests of 8 KV heads 323 and 224; what few requests read comes
// from the memory-side cache either way, and their splits cost more (one over 131,072
// keys 36 and 38 us, 4 over 4,000 14 and 15).
int heads_together(const ll_paged_attention_args &a) {
  if (a.head_dim == 256 || a.num_requests * a.num_kv_heads < 32) return 1;
  if (a.head_dim == 64 && a.num_kv_heads % 4 == 0) return 4;
  return a.num_kv_heads % 2 == 0 ? 2 : 1;
}

template <int D, typename E>
int launch_all(const QuantizedParams &p, const Launch &x, int heads, hipStream_t s) {
  const unsigned units = static_cast<unsigned>(x.max_units);
  launch_plan(p, x, s);
  if (x.wide) {
    quantized_wide_kernel<D, E><<<units * static_cast<unsigned>(p.hkv), Wide8<D>::kThreads, 0, s>>>(p);
  } else {
    const unsigned grid = units * static_cast<unsigned>(p.hkv / heads);
    if (heads == 1) quantized_narrow_kernel<D, E, 1><<<grid, Narrow8<D>::kThreads, 0, s>>>(p);
    if constexpr (D < 256)
      if (heads == 2) quantized_narrow_kernel<D, E, 2><<<grid, Narrow8<D>::kThreads, 0, s>>>(p);
    if constexpr (D == 64)
      if (heads == 4) quantized_narrow_kernel<D, E, 4><<<grid, Narrow8<D>::kThreads, 0, s>>>(p);
  }
  return launch_join<D, E>(p, x, s);
}

int check_quantized(const ll_quantized_attention_args *a) {
  if (a == nullptr) return fail(LL_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->struct_size != static_cast<int64_t>(sizeof(*a)))
    return fail(LL_ERR_INVALID_ARGUMENT, "struct_size %lld, expected %lld", static_cast<long long>(a->struct_size),
                static_cast<long long>(sizeof(*a)));
  const int rc = check_args(&a->paged);
  if (rc != LL_OK) return rc;
  if (a->scale_block < kGroupKeys || a->scale_block > 128 || (a->scale_block & (a->scale_block - 1)) != 0)
    return fail(LL_ERR_INVALID_ARGUMENT, "scale_block must be 16, 32, 64 or 128");
  if (a->paged.page_size % a->scale_block != 0 || a->paged.num_slots % a->scale_block != 0)
    return fail(LL_ERR_INVALID_ARGUMENT, "pages and the pool must be whole blocks");
  if (a->paged.num_queries > 0 && a->paged.num_requests > 0 && a->paged.num_slots > 0 &&
      (a->key_scales == nullptr || a->value_scales == nullptr))
    return fail(LL_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
  return LL_OK;
}

}  // namespace

extern "C" {

int64_t ll_quantized_attention_args_size(void) { return static_cast<int64_t>(sizeof(ll_quantized_attention_args)); }

int64_t ll_quantized_attention_workspace_bytes(const ll_quantized_attention_args *a) {
  const int rc = check_quantized(a);
  if (rc != LL_OK) return rc;
  if (a->paged.num_queries == 0 || a->paged.num_requests == 0) return 0;
  return plan_launch(&a->paged, heads_together(a->paged), true).ws_floats * 4;
}

int ll_quantized_attention(const ll_quantized_attention_args *a, ll_stream_t stream) {
  int rc = check_quantized(a);
  if (rc != LL_OK || a->paged.num_queries == 0 || a->paged.num_requests == 0) return rc;
  const Launch x = plan_launch(&a->paged, heads_together(a->paged), true);
  QuantizedParams p;
  memset(&p, 0, sizeof(p));
  rc = fill_params(&a->paged, x, &p);
  if (rc != LL_OK) return rc;
  p.k8 = static_cast<const uint8_t *>(a->paged.key_buffer);
  p.v8 = static_cast<const uint8_t *>(a->paged.value_buffer);
  p.row_bytes = static_cast<unsigned>(a->paged.num_kv_heads * a->paged.head_dim);
  p.k_scales = static_cast<const uint8_t *>(a->key_scales);
  p.v_scales = static_cast<const uint8_t *>(a->value_scales);
  while ((1ll << p.block_shift) < a->scale_block) ++p.block_shift;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool f16 = a->paged.kv_dtype == LL_DTYPE_FLOAT16;
  const int heads = heads_together(a->paged);
  if (a->paged.head_dim == 64) return f16 ? launch_all<64, F16>(p, x, heads, s) : launch_all<64, Bf16>(p, x, heads, s);
  if (a->paged.head_dim == 128)
    return f16 ? launch_all<128, F16>(p, x, heads, s) : launch_all<128, Bf16>(p, x, heads, s);
  return f16 ? launch_all<256, F16>(p, x, heads, s) : launch_all<256, Bf16>(p, x, heads, s);
}

}  // extern "C"
