// Device pieces that the library's attention kernels share: the 16-bit element
// types with their MFMAs and roundings, exchanges between the lanes of a column,
// and gathers of rows straight into LDS.
#ifndef ATTENTION_DEVICE_H
#define ATTENTION_DEVICE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) short i16x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

// The 16-bit element types of queries, keys, values and outputs: the MFMA
// that takes them (fp32 accumulation) and the rounding of fp32 results back
// to them (two at a time, round to nearest even).
struct Bf16 {
  typedef bf16x8 frag;
  static constexpr uint32_t kOnes = 0x3F803F80u;  // two 1.0s
  static constexpr float kWeightShift = 0.f;      // log2 of what paged attention scales its weights by
  __device__ static uint32_t pack(float lo, float hi) {  // one v_cvt_pk_bf16_f32
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
  }
  static constexpr uint32_t kExponent = 0x7F80u;  // of one value's bits
  __device__ static f32x16 mfma32(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  __device__ static f32x4 mfma16(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  __device__ static float dot2_ones(uint32_t pair, float acc) {  // acc + lo + hi, one v_dot2_f32_bf16
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), __builtin_bit_cast(bf16x2, kOnes),
                                           acc, false);
  }
  __device__ static f32x2 unpack(uint32_t pair) {  // exact
    return f32x2{__uint_as_float(pair << 16), __uint_as_float(pair & 0xffff0000u)};
  }
};

struct F16 {
  typedef f16x8 frag;
  static constexpr uint32_t kOnes = 0x3C003C00u;
  static constexpr float kWeightShift = 7.f;
  __device__ static uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, f16x2));
  }
  static constexpr uint32_t kExponent = 0x7C00u;
  __device__ static f32x16 mfma32(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  __device__ static f32x4 mfma16(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  __device__ static float dot2_ones(uint32_t pair, float acc) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pair), __builtin_bit_cast(f16x2, kOnes), acc, false);
  }
  __device__ static f32x2 unpack(uint32_t pair) {  // exact
    return __builtin_convertvector(__builtin_bit_cast(f16x2, pair), f32x2);
  }
};

// v_permlane32_swap a, b exchanges the upper half of a with the lower half of
// b: from two copies of x it leaves (x[l], x[l ^ 32]) in the lane, up to
// order -- the operands of an xor shuffle 32.  (Inline assembly: the compiler
// builtin loses the second result when both operands hold the same value.)
// The s_nop covers the wait states between a VALU write of an operand and the
// permute.
__device__ inline void permlane32_swap(unsigned &a, unsigned &b) {
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
}

// The same for an xor shuffle 16.
__device__ inline void permlane16_swap(unsigned &a, unsigned &b) {
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
}

// v_max_f32 straight from assembly: fmaxf would first quiet its operands
// (which come out of inline assembly) with two more instructions.  Scores
// reaching here are never NaN (masked ones are -inf).
__device__ inline float max_f32(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}

typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

// Two 16-byte-per-lane gathers into LDS (global_load_lds_dwordx4: lane l's
// bytes land at the LDS base in M0 + 16 l).  They are issued from inline
// assembly so that the compiler, which cannot tell the ring's stages apart,
// does not add waits for every outstanding gather before each LDS access:
// the kernels' loops order the stages themselves with explicit vmcnt waits and
// barriers.  M0 is saved and restored around them.
__device__ inline void dma_pair(const void *src0, void *lds0, const void *src1, void *lds1) {
  const unsigned base0 = __builtin_amdgcn_readfirstlane(
      static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void *)lds0)));
  const unsigned base1 = __builtin_amdgcn_readfirstlane(
      static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void *)lds1)));
  unsigned saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %3\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, off\n\t"
      "s_mov_b32 m0, %4\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %2, off\n\t"
      "s_nop 0\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "v"(src0), "v"(src1), "s"(base0), "s"(base1)
      : "memory");
}

// The LDS address of what a generic pointer into LDS points to.
__device__ inline unsigned lds_offset(void *lds) {
  return static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void *)lds));
}

// One of them, to the LDS address `base` (the same in every lane).  M0 is the
// compiler's to restore.
__device__ inline void dma_row(const void *src, unsigned base) {
  asm volatile(
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %0, off"
      :
      : "v"(src), "s"(base)
      : "memory", "m0");
}

// dma_pair with 32-bit byte offsets into the K and V buffers (buffer loads:
// one multiply-add per address instead of 64-bit address arithmetic), for
// pools whose K and V buffers each fit in 4 GiB.  The resources hold the
// buffer's base and size (loads past it would read zeros; the offsets used
// stay inside).
typedef int i32x4r __attribute__((ext_vector_type(4)));
__device__ inline i32x4r buffer_resource(const void *base, unsigned bytes) {
  const unsigned long long address = reinterpret_cast<unsigned long long>(base);
  i32x4r r;
  r[0] = static_cast<int>(static_cast<unsigned>(address));
  r[1] = static_cast<int>(static_cast<unsigned>(address >> 32) & 0xffffu);  // stride 0
  r[2] = static_cast<int>(bytes);
  r[3] = 0x00020000;  // raw 32-bit dwords
  return r;
}

__device__ inline void dma_pair_buffer(unsigned off0, void *lds0, i32x4r res0, unsigned off1, void *lds1,
                                       i32x4r res1) {
  const unsigned base0 = __builtin_amdgcn_readfirstlane(
      static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void *)lds0)));
  const unsigned base1 = __builtin_amdgcn_readfirstlane(
      static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void *)lds1)));
  unsigned saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %3\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %5, 0 offen lds\n\t"
      "s_mov_b32 m0, %4\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %2, %6, 0 offen lds\n\t"
      "s_nop 0\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "v"(off0), "v"(off1), "s"(base0), "s"(base1), "s"(res0), "s"(res1)
      : "memory");
}

// s_barrier without __syncthreads()'s wait for all outstanding memory
// operations (which would drain the gathers in flight); the empty asm keeps
// the compiler from moving LDS accesses across it.
__device__ inline void workgroup_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

}  // namespace

#endif  // ATTENTION_DEVICE_H
