// Shared pieces of the transformer-block kernels (blk_gemm.hip, blk_attn.hip): operand types, the matrix instruction behind a
// 16-byte fragment, asynchronous copies into LDS, activations.
#pragma once
#include "common.h"

typedef __bf16 bf16;
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

#define MG_LDS __attribute__((address_space(3)))
#define MG_GLB __attribute__((address_space(1)))

#define BLK_F32 0
#define BLK_BF16 1

// activation codes beyond those of common.h
#define ACT_SILU 4
#define ACT_GELU 5

// D[i][j] += sum_k A[i][k] B[k][j] over the 64 bytes of a row that the four 16-lane groups hold, 16 bytes a lane: lane l = 16 g + i
// holds row i's chunk g of both operands.  bf16: one 16x16x32 instruction (k = 8 g + t); f32: four 16x16x4 instructions, number t
// takes element t of every lane's chunk (k = 4 g + t: a sum over k may take its terms in any order that both operands share).
template <class T>
struct Mf;
template <>
struct Mf<bf16> {
  static constexpr int CH = 8;  // elements of a 16-byte chunk
  static __device__ __forceinline__ f32x4 step(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Mf<float> {
  static constexpr int CH = 4;
  static __device__ __forceinline__ f32x4 step(u32x4 a, u32x4 b, f32x4 c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[t], y[t], c, 0, 0, 0);
    return c;
  }
};

// 16 bytes a lane from global memory straight into LDS: lane l's data lands at `lds` + 16 l (`lds` is the wave's, not the lane's).
__device__ __forceinline__ void lds_copy16(const void* g, void* lds) {
  __builtin_amdgcn_global_load_lds((MG_GLB const void*)g, (MG_LDS void*)lds, 16, 0, 0);
}

// Copies into LDS are waited for by hand: copies_done() for all of them, a counted wait where some may stay under way.  Left to itself the
// compiler waits for every copy before any read that might meet one, the next tile's included, which undoes the double buffer.  It does not
// where a kernel has one __shared__ object and where the pointer of a transposing read is its own (__restrict: nothing is written while
// the function runs).  Training pass of the gated layer, 8,192 rows of 4,096: 2.95 -> 2.79 ms; attention's forward pass at width 128: 854 -> 830 us.
__device__ __forceinline__ void copies_done() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// The transposing read: four 16-bit values of each of the lane's group's rows.
__device__ __forceinline__ s16x4 lds_transposed(const char* __restrict p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((MG_LDS s16x4*)p); }

// Activation and derivative by its INPUT z.  exp through __expf, whose error grows with its argument: (8 + |z|) 2^-23 of the value at most.
// gelu is the exact form z Phi(z), Phi by erf: a few 2^-24 of |z|.
__device__ __forceinline__ float blk_act(float z, int act, float slope) {
  switch (act) {
    case ACT_LEAKY: return z > 0.f ? z : z * slope;
    case ACT_SIGMOID: return mg_sigmoid(z);
    case ACT_SILU: return z * mg_sigmoid(z);
    case ACT_GELU: return z * (0.5f + 0.5f * erff(z * 0.70710678f));
    default: return z;
  }
}
__device__ __forceinline__ float blk_act_grad(float z, int act, float slope) {
  switch (act) {
    case ACT_LEAKY: return z > 0.f ? 1.f : slope;
    case ACT_SIGMOID: {
      const float s = mg_sigmoid(z);
      return s * (1.f - s);
    }
    case ACT_SILU: {
      const float s = mg_sigmoid(z);
      return s * (1.f + z * (1.f - s));
    }
    case ACT_GELU: return 0.5f + 0.5f * erff(z * 0.70710678f) + z * 0.39894228f * __expf(-0.5f * z * z);
    default: return 1.f;
  }
}
