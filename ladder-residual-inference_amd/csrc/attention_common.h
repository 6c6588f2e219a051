// What the prompts' attentions on the matrix cores share, that of a contiguous cache (attention.hip) and that of a paged one (paged_attention.hip).
#pragma once
#include "lr_common.h"

typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));

// e^x through the hardware exp2 (1 ulp in fp32: far below the bf16 rounding of the output), with the score scale
// folded into its argument; the library expf costs ~15 VALU instructions, and these kernels are VALU-bound next to
// their MFMAs
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
// max(a, b) as the median of {a, b, +inf}: one instruction (fmaxf makes the compiler canonicalise both operands
// first, an instruction each, when they come out of a matrix-core product).  Which of the two it is where one is NaN is left open.
// (No inline assembler here: the compiler does not count the wait states between a matrix-core instruction and
// an assembler statement that reads its result, and the statement then reads the registers too early.)
__device__ __forceinline__ float max_med3(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, INFINITY); }

// Keys and values in LDS: the place among a row's 16-byte pieces is the piece's number XOR this: 16 lanes reading one piece of 16 consecutive keys,
// and 16 reading four neighbouring pieces (32 dimensions) of four keys, touch every bank once
template <int HD>
__device__ __forceinline__ int key_swizzle(int key) { return HD == 128 ? key & 15 : (key >> 1) & 7; }
template <int HD>
__device__ __forceinline__ int value_swizzle(int key) { return HD == 128 ? (key & 3) << 2 : ((key >> 1) & 1) << 2; }
