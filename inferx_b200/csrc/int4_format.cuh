// Weights held in four bits: how a matrix is laid out, and how codes become numbers.
//
// A row is cut along K into groups of 32, 64 or 128 entries; entry = scale * (code - zero) with a
// code and a zero point in 0..15 and a bfloat16 scale per row and group.
//
// Blocks.  [matrix][chunk of 128 k][strip of 16 rows], K padded to whole chunks and rows to whole
// strips; a block is 256 words of codes and 16 x (128 / group) words of parameters behind them.  So the
// strips that a tile of weight rows takes of a chunk are one piece of memory (one bulk copy), and a
// strip's share of it is 1 KB and its parameters.
//
// Codes.  [tile of 64 k][lane 0..31][word 0..3].  Word j of lane 4 g + t has the entries k = 16 j +
// 4 t .. + 3 of rows g and g + 8.  Nibbles i and i + 4 of a word are a pair of neighbouring k: i = 0, 1:
// the first pair of rows g and g + 8; i = 2, 3: the second.  So a word is the A side of one
// mma.m16n8k16 (k in an order that the activations' 8-byte loads follow too), and, as four registers of
// pairs, sixteen rows by sixteen k of an operand in tensor memory (the 16x256b shape).
//
// Parameters.  [row 0..15][group of the chunk]: one word, the scale times 2^11 in the low half, 2^-4 +
// zero * 2^-11 as bfloat16 in the high half.  (The zero point as a nibble would be 1.5 of 67 bytes a
// group less; the word needs no arithmetic before its use.)
//
// A code c becomes the bfloat16 2^-4 + c * 2^-11 by setting its bits below 0x3d80, and the difference
// to 2^-4 + zero * 2^-11 is exact: products of activations with codes are formed from multiples of
// 2^-11 up to 15 * 2^-11, summed in fp32 over a group, and the group's scale multiplies the sum in
// fp32.  128 of them are less than one, so the sum of a group does not overflow where the activations
// have not (as whole numbers up to 15 they did from 1.7e35 on), and down to activations of 2^-133, the
// last bit that bfloat16 has, their products are numbers that fp32 holds.  A scale that 2^11 would
// take out of bfloat16's range is held as it is, over codes as whole numbers: 128 + zero (0x4300 +
// zero) in the high half says so.
// Padding codes equal their group's zero point, padding rows and groups have scale 0.
#pragma once
#include "common.cuh"

#define I4_STRIP 16                    // rows of a strip
#define I4_TILE_WORDS 128              // 16 rows x 64 k
#define I4_CHUNK_K 128                 // k of a chunk
#define I4_CODE_WORDS 256              // a block's codes

// words of a block
__host__ __device__ constexpr int i4_block_words(int group) { return I4_CODE_WORDS + 16 * (128 / group); }

// A matrix, or one per expert, as the products' entry points take it (filled in by the caller).
struct I4Weight {
  const unsigned* data;
  int N;                               // columns of the product: rows of a matrix
  int E;                               // experts
  int group;
  int dual;                            // a gate and an up matrix per expert
  int settled;                         // nothing on the device writes it any more
};

// Shared memory beyond 48 KB has to be asked for once per kernel and device.
template <typename F> static inline cudaError_t i4_allow_smem(F kern, int bytes, unsigned* done) {
  int dev = 0;
  cudaGetDevice(&dev);
  const unsigned bit = 1u << (dev & 31);
  if (*done & bit) return cudaSuccess;
  const cudaError_t e =
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) *done |= bit;
  return e;
}

__host__ __device__ static inline long long i4_strips(long long rows) {
  return (rows + I4_STRIP - 1) / I4_STRIP;
}
__host__ __device__ static inline long long i4_chunks(long long k) {
  return (k + I4_CHUNK_K - 1) / I4_CHUNK_K;
}

#define I4_UNIT 0x3d80u                // 2^-4, whose last bit is 2^-11
#define I4_WHOLE 0x4300u               // 128, whose last bit is 1

// scale (bfloat16) and zero point as a parameter, and back
__device__ __forceinline__ unsigned i4_param(__nv_bfloat16 scale, int zero) {
  const float s = __bfloat162float(scale);
  // (2^11 is exact: a smaller scale only leaves the subnormal numbers)
  if (fabsf(s) < 0x1p116f)
    return (unsigned)__bfloat16_as_ushort(__float2bfloat16_rn(s * 2048.f)) |
           ((I4_UNIT + (unsigned)zero) << 16);
  return (unsigned)__bfloat16_as_ushort(scale) | ((I4_WHOLE + (unsigned)zero) << 16);
}
__device__ __forceinline__ int i4_param_zero(unsigned param) { return (param >> 16) & 15; }
__device__ __forceinline__ unsigned short i4_param_scale(unsigned param) {
  const float s = __uint_as_float(param << 16);
  return (param >> 20) == (I4_UNIT >> 4)
             ? __bfloat16_as_ushort(__float2bfloat16_rn(s * (1.f / 2048.f)))
             : (unsigned short)param;
}

__device__ __forceinline__ float i4_scale(unsigned param) { return __uint_as_float(param << 16); }
// the zero point's number in both halves
__device__ __forceinline__ unsigned i4_sub(unsigned param) { return __byte_perm(param, 0, 0x3232); }

// Nibbles i and i + 4 of a word, less the zero point: two neighbouring k.
__device__ __forceinline__ unsigned i4_pair(unsigned word, int i, unsigned sub) {
  unsigned q = ((word >> (4 * i)) & 0x000f000fu) | (sub & 0xfff0fff0u);
  const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&q),
                                   *reinterpret_cast<const __nv_bfloat162*>(&sub));
  return *reinterpret_cast<const unsigned*>(&d);
}

// An fp32 number as three bfloat16 terms by cutting off: 8 + 8 + 8 bits, nothing is left over (down
// to 2^-133, the last bit that bfloat16 has).  An infinity is its first term alone.
__device__ __forceinline__ void i4_terms2(float a, float b, unsigned& t1, unsigned& t2,
                                          unsigned& t3) {
  const unsigned a1 = __float_as_uint(a) & 0xffff0000u, b1 = __float_as_uint(b) & 0xffff0000u;
  t1 = __byte_perm(a1, b1, 0x7632);
  a = fabsf(a) == INFINITY ? 0.f : a - __uint_as_float(a1);
  b = fabsf(b) == INFINITY ? 0.f : b - __uint_as_float(b1);
  const unsigned a2 = __float_as_uint(a) & 0xffff0000u, b2 = __float_as_uint(b) & 0xffff0000u;
  t2 = __byte_perm(a2, b2, 0x7632);
  a -= __uint_as_float(a2);
  b -= __uint_as_float(b2);
  t3 = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
}
