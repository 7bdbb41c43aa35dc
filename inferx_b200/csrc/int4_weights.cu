// Making, laying out and reading back matrices of four-bit codes (int4_format.cuh).
//
// Quantising a group: lo = min(0, least entry), hi = max(0, greatest), scale = (hi - lo) / 15 rounded
// once to bfloat16, zero = rint(-lo / scale), code = rint(entry / scale) + zero, both kept in 0..15.
// A group of zeros (or so small that its scale is 0) has scale, zero point and codes 0; a group that
// holds an infinity or a NaN has scale NaN, so that products say so.
//
// One warp takes 16 rows by 128 k: a lane holds the 64 entries whose codes it packs, least and greatest
// entries are joined over the four lanes of a row by shuffles, nothing passes through shared memory, and
// each entry is read once.  Measured: 6,144 x 2,048 bfloat16 15 us, fp32 20 (the bytes alone 5 and 9):
// finding the extremes and the two comparisons of an entry's remainder, not the bytes, set the pace.
#include "int4_format.cuh"

#define I4_WARPS 8

// The nearest whole number to v / s (ties to even) for |v| <= 16 s, r near 1 / s.  The product is off by
// a step at most, and the remainder (exact: v has 24 bits, s has 8) says which way.
__device__ __forceinline__ int i4_rint_ratio(float v, float s, float r) {
  const float t = fmaf(v, r, 12582912.f);          // its last bit is 1: a whole number in the low bits
  int q = __float_as_int(t) - 0x4b400000;
  const float left = fmaf(12582912.f - t, s, v), half = 0.5f * s;
  if (fabsf(left) >= half) {
    const bool odd = q & 1;
    if (left > half || (left == half && odd)) ++q;
    else if (left < -half || (left == -half && odd)) --q;
  }
  return q;
}

// (hi - lo) / 15 rounded once to bfloat16.  In 32 bits the quotient is off by less than two of its
// steps, which matters only where it lies as near to the middle of two bfloat16 numbers (or is too small
// for 24 bits): there it is formed in 64 bits, cut to 32 with the last bit set where something was cut
// off, and rounded from that.
__device__ __forceinline__ bf16 i4_group_scale(float lo, float hi) {
  float t = __fdiv_rn(hi - lo, 15.f);
  const int from_middle = (int)(__float_as_uint(t) & 0xffffu) - 0x8000;
  if ((unsigned)(from_middle + 4) <= 8u || t < 1e-30f || t > 1e37f) {
    const double q = ((double)hi - (double)lo) / 15.0;
    unsigned u = __float_as_uint(__double2float_rz(q));
    if ((double)__uint_as_float(u) != q) u |= 1u;
    t = __uint_as_float(u);
  }
  return __float2bfloat16_rn(t);
}

// Where a warp works: matrix, strip, chunk; false behind the last.
struct I4Place {
  long long m;
  int strip, chunk;
};
__device__ __forceinline__ bool i4_place(I4Place& p, long long matrices, int strips, int chunks) {
  const long long w = (long long)blockIdx.x * I4_WARPS + (threadIdx.x >> 5);
  if (w >= matrices * strips * chunks) return false;
  p.chunk = (int)(w % chunks);               // (neighbouring warps read a row's neighbouring k)
  const long long s = w / chunks;
  p.strip = (int)(s % strips);
  p.m = s / strips;
  return true;
}
__device__ __forceinline__ size_t i4_block(const I4Place& p, int strips, int chunks) {
  return ((size_t)p.m * chunks + p.chunk) * strips + p.strip;
}

// The 32 entries of a row that a lane of `t` holds of a chunk, four of every sixteen, from `src` (the
// row, or null: zeros), in their own type: 16 registers of bfloat16 pairs leave room for twice the warps
// that 32 numbers would.
template <typename T> struct I4Entries;
template <> struct I4Entries<float> {
  float v[32];
  __device__ __forceinline__ float at(int i) const { return v[i]; }
  __device__ __forceinline__ void load(const float* src, int k0, int K, int t, bool vec) {
#pragma unroll
    for (int b = 0; b < 8; ++b) {                  // blocks of 16 k
      const int k = k0 + b * 16 + t * 4;
      if (vec) {                                   // K is a multiple of 4
        const float4 r = src && k < K ? *reinterpret_cast<const float4*>(src + k)
                                      : make_float4(0.f, 0.f, 0.f, 0.f);
        v[b * 4] = r.x;
        v[b * 4 + 1] = r.y;
        v[b * 4 + 2] = r.z;
        v[b * 4 + 3] = r.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[b * 4 + i] = src && k + i < K ? src[k + i] : 0.f;
      }
    }
  }
};
template <> struct I4Entries<bf16> {
  unsigned v[16];
  __device__ __forceinline__ float at(int i) const {
    return __uint_as_float((i & 1) ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16);
  }
  __device__ __forceinline__ void load(const bf16* src, int k0, int K, int t, bool vec) {
    const unsigned short* bits = reinterpret_cast<const unsigned short*>(src);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const int k = k0 + b * 16 + t * 4;
      if (vec) {
        const uint2 r = src && k < K ? *reinterpret_cast<const uint2*>(bits + k) : make_uint2(0, 0);
        v[b * 2] = r.x;
        v[b * 2 + 1] = r.y;
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const unsigned lo = src && k + 2 * i < K ? bits[k + 2 * i] : 0u;
          const unsigned hi = src && k + 2 * i + 1 < K ? bits[k + 2 * i + 1] : 0u;
          v[b * 2 + i] = lo | (hi << 16);
        }
      }
    }
  }
};

// codes of rows g and g + 8 (32 each, in the order of I4Entries) to the lane's words
__device__ __forceinline__ void i4_store_words(unsigned* dst, int lane, const unsigned char* ca,
                                               const unsigned char* cb) {
#pragma unroll
  for (int tile = 0; tile < 2; ++tile) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = tile * 16 + i * 4;
      w[i] = (unsigned)ca[at] | ((unsigned)ca[at + 1] << 16) | ((unsigned)cb[at] << 4) |
             ((unsigned)cb[at + 1] << 20) | ((unsigned)ca[at + 2] << 8) |
             ((unsigned)ca[at + 3] << 24) | ((unsigned)cb[at + 2] << 12) |
             ((unsigned)cb[at + 3] << 28);
    }
    *reinterpret_cast<uint4*>(dst + tile * I4_TILE_WORDS + lane * 4) =
        make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <typename T, int GROUP>
__global__ void __launch_bounds__(I4_WARPS * 32, sizeof(T) == 2 ? 4 : 2)
i4_quantize_kernel(const T* __restrict__ w, unsigned* __restrict__ data,
                   long long matrices, int rows, int K, int strips,
                   int chunks, int vec) {
  constexpr int PER = GROUP / 32, NG = 4 / PER;    // blocks of 32 a group, groups a chunk
  I4Place p;
  if (!i4_place(p, matrices, strips, chunks)) return;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int k0 = p.chunk * I4_CHUNK_K;
  const size_t block = i4_block(p, strips, chunks) * i4_block_words(GROUP);
  I4Entries<T> v[2];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const int row = p.strip * I4_STRIP + g + side * 8;
    v[side].load(row < rows ? w + ((size_t)p.m * rows + row) * K : nullptr, k0, K, t, vec != 0);
  }
  unsigned word[8];                                // of sixteen k each
#pragma unroll
  for (int side = 0; side < 2; ++side) {
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const int first = n * PER * 8;
      float lo = 0.f, hi = 0.f, odd_one = 0.f;     // the last is NaN where an entry is not finite
#pragma unroll
      for (int i = 0; i < PER * 8; ++i) {
        const float e = v[side].at(first + i);
        lo = fminf(lo, e);
        hi = fmaxf(hi, e);
        odd_one = fmaf(e, 0.f, odd_one);
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        odd_one += __shfl_xor_sync(0xffffffffu, odd_one, o);
      }
      const bf16 scale = odd_one != 0.f ? __ushort_as_bfloat16(0x7fc0) : i4_group_scale(lo, hi);
      float s = __bfloat162float(scale);
      const bool some = s > 0.f;                   // false for 0 and for NaN
      int zero = 0;
      // (so that 1 / s is a number, a group whose scale is tiny is taken 2^100 times as large)
      auto quantize = [&](float up) {
        s *= up;
        const float r = some ? __frcp_rn(s) : 0.f;
        zero = some ? min(max(i4_rint_ratio(-lo * up, s, r), 0), 15) : 0;
#pragma unroll
        for (int i = 0; i < PER * 2; ++i) {
          unsigned c[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float e = v[side].at(first + 4 * i + j) * up;
            const int q = min(max(i4_rint_ratio(e, s, r) + zero, 0), 15);
            c[j] = some ? (unsigned)q : 0u;
          }
          const unsigned half = (c[0] | (c[1] << 16)) | ((c[2] << 8) | (c[3] << 24));
          unsigned& at = word[n * PER * 2 + i];
          at = side ? at | (half << 4) : half;
        }
      };
      if (s < 1e-30f) quantize(1.2676506e30f);
      else quantize(1.f);
      if (t == 0)
        data[block + I4_CODE_WORDS + (g + side * 8) * NG + n] = i4_param(scale, zero);
    }
  }
#pragma unroll
  for (int tile = 0; tile < 2; ++tile)
    *reinterpret_cast<uint4*>(data + block + tile * I4_TILE_WORDS + lane * 4) = make_uint4(
        word[tile * 4], word[tile * 4 + 1], word[tile * 4 + 2], word[tile * 4 + 3]);
}

// Codes, scales and zero points of a caller's own into the layout.
template <int GROUP>
__global__ void __launch_bounds__(I4_WARPS * 32)
i4_pack_kernel(const unsigned char* __restrict__ in, const bf16* __restrict__ scales,
               const unsigned char* __restrict__ zeros, unsigned* __restrict__ data,
               long long matrices, int rows, int K, int strips,
               int chunks, int vec) {
  constexpr int PER = GROUP / 32, NG = 4 / PER;
  I4Place p;
  if (!i4_place(p, matrices, strips, chunks)) return;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int k0 = p.chunk * I4_CHUNK_K, groups = (K + GROUP - 1) / GROUP;
  const size_t block = i4_block(p, strips, chunks) * i4_block_words(GROUP);
  unsigned char code[2][32];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const int row = p.strip * I4_STRIP + g + side * 8;
    const size_t r = (size_t)p.m * rows + row;
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const int group = p.chunk * NG + n;
      const bool there = row < rows && group < groups;
      const bf16 scale = there ? scales[r * groups + group] : __ushort_as_bfloat16(0);
      const int zero = there ? zeros[r * groups + group] & 15 : 0;
#pragma unroll
      for (int b = 0; b < 2 * PER; ++b) {          // blocks of 16 k
        const int at = (n * 2 * PER + b) * 4, k = k0 + (n * 2 * PER + b) * 16 + t * 4;
        if (vec && there && k < K) {               // K is a multiple of 4
          const unsigned q = *reinterpret_cast<const unsigned*>(in + r * K + k);
#pragma unroll
          for (int i = 0; i < 4; ++i) code[side][at + i] = (q >> (8 * i)) & 15;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            code[side][at + i] = there && k + i < K ? in[r * K + k + i] & 15 : zero;
        }
      }
      if (t == 0)
        data[block + I4_CODE_WORDS + (g + side * 8) * NG + n] = i4_param(scale, zero);
    }
  }
  i4_store_words(data + block, lane, code[0], code[1]);
}

// The layout back to codes, scales and zero points.
template <int GROUP>
__global__ void __launch_bounds__(I4_WARPS * 32)
i4_unpack_kernel(const unsigned* __restrict__ data, unsigned char* __restrict__ out, bf16* __restrict__ scales,
                 unsigned char* __restrict__ zeros, long long matrices, int rows, int K, int strips,
                 int chunks, int whole) {
  constexpr int NG = 128 / GROUP;
  I4Place p;
  if (!i4_place(p, matrices, strips, chunks)) return;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int k0 = p.chunk * I4_CHUNK_K, groups = (K + GROUP - 1) / GROUP;
  const size_t block = i4_block(p, strips, chunks) * i4_block_words(GROUP);
  uint4 w[2];
#pragma unroll
  for (int tile = 0; tile < 2; ++tile)
    w[tile] = *reinterpret_cast<const uint4*>(data + block +
                                              tile * I4_TILE_WORDS + lane * 4);
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const int row = p.strip * I4_STRIP + g + side * 8;
    const size_t r = (size_t)p.m * rows + row;
#pragma unroll
    for (int h = 0; h < 2; ++h) {                  // 64 k: a lane's four codes of each sixteen
      const unsigned from[4] = {w[h].x, w[h].y, w[h].z, w[h].w};
      unsigned o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned u = from[j] >> (4 * side);
        o[j] = __byte_perm(u & 0x0f0f0f0fu, 0, 0x3120);
      }
      if (whole) {
        // the four lanes of a row trade, so that lane t has sixteen codes beside each other
        const bool up = t & 2, right = t & 1;
        unsigned a0 = up ? o[0] : o[2], a1 = up ? o[1] : o[3];
        a0 = __shfl_xor_sync(0xffffffffu, a0, 2);
        a1 = __shfl_xor_sync(0xffffffffu, a1, 2);
        const unsigned m[4] = {up ? a0 : o[0], up ? a1 : o[1], up ? o[2] : a0, up ? o[3] : a1};
        unsigned b0 = right ? m[0] : m[1], b1 = right ? m[2] : m[3];
        b0 = __shfl_xor_sync(0xffffffffu, b0, 1);
        b1 = __shfl_xor_sync(0xffffffffu, b1, 1);
        const uint4 r4 = make_uint4(right ? b0 : m[0], right ? m[1] : b0, right ? b1 : m[2],
                                    right ? m[3] : b1);
        const int k = k0 + h * 64 + t * 16;
        if (row < rows && k < K) *reinterpret_cast<uint4*>(out + r * K + k) = r4;
      } else if (row < rows) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = k0 + h * 64 + j * 16 + t * 4;
          if (K % 4 == 0 && ((uintptr_t)out & 3) == 0) {
            if (k < K) *reinterpret_cast<unsigned*>(out + r * K + k) = o[j];
            continue;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (k + i < K) out[r * K + k + i] = (unsigned char)(o[j] >> (8 * i));
        }
      }
    }
    if (row >= rows) continue;
    for (int n = t; n < NG; n += 4) {
      const int group = p.chunk * NG + n;
      if (group >= groups) continue;
      const unsigned param = data[block + I4_CODE_WORDS + (g + side * 8) * NG + n];
      scales[r * groups + group] = __ushort_as_bfloat16(i4_param_scale(param));
      zeros[r * groups + group] = (unsigned char)i4_param_zero(param);
    }
  }
}

static int i4_grid(long long matrices, int rows, int K, int& strips, int& chunks, unsigned& grid) {
  if (matrices <= 0 || rows <= 0 || K <= 0) return IX_ERR_SIZE;
  strips = (int)i4_strips(rows);
  chunks = (int)i4_chunks(K);
  const long long blocks = (matrices * strips * chunks + I4_WARPS - 1) / I4_WARPS;
  if (blocks > 0x7fffffffLL) return IX_ERR_SIZE;
  grid = (unsigned)blocks;
  return IX_OK;
}

#define I4_GROUPS(G, ...)                                                      \
  do {                                                                         \
    if (group == 128) { constexpr int G = 128; __VA_ARGS__; }                  \
    else if (group == 64) { constexpr int G = 64; __VA_ARGS__; }               \
    else if (group == 32) { constexpr int G = 32; __VA_ARGS__; }               \
    else return IX_ERR_UNSUPPORTED;                                            \
  } while (0)

// w: [matrices, rows, K] fp32 or bf16.  data: [matrices, chunks, strips, words of a block].
IX_API int ix_int4_quantize(const void* w, int dtype, void* data, long long matrices, int rows, int K,
                            int group, cudaStream_t stream) {
  int strips, chunks;
  unsigned grid;
  const int rc = i4_grid(matrices, rows, K, strips, chunks, grid);
  if (rc != IX_OK) return rc;
  const int vec = K % 4 == 0 && ((uintptr_t)w & 15) == 0;
  IX_DISPATCH_DTYPE(dtype, T, {
    I4_GROUPS(G, i4_quantize_kernel<T, G><<<grid, I4_WARPS * 32, 0, stream>>>(
                     (const T*)w, (unsigned*)data, matrices, rows, K, strips,
                     chunks, vec));
  });
  return ix_launch_status();
}

// in: [matrices, rows, K] bytes; scales bf16 and zeros bytes: [matrices, rows, ceil(K / group)].
IX_API int ix_int4_pack(const void* in, const void* scales, const void* zeros, void* data,
                        long long matrices, int rows, int K, int group,
                        cudaStream_t stream) {
  int strips, chunks;
  unsigned grid;
  const int rc = i4_grid(matrices, rows, K, strips, chunks, grid);
  if (rc != IX_OK) return rc;
  const int vec = K % 4 == 0 && ((uintptr_t)in & 3) == 0;
  I4_GROUPS(G, i4_pack_kernel<G><<<grid, I4_WARPS * 32, 0, stream>>>(
                   (const unsigned char*)in, (const bf16*)scales, (const unsigned char*)zeros,
                   (unsigned*)data, matrices, rows, K, strips, chunks, vec));
  return ix_launch_status();
}

IX_API int ix_int4_unpack(const void* data, void* out, void* scales,
                          void* zeros, long long matrices, int rows, int K, int group,
                          cudaStream_t stream) {
  int strips, chunks;
  unsigned grid;
  const int rc = i4_grid(matrices, rows, K, strips, chunks, grid);
  if (rc != IX_OK) return rc;
  const int whole = K % 16 == 0 && ((uintptr_t)out & 15) == 0;
  I4_GROUPS(G, i4_unpack_kernel<G><<<grid, I4_WARPS * 32, 0, stream>>>(
                   (const unsigned*)data, (unsigned char*)out, (bf16*)scales,
                   (unsigned char*)zeros, matrices, rows, K, strips, chunks, whole));
  return ix_launch_status();
}

// Activation rows as the products want them: gathered where `rows` names them, with zeros from K up to
// Kp, in their own type (TERMS 1) or as three planes of bfloat16 terms (fp32, TERMS 3).
template <typename T, int TERMS>
__global__ void __launch_bounds__(128)
i4_rows_kernel(const T* __restrict__ x, const int* __restrict__ rows, void* __restrict__ out, int R,
               int K, int Kp) {
  IX_PDL_WAIT();
  const size_t r = blockIdx.x, src = rows ? (size_t)rows[r] : r;
  for (int k = 2 * threadIdx.x; k < Kp; k += 256) {    // Kp is even
    const float a = k < K ? to_f32<T>(x[src * K + k]) : 0.f;
    const float b = k + 1 < K ? to_f32<T>(x[src * K + k + 1]) : 0.f;
    if (TERMS == 3) {
      unsigned t1, t2, t3;
      i4_terms2(a, b, t1, t2, t3);
      unsigned* o = (unsigned*)out + (r * Kp + k) / 2;
      const size_t plane = (size_t)R * Kp / 2;
      o[0] = t1;
      o[plane] = t2;
      o[2 * plane] = t3;
    } else {
      T* o = (T*)out + r * Kp + k;
      o[0] = from_f32<T>(a);
      o[1] = from_f32<T>(b);
    }
  }
}

IX_API int ix_int4_rows(const void* x, int dtype, const int* rows, void* out, int R, int K, int Kp,
                        int terms, cudaStream_t stream) {
  if (R <= 0) return IX_OK;
  if (K <= 0 || Kp < K || Kp % 8) return IX_ERR_SIZE;
  if ((uintptr_t)out & 15) return IX_ERR_ALIGN;
  if (terms == 3 && dtype == IX_F32)
    ix_launch(i4_rows_kernel<float, 3>, dim3(R), dim3(128), 0, stream, (const float*)x, rows, out, R,
              K, Kp);
  else if (terms == 1 && dtype == IX_F32)
    ix_launch(i4_rows_kernel<float, 1>, dim3(R), dim3(128), 0, stream, (const float*)x, rows, out, R,
              K, Kp);
  else if (terms == 1 && dtype == IX_BF16)
    ix_launch(i4_rows_kernel<bf16, 1>, dim3(R), dim3(128), 0, stream, (const bf16*)x, rows, out, R,
              K, Kp);
  else
    return IX_ERR_UNSUPPORTED;
  return ix_launch_status();
}
