// Products with four-bit weights for few rows (decode steps): the codes are read once, as they lie,
// and become tensor-core fragments in registers.
//
//   out[r, j] = sum_k x[src(r), k] * w[e(r), j, k]           (plain, an activation may follow)
//   out[r, j] = silu(x . wg[e, j]) * (x . wu[e, j])          (DUAL: gate and up matrices)
//   w[j, k] = scale[j, k / group] * (code[j, k] - zero[j, k / group])      (int4_format.cuh)
//
// Groups of rows are the experts of a mixture (ragged ranges from `offsets`, source rows from `rows`)
// or a single matrix with a few rows (E = 1).
//
// Mapping: out^T = w . x^T with mma.sync.m16n8k16, sixteen weight rows the M side, eight activation
// rows the N side.  A warp holds two strips of 16 weight rows (DUAL: a gate strip and the up strip of
// the same columns) against 8 NT activation rows, so an activation fragment serves both.  Per chunk of
// 128 k a lane loads 2 x 2 x 16 bytes of codes, turns each word into the A side of one mma with three
// shifts, four logic operations and four exact subtractions, and multiplies the fp32 sums of each
// group by the group's scale.  fp32 activations are three bfloat16 terms that are multiplied into the
// same sums.  The warps of a block split K by chunks and join their sums through shared memory in warp
// order, so a row's result does not depend on which rows share its tile.
#include "int4_format.cuh"

#define I4S_THREADS 256
#define I4S_WARPS 8

__device__ __forceinline__ uint4 i4s_ld16(const unsigned* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}
__device__ __forceinline__ void i4s_mma(float* c, const unsigned* a, unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// NG words (1, 2 or 4) that lie beside each other
template <int NG> __device__ __forceinline__ void i4s_params(const unsigned* p, unsigned* v) {
  if (NG == 1) v[0] = __ldg(p);
  if (NG == 2) {
    const uint2 r = __ldg(reinterpret_cast<const uint2*>(p));
    v[0] = r.x;
    v[NG - 1] = r.y;
  }
  if (NG == 4) {
    const uint4 r = __ldg(reinterpret_cast<const uint4*>(p));
    v[0] = r.x;
    v[NG > 1 ? 1 : 0] = r.y;
    v[NG > 2 ? 2 : 0] = r.z;
    v[NG - 1] = r.w;
  }
}

// Eight activations of a row as fragments: [term][pair of k].
template <typename XT> struct I4Frag;
template <> struct I4Frag<bf16> {
  static constexpr int TERMS = 1;
  uint4 r;
  __device__ __forceinline__ void load(const bf16* p, bool ok) {
    r = ok ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void terms(unsigned (*b)[4]) const {
    b[0][0] = r.x;
    b[0][1] = r.y;
    b[0][2] = r.z;
    b[0][3] = r.w;
  }
};
template <> struct I4Frag<float> {
  static constexpr int TERMS = 3;
  float4 lo, hi;
  __device__ __forceinline__ void load(const float* p, bool ok) {
    lo = ok ? *reinterpret_cast<const float4*>(p) : make_float4(0.f, 0.f, 0.f, 0.f);
    hi = ok ? *reinterpret_cast<const float4*>(p + 4) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ void terms(unsigned (*b)[4]) const {
    i4_terms2(lo.x, lo.y, b[0][0], b[1][0], b[2][0]);
    i4_terms2(lo.z, lo.w, b[0][1], b[1][1], b[2][1]);
    i4_terms2(hi.x, hi.y, b[0][2], b[1][2], b[2][2]);
    i4_terms2(hi.z, hi.w, b[0][3], b[1][3], b[2][3]);
  }
};

struct I4Out {
  void* out;
  int wide;                 // fp32 results, otherwise bfloat16
  const float* row_scale;   // DUAL: one factor per output row on both products, or null
  int plain;                // not DUAL: IX_ACT_*
};

template <bool DUAL>
__device__ __forceinline__ void i4s_store(const I4Out& o, size_t r, int j, int N, float v, float u) {
  if (DUAL) {
    if (o.row_scale) {
      const float f = o.row_scale[r];
      v *= f;
      u *= f;
    }
    v = v / (1.0f + (o.wide ? expf(-v) : __expf(-v))) * u;
  } else if (o.plain) {
    v = o.wide ? ix_act<float>(v, o.plain) : ix_act<bf16>(v, o.plain);
  }
  if (o.wide) ((float*)o.out)[r * N + j] = v;
  else ((bf16*)o.out)[r * N + j] = __float2bfloat16_rn(v);
}

template <typename XT, bool DUAL, int NT, int GROUP>
__global__ void __launch_bounds__(I4S_THREADS)
int4_stream_kernel(const XT* __restrict__ x, const int* __restrict__ rows,
                   const int* __restrict__ offsets, const unsigned* __restrict__ codes,
                   const unsigned* __restrict__ params, I4Out out, int M_single, int N, int K,
                   int strips, int chunks, int ksplit, int offsets_settled) {
  constexpr int NG = 128 / GROUP, PER = GROUP / 32, D = 2;
  constexpr int TERMS = I4Frag<XT>::TERMS;
  __shared__ float red[2][I4S_WARPS][NT][4][32];
  const int e = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int tiles = I4S_WARPS / ksplit;
  const int tile = warp / ksplit, ks = warp % ksplit;
  const int pos = blockIdx.x * tiles + tile;
  // the warp's two strips; where there is none its loads go to the first and are not stored
  const int s0 = DUAL ? pos : 2 * pos, s1 = DUAL ? pos : 2 * pos + 1;
  const size_t matrix = (size_t)e * (DUAL ? 2 : 1);
  const size_t b0 = (matrix * strips + (s0 < strips ? s0 : 0)) * chunks;
  const size_t b1 = ((matrix + (DUAL ? 1 : 0)) * strips + (s1 < strips ? s1 : 0)) * chunks;
  const unsigned* cw[2] = {codes + b0 * I4_CHUNK_WORDS + lane * 4,
                           codes + b1 * I4_CHUNK_WORDS + lane * 4};
  const unsigned* cp[2] = {params + (b0 * I4_STRIP + g) * NG, params + (b1 * I4_STRIP + g) * NG};
  uint4 w[D][2][2];
  unsigned prm[D][2][2][NG];
  auto fetch_w = [&](int u, int c) {
    if (c < chunks) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        w[u][s][0] = i4s_ld16(cw[s] + (size_t)c * I4_CHUNK_WORDS);
        w[u][s][1] = i4s_ld16(cw[s] + (size_t)c * I4_CHUNK_WORDS + I4_TILE_WORDS);
        i4s_params<NG>(cp[s] + (size_t)c * I4_STRIP * NG, prm[u][s][0]);
        i4s_params<NG>(cp[s] + ((size_t)c * I4_STRIP + 8) * NG, prm[u][s][1]);
      }
    }
  };
  // Weights are never written on the device while steps run: the first loads go out before the
  // wait on the predecessor where the range of rows is known already.
  const bool early = offsets == nullptr || offsets_settled != 0;
  int lo = 0, hi = M_single;
  if (early) {
    if (offsets) {
      lo = offsets[e];
      hi = offsets[e + 1];
    }
    if (lo >= hi) return;
#pragma unroll
    for (int u = 0; u < D; ++u) fetch_w(u, ks + u * ksplit);
  }
  IX_PDL_WAIT();
  if (!early) {
    lo = offsets[e];
    hi = offsets[e + 1];
    if (lo >= hi) return;
  }
  for (int r0 = lo; r0 < hi; r0 += 8 * NT) {
    const XT* xrow[NT];
    bool xok[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int r = r0 + i * 8 + g;
      xok[i] = r < hi;
      const size_t src = xok[i] ? (rows ? (size_t)rows[r] : (size_t)r) : 0;
      xrow[i] = x + src * K + t * 8;
    }
    float tot[2][NT][4];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) tot[s][i][c] = 0.f;
    if (!(early && r0 == lo)) {
#pragma unroll
      for (int u = 0; u < D; ++u) fetch_w(u, ks + u * ksplit);
    }
    for (int c0 = ks; c0 < chunks; c0 += D * ksplit) {
#pragma unroll
      for (int u = 0; u < D; ++u) {
        const int c = c0 + u * ksplit;
        if (c < chunks) {
          I4Frag<XT> f[4][NT];
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int i = 0; i < NT; ++i) {
              const int k = c * I4_CHUNK_K + b * 32;
              f[b][i].load(xrow[i] + k, xok[i] && k + t * 8 < K);
            }
          float acc[2][NT][4];
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            if (b % PER == 0) {
#pragma unroll
              for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                  for (int q = 0; q < 4; ++q) acc[s][i][q] = 0.f;
            }
            unsigned a[2][2][4];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              const uint4 v = w[u][s][b >> 1];
              const unsigned word[2] = {(b & 1) ? v.z : v.x, (b & 1) ? v.w : v.y};
              const unsigned sa = i4_sub(prm[u][s][0][b / PER]), sb = i4_sub(prm[u][s][1][b / PER]);
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                a[s][j][0] = i4_pair(word[j], 0, sa);
                a[s][j][1] = i4_pair(word[j], 1, sb);
                a[s][j][2] = i4_pair(word[j], 2, sa);
                a[s][j][3] = i4_pair(word[j], 3, sb);
              }
            }
#pragma unroll
            for (int i = 0; i < NT; ++i) {
              unsigned xb[TERMS][4];
              f[b][i].terms(xb);
#pragma unroll
              for (int m = 0; m < TERMS; ++m)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                  i4s_mma(acc[s][i], a[s][0], xb[m][0], xb[m][1]);
                  i4s_mma(acc[s][i], a[s][1], xb[m][2], xb[m][3]);
                }
            }
            if (b % PER == PER - 1) {
#pragma unroll
              for (int s = 0; s < 2; ++s) {
                const float fa = i4_scale(prm[u][s][0][b / PER]);
                const float fb = i4_scale(prm[u][s][1][b / PER]);
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                  tot[s][i][0] = fmaf(fa, acc[s][i][0], tot[s][i][0]);
                  tot[s][i][1] = fmaf(fa, acc[s][i][1], tot[s][i][1]);
                  tot[s][i][2] = fmaf(fb, acc[s][i][2], tot[s][i][2]);
                  tot[s][i][3] = fmaf(fb, acc[s][i][3], tot[s][i][3]);
                }
              }
            }
          }
        }
        fetch_w(u, c + D * ksplit);
      }
    }
    // c0, c1: column g of the strip, rows 2t and 2t + 1; c2, c3: column g + 8
    if (ksplit == 1) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int col = (c & 2) ? g + 8 : g;
          const int r = r0 + i * 8 + 2 * t + (c & 1);
          if (r >= hi) continue;
          if (s0 * I4_STRIP + col < N)
            i4s_store<DUAL>(out, r, s0 * I4_STRIP + col, N, tot[0][i][c], tot[1][i][c]);
          if (!DUAL && s1 * I4_STRIP + col < N)
            i4s_store<DUAL>(out, r, s1 * I4_STRIP + col, N, tot[1][i][c], 0.f);
        }
    } else {
      __syncthreads();   // the previous pass has read its sums
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) red[s][warp][i][c][lane] = tot[s][i][c];
      __syncthreads();
      for (int idx = threadIdx.x; idx < tiles * NT * 128; idx += I4S_THREADS) {
        const int l = idx & 31, c = (idx >> 5) & 3, i = (idx >> 7) % NT, ti = idx / (NT * 128);
        float v = 0.f, v2 = 0.f;
        for (int q = 0; q < ksplit; ++q) {
          v += red[0][ti * ksplit + q][i][c][l];
          v2 += red[1][ti * ksplit + q][i][c][l];
        }
        const int p = blockIdx.x * tiles + ti;
        const int col = (l >> 2) + ((c & 2) ? 8 : 0);
        const int r = r0 + i * 8 + 2 * (l & 3) + (c & 1);
        if (r >= hi) continue;
        const int j0 = (DUAL ? p : 2 * p) * I4_STRIP + col;
        if (j0 < N) i4s_store<DUAL>(out, r, j0, N, v, v2);
        if (!DUAL && j0 + I4_STRIP < N) i4s_store<DUAL>(out, r, j0 + I4_STRIP, N, v2, 0.f);
      }
    }
  }
}

template <typename XT, bool DUAL, int NT, int GROUP>
static int i4s_launch(const void* x, const int* rows, const int* offsets, const void* codes,
                      const void* params, I4Out out, int M, int N, int K, int E, int active,
                      int settled, cudaStream_t stream) {
  const int strips = (int)i4_strips(N), chunks = (int)i4_chunks(K);
  const int pairs = DUAL ? strips : (strips + 1) / 2;
  // K is split over the warps of a block until every SM has eight warps
  int ksplit = 1;
  while (ksplit < 8 && ksplit < chunks && (long long)pairs * active * ksplit < 148 * 8) ksplit *= 2;
  const int tiles = I4S_WARPS / ksplit;
  ix_launch(int4_stream_kernel<XT, DUAL, NT, GROUP>, dim3((pairs + tiles - 1) / tiles, E),
            dim3(I4S_THREADS), 0, stream, (const XT*)x, rows, offsets, (const unsigned*)codes,
            (const unsigned*)params, out, offsets ? 0 : M, N, K, strips, chunks, ksplit, settled);
  return ix_launch_status();
}

// x: [*, K] fp32 or bf16, K a multiple of 8, 16-byte aligned; codes and params as int4_format.cuh
// lays them out, [E or 2 E matrices]; out: [rows, N] fp32 (wide) or bf16.  offsets == null: one
// matrix with M rows.  active: how many of the E groups are expected to have rows.
// offsets_settled: nonzero when `offsets` was written at least two launches back in the stream.
IX_API int ix_int4_stream(const void* x, int x_dtype, const int* rows, const int* offsets,
                          const void* codes, const void* params, void* out, int wide, int dual,
                          int M, int N, int K, int E, int group, int rows_per_pass, int active,
                          int offsets_settled, const float* row_scale, int plain,
                          cudaStream_t stream) {
  if ((row_scale && !dual) || (plain && dual)) return IX_ERR_UNSUPPORTED;
  if (N <= 0 || K <= 0 || E <= 0 || E > 65535) return IX_ERR_SIZE;
  if (K % 8 != 0) return IX_ERR_UNSUPPORTED;
  if (!offsets && E != 1) return IX_ERR_SIZE;
  if (!offsets && M <= 0) return IX_OK;
  if ((uintptr_t)x & 15) return IX_ERR_ALIGN;
  if (active <= 0 || active > E) active = E;
  const I4Out o = {out, wide, row_scale, plain};
  const int nt = rows_per_pass > 16 ? 4 : rows_per_pass > 8 ? 2 : 1;
#define I4S_GO(T, D, NT, G) \
  return i4s_launch<T, D, NT, G>(x, rows, offsets, codes, params, o, M, N, K, E, active, offsets_settled, stream)
// (32 rows of three terms each would not fit the registers: fp32 takes 16 a pass)
#define I4S_NT(T, D, G)                                             \
  do {                                                              \
    if (nt == 4 && sizeof(T) == 2) I4S_GO(T, D, sizeof(T) == 2 ? 4 : 2, G); \
    if (nt >= 2) I4S_GO(T, D, 2, G);                                \
    I4S_GO(T, D, 1, G);                                             \
  } while (0)
#define I4S_G(T, D)                    \
  do {                                 \
    if (group == 128) I4S_NT(T, D, 128); \
    if (group == 64) I4S_NT(T, D, 64);   \
    if (group == 32) I4S_NT(T, D, 32);   \
    return IX_ERR_UNSUPPORTED;           \
  } while (0)
  if (x_dtype == IX_BF16) {
    if (dual) I4S_G(bf16, true);
    I4S_G(bf16, false);
  }
  if (x_dtype == IX_F32) {
    if (dual) I4S_G(float, true);
    I4S_G(float, false);
  }
  return IX_ERR_DTYPE;
}
