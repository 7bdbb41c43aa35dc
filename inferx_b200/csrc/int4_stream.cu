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
// rows the N side.  A warp holds S strips of 16 weight rows (DUAL: a gate strip and the up strip of the
// same columns) against 8 NT activation rows, so an activation fragment serves them all.  Blocks of
// 128 k come by cp.async into a ring of the warp's own (nobody else reads it: no barrier in the loop),
// R - 1 of them in flight; the next chunk's activations are loaded ahead into registers.  Each word of
// codes becomes the A side of one mma by three shifts, four logic operations and four exact
// subtractions, and the fp32 sums of a group are multiplied by the group's scale.  fp32 activations are
// three bfloat16 terms, the two small ones summed apart from the first.  The warps of a block split K by
// chunks and join their sums through shared memory in warp order, so a row's result does not depend on
// which rows share its tile.
#include "int4_format.cuh"

#define I4S_THREADS 256
#define I4S_WARPS 8

__device__ __forceinline__ void i4s_copy16(unsigned to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void i4s_mma(float* c, const unsigned* a, unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four activations of a row as fragments: [term][pair of k].
template <typename XT> struct I4Frag;
template <> struct I4Frag<bf16> {
  static constexpr int TERMS = 1;
  uint2 r;
  __device__ __forceinline__ void load(const bf16* p, bool ok) {
    r = ok ? *reinterpret_cast<const uint2*>(p) : make_uint2(0, 0);
  }
  __device__ __forceinline__ void terms(unsigned (*b)[2]) const {
    b[0][0] = r.x;
    b[0][1] = r.y;
  }
};
template <> struct I4Frag<float> {
  static constexpr int TERMS = 3;
  float4 r;
  __device__ __forceinline__ void load(const float* p, bool ok) {
    r = ok ? *reinterpret_cast<const float4*>(p) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ void terms(unsigned (*b)[2]) const {
    i4_terms2(r.x, r.y, b[0][0], b[1][0], b[2][0]);
    i4_terms2(r.z, r.w, b[0][1], b[1][1], b[2][1]);
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

template <int NT, int GROUP, int S> struct I4SCfg {
  static constexpr int BYTES = i4_block_words(GROUP) * 4;          // a strip's share of a chunk
  static constexpr int R = S == 1 ? 8 : 6;                         // stages of a warp's ring
  static constexpr int RING = I4S_WARPS * R * S * BYTES;
  static constexpr int SMEM = RING + S * I4S_WARPS * NT * 128 * 4; // and the sums that are joined
};

template <typename XT, bool DUAL, int NT, int GROUP, int S>
__global__ void __launch_bounds__(I4S_THREADS, NT == 1 && sizeof(XT) == 2 ? 2 : 1)
int4_stream_kernel(const XT* __restrict__ x, const int* __restrict__ rows,
                   const int* __restrict__ offsets, const unsigned* __restrict__ data, I4Out out,
                   int M_single, int N, int K, int strips, int chunks, int ksplit,
                   int offsets_settled) {
  typedef I4SCfg<NT, GROUP, S> C;
  constexpr int NG = 128 / GROUP, PER = GROUP / 16;
  constexpr int TERMS = I4Frag<XT>::TERMS, ACCS = TERMS == 3 ? 2 : 1;
  static_assert(!DUAL || S == 2, "a gate strip and its up strip");
  extern __shared__ __align__(16) unsigned char smem[];
  float* red = reinterpret_cast<float*>(smem + C::RING);           // [S][warp][NT][4][32]
  const int e = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int tiles = I4S_WARPS / ksplit;
  const int tile = warp / ksplit, ks = warp % ksplit;
  const int pos = blockIdx.x * tiles + tile;
  // the warp's strips; where there is none its copies come from the first and are not stored
  const size_t pitch = (size_t)strips * C::BYTES;                  // from chunk to chunk
  const unsigned char* base = reinterpret_cast<const unsigned char*>(data) +
                              (size_t)e * (DUAL ? 2 : 1) * chunks * pitch;
  const unsigned char* from[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int strip = DUAL ? pos : S * pos + s;
    from[s] = base + (DUAL && s ? chunks * pitch : 0) +
              (size_t)(strip < strips ? strip : 0) * C::BYTES;
  }
  // parameters of a strip: 4 NG pieces of 16 bytes, lanes 0.. for the first strip, 16.. for the second
  const bool copies_params = (lane & 15) < 4 * NG && (lane >> 4) < S;
  const unsigned char* from_params =
      from[S == 2 ? lane >> 4 : 0] + I4_CODE_WORDS * 4 + (lane & 15) * 16;
  const unsigned params_at = (S == 2 ? (lane >> 4) * C::BYTES : 0) + I4_CODE_WORDS * 4 + (lane & 15) * 16;
  unsigned char* ring = smem + warp * (C::R * S * C::BYTES);
  const unsigned ring_at = (unsigned)__cvta_generic_to_shared(ring);
  const int n = chunks > ks ? (chunks - ks + ksplit - 1) / ksplit : 0;   // chunks of this warp
  auto fetch = [&](int i) {                        // its i-th chunk, if there is one
    if (i < n) {
      const size_t c = (size_t)(ks + i * ksplit) * pitch;
      const unsigned at = ring_at + (i % C::R) * (S * C::BYTES);
#pragma unroll
      for (int s = 0; s < S; ++s) {
        i4s_copy16(at + s * C::BYTES + lane * 16, from[s] + c + lane * 16);
        i4s_copy16(at + s * C::BYTES + I4_TILE_WORDS * 4 + lane * 16,
                   from[s] + c + I4_TILE_WORDS * 4 + lane * 16);
      }
      if (copies_params) i4s_copy16(at + params_at, from_params + c);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // Weights are never written on the device while steps run: the first copies go out before the
  // wait on the predecessor where the range of rows is known already.
  const bool early = offsets == nullptr || offsets_settled != 0;
  int lo = 0, hi = M_single;
  if (early) {
    if (offsets) {
      lo = offsets[e];
      hi = offsets[e + 1];
    }
    if (lo >= hi) return;
    for (int i = 0; i < C::R - 1; ++i) fetch(i);
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
      xrow[i] = x + src * K + t * 4;
    }
    float tot[S][NT][4];
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) tot[s][i][c] = 0.f;
    if (!(early && r0 == lo)) {
      __syncwarp();                                // the previous pass has read its parameters
      for (int i = 0; i < C::R - 1; ++i) fetch(i);
    }
    I4Frag<XT> f[8][NT], f_next[8][NT];
    auto fetch_x = [&](int i) {
      const int k0 = (ks + i * ksplit) * I4_CHUNK_K;
#pragma unroll
      for (int b = 0; b < 8; ++b)
#pragma unroll
        for (int j = 0; j < NT; ++j)
          f_next[b][j].load(xrow[j] + k0 + b * 16, xok[j] && i < n && k0 + b * 16 + t * 4 < K);
    };
    fetch_x(0);
    for (int i = 0; i < n; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(C::R - 2) : "memory");
      __syncwarp();            // parameters were copied by other lanes; the last chunk's are read
      fetch(i + C::R - 1);
#pragma unroll
      for (int b = 0; b < 8; ++b)
#pragma unroll
        for (int j = 0; j < NT; ++j) f[b][j] = f_next[b][j];
      fetch_x(i + 1);
      const unsigned* block = reinterpret_cast<const unsigned*>(ring + (i % C::R) * (S * C::BYTES));
      uint4 w[S][2];
      unsigned pa[S][NG], pb[S][NG];
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const unsigned* at = block + s * (C::BYTES / 4);
        w[s][0] = *reinterpret_cast<const uint4*>(at + lane * 4);
        w[s][1] = *reinterpret_cast<const uint4*>(at + I4_TILE_WORDS + lane * 4);
#pragma unroll
        for (int q = 0; q < NG; ++q) {
          pa[s][q] = at[I4_CODE_WORDS + g * NG + q];
          pb[s][q] = at[I4_CODE_WORDS + (g + 8) * NG + q];
        }
      }
      float acc[ACCS][S][NT][4];
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        if (b % PER == 0) {
#pragma unroll
          for (int a = 0; a < ACCS; ++a)
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[a][s][j][q] = 0.f;
        }
        unsigned a[S][4];
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const uint4 v = w[s][b >> 2];
          const unsigned word = (b & 3) == 0 ? v.x : (b & 3) == 1 ? v.y : (b & 3) == 2 ? v.z : v.w;
          const unsigned sa = i4_sub(pa[s][b / PER]), sb = i4_sub(pb[s][b / PER]);
          a[s][0] = i4_pair(word, 0, sa);
          a[s][1] = i4_pair(word, 1, sb);
          a[s][2] = i4_pair(word, 2, sa);
          a[s][3] = i4_pair(word, 3, sb);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          unsigned xb[TERMS][2];
          f[b][j].terms(xb);
#pragma unroll
          for (int m = TERMS - 1; m >= 0; --m)
#pragma unroll
            for (int s = 0; s < S; ++s)
              i4s_mma(acc[m > 0 ? ACCS - 1 : 0][s][j], a[s], xb[m][0], xb[m][1]);
        }
        if (b % PER == PER - 1) {
#pragma unroll
          for (int s = 0; s < S; ++s) {
            const float fa = i4_scale(pa[s][b / PER]), fb = i4_scale(pb[s][b / PER]);
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                float v = acc[0][s][j][q];
                if (ACCS == 2) v += acc[ACCS - 1][s][j][q];
                tot[s][j][q] = fmaf(q < 2 ? fa : fb, v, tot[s][j][q]);
              }
          }
        }
      }
    }
    // q = 0, 1: column g of the strip, rows 2t and 2t + 1; q = 2, 3: column g + 8
    auto store = [&](int p, int col, int r, float v, float u) {
      if (r >= hi) return;
      const int j = (DUAL ? p : S * p) * I4_STRIP + col;
      if (j < N) i4s_store<DUAL>(out, r, j, N, v, u);
      if (S == 2 && !DUAL && j + I4_STRIP < N) i4s_store<DUAL>(out, r, j + I4_STRIP, N, u, 0.f);
    };
    if (ksplit == 1) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          store(pos, (q & 2) ? g + 8 : g, r0 + j * 8 + 2 * t + (q & 1), tot[0][j][q],
                tot[S - 1][j][q]);
    } else {
      __syncthreads();   // the previous pass has read its sums
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            red[(((s * I4S_WARPS + warp) * NT + j) * 4 + q) * 32 + lane] = tot[s][j][q];
      __syncthreads();
      for (int idx = threadIdx.x; idx < tiles * NT * 128; idx += I4S_THREADS) {
        const int l = idx & 31, q = (idx >> 5) & 3, j = (idx >> 7) % NT, ti = idx / (NT * 128);
        float v = 0.f, u = 0.f;
        for (int k = 0; k < ksplit; ++k) {
          const int at = ((ti * ksplit + k) * NT + j) * 128 + q * 32 + l;
          v += red[at];
          if (S == 2) u += red[I4S_WARPS * NT * 128 + at];
        }
        store(blockIdx.x * tiles + ti, (l >> 2) + ((q & 2) ? 8 : 0),
              r0 + j * 8 + 2 * (l & 3) + (q & 1), v, u);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

struct I4SCall {
  const void* x;
  const int *rows, *offsets;
  const void* data;
  I4Out out;
  int M, N, K, E, active, settled;
};

template <typename XT, bool DUAL, int NT, int GROUP, int S>
static int i4s_launch2(const I4SCall& c, cudaStream_t stream) {
  typedef I4SCfg<NT, GROUP, S> C;
  const int strips = (int)i4_strips(c.N), chunks = (int)i4_chunks(c.K);
  const int sets = DUAL ? strips : (strips + S - 1) / S;
  // K is split over the warps of a block until every SM has sixteen warps
  int ksplit = 1;
  while (ksplit < 8 && ksplit < chunks && (long long)sets * c.active * ksplit < 148 * 16) ksplit *= 2;
  const int tiles = I4S_WARPS / ksplit;
  auto kern = int4_stream_kernel<XT, DUAL, NT, GROUP, S>;
  const cudaError_t e =
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return (int)e;
  ix_launch(kern, dim3((sets + tiles - 1) / tiles, c.E), dim3(I4S_THREADS), C::SMEM, stream,
            (const XT*)c.x, c.rows, c.offsets, (const unsigned*)c.data, c.out, c.offsets ? 0 : c.M,
            c.N, c.K, strips, chunks, ksplit, c.settled);
  return ix_launch_status();
}

template <typename XT, bool DUAL, int NT, int GROUP>
static int i4s_launch(const I4SCall& c, cudaStream_t stream) {
  if constexpr (!DUAL) {
    // one strip a warp while pairs of them would not reach every SM
    if (i4_strips(c.N) * c.active < 2 * 148 * 2)
      return i4s_launch2<XT, false, NT, GROUP, 1>(c, stream);
  }
  return i4s_launch2<XT, DUAL, NT, GROUP, 2>(c, stream);
}

// x: [*, K] fp32 or bf16, K a multiple of 8, 16-byte aligned; data as int4_format.cuh lays
// it out, [E or 2 E matrices]; out: [rows, N] fp32 (wide) or bf16.  offsets == null: one
// matrix with M rows.  active: how many of the E groups are expected to have rows.
// offsets_settled: nonzero when `offsets` was written at least two launches back in the stream.
IX_API int ix_int4_stream(const void* x, int x_dtype, const int* rows, const int* offsets,
                          const void* data, void* out, int wide, int dual, int M, int N, int K, int E,
                          int group, int rows_per_pass, int active, int offsets_settled,
                          const float* row_scale, int plain,
                          cudaStream_t stream) {
  if ((row_scale && !dual) || (plain && dual)) return IX_ERR_UNSUPPORTED;
  if (N <= 0 || K <= 0 || E <= 0 || E > 65535) return IX_ERR_SIZE;
  if (K % 8 != 0) return IX_ERR_UNSUPPORTED;
  if (!offsets && E != 1) return IX_ERR_SIZE;
  if (!offsets && M <= 0) return IX_OK;
  if ((uintptr_t)x & 15) return IX_ERR_ALIGN;
  if (active <= 0 || active > E) active = E;
  const I4SCall c = {x, rows, offsets, data, {out, wide, row_scale, plain}, M, N, K, E, active,
                     offsets_settled};
  const int nt = rows_per_pass > 16 ? 4 : rows_per_pass > 8 ? 2 : 1;
#define I4S_GO(T, D, NT, G) return i4s_launch<T, D, NT, G>(c, stream)
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
