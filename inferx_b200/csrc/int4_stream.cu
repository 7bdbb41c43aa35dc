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
// codes and the activations of the same 128 k come by cp.async into a ring of the warp's own (nobody
// else reads it: no barrier in the loop), R - 1 chunks in flight.  Each word of codes becomes the A side
// of one mma by three shifts, four logic operations and four exact subtractions, and the fp32 sums of a
// group are multiplied by the group's scale.  fp32 activations are three bfloat16 terms, the two small
// ones summed apart from the first.  The warps of a block split K by chunks and join their sums through
// shared memory in warp order, so a row's result does not depend on which rows share its tile.
//
// Measured (bfloat16, groups of 128, weights from DRAM; us, GB/s of codes): one row, 2,048 -> 2,048 3.5
// (600), gated 2,048 -> 2 x 5,632 7.6 (1,520); eight rows, 5,632 -> 2,048 5.3 (1,100), gated 3,584 -> 2 x
// 20,480 25.0 (2,930); eight tokens of 4 of 60 experts of 2 x 1,408 x 2,048 27.1 up and 14.9 down (2,900
// and 2,600).  What bounds it is latency: the short calls are one chain (launch, first copies, a few chunks,
// the join: 19 % of issue slots used, memory 16 % busy), and in the long ones nothing is busy either
// (issue slots 44 %, ALU pipe 41 %, memory 37 %).  Registers (120 a thread) and rings let two blocks onto
// an SM, 14.7 warps in the mean, and a warp is ready every sixth cycle: its time goes in about equal
// parts to the ring's loads, results of fixed latency, the ALU's turns and the other warps'.  In 32 bits
// three terms and their sums leave one block an SM: eight tokens of the experts 57 us up, 29 down.  One
// pass over the codes serves up to 32 rows; tcgen05 would want 128 weight rows by 128 k unpacked into
// tensor memory before its first product, which is the other kernel's business.  Blocks that stay and
// take one piece of work after the other were built and are slower, and so were shifts by multiplication.
#include "int4_format.cuh"

#define I4S_THREADS 256
#define I4S_WARPS 8

__device__ __forceinline__ void i4s_copy16(unsigned to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// the first `bytes` of 16, zeros behind them
__device__ __forceinline__ void i4s_copy16(unsigned to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes)
               : "memory");
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
  __device__ __forceinline__ void load(const unsigned char* p) {
    r = *reinterpret_cast<const uint2*>(p);
  }
  __device__ __forceinline__ void terms(unsigned (*b)[2]) const {
    b[0][0] = r.x;
    b[0][1] = r.y;
  }
};
template <> struct I4Frag<float> {
  static constexpr int TERMS = 3;
  float4 r;
  __device__ __forceinline__ void load(const unsigned char* p) {
    r = *reinterpret_cast<const float4*>(p);
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

template <typename XT, int NT, int GROUP, int S> struct I4SCfg {
  static constexpr int BYTES = i4_block_words(GROUP) * 4;          // a strip's share of a chunk
  // a row's activations of a chunk, padded so that the rows of a load meet different banks
  static constexpr int X_PITCH = I4_CHUNK_K * sizeof(XT) + 16 * sizeof(XT);
  static constexpr int STAGE = S * BYTES + 8 * NT * X_PITCH;
  static constexpr int R = NT * sizeof(XT) >= 8 ? 2 : 3;                      // stages of a warp's ring
  static constexpr int RING = I4S_WARPS * R * STAGE;
  static constexpr int RED = S * I4S_WARPS * NT * 128 * 4;         // and the sums that are joined
  static constexpr int SMEM = RING + RED;
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

template <typename XT, bool DUAL, int NT, int GROUP, int S>
__global__ void __launch_bounds__(I4S_THREADS, NT == 1 && sizeof(XT) == 2 ? 2 : 1)
int4_stream_kernel(const XT* __restrict__ x, const int* __restrict__ rows,
                   const int* __restrict__ offsets, const unsigned* __restrict__ data, I4Out out,
                   int M_single, int N, int K, int E, int strips, int chunks, int klog, int early) {
  typedef I4SCfg<XT, NT, GROUP, S> C;
  constexpr int NG = 128 / GROUP, PER = GROUP / 16;
  constexpr int TERMS = I4Frag<XT>::TERMS, ACCS = TERMS == 3 ? 2 : 1;
  // 16-byte pieces of activations: so many lanes take a row's, so many rows go by at once
  constexpr int PIECES = I4_CHUNK_K * sizeof(XT) / 16, AT_ONCE = 32 / PIECES;
  constexpr int PASSES = 8 * NT / AT_ONCE;
  static_assert(!DUAL || S == 2, "a gate strip and its up strip");
  extern __shared__ __align__(16) unsigned char smem[];
  float* red = reinterpret_cast<float*>(smem + C::RING);           // [S][warp][NT][4][32]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int ksplit = 1 << klog, tiles = I4S_WARPS >> klog;
  const int tile = warp >> klog, ks = warp & (ksplit - 1);
  const int pos = blockIdx.x * tiles + tile;
  // The first copies of codes go out before the wait on the predecessor where the caller says that
  // nothing on the device still writes the weights and the range of rows is known already.
  if (!early) IX_PDL_WAIT();
  int e = 0, lo = 0, hi = M_single;
  if (offsets) {
    // blockIdx.y counts the groups that have rows (a grid over all of them costs more than their
    // products where a step's tokens reach few: 4 of 60 experts)
    int left = blockIdx.y;
    e = -1;
    for (int e0 = 0; e0 < E && e < 0; e0 += 32) {
      const bool some = e0 + lane < E && offsets[e0 + lane + 1] > offsets[e0 + lane];
      unsigned mask = __ballot_sync(0xffffffffu, some);
      if (left < __popc(mask)) {
        for (; left > 0; --left) mask &= mask - 1;
        e = e0 + __ffs(mask) - 1;
      } else {
        left -= __popc(mask);
      }
    }
    if (e < 0) return;
    lo = offsets[e];
    hi = offsets[e + 1];
  }
  // the warp's strips; where there is none its copies come from the first and are not stored
  const size_t pitch = (size_t)strips * C::BYTES;                  // from chunk to chunk
  const unsigned char* base = reinterpret_cast<const unsigned char*>(data) +
                              ((size_t)e * (DUAL ? 2 : 1) * chunks + ks) * pitch;
  const size_t step = pitch << klog;
  const unsigned char* from[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int strip = DUAL ? pos : S * pos + s;
    from[s] = base + (DUAL && s ? chunks * pitch : 0) +
              (size_t)(strip < strips ? strip : 0) * C::BYTES + lane * 16;
  }
  // parameters of a strip: 4 NG pieces of 16 bytes, lanes 0.. for the first strip, 16.. for the second
  const bool copies_params = (lane & 15) < 4 * NG && (lane >> 4) < S;
  const int params_off = I4_CODE_WORDS * 4 + (lane & 15) * 16 - lane * 16;
  const unsigned char* from_params = from[S == 2 ? lane >> 4 : 0] + params_off;
  const unsigned params_at = (S == 2 ? (lane >> 4) * C::BYTES : 0) + params_off;
  unsigned char* ring = smem + warp * (C::R * C::STAGE);
  const unsigned ring_at = (unsigned)__cvta_generic_to_shared(ring) + lane * 16;
  const int n = (chunks - ks + ksplit - 1) >> klog;   // chunks of this warp
  // One chunk's codes, or its activations, into stage u (chunks are asked for in order).
  const unsigned char *next_w[S], *next_params;
  auto fetch_w = [&](int u) {
    const unsigned at = ring_at + u * C::STAGE;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      i4s_copy16(at + s * C::BYTES, next_w[s]);
      i4s_copy16(at + s * C::BYTES + I4_TILE_WORDS * 4, next_w[s] + I4_TILE_WORDS * 4);
      next_w[s] += step;
    }
    if (copies_params) i4s_copy16(at + params_at, next_params);
    next_params += step;
  };
  auto start_w = [&]() {
#pragma unroll
    for (int s = 0; s < S; ++s) next_w[s] = from[s];
    next_params = from_params;
  };
  if (early) {
    start_w();
    for (int i = 0; i < C::R - 1; ++i)
      if (i < n) fetch_w(i);
    IX_PDL_WAIT();
  }
  for (int r0 = lo; r0 < hi; r0 += 8 * NT) {
    // this lane's pieces of the activations: rows r0 + lane / PIECES + AT_ONCE * q.  Rows behind the
    // last are not copied: what stands there meets columns of the product that are not stored.
    const int first_k = (lane % PIECES) * (16 / (int)sizeof(XT));
    const unsigned x_at = ring_at - lane * 16 + S * C::BYTES + (lane / PIECES) * C::X_PITCH +
                          (lane % PIECES) * 16;
    const XT* xrow[PASSES];
#pragma unroll
    for (int q = 0; q < PASSES; ++q) {
      const int r = r0 + lane / PIECES + AT_ONCE * q;
      const size_t src = r < hi ? (rows ? (size_t)rows[r] : (size_t)r) : 0;
      xrow[q] = x + src * K + ks * I4_CHUNK_K + first_k;
    }
    const int here = hi - r0 - lane / PIECES;      // rows left from this lane's first
    int next_k = ks * I4_CHUNK_K + first_k;
    auto fetch_x = [&](int u) {
      const int bytes = next_k < K ? 16 : 0;       // K is a multiple of 8
#pragma unroll
      for (int q = 0; q < PASSES; ++q) {
        if (AT_ONCE * q < here)
          i4s_copy16(x_at + u * C::STAGE + AT_ONCE * q * C::X_PITCH, xrow[q], bytes);
        xrow[q] += ksplit * I4_CHUNK_K;
      }
      next_k += ksplit * I4_CHUNK_K;
    };
    float tot[S][NT][4];
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) tot[s][i][c] = 0.f;
    if (!(early && r0 == lo)) {
      __syncwarp();                                // the previous pass has read its stages
      start_w();
      for (int i = 0; i < C::R - 1; ++i)
        if (i < n) fetch_w(i);
    }
    for (int i = 0; i < C::R - 1; ++i) {
      if (i < n) fetch_x(i);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    int u = 0, ahead = C::R - 1;                   // the stage of chunk i, and of chunk i + R - 1
    for (int i = 0; i < n; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(C::R - 2) : "memory");
      __syncwarp();            // pieces were copied by other lanes; the last chunk's stage is read
      if (i + C::R - 1 < n) {
        fetch_w(ahead);
        fetch_x(ahead);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      const unsigned char* block = ring + u * C::STAGE;
      const unsigned char* xs = block + S * C::BYTES + g * C::X_PITCH + t * (4 * sizeof(XT));
      uint4 w[S][2];
      unsigned pa[S][NG], pb[S][NG];
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const unsigned* at = reinterpret_cast<const unsigned*>(block + s * C::BYTES);
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
        I4Frag<XT> f[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) f[j].load(xs + j * 8 * C::X_PITCH + b * (16 * sizeof(XT)));
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
          f[j].terms(xb);
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
      u = u + 1 == C::R ? 0 : u + 1;
      ahead = ahead + 1 == C::R ? 0 : ahead + 1;
    }
    // q = 0, 1: column g of the strip, rows 2t and 2t + 1; q = 2, 3: column g + 8
    auto store = [&](int p, int col, int r, float v, float u) {
      if (r >= hi) return;
      const int j = (DUAL ? p : S * p) * I4_STRIP + col;
      if (j < N) i4s_store<DUAL>(out, r, j, N, v, u);
      if (S == 2 && !DUAL && j + I4_STRIP < N) i4s_store<DUAL>(out, r, j + I4_STRIP, N, u, 0.f);
    };
    if (klog == 0) {
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
  int M, N, K, E, active, early;
};

template <typename XT, bool DUAL, int NT, int GROUP, int S>
static int i4s_launch2(const I4SCall& c, cudaStream_t stream) {
  typedef I4SCfg<XT, NT, GROUP, S> C;
  const int strips = (int)i4_strips(c.N), chunks = (int)i4_chunks(c.K);
  const int sets = DUAL ? strips : (strips + S - 1) / S;
  // K is split over the warps of a block until there are 32 warps for every SM, as long as a warp
  // keeps four chunks (us at 8 rows, 1 / 2 / 4 / 8 warps: gated 3584 x 20480 36 / 29 / 26 / 27; 27
  // experts of 2 x 1408 x 2048 29 / 27 / 29 / 34); where that leaves SMs idle it is split further (2048
  // x 6144 9.1 / 6.5 / 6.2 / 6.5, 2048 x 2048 8.8 / 6.0 / 4.3 / 3.6).
  int klog = 0;
  const long long warps = (long long)sets * c.active;
  while (klog < 3 && (1 << klog) < chunks && (warps << klog) < 148 * 32 &&
         (chunks >= (8 << klog) || (warps << klog) < 148 * 8))
    ++klog;
  const int tiles = I4S_WARPS >> klog;
  auto kern = int4_stream_kernel<XT, DUAL, NT, GROUP, S>;
  static unsigned done = 0;
  const cudaError_t e = i4_allow_smem(kern, C::SMEM, &done);
  if (e != cudaSuccess) return (int)e;
  ix_launch(kern, dim3((sets + tiles - 1) / tiles, c.active), dim3(I4S_THREADS), C::SMEM, stream,
            (const XT*)c.x, c.rows, c.offsets, (const unsigned*)c.data, c.out, c.offsets ? 0 : c.M,
            c.N, c.K, c.E, strips, chunks, klog, c.early);
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

// x: [*, K] fp32 or bf16, K a multiple of 8 that ends in the weight's last chunk, 16-byte aligned;
// out: [rows, N] fp32 (wide) or bf16.  offsets == null: one matrix with M rows.  active: the most
// groups that can have rows (0: all).  offsets_settled: nonzero when `offsets` was written at least two
// launches back in the stream.  w->settled: the same of the weights, for good; where it is 0 (they have
// just been quantised or packed, perhaps by the launch before) they are read behind the wait.
IX_API int ix_int4_stream(const I4Weight* w, const void* x, int x_dtype, const int* rows,
                          const int* offsets, void* out, int wide, int M, int K, int rows_per_pass,
                          int active, int offsets_settled, const float* row_scale, int plain,
                          cudaStream_t stream) {
  const int E = w->E, group = w->group, dual = w->dual;
  if ((row_scale && !dual) || (plain && dual)) return IX_ERR_UNSUPPORTED;
  if (w->N <= 0 || K <= 0 || E <= 0 || E > 65535) return IX_ERR_SIZE;
  if (K % 8 != 0) return IX_ERR_UNSUPPORTED;
  if (!offsets && E != 1) return IX_ERR_SIZE;
  if (!offsets && M <= 0) return IX_OK;
  if (((uintptr_t)x | (uintptr_t)w->data) & 15) return IX_ERR_ALIGN;
  if (active <= 0 || active > E) active = E;
  const I4SCall c = {x, rows, offsets, w->data, {out, wide, row_scale, plain}, M, w->N, K, E, active,
                     w->settled != 0 && (!offsets || offsets_settled != 0)};
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
