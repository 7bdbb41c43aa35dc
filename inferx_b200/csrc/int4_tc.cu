// Products with four-bit weights for many rows (prompts) on the 5th-generation tensor cores.
//
//   out[r, j] = sum_k a[r, k] * w[e(r), j, k]                (plain, an activation may follow)
//   out[r, j] = silu(a . wg[e, j]) * (a . wu[e, j])          (DUAL)
//   w[j, k] = scale[j, k / group] * (code[j, k] - zero[j, k / group])      (int4_format.cuh)
//
// `a` holds bfloat16 rows grouped by expert (offsets), or the rows of a single matrix; fp32 rows come
// as three planes of bfloat16 terms that are multiplied into the same sums.
//
// The weights are the M side of tcgen05.mma and the rows the N side.  An item of work is 128 weight
// rows (DUAL: 64 gate rows and the up rows of the same columns) for a tile of up to BT rows of one
// expert; blocks are persistent, one per SM, and take items round robin, the weight tiles of one row
// tile beside each other.  Roles:
//   warp 0      brings the rows, 64 k at a time, into a ring of stages (TMA, 128-byte swizzle);
//   warp 1      issues the MMAs, a group of k into one of two accumulators in tensor memory;
//   warps 2-9   load their strip's codes straight into registers (a lane's 16 bytes are eight
//               neighbouring k of two rows, twice), subtract the zero points, and write whole numbers
//               as a swizzled operand tile into a ring of their own; and take each finished group's
//               sums out of tensor memory, a weight row a lane, and add scale * sum to fp32 registers.
// So the operands of the tensor cores are exact (a code less its zero point has five bits), sums of a
// group are the tensor cores' fp32, and a group's scale multiplies in fp32: no weight is rounded to
// bfloat16.  The warps unpack the next chunk of 128 k before they take the sums of the last one, also
// across items, so the MMAs run meanwhile.
//
// Columns past the tile and weight rows past N are computed on whatever is there and never stored.
// Every wait on an mbarrier is bounded: the waiter records a code in `status` (51 copies, 52 MMAs, 53
// the unpacking warps), raises a flag that ends the other roles, and the block frees its tensor memory.
#include "int4_format.cuh"
#include "tcgen05_common.cuh"
#include "tma_common.cuh"

#define I4T_THREADS 320
#define I4T_WORKERS 8
#define I4T_BOX 32                        // rows of a TMA box
#define I4T_A_BYTES (128 * 64 * 2)        // an operand tile of weights
#define I4T_MAX_EXPERTS 1024              // the prefix of tiles lives in shared memory
#define I4T_EXCHANGE (4 * 32 * 33 * 4)    // DUAL: up sums on their way to the gate's warps

enum { I4T_ERR_COPY = 51, I4T_ERR_MMA = 52, I4T_ERR_WORK = 53 };

struct I4TArgs {
  const int* offsets;       // null: one matrix with `rows` rows
  const unsigned* codes;
  const unsigned* params;
  void* out;
  int wide;                 // fp32 results, otherwise bfloat16
  const float* row_scale;
  int plain;
  int rows, N, strips, chunks, E;
  int tile_rows;            // one matrix: rows of a tile, a multiple of 16
  int plane_rows;           // rows of one plane of terms
  int* status;
};

struct I4TItem {
  int e, m0, n, f0;
};

template <int TERMS, bool DUAL, int BT, int GROUP> struct I4TCfg {
  static constexpr int X_BYTES = BT * 64 * 2;                  // a term's rows of a stage
  static constexpr int A_RING = TERMS == 3 ? 3 : 4;
  static constexpr int X_RING = TERMS == 3 ? 3 : BT == 256 ? 4 : 6;
  static constexpr int SMEM = X_RING * TERMS * X_BYTES + A_RING * I4T_A_BYTES +
                              (DUAL ? I4T_EXCHANGE : 0) + 1024;
  static constexpr unsigned TMEM_COLS = 2 * BT;
  static constexpr int F = DUAL ? 64 : 128;                    // output columns of an item
};

template <int BT>
__device__ __forceinline__ int i4t_tiles(int rows) { return (rows + BT - 1) / BT; }

template <int TERMS, bool DUAL, int BT, int GROUP>
__global__ void __launch_bounds__(I4T_THREADS, 1)
int4_tc_kernel(const __grid_constant__ CUtensorMap map_x, const I4TArgs p) {
  typedef I4TCfg<TERMS, DUAL, BT, GROUP> C;
  constexpr int NG = 128 / GROUP;
  constexpr int F = C::F;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* xs =
      reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* as = xs + C::X_RING * TERMS * C::X_BYTES;
  float* exchange = reinterpret_cast<float*>(as + C::A_RING * I4T_A_BYTES);
  __shared__ __align__(8) unsigned long long full_x[C::X_RING], empty_x[C::X_RING];
  __shared__ __align__(8) unsigned long long full_a[C::A_RING], empty_a[C::A_RING];
  __shared__ __align__(8) unsigned long long acc_full[2], acc_empty[2];
  __shared__ __align__(8) unsigned long long ex_full[4], ex_empty[4];
  __shared__ unsigned tmem_holder;
  __shared__ int abort_flag;
  __shared__ int tile_start[I4T_MAX_EXPERTS + 1];

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int f_tiles = (p.N + F - 1) / F;
  if (warp == 2) {                           // tiles before each expert
    if (p.offsets) {
      int carry = 0;
      for (int e0 = 0; e0 < p.E; e0 += 32) {
        const int e = e0 + lane;
        const int t = e < p.E ? i4t_tiles<BT>(p.offsets[e + 1] - p.offsets[e]) : 0;
        int incl = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += v;
        }
        if (e < p.E) tile_start[e] = carry + incl - t;
        carry += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (lane == 0) tile_start[p.E] = carry;
    } else if (lane == 0) {
      tile_start[0] = 0;
      tile_start[1] = (p.rows + p.tile_rows - 1) / p.tile_rows;
    }
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::X_RING; ++s) {
      mbar_init(&full_x[s], 1);
      mbar_init(&empty_x[s], 1);
    }
    for (int s = 0; s < C::A_RING; ++s) {
      mbar_init(&full_a[s], I4T_WORKERS);
      mbar_init(&empty_a[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], I4T_WORKERS);
    }
    for (int b = 0; b < 4; ++b) {
      mbar_init(&ex_full[b], 1);
      mbar_init(&ex_empty[b], 1);
    }
    abort_flag = 0;
    mbar_init_fence();
    fence_proxy_async();
  }
  if (warp == 1) tc_alloc<false>(&tmem_holder, C::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem_base = __shfl_sync(0xffffffffu, tmem_holder, 0);
  volatile int* abortp = &abort_flag;
  const int n_items = tile_start[p.E] * f_tiles;

  auto item_of = [&](int w) {
    const int tt = w / f_tiles;
    I4TItem it;
    it.f0 = (w - tt * f_tiles) * F;
    if (p.offsets) {
      int lo = 0, hi = p.E;                  // the last e with tile_start[e] <= tt
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tile_start[mid] <= tt) lo = mid; else hi = mid;
      }
      it.e = lo;
      const int r0 = p.offsets[lo], rows = p.offsets[lo + 1] - r0;
      const int cuts = i4t_tiles<BT>(rows);
      const int per = ((rows + cuts - 1) / cuts + 15) & ~15;
      it.m0 = r0 + (tt - tile_start[lo]) * per;
      it.n = max(0, min(r0 + rows - it.m0, per));
    } else {
      it.e = 0;
      it.m0 = tt * p.tile_rows;
      it.n = min(p.rows - it.m0, p.tile_rows);
    }
    it.e = __shfl_sync(0xffffffffu, it.e, 0);
    it.m0 = __shfl_sync(0xffffffffu, it.m0, 0);
    it.n = __shfl_sync(0xffffffffu, it.n, 0);
    it.f0 = __shfl_sync(0xffffffffu, it.f0, 0);
    return it;
  };

  if (warp == 0) {
    int fill = 0;
    bool ok = true;
    for (int w = blockIdx.x; w < n_items && ok; w += gridDim.x) {
      const I4TItem it = item_of(w);
      if (it.n <= 0) continue;
      const int boxes = (((it.n + 15) & ~15) + I4T_BOX - 1) / I4T_BOX;
      const unsigned tx = (unsigned)(TERMS * boxes * I4T_BOX * 64 * 2);
      for (int kt = 0; kt < 2 * p.chunks; ++kt, ++fill) {
        const int s = fill % C::X_RING;
        ok = __all_sync(0xffffffffu, mbar_wait(&empty_x[s], ((fill / C::X_RING) & 1) ^ 1, abortp));
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(&full_x[s], tx);
          for (int t = 0; t < TERMS; ++t)
            for (int b = 0; b < boxes; ++b)
              tma_load_2d(xs + (s * TERMS + t) * C::X_BYTES + b * (I4T_BOX * 64 * 2), &map_x,
                          kt * 64, t * p.plane_rows + it.m0 + b * I4T_BOX, &full_x[s]);
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) {
      if (!*abortp) { atomicExch(p.status, I4T_ERR_COPY); *abortp = 1; }
      // copies in flight land before the block's shared memory goes away
      for (int f = max(0, fill - C::X_RING); f < fill; ++f)
        mbar_drain(&full_x[f % C::X_RING], (f / C::X_RING) & 1);
    }
  } else if (warp == 1) {
    int tile = 0, group = 0;                 // tiles of 64 k and groups so far, over all items
    bool ok = true;
    for (int w = blockIdx.x; w < n_items && ok; w += gridDim.x) {
      const I4TItem it = item_of(w);
      if (it.n <= 0) continue;
      // kind::f16: fp32 sums, both sides bfloat16 and K-major, M 128, N the tile's rows in sixteens
      const unsigned idesc = (1u << 4) | (1u << 7) | (1u << 10) |
                             ((unsigned)(((it.n + 15) & ~15) >> 3) << 17) | (8u << 24);
      for (int kt = 0; kt < 2 * p.chunks && ok; ++kt, ++tile) {
        const int sx = tile % C::X_RING, sa = tile % C::A_RING;
        ok = __all_sync(0xffffffffu, mbar_wait(&full_a[sa], (tile / C::A_RING) & 1, abortp)) &&
             __all_sync(0xffffffffu, mbar_wait(&full_x[sx], (tile / C::X_RING) & 1, abortp));
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int k4 = 0; k4 < 4; ++k4) {
          const int at = (kt & 1) * 4 + k4;            // sixteens of k into the chunk
          const bool first = at % (GROUP / 16) == 0, last = at % (GROUP / 16) == GROUP / 16 - 1;
          const int buf = group & 1;
          if (first) {
            ok = __all_sync(0xffffffffu,
                            mbar_wait(&acc_empty[buf], ((group >> 1) & 1) ^ 1, abortp));
            if (!ok) break;
            tc_fence_after();
          }
          if (lane == 0) {
            const unsigned long long ad = umma_desc(as + sa * I4T_A_BYTES) + 2 * k4;
#pragma unroll
            for (int t = TERMS - 1; t >= 0; --t)       // small terms first
              tc_mma(tmem_base + buf * BT, ad,
                     umma_desc(xs + (sx * TERMS + t) * C::X_BYTES) + 2 * k4, idesc,
                     (first && t == TERMS - 1) ? 0u : 1u);
            if (last) tc_commit(&acc_full[buf]);
            if (k4 == 3) {
              tc_commit(&empty_a[sa]);
              tc_commit(&empty_x[sx]);
            }
          }
          __syncwarp();
          if (last) ++group;
        }
      }
    }
    if (!ok && lane == 0 && !*abortp) { atomicExch(p.status, I4T_ERR_MMA); *abortp = 1; }
  } else {
    const int worker = warp - 2;
    const int quarter = warp & 3, half = worker >> 2;  // lanes of tensor memory; every second 32 rows
    const int g = lane >> 2, t = lane & 3;
    const bool odd = g & 1;
    bool ok = true;
    // strip s (0..7) of an item, as a block of the layout; strips past the last read the last
    auto block_of = [&](const I4TItem& it, int s) {
      const int strip = min(it.f0 / I4_STRIP + (DUAL ? (s & 3) : s), p.strips - 1);
      const size_t matrix = DUAL ? 2 * (size_t)it.e + (s >> 2) : (size_t)it.e;
      return (matrix * p.strips + strip) * p.chunks;
    };
    // -- the unpacking side: where the next chunk is, its codes and parameters in registers
    int next_w = blockIdx.x, next_c = 0, tile = 0;
    const unsigned *code_at = nullptr, *param_at = nullptr, *scale_at = nullptr;
    uint4 code[2];
    unsigned pa[NG], pb[NG], ps[NG];
    auto words = [&](const unsigned* at, unsigned* v) {
#pragma unroll
      for (int i = 0; i < NG; ++i) v[i] = __ldg(at + i);
    };
    auto fetch = [&]() {                     // the chunk at (next_w, next_c)
      code[0] = __ldg(reinterpret_cast<const uint4*>(code_at));
      code[1] = __ldg(reinterpret_cast<const uint4*>(code_at + I4_TILE_WORDS));
      words(param_at, pa);
      words(param_at + 8 * NG, pb);
      words(scale_at, ps);
    };
    auto enter = [&]() {                     // the first chunk of the next item with rows
      while (next_w < n_items) {
        const I4TItem it = item_of(next_w);
        if (it.n > 0) {
          const size_t own = block_of(it, worker), row = block_of(it, 2 * quarter + (lane >> 4));
          code_at = p.codes + own * I4_CHUNK_WORDS + lane * 4;
          param_at = p.params + (own * I4_STRIP + g) * NG;
          scale_at = p.params + (row * I4_STRIP + (lane & 15)) * NG;
          next_c = 0;
          fetch();
          return;
        }
        next_w += gridDim.x;
      }
    };
    float scale_next[NG];
    auto unpack = [&]() {                    // the chunk in registers into two operand tiles
#pragma unroll
      for (int i = 0; i < NG; ++i) scale_next[i] = i4_scale(ps[i]);
#pragma unroll
      for (int h = 0; h < 2; ++h, ++tile) {
        const int s = tile % C::A_RING;
        ok = __all_sync(0xffffffffu, mbar_wait(&empty_a[s], ((tile / C::A_RING) & 1) ^ 1, abortp));
        if (!ok) return;
        unsigned char* at = as + s * I4T_A_BYTES + worker * 2048 + g * 128;
#pragma unroll
        for (int run = 0; run < 2; ++run) {
          // lanes of odd rows take the two runs of eight k the other way round, so that the
          // eight lanes of a store phase meet all banks
          const bool second = (run == 1) != odd;
          const unsigned w0 = second ? code[h].z : code[h].x;
          const unsigned w1 = second ? code[h].w : code[h].y;
          unsigned sa, sb;
          if (GROUP == 32) {
            sa = i4_sub(second ? pa[(2 * h + 1) % NG] : pa[2 * h % NG]);
            sb = i4_sub(second ? pb[(2 * h + 1) % NG] : pb[2 * h % NG]);
          } else {
            sa = i4_sub(pa[GROUP == 64 ? h % NG : 0]);
            sb = i4_sub(pb[GROUP == 64 ? h % NG : 0]);
          }
          const int where = (((second ? 4 : 0) + t) ^ g) * 16;
          *reinterpret_cast<uint4*>(at + where) = make_uint4(
              i4_pair(w0, 0, sa), i4_pair(w0, 2, sa), i4_pair(w1, 0, sa), i4_pair(w1, 2, sa));
          *reinterpret_cast<uint4*>(at + 1024 + where) = make_uint4(
              i4_pair(w0, 1, sb), i4_pair(w0, 3, sb), i4_pair(w1, 1, sb), i4_pair(w1, 3, sb));
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full_a[s]);
      }
      if (++next_c < p.chunks) {
        code_at += I4_CHUNK_WORDS;
        param_at += I4_STRIP * NG;
        scale_at += I4_STRIP * NG;
        fetch();
      } else {
        next_w += gridDim.x;
        enter();
      }
    };
    // -- the summing side
    int group = 0, handed = 0;
    float sum[BT / 64][32];
    enter();
    if (next_w < n_items) unpack();
    for (int w = blockIdx.x; w < n_items && ok; w += gridDim.x) {
      const I4TItem it = item_of(w);
      if (it.n <= 0) continue;
#pragma unroll
      for (int i = 0; i < BT / 64; ++i)
#pragma unroll
        for (int j = 0; j < 32; ++j) sum[i][j] = 0.f;
      const unsigned lanes = tmem_base + ((unsigned)(quarter * 32) << 16);
      for (int c = 0; c < p.chunks && ok; ++c) {
        float scale[NG];
#pragma unroll
        for (int i = 0; i < NG; ++i) scale[i] = scale_next[i];
        if (next_w < n_items) unpack();
        if (!ok) break;
#pragma unroll
        for (int n = 0; n < NG; ++n, ++group) {
          const int buf = group & 1;
          ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[buf], (group >> 1) & 1, abortp));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < BT / 64; ++i) {
            const int col = 64 * i + 32 * half;
            if (col < it.n) {
              float v[32];
              tc_ld32(lanes + buf * BT + col, v);
#pragma unroll
              for (int j = 0; j < 32; ++j) sum[i][j] = fmaf(scale[n], v[j], sum[i][j]);
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty[buf]);
        }
      }
      if (!ok) break;
      // -- a lane holds one weight row for 32 rows at a time: 64- or 128-byte stores of a warp
      if (DUAL) {
        // the warps of the up rows (quarters 2, 3) hand their sums to those of the gate rows
        const int pair = (quarter & 1) + 2 * half;
        float* mine = exchange + pair * (32 * 33);
        const int f = it.f0 + (quarter & 1) * 32 + lane;
#pragma unroll
        for (int i = 0; i < BT / 64; ++i) {
          const int col = 64 * i + 32 * half;
          if (col >= it.n) continue;
          if (quarter >= 2) {
            ok = __all_sync(0xffffffffu, mbar_wait(&ex_empty[pair], (handed & 1) ^ 1, abortp));
            if (!ok) break;
#pragma unroll
            for (int j = 0; j < 32; ++j) mine[j * 33 + lane] = sum[i][j];
            __syncwarp();
            if (lane == 0) mbar_arrive(&ex_full[pair]);
            ++handed;
          } else {
            ok = __all_sync(0xffffffffu, mbar_wait(&ex_full[pair], handed & 1, abortp));
            if (!ok) break;
            ++handed;
            const float rs = p.row_scale && col + lane < it.n ? p.row_scale[it.m0 + col + lane] : 1.f;
            float y[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float s = __shfl_sync(0xffffffffu, rs, j);
              const float a = sum[i][j] * s, u = mine[j * 33 + lane] * s;
              y[j] = p.wide ? a / (1.0f + expf(-a)) * u : __fdividef(a, 1.0f + __expf(-a)) * u;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&ex_empty[pair]);
            const int n_here = f < p.N ? it.n - col : 0;
            const size_t at = (size_t)(it.m0 + col) * p.N + f;
            if (p.wide) {
              float* o = (float*)p.out + at;
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (j < n_here) o[(size_t)j * p.N] = y[j];
            } else {
              bf16* o = (bf16*)p.out + at;
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (j < n_here) o[(size_t)j * p.N] = __float2bfloat16_rn(y[j]);
            }
          }
        }
      } else {
        const int f = it.f0 + quarter * 32 + lane;
#pragma unroll
        for (int i = 0; i < BT / 64; ++i) {
          const int col = 64 * i + 32 * half;
          if (col >= it.n) continue;
          const int n_here = f < p.N ? it.n - col : 0;
          const size_t at = (size_t)(it.m0 + col) * p.N + f;
          if (p.plain) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              sum[i][j] = p.wide ? ix_act<float>(sum[i][j], p.plain) : ix_act<bf16>(sum[i][j], p.plain);
          }
          if (p.wide) {
            float* o = (float*)p.out + at;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j < n_here) o[(size_t)j * p.N] = sum[i][j];
          } else {
            bf16* o = (bf16*)p.out + at;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j < n_here) o[(size_t)j * p.N] = __float2bfloat16_rn(sum[i][j]);
          }
        }
      }
    }
    if (!ok && lane == 0 && !*abortp) { atomicExch(p.status, I4T_ERR_WORK); *abortp = 1; }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tc_dealloc<false>(tmem_base, C::TMEM_COLS);
}

template <int TERMS, bool DUAL, int BT, int GROUP>
static int i4t_launch(const void* x, int x_rows, int Kp, I4TArgs p, int sms, cudaStream_t stream) {
  typedef I4TCfg<TERMS, DUAL, BT, GROUP> C;
  CUtensorMap map;
  const int rc = ix_tensor_map_bf16_2d(&map, x, (long long)TERMS * x_rows, Kp, 64, I4T_BOX);
  if (rc != IX_OK) return rc;
  const long long tiles = p.offsets ? (p.rows + BT - 1) / BT + (long long)p.E
                                    : (p.rows + p.tile_rows - 1) / p.tile_rows;
  const long long items = tiles * ((p.N + C::F - 1) / C::F);
  if (items > 0x7fffffffLL) return IX_ERR_SIZE;
  auto kern = int4_tc_kernel<TERMS, DUAL, BT, GROUP>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return (int)e;
  kern<<<(int)(items < sms ? items : sms), I4T_THREADS, C::SMEM, stream>>>(map, p);
  return ix_launch_status();
}

// x: [rows, Kp] bf16, or [3, rows, Kp] terms of fp32 rows; Kp a multiple of 8 that ends in the last
// chunk.  out: [rows, N] fp32 (wide) or bf16.  offsets == null: one matrix.  status: one int, zero
// before the first call.
IX_API int ix_int4_tc(const void* x, int terms, const int* offsets, const void* codes,
                      const void* params, void* out, int wide, int dual, int rows, int N, int Kp,
                      int E, int group, const float* row_scale, int plain, int* status,
                      cudaStream_t stream) {
  if ((row_scale && !dual) || (plain && dual)) return IX_ERR_UNSUPPORTED;
  if (rows <= 0) return IX_OK;
  if (N <= 0 || Kp <= 0 || E <= 0 || status == nullptr) return IX_ERR_SIZE;
  if (Kp % 8 != 0 || E > I4T_MAX_EXPERTS || (!offsets && E != 1)) return IX_ERR_UNSUPPORTED;
  if ((uintptr_t)x & 15) return IX_ERR_ALIGN;
  if (3LL * rows > 0x7fffffffLL) return IX_ERR_SIZE;
  static int sms = 0;
  if (sms == 0) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
      sms = 148;
  }
  I4TArgs p = {offsets, (const unsigned*)codes, (const unsigned*)params, out, wide, row_scale, plain,
               rows, N, (int)i4_strips(N), (int)i4_chunks(Kp), E, 0, rows, status};
  const int f = dual ? 64 : 128;
  bool large;
  if (offsets) {
    large = 1.15 * rows / E > 128.0;      // the mean rows of an expert, and some for imbalance
  } else {
    large = rows > 128;
    const int most = large && terms == 1 ? 256 : 128;
    // as many tiles as give the least work: waves of blocks times the rows of a tile (and some
    // that a tile costs whatever its rows)
    const int f_tiles = (N + f - 1) / f;
    long long best = -1;
    for (int cuts = (rows + most - 1) / most; cuts <= (rows + most - 1) / most + 8; ++cuts) {
      const int per = ((rows + cuts - 1) / cuts + 15) & ~15;
      const long long items = (long long)((rows + per - 1) / per) * f_tiles;
      const long long cost = (items + sms - 1) / sms * (per + 32);
      if (best < 0 || cost < best) {
        best = cost;
        p.tile_rows = per;
      }
      if (per <= 16) break;
    }
    large = p.tile_rows > 128;
  }
#define I4T_BT(T, D, B)                                                               \
  do {                                                                                \
    if (group == 128) return i4t_launch<T, D, B, 128>(x, rows, Kp, p, sms, stream);   \
    if (group == 64) return i4t_launch<T, D, B, 64>(x, rows, Kp, p, sms, stream);     \
    if (group == 32) return i4t_launch<T, D, B, 32>(x, rows, Kp, p, sms, stream);     \
    return IX_ERR_UNSUPPORTED;                                                        \
  } while (0)
  if (terms == 1) {
    if (dual) {
      if (large) I4T_BT(1, true, 256);
      I4T_BT(1, true, 128);
    }
    if (large) I4T_BT(1, false, 256);
    I4T_BT(1, false, 128);
  }
  if (terms == 3) {
    if (dual) I4T_BT(3, true, 128);
    I4T_BT(3, false, 128);
  }
  return IX_ERR_UNSUPPORTED;
}
