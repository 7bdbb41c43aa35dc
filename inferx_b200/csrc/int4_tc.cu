// Products with four-bit weights for many rows (prompts) on the 5th-generation tensor cores.
//
//   out[r, j] = sum_k a[r, k] * w[e(r), j, k]                (plain, an activation may follow)
//   out[r, j] = silu(a . wg[e, j]) * (a . wu[e, j])          (DUAL)
//   w[j, k] = scale[j, k / group] * (code[j, k] - zero[j, k / group])      (int4_format.cuh)
//
// `a` holds bfloat16 rows grouped by expert (offsets), or the rows of a single matrix; fp32 rows come
// as three planes of bfloat16 terms that are multiplied into the same sums.
//
// The weights are the M side of tcgen05.mma, read from tensor memory, and the rows the N side, read from
// shared memory.  Two SMs work on one item (cta_group::2): 256 weight rows (DUAL: 128 gate rows and the
// up rows of the same columns) for a tile of up to BT rows of one expert, over all of K or one of
// `splits` runs of it.  A block holds 128 of the weight rows and half of the tile's rows, so each of the
// two halves is brought once.  Pairs are persistent and take items round robin.  Roles of a block's
// warps, a chunk of 128 k at a time:
//   0      brings the rows into a ring of stages (TMA, 128-byte swizzle);
//   1      the first block's issues the MMAs for both, a group of k into one of two accumulators in
//          tensor memory; the second block's tells the first that its weights are there and its sums
//          taken (its rows' copies report to the first block's barrier themselves);
//   2      brings the codes and parameters of the block's eight strips (one bulk copy, DUAL two);
//   4-11   take each finished group's sums out of tensor memory, a weight row a lane, add scale * sum to
//          fp32 registers, and leave an item's results in shared memory;
//   12-19  unpack, four the even chunks and four the odd ones, two strips a warp: a lane's sixteen bytes
//          of codes, less their zero points, are numbers of five bits that lie in registers as tensor memory
//          wants them (16 rows by 256 bits);
//   20-23  finish and store the results of an item while the next one is under way.
// Rows of a DUAL item lie as 16 gate rows, the 16 up rows of the same columns, and so on.
// So the operands of the tensor cores are exact (a code less its zero point has five bits), the sums of
// a group are the tensor cores' fp32, and a group's scale multiplies in fp32: no weight is rounded to
// bfloat16.
//
// Measured (bfloat16, groups of 128): 2,048 rows, 2,048 -> 6,144 57.7 us (893 TFLOP/s); 4,096 rows, 3,584 ->
// 4,096 111 us (1,081; a bfloat16 library product alone reaches 1,670); gated, 2,048 rows, 2,048 -> 2 x
// 5,632 97 us (976); 60 experts of 2 x 1,408 x 2,048 with 137 rows each 132 us (715).  What bounds it: a chunk
// of 192 rows takes 1,330 cycles where its MMAs are 768.  The summing warps need 700 for their 96 columns
// and 630 more from one accumulator to the next (the arrival, two waits), and an operand stage is full
// again 1,300 after its MMAs have run; tensor memory has room for two accumulators and two stages.
// Groups of 64 or 32 have two or four sums a chunk to take: 2,048 -> 6,144 80.6 and 139 us.  fp32 rows
// have three times the MMAs for the same sums: 118 us, 437 TFLOP/s of 557.
// Built and slower: every warp of the second block arriving at the first's barrier by itself (64 us
// where the one relay had 60), sixteen columns of sums on their way while sixteen are added (61 against
// 59), polling barriers instead of sleeping on them (63 against 59).
//
// Columns past the tile and weight rows past N are computed on whatever is there and never stored.
// Every wait on an mbarrier is bounded: the waiter records a code in `status` (51 and 54 copies, 52
// MMAs, 53 unpacking, 55 sums, 56 results), raises a flag that ends its block's other roles, and the pair meets at
// its end, where tensor memory is freed.
#include <type_traits>

#include "int4_format.cuh"
#include "tcgen05_common.cuh"
#include "tma_common.cuh"

#define I4T_THREADS 768
#define I4T_MAX_EXPERTS 1024              // the prefix of tiles lives in shared memory
#define I4T_NAP 20000                     // ns
#define I4T_WAIT_CLOCKS 4000000000LL      // about two seconds
#define I4T_DONE 4                        // barriers of finished chunks

enum {
  I4T_ERR_COPY = 51, I4T_ERR_MMA = 52, I4T_ERR_UNPACK = 53, I4T_ERR_CODES = 54, I4T_ERR_SUM = 55,
  I4T_ERR_STORE = 56
};

struct I4TArgs {
  const int* offsets;       // null: one matrix with `rows` rows
  const unsigned* data;
  void* out;
  float* part;              // splits > 1: [splits][rows][columns of both halves] sums
  int wide;                 // fp32 results, otherwise bfloat16
  const float* row_scale;
  int plain;
  int rows, N, strips, chunks, E;
  int tile_rows;            // one matrix: rows of a tile, a multiple of 32
  int splits, run;          // runs of K, chunks of a run
  int plane_rows;           // rows of one plane of terms
  int* status;
};

struct I4TItem {
  int e, m0, n, f0, c0, c1, z;
};

template <int TERMS, bool DUAL, int BT, int GROUP> struct I4TCfg {
  static constexpr int X_TILE = BT / 2 * 64 * 2;               // 64 k of a block's rows, one term
  static constexpr int X_STAGE = TERMS * 2 * X_TILE;
  static constexpr int BOX = BT / 4;                           // rows of a TMA box
  static constexpr int C_BYTES = i4_block_words(GROUP) * 4;    // a strip's codes and parameters
  static constexpr int X_RING = TERMS == 3 ? 2 : 4;
  static constexpr int C_RING = BT == 128 ? 4 : GROUP == 128 ? 3 : 2;
  // Tensor memory: two accumulators of BT columns, and operand stages of 128 k (64 columns)
  static constexpr int A_RING = (512 - 2 * BT) / 64;
  // Scales are written once the MMAs of A_RING chunks before have run, and those had waited for the
  // sums of two chunks before them to be taken: a slot is read by then.
  static constexpr int S_RING = A_RING + 2;
  static constexpr int SMEM = X_RING * X_STAGE + BT * 128 * 4 + C_RING * 8 * C_BYTES +
                              S_RING * 128 * (128 / GROUP) * 2 + 1024;
  static_assert(SMEM + 4608 <= 227 * 1024, "shared memory");
  static_assert(X_RING <= I4T_DONE && A_RING <= I4T_DONE, "a stage's last use is still to be seen");
  static_assert(A_RING % 2 == 0 && S_RING % 2 == 0, "a stage's chunks are the same four warps'");
  static_assert(BT % 64 == 0 && 2 * BT + 64 * A_RING <= 512, "tensor memory");
  static constexpr int F = DUAL ? 128 : 256;                   // output columns of an item
};

// bytes (a multiple of 16, both sides 16-byte aligned) into shared memory, counted at `bar`
__device__ __forceinline__ void i4t_copy(void* to, const void* from, unsigned bytes,
                                         unsigned long long* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(to)),
      "l"(from), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}
// Bounded wait; its polls sleep in the barrier unit, up to I4T_NAP ns each.  PAIR: for a barrier that
// the other block and its copies arrive at too.
template <bool PAIR>
__device__ __forceinline__ bool i4t_try(unsigned long long* bar, unsigned parity) {
  unsigned ok;
  if (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(I4T_NAP)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(I4T_NAP)
        : "memory");
  return ok != 0;
}
template <bool PAIR = false>
__device__ __forceinline__ bool i4t_wait(unsigned long long* bar, unsigned parity,
                                         volatile int* abort_flag) {
  if (i4t_try<PAIR>(bar, parity)) return true;
  const long long begin = clock64();
  while (clock64() - begin < I4T_WAIT_CLOCKS) {
    if (i4t_try<PAIR>(bar, parity)) return true;
    if (*abort_flag) return false;
  }
  return false;
}
// One lane of the warp, known to the compiler to be one: with `lane == 0` the eight MMAs of a chunk
// take 700 cycles to issue, with this 250.
__device__ __forceinline__ bool i4t_elect() {
  unsigned ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok));
  return ok != 0;
}
// The pair's MMA with the weights in tensor memory (each block's rows in its own).
__device__ __forceinline__ void i4t_mma(unsigned d, unsigned a, unsigned long long bdesc,
                                        unsigned idesc, unsigned accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accum)
      : "memory");
}
// Sixteen rows by 64 k of an operand: four registers a lane for every sixteen k.
__device__ __forceinline__ void i4t_put(unsigned taddr, const unsigned* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
// sixteen columns of this thread's lane
__device__ __forceinline__ void i4t_ld16(unsigned taddr, float* v) {
  unsigned r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
// two fp32 numbers as one 64-bit register, and a * b + c on both
__device__ __forceinline__ unsigned long long i4t_pack(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void i4t_unpack(unsigned long long v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ void i4t_fma2(unsigned long long& c, unsigned long long a,
                                         unsigned long long b) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(a), "l"(b));
}

// the low halves of NG parameters beside each other
template <int NG> __device__ __forceinline__ void i4t_scales(unsigned short* to, const unsigned* v) {
  if (NG == 1) *to = (unsigned short)v[0];
  if (NG == 2) *reinterpret_cast<unsigned*>(to) = __byte_perm(v[0], v[NG - 1], 0x5410);
  if (NG == 4)
    *reinterpret_cast<uint2*>(to) =
        make_uint2(__byte_perm(v[0], v[NG > 1 ? 1 : 0], 0x5410),
                   __byte_perm(v[NG > 2 ? 2 : 0], v[NG - 1], 0x5410));
}
// sum += scale * (32 columns of this thread's lane)
__device__ __forceinline__ void i4t_add(unsigned long long* sum, unsigned long long scale,
                                        unsigned taddr) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float v[16];
    i4t_ld16(taddr + 16 * h, v);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      i4t_fma2(sum[8 * h + j], scale, i4t_pack(v[2 * j], v[2 * j + 1]));
  }
}

template <int BT>
__device__ __forceinline__ int i4t_tiles(int rows) { return (rows + BT - 1) / BT; }

template <int TERMS, bool DUAL, int BT, int GROUP>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(I4T_THREADS, 1)
int4_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ I4TArgs p) {
  typedef I4TCfg<TERMS, DUAL, BT, GROUP> C;
  constexpr int NG = 128 / GROUP;
  constexpr int F = C::F;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* xs =
      reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* stage = reinterpret_cast<float*>(xs + C::X_RING * C::X_STAGE);   // [row of the tile][128]
  unsigned char* cs = reinterpret_cast<unsigned char*>(stage + BT * 128);
  unsigned short* scales = reinterpret_cast<unsigned short*>(cs + C::C_RING * 8 * C::C_BYTES);
  // A group may be multiplied: on a chunk's first group the block's weights are there (four unpacking
  // warps), an accumulator's sums are taken (eight warps), and, in the first block, the second one is as
  // far and both blocks' rows are there.  One barrier for all of it, as a wait costs the issuing warp
  // hundreds of cycles even where nothing is waited for.
  // The second block's arrival is relaxed: its threads' weights and sums are tensor memory, which the
  // tcgen05 fences on both sides order.  Its rows lie in shared memory, and their copies report
  // to the first block's barrier themselves, which releases them to the cluster.  (An arrival that
  // releases what threads have written takes some 1,400 cycles, more than a chunk's MMAs; 2,048 rows,
  // 2,048 -> 6,144 with the rows announced that way from a warp of their own 61.8 us, as it is 57.4.)
  __shared__ __align__(8) unsigned long long go[I4T_DONE][NG];
  // Codes of a chunk are there.  Two barriers for every stage, chunks in turn, so that a barrier's
  // chunks are all unpacked by the same four warps: a wait for a phase is only right where the phase
  // before has been waited for, and with three stages and one barrier each the phase before belongs to
  // the other four warps, whose copy may land later.
  __shared__ __align__(8) unsigned long long full_c[2 * C::C_RING], empty_c[C::C_RING];
  __shared__ __align__(8) unsigned long long done[I4T_DONE];     // a chunk's MMAs have run
  __shared__ __align__(8) unsigned long long full_s[C::S_RING];  // a chunk's scales are there
  __shared__ __align__(8) unsigned long long acc_full[2];
  __shared__ __align__(8) unsigned long long stage_full, stage_empty;
  __shared__ unsigned tmem_holder;
  __shared__ int abort_flag;
  __shared__ int tile_start[I4T_MAX_EXPERTS + 1];

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = (int)tc_rank();
  const int f_tiles = (p.N + F - 1) / F;
  if (warp == 3) {                           // tiles before each expert
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
    for (int s = 0; s < I4T_DONE; ++s)
      for (int q = 0; q < NG; ++q)
        mbar_init(&go[s][q], q == 0 ? (rank == 0 ? 14 : 12) : (rank == 0 ? 9 : 8));
    for (int s = 0; s < 2 * C::C_RING; ++s) mbar_init(&full_c[s], 1);
    for (int s = 0; s < C::C_RING; ++s) mbar_init(&empty_c[s], 4);
    for (int s = 0; s < I4T_DONE; ++s) mbar_init(&done[s], 1);
    for (int s = 0; s < C::S_RING; ++s) mbar_init(&full_s[s], 4);
    for (int b = 0; b < 2; ++b) mbar_init(&acc_full[b], 1);
    mbar_init(&stage_full, 8);
    mbar_init(&stage_empty, 4);
    abort_flag = 0;
    mbar_init_fence();
    fence_proxy_async();
  }
  if (warp == 1) tc_alloc<true>(&tmem_holder, 512);
  tc_fence_before();
  __syncthreads();
  tc_cluster_sync();
  tc_fence_after();
  const unsigned tmem_base = __shfl_sync(0xffffffffu, tmem_holder, 0);
  volatile int* abortp = &abort_flag;
  const int n_items = tile_start[p.E] * f_tiles * p.splits;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

  auto item_of = [&](int w) {
    I4TItem it;
    it.z = w % p.splits;
    w /= p.splits;
    const int tt = w / f_tiles;
    it.f0 = (w - tt * f_tiles) * F;
    it.c0 = min(p.chunks, it.z * p.run);     // (roles count chunks: c1 - c0 is never negative)
    it.c1 = min(p.chunks, it.c0 + p.run);
    if (p.offsets) {
      int lo = 0, hi = p.E;                  // the last e with tile_start[e] <= tt
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tile_start[mid] <= tt) lo = mid; else hi = mid;
      }
      it.e = lo;
      const int r0 = p.offsets[lo], rows = p.offsets[lo + 1] - r0;
      const int cuts = i4t_tiles<BT>(rows);
      const int per = ((rows + cuts - 1) / cuts + 31) & ~31;
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
    it.c0 = __shfl_sync(0xffffffffu, it.c0, 0);
    it.c1 = __shfl_sync(0xffffffffu, it.c1, 0);
    return it;
  };
  auto wait = [&](unsigned long long* bar, int parity) {
    return (bool)__all_sync(0xffffffffu, i4t_wait(bar, parity, abortp));
  };

  // Registers go from the roles that need few to the warps that hold up to 96 sums a lane (768
  // threads at 80: 128 x 32 + 256 x 136 + 256 x 56 + 128 x 56).
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
    if (warp == 0) {
      const unsigned first_block = tc_of_rank(&go[0][0], 0);
      int n = 0;                             // chunks so far, over all items
      bool ok = true;
      for (int w = first; w < n_items && ok; w += step) {
        const I4TItem it = item_of(w);
        if (it.n <= 0) continue;
        const int half = ((it.n + 31) & ~31) / 2;              // rows of this block
        const int boxes = (half + C::BOX - 1) / C::BOX;
        // a lane a box: term, 64 k, a quarter of the tile's rows
        const int box = lane % boxes, sub = lane / boxes & 1, term = lane / (2 * boxes);
        for (int c = it.c0; c < it.c1; ++c, ++n) {
          const int s = n % C::X_RING;
          if (n >= C::X_RING) {
            const int before = n - C::X_RING;
            ok = wait(&done[before % I4T_DONE], before / I4T_DONE & 1);
            if (!ok) break;
          }
          // both blocks' bytes (the second's may land before they are expected: the phase is not over
          // without this arrival, and its copies are not sent before the last phase is)
          if (rank == 0 && lane == 0)
            mbar_expect_tx(&go[n % I4T_DONE][0],
                           (unsigned)(2 * TERMS * 2 * boxes * C::BOX * 64 * 2));
          __syncwarp();
          if (term < TERMS)
            tc_load_pair(xs + s * C::X_STAGE + (term * 2 + sub) * C::X_TILE +
                             box * (C::BOX * 64 * 2),
                         &map_x, c * 128 + sub * 64,
                         term * p.plane_rows + it.m0 + rank * half + box * C::BOX,
                         first_block + (n % I4T_DONE) * NG * 8);
          __syncwarp();
        }
      }
      if (lane == 0) {
        if (!ok && !*abortp) { atomicExch(p.status, I4T_ERR_COPY); *abortp = 1; }
        // copies in flight land before the block's shared memory goes away, whatever the others do
        // (a wait that nothing ends takes its full limit, thousands of times as long as a copy)
        if (!ok)
          for (int f = max(0, n - C::X_RING); f < n; ++f)
            mbar_drain(&done[f % I4T_DONE], f / I4T_DONE & 1);
        else if (n > 0)
          mbar_drain(&done[(n - 1) % I4T_DONE], (n - 1) / I4T_DONE & 1);
      }
    } else if (warp == 1) {
      const unsigned first_block = tc_of_rank(&go[0][0], 0);
      int n = 0, group = 0;
      bool ok = true;
      for (int w = first; w < n_items && ok; w += step) {
        const I4TItem it = item_of(w);
        if (it.n <= 0) continue;
        // kind::f16: fp32 sums, both sides bfloat16 and K-major, M 256, N the tile's rows
        const unsigned idesc = (1u << 4) | (1u << 7) | (1u << 10) |
                               ((unsigned)(((it.n + 31) & ~31) >> 3) << 17) | (16u << 24);
        for (int c = it.c0; c < it.c1 && ok; ++c, ++n) {
          const int slot = n % I4T_DONE;
          const unsigned ad = tmem_base + 2 * BT + (n % C::A_RING) * 64;
          const unsigned long long xd = umma_desc(xs + (n % C::X_RING) * C::X_STAGE);
          for (int q = 0; q < NG; ++q, ++group) {
            // (one wait for both blocks: with a wait in either branch a chunk takes 3 % longer, and
            // with groups of 64 17 %)
            ok = __all_sync(0xffffffffu,
                            i4t_wait<true>(&go[slot][q], n / I4T_DONE & 1, abortp));
            if (!ok) break;
            tc_fence_after();
            if (rank != 0) {
              tc_fence_before();
              if (i4t_elect()) tc_arrive_relaxed_at(first_block + (slot * NG + q) * 8);
              __syncwarp();
              continue;
            }
            const int buf = group & 1;
            const unsigned sums = tmem_base + buf * BT;
            if (i4t_elect()) {
#pragma unroll
              for (int i = 0; i < GROUP / 16; ++i) {
                // sixteens of k into the chunk: eight columns of weights, 32 bytes of a row
                const int at = q * (GROUP / 16) + i;
#pragma unroll
                for (int t = TERMS - 1; t >= 0; --t)           // small terms first
                  i4t_mma(sums, ad + at * 8,
                          xd + (t * 2 + (at >> 2)) * (C::X_TILE >> 4) + (at & 3) * 2, idesc,
                          i == 0 && t == TERMS - 1 ? 0u : 1u);
              }
              if (NG > 1) tc_commit_pair(&acc_full[buf]);
              if (q == NG - 1) tc_commit_pair(&done[slot]);
            }
            __syncwarp();
          }
        }
      }
      if (!ok && lane == 0 && !*abortp) { atomicExch(p.status, I4T_ERR_MMA); *abortp = 1; }
    } else if (warp == 2) {
      int n = 0;
      bool ok = true;
      for (int w = first; w < n_items && ok; w += step) {
        const I4TItem it = item_of(w);
        if (it.n <= 0) continue;
        // strips past the last one stay as they are in shared memory: their sums are not stored
        const int s0 = (it.f0 + rank * (F / 2)) / I4_STRIP;
        const int count = max(0, min(DUAL ? 4 : 8, p.strips - s0));
        const unsigned bytes = (unsigned)(count * C::C_BYTES);
        const size_t pitch = (size_t)p.strips * C::C_BYTES;
        const unsigned char* from = reinterpret_cast<const unsigned char*>(p.data) +
                                    ((size_t)it.e * (DUAL ? 2 : 1) * p.chunks + it.c0) * pitch +
                                    (size_t)s0 * C::C_BYTES;
        for (int c = it.c0; c < it.c1; ++c, ++n, from += pitch) {
          const int s = n % C::C_RING;
          ok = wait(&empty_c[s], (n / C::C_RING & 1) ^ 1);
          if (!ok) break;
          if (lane == 0) {
            unsigned char* to = cs + s * 8 * C::C_BYTES;
            unsigned long long* full = &full_c[n % (2 * C::C_RING)];
            mbar_expect_tx(full, DUAL ? 2 * bytes : bytes);
            if (bytes) {
              i4t_copy(to, from, bytes, full);
              if (DUAL) i4t_copy(to + 4 * C::C_BYTES, from + p.chunks * pitch, bytes, full);
            }
          }
          __syncwarp();
        }
      }
      if (lane == 0) {
        if (!ok && !*abortp) { atomicExch(p.status, I4T_ERR_CODES); *abortp = 1; }
        for (int f = max(0, n - C::C_RING); f < n; ++f)
          mbar_drain(&full_c[f % (2 * C::C_RING)], f / (2 * C::C_RING) & 1);
      }
    }
  } else if (warp >= 20) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    // Units of eight neighbouring columns of one row: sixteen a row (DUAL: eight), so 128 threads take
    // eight (sixteen) rows a pass; consecutive threads take consecutive units.
    constexpr int COLS = F / 2, UNITS = COLS / 8;
    const int thread = threadIdx.x - 20 * 32;
    const int unit = thread % UNITS;
    const int at = DUAL ? (unit >> 1) * 32 + (unit & 1) * 8 : unit * 8;      // its first entry of a row
    const bool whole = p.N % 8 == 0 && ((uintptr_t)p.out & 15) == 0;
    int k = 0;                               // items so far
    bool ok = true;
    for (int w = first; w < n_items && ok; w += step) {
      const I4TItem it = item_of(w);
      if (it.n <= 0) continue;
      ok = wait(&stage_full, k & 1);
      if (!ok) break;
      const int f = it.f0 + rank * COLS + unit * 8;
      const int cols = min(8, p.N - f);
      if (cols > 0)
        for (int r = thread / UNITS; r < it.n; r += 128 / UNITS) {
          float v[8], u[8];
          *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(stage + r * 128 + at);
          *reinterpret_cast<float4*>(v + 4) =
              *reinterpret_cast<const float4*>(stage + r * 128 + at + 4);
          if (DUAL) {
            *reinterpret_cast<float4*>(u) = *reinterpret_cast<const float4*>(stage + r * 128 + at + 16);
            *reinterpret_cast<float4*>(u + 4) =
                *reinterpret_cast<const float4*>(stage + r * 128 + at + 20);
          }
          const size_t row = (size_t)(it.m0 + r);
          if (p.part) {                      // sums of a run of K: the halves' columns beside each other
            const size_t width = DUAL ? 2 * (size_t)p.N : (size_t)p.N;
            float* o = p.part + ((size_t)it.z * p.rows + row) * width + f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (i < cols) {
                o[i] = v[i];
                if (DUAL) o[p.N + i] = u[i];
              }
            continue;
          }
          if (DUAL) {
            const float s = p.row_scale ? p.row_scale[row] : 1.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float a = v[i] * s;
              v[i] = p.wide ? a / (1.0f + expf(-a)) * (u[i] * s)
                            : __fdividef(a, 1.0f + __expf(-a)) * (u[i] * s);
            }
          } else if (p.plain) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              v[i] = p.wide ? ix_act<float>(v[i], p.plain) : ix_act<bf16>(v[i], p.plain);
          }
          const size_t to = row * p.N + f;
          if (p.wide) {
            float* o = (float*)p.out + to;
            if (whole) {
              *reinterpret_cast<float4*>(o) = *reinterpret_cast<float4*>(v);
              *reinterpret_cast<float4*>(o + 4) = *reinterpret_cast<float4*>(v + 4);
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (i < cols) o[i] = v[i];
            }
          } else {
            bf16* o = (bf16*)p.out + to;
            if (whole) {
              __nv_bfloat162 h[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
              *reinterpret_cast<uint4*>(o) = *reinterpret_cast<uint4*>(h);
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (i < cols) o[i] = __float2bfloat16_rn(v[i]);
            }
          }
        }
      __syncwarp();
      if (lane == 0) mbar_arrive(&stage_empty);
      ++k;
    }
    if (!ok && lane == 0 && !*abortp) { atomicExch(p.status, I4T_ERR_STORE); *abortp = 1; }
  } else if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    // its strips: the two that the warp's lanes of tensor memory hold
    const int quarter = warp & 3, turn = (warp - 12) >> 2;
    const int g = lane >> 2, t = lane & 3;
    const unsigned to = tmem_base + 2 * BT + ((unsigned)(quarter * 32) << 16);
    int n = 0;
    bool ok = true;
    for (int w = first; w < n_items && ok; w += step) {
      const I4TItem it = item_of(w);
      if (it.n <= 0) continue;
      const int chunks = it.c1 - it.c0, end = n + chunks;
      for (n += (n & 1) != turn; n < end; n += 2) {
        const int sc = n % C::C_RING, sa = n % C::A_RING;
        ok = wait(&full_c[n % (2 * C::C_RING)], n / (2 * C::C_RING) & 1);
        if (!ok) break;
        // (DUAL: four gate strips were copied, then four up strips)
        const unsigned* own[2];
        uint4 code[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          own[i] = reinterpret_cast<const unsigned*>(
              cs + (sc * 8 + (DUAL ? i * 4 + quarter : 2 * quarter + i)) * C::C_BYTES);
          code[i][0] = *reinterpret_cast<const uint4*>(own[i] + lane * 4);
          code[i][1] = *reinterpret_cast<const uint4*>(own[i] + I4_TILE_WORDS + lane * 4);
        }
        // (parameters of groups of 64 or 32 are read when their strip's turn comes: there are not the
        // registers to hold them all)
        unsigned pa[2][NG], pb[2][NG];
        auto params = [&](int i) {
#pragma unroll
          for (int j = 0; j < NG; ++j) {
            pa[i][j] = own[i][I4_CODE_WORDS + g * NG + j];
            pb[i][j] = own[i][I4_CODE_WORDS + (g + 8) * NG + j];
          }
          if (i == 1) {
            // The next copy into this stage may not pass the reads, which no instruction has waited
            // for yet: where the load unit is busy with results an arrival overtakes them by a
            // microsecond, and the codes of three chunks on are what is read.
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty_c[sc]);
          }
        };
        if (NG == 1) {
          params(0);
          params(1);
        }
        if (n >= C::A_RING) {
          const int before = n - C::A_RING;
          ok = wait(&done[before % I4T_DONE], before / I4T_DONE & 1);
          if (!ok) break;
        }
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (NG > 1) params(i);
          // the scales, by row and group, to the warps that add up
          if (t == 0) {
            unsigned short* row = scales + ((n % C::S_RING) * 128 + quarter * 32 + i * 16 + g) * NG;
            i4t_scales<NG>(row, pa[i]);
            i4t_scales<NG>(row + 8 * NG, pb[i]);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const unsigned word[4] = {code[i][h].x, code[i][h].y, code[i][h].z, code[i][h].w};
            unsigned v[16];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int group = (h * 4 + j) * 16 / GROUP;
              const unsigned sa2 = i4_sub(pa[i][group]), sb2 = i4_sub(pb[i][group]);
              v[4 * j] = i4_pair(word[j], 0, sa2);
              v[4 * j + 1] = i4_pair(word[j], 2, sa2);
              v[4 * j + 2] = i4_pair(word[j], 1, sb2);
              v[4 * j + 3] = i4_pair(word[j], 3, sb2);
            }
            i4t_put(to + ((unsigned)(i * 16) << 16) + sa * 64 + h * 32, v);
          }
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&go[n % I4T_DONE][0]);
          mbar_arrive(&full_s[n % C::S_RING]);
        }
      }
      n = end;
    }
    if (!ok && lane == 0 && !*abortp) { atomicExch(p.status, I4T_ERR_UNPACK); *abortp = 1; }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
    const int quarter = warp & 3, half = (warp - 4) >> 2;  // lanes of tensor memory; every second 32 rows
    const unsigned lanes = tmem_base + ((unsigned)(quarter * 32) << 16);
    int n = 0, group = 0, items = 0;
    bool ok = true;
    // group g's accumulator is free
    auto free_for = [&](int g) {
      if (lane == 0) mbar_arrive(&go[g / NG % I4T_DONE][g % NG]);
    };
    free_for(0);
    free_for(1);
    unsigned long long sum[BT / 64][16];     // pairs of rows
    for (int w = first; w < n_items && ok; w += step) {
      const I4TItem it = item_of(w);
      if (it.n <= 0) continue;
#pragma unroll
      for (int i = 0; i < BT / 64; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) sum[i][j] = 0;
      for (int c = it.c0; c < it.c1 && ok; ++c, ++n) {
        ok = wait(&full_s[n % C::S_RING], n / C::S_RING & 1);
        if (!ok) break;
        unsigned long long scale[NG];
#pragma unroll
        for (int q = 0; q < NG; ++q) {
          const float v = i4_scale(scales[((n % C::S_RING) * 128 + quarter * 32 + lane) * NG + q]);
          scale[q] = i4t_pack(v, v);
        }
#pragma unroll
        for (int q = 0; q < NG; ++q, ++group) {
          const int buf = group & 1;
          ok = NG == 1 ? wait(&done[n % I4T_DONE], n / I4T_DONE & 1)
                       : wait(&acc_full[buf], group >> 1 & 1);
          if (!ok) break;
          tc_fence_after();
          // (a tile that fills its columns takes them without a branch between)
          if (it.n > BT - 64) {
#pragma unroll
            for (int i = 0; i < BT / 64; ++i)
              i4t_add(sum[i], scale[q], lanes + buf * BT + 64 * i + 32 * half);
          } else {
#pragma unroll
            for (int i = 0; i < BT / 64 - 1; ++i)
              if (64 * i + 32 * half < it.n)
                i4t_add(sum[i], scale[q], lanes + buf * BT + 64 * i + 32 * half);
          }
          tc_fence_before();
          __syncwarp();
          free_for(group + 2);
        }
      }
      if (!ok) break;
      // the item's results, a weight row a lane, to the warps that store them
      ok = wait(&stage_empty, (items & 1) ^ 1);
      if (!ok) break;
      float* mine = stage + quarter * 32 + lane;
#pragma unroll
      for (int i = 0; i < BT / 64; ++i) {
        const int col = 64 * i + 32 * half;
        if (col >= it.n) continue;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          float a, b;
          i4t_unpack(sum[i][j], a, b);
          mine[(col + 2 * j) * 128] = a;
          mine[(col + 2 * j + 1) * 128] = b;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&stage_full);
      ++items;
    }
    if (!ok && lane == 0 && !*abortp) { atomicExch(p.status, I4T_ERR_SUM); *abortp = 1; }
  }
  tc_fence_before();
  __syncthreads();
  // neither block ends while the other can still reach its barriers, tiles or accumulators
  tc_cluster_sync();
  if (warp == 1) tc_dealloc<true>(tmem_base, 512);
}

// The runs' sums in ascending order, and what follows them.
template <bool DUAL>
__global__ void __launch_bounds__(256)
int4_join_kernel(const I4TArgs p) {
  const int f = blockIdx.x * 256 + threadIdx.x;
  if (f >= p.N) return;
  const size_t width = DUAL ? 2 * (size_t)p.N : (size_t)p.N, plane = (size_t)p.rows * width;
  for (size_t r = blockIdx.y; r < (size_t)p.rows; r += gridDim.y) {
    const float* from = p.part + r * width + f;
    float a = 0.f, u = 0.f;
    for (int z = 0; z < p.splits; ++z, from += plane) {
      a += from[0];
      if (DUAL) u += from[p.N];
    }
    if (DUAL) {
      if (p.row_scale) {
        a *= p.row_scale[r];
        u *= p.row_scale[r];
      }
      a = p.wide ? a / (1.0f + expf(-a)) * u : __fdividef(a, 1.0f + __expf(-a)) * u;
    } else if (p.plain) {
      a = p.wide ? ix_act<float>(a, p.plain) : ix_act<bf16>(a, p.plain);
    }
    if (p.wide) ((float*)p.out)[r * p.N + f] = a;
    else ((bf16*)p.out)[r * p.N + f] = __float2bfloat16_rn(a);
  }
}

template <int TERMS, bool DUAL, int BT, int GROUP>
static int i4t_launch(const void* x, int Kp, const I4TArgs& p, int sms, cudaStream_t stream) {
  typedef I4TCfg<TERMS, DUAL, BT, GROUP> C;
  CUtensorMap map;
  const int rc = ix_tensor_map_bf16_2d(&map, x, (long long)TERMS * p.rows, Kp, 64, C::BOX);
  if (rc != IX_OK) return rc;
  const long long tiles = p.offsets ? (p.rows + BT - 1) / BT + (long long)p.E
                                    : (p.rows + p.tile_rows - 1) / p.tile_rows;
  const long long items = tiles * ((p.N + C::F - 1) / C::F) * p.splits;
  if (items > 0x7fffffffLL) return IX_ERR_SIZE;
  auto kern = int4_tc_kernel<TERMS, DUAL, BT, GROUP>;
  static unsigned done = 0;
  const cudaError_t e = i4_allow_smem(kern, C::SMEM, &done);
  if (e != cudaSuccess) return (int)e;
  const int pairs = sms / 2;
  kern<<<2 * (int)(items < pairs ? items : pairs), I4T_THREADS, C::SMEM, stream>>>(map, p);
  if (p.part)
    int4_join_kernel<DUAL><<<dim3((p.N + 255) / 256, p.rows < 16384 ? p.rows : 16384), 256, 0,
                             stream>>>(p);
  return ix_launch_status();
}

static int i4t_sms() {
  static int sms = 0;
  if (sms == 0) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
      sms = 148;
  }
  return sms;
}

// How a call is cut: rows of a tile (one matrix) and runs of K.
struct I4TPlan {
  int tile_rows, splits;
  bool large;
};

static I4TPlan i4t_plan(int rows, int N, int Kp, int E, bool grouped, bool dual, int terms) {
  const int pairs = i4t_sms() / 2, f = dual ? 128 : 256, chunks = (int)i4_chunks(Kp);
  const long long f_tiles = (N + f - 1) / f;
  I4TPlan plan = {0, 1, false};
  double best = -1;
  if (grouped) {
    // the mean rows of an expert, and some for imbalance
    plan.large = terms == 1 && 1.15 * rows / E > 128.0;
    plan.tile_rows = plan.large ? 192 : 128;
    const long long tiles = (rows < E ? rows : E) * f_tiles;
    while (rows <= 4096 && plan.splits < 16 && tiles * plan.splits * 2 <= pairs && chunks / (plan.splits * 2) >= 2)
      plan.splits *= 2;
    // no run begins at or behind the last chunk (20 chunks in runs of 3 are seven runs, not eight)
    const int run = (chunks + plan.splits - 1) / plan.splits;
    plan.splits = (chunks + run - 1) / run;
    return plan;
  }
  const int most = rows > 128 && terms == 1 ? 192 : 128;
  const int cuts0 = (rows + most - 1) / most;
  for (int cuts = cuts0; cuts <= cuts0 + 8; ++cuts) {
    const int per = ((rows + cuts - 1) / cuts + 31) & ~31;
    for (int splits = 1; splits <= (rows > 4096 ? 1 : 16) && splits <= chunks; ++splits) {
      const int run = (chunks + splits - 1) / splits;
      if ((long long)run * (splits - 1) >= chunks) continue;      // an empty last run
      // Least squares over 166 timed cuts of eight products, each in both types (64 to 2,048 rows, 2 to
      // 37 MB of codes): half of them off by 5 % at most, eight in ten by 9 %, and the cut with the
      // lowest estimate was the fastest of those timed for every one of the sixteen.
      const long long items = (long long)((rows + per - 1) / per) * f_tiles * splits;
      const double waves = (double)((items + pairs - 1) / pairs);
      const double chunk = terms == 3 ? 0.55 + 0.0058 * per : 0.40 + 0.0017 * per;
      const double join = (terms == 3 ? 0.55 : 0.34) * 4e-6 * splits * (double)rows * N * (dual ? 2 : 1);
      const double us = waves * (run * chunk + (terms == 3 ? 0.1 : 1.1)) + 6.0 +
                        (splits > 1 ? 3.4 + join : 0.0);
      if (best < 0 || us < 0.98 * best) {
        best = us;
        plan.tile_rows = per;
        plan.splits = splits;
      }
    }
    if (per <= 32) break;
  }
  plan.large = plan.tile_rows > 128;
  return plan;
}

// fp32 entries of scratch that a call of these sizes wants (0: none)
IX_API long long ix_int4_tc_scratch(const I4Weight* w, int rows, int Kp, int grouped, int terms) {
  if (rows <= 0 || w->N <= 0 || Kp <= 0 || w->E <= 0) return 0;
  const I4TPlan plan = i4t_plan(rows, w->N, Kp, w->E, grouped != 0, w->dual != 0, terms);
  return plan.splits > 1 ? (long long)plan.splits * rows * w->N * (w->dual ? 2 : 1) : 0;
}

// x: [rows, Kp] bf16, or [3, rows, Kp] terms of fp32 rows; Kp a multiple of 8 that ends in the weight's
// last chunk.  out: [rows, N] fp32 (wide) or bf16.  offsets == null: one matrix.  part: scratch of the
// size that ix_int4_tc_scratch names, or null where it names none.  status: one int, zero before the
// first call.
IX_API int ix_int4_tc(const I4Weight* w, const void* x, int terms, const int* offsets, void* out,
                      float* part, int wide, int rows, int Kp, const float* row_scale, int plain,
                      int* status, cudaStream_t stream) {
  const int N = w->N, E = w->E, group = w->group, dual = w->dual;
  if ((row_scale && !dual) || (plain && dual)) return IX_ERR_UNSUPPORTED;
  if (rows <= 0) return IX_OK;
  if (N <= 0 || Kp <= 0 || E <= 0 || status == nullptr) return IX_ERR_SIZE;
  if (Kp % 8 != 0 || E > I4T_MAX_EXPERTS || (!offsets && E != 1)) return IX_ERR_UNSUPPORTED;
  if (((uintptr_t)x | (uintptr_t)w->data) & 15) return IX_ERR_ALIGN;
  if (3LL * rows > 0x7fffffffLL || N > 0x3fffff00) return IX_ERR_SIZE;
  const I4TPlan plan = i4t_plan(rows, N, Kp, E, offsets != nullptr, dual != 0, terms);
  if (plan.splits > 1) {
    if (part == nullptr) return IX_ERR_SIZE;
  } else {
    part = nullptr;
  }
  const int chunks = (int)i4_chunks(Kp);
  const I4TArgs p = {offsets, w->data, out, part, wide, row_scale, plain, rows, N,
                     (int)i4_strips(N), chunks, E, plan.tile_rows, plan.splits,
                     (chunks + plan.splits - 1) / plan.splits, rows, status};
  const int sms = i4t_sms();
#define I4T_BT(T, D, B)                                                       \
  do {                                                                        \
    if (group == 128) return i4t_launch<T, D, B, 128>(x, Kp, p, sms, stream); \
    if (group == 64) return i4t_launch<T, D, B, 64>(x, Kp, p, sms, stream);   \
    if (group == 32) return i4t_launch<T, D, B, 32>(x, Kp, p, sms, stream);   \
    return IX_ERR_UNSUPPORTED;                                                \
  } while (0)
  if (terms == 1) {
    if (dual) {
      if (plan.large) I4T_BT(1, true, 192);
      I4T_BT(1, true, 128);
    }
    if (plan.large) I4T_BT(1, false, 192);
    I4T_BT(1, false, 128);
  }
  if (terms == 3) {
    if (dual) I4T_BT(3, true, 128);
    I4T_BT(3, false, 128);
  }
  return IX_ERR_UNSUPPORTED;
}
