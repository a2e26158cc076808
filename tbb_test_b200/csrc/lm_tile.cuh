// Tiles of matrix products for the operators around a language model's layers (xent.cu, muon.cu): a persistent kernel of
// CTA pairs on the tensor cores whose operator Op says which tiles there are and what happens to their elements.
//
// A pair (a cluster of two CTAs on neighbouring SMs) computes 256 x BN of C = A B' with tcgen05.mma.cta_group::2: CTA r holds
// rows [128 r, 128 r + 128) of A's slab and the r-th half of B's, the leader issues every MMA, and each CTA's tensor
// memory receives its own 128 rows. Operands are 16-bit, either with K contiguous or with M/N contiguous, and come by TMA in
// slabs of 64 k. Two accumulators take turns, so that one tile's elements are worked on while the next is summed.
//
// Two forms:
//   plain   bf16 operands, BN = 256, six stages of 32 KB
//   split   every operand is a pair of fp16 matrices x = hi + 2^-11 lo, 22 bits together; hi hi' goes to one
//           accumulator, hi lo' + lo hi' to another behind it (lo lo' is 2^-22 of the product and left out). BN = 128, four
//           stages of 48 KB. Three MMAs at the full fp16 rate give what three tf32 MMAs give at half of it, provided the
//           caller scales its matrices into fp16's range; with lo as large as hi, 22 bits are kept down to magnitudes of
//           2^-13 and what lies below is held to 2^-36. The tensor core truncates when it adds to an
//           accumulator (about 2e-8 of the sum each time, and always towards zero), so a sum is handed over every
//           Op::SUM k-blocks and added up in fp32 registers, rounded to nearest.
//
// Where there are no more tiles than SMs, single CTAs (ONE) with tcgen05.mma.cta_group::1 and tiles of a quarter of the size take less
// time: more SMs have work, and a call's products, which wait for one another, start and end sooner without a cluster (15 products of 256 x
// 256 x 256: 144 -> 99 us; of 1024 x 1024 x 1024 249 -> 184). With more tiles pairs do, which read half of B's slab each: 1536 x 1536 in
// two rounds of single CTAs 393 us, in one of pairs 324. The plain form's single CTAs take 128 x 128.
//
// Warps: 0 loads, 1 allocates tensor memory and (in the leader) issues, the others work on elements: those of a lane quarter share
// its columns. There are 16 of them in the split form, where small matrices wait for nothing else as long (256 x 256 in pairs: 154 ->
// 144 us), and 8 in the plain one, which the power limit binds (with 16 and five stages 8192 x 2048 x 65536 took 6.2 ms for 6.0).
#pragma once

#include <cuda_fp16.h>

#include <atomic>

#include "lm.cuh"
#include "tcgen05.cuh"

namespace b2 {
namespace {

constexpr int TILE_M = 256, TILE_K = 64;
constexpr float LO_UP = 2048.f;  // lo = 2^11 (x - hi)
constexpr uint32_t ACC_COLS = 256;  // tensor-memory columns of an accumulator stage
constexpr int TILE_MAX_STAGES = 6;

// CTAs in which a wait gave up, and the number of the role that was first to; never cleared (b2_lm_sync reports what is new).
struct TileReport {
  unsigned int count, role;
};
__device__ TileReport tile_report;

template <bool SPLIT_, bool ONE_ = false>
struct TileForm {
  static constexpr bool SPLIT = SPLIT_, ONE = ONE_;
  static constexpr int CTAS = ONE ? 1 : 2;       // that share a tile
  static constexpr int M = CTAS * 128;
  static constexpr int BN = (SPLIT ? 64 : 128) * CTAS;
  static constexpr int B_ROWS = BN / CTAS;       // of B's slab, in a CTA
  static constexpr int STAGES = SPLIT ? 4 : 6;
  static constexpr uint32_t A_BYTES = 128 * 128, B_BYTES = B_ROWS * 128;
  static constexpr uint32_t SLABS = (A_BYTES + B_BYTES) * (SPLIT ? 2 : 1);  // of a stage
  static constexpr int WARPS = SPLIT ? 16 : 8;   // on elements
  static constexpr int PARTS = WARPS / 4;        // warps that share a row's columns
  static constexpr int COLS = BN / PARTS;        // columns of a warp
  static constexpr int CHUNK = SPLIT ? 16 : 32;  // columns that it works on at a time
  static constexpr int STAGE = 32 * CHUNK * 4;   // bytes of its buffer for that
  static constexpr int THREADS = 64 + 32 * WARPS;
  static constexpr int BOUND = SPLIT ? 640 : THREADS;  // registers are handed out as if 18 warps were 20
  static constexpr size_t SMEM = 1024 + STAGES * SLABS + WARPS * STAGE;
};

struct TileMaps {
  CUtensorMap a, a_lo, b, b_lo;
  CUtensorMap c;  // of a result that leaves by TMA stores, where the operator has one
};
struct TileLayout {
  int a_form, b_form;  // SlabForm
  uint32_t a_lbo, a_kstep, b_lbo, b_kstep;
  uint32_t idesc;
};
// One tile: rows and columns of C from m0, n0 on; where its slabs lie in A and B along M/N and along K.
struct Tile {
  int m0, n0;
  int a_mn, b_mn, a_k, b_k;
  int kblocks;  // 0: nothing to sum, the elements are zeros
  int z;        // the operator's own
};

// Finished columns of this lane's row.
__device__ __forceinline__ void tile_read(uint32_t from, uint32_t (&r)[32]) { tmem_ld32(from, r); }
__device__ __forceinline__ void tile_read(uint32_t from, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(from)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tile_add16(uint32_t from, float* sum) {
  uint32_t r[16];
  tile_read(from, r);
#pragma unroll
  for (int j = 0; j < 16; ++j) sum[j] += __uint_as_float(r[j]);
}
template <bool PAIR>
__device__ __forceinline__ void tile_commit(uint32_t bar) {
  if (PAIR) tc_commit_pair(bar);
  else tc_commit(bar);
}
// All 512 columns of tensor memory, by one whole warp (of each CTA of a pair).
template <bool PAIR>
__device__ __forceinline__ void tmem_take(uint32_t* base) {
#define B2_TAKE(GROUP)                                                                                                             \
  asm volatile("tcgen05.alloc." GROUP ".sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(base)), "r"(512u) : "memory"); \
  asm volatile("tcgen05.relinquish_alloc_permit." GROUP ".sync.aligned;" ::: "memory")
  if (PAIR) {
    B2_TAKE("cta_group::2");
  } else {
    B2_TAKE("cta_group::1");
  }
#undef B2_TAKE
}
template <bool PAIR>
__device__ __forceinline__ void tmem_give(uint32_t base) {
  if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(512u) : "memory");
  else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(512u) : "memory");
}

// Op: struct Params; typedef TileForm<...> Form; Op(const Params&, const TileMaps&); int tiles(); Tile tile(int t);
//     and in the element warps: void begin(const Tile&, int row, int col, int lane) before the sums are there, for the warp's
//     first row and column; void chunk(const Tile&, int row0, int col0, float (&v)[CHUNK], uint8_t* stage, int lane) for CHUNK columns of
//     rows row0 + lane; void end(const Tile&, int row, int part) for the thread's row and its warp's part of the columns;
//     static constexpr bool STORES: it issues TMA stores from `stage`; static constexpr bool LONG: sums are handed over every SUM
//     (static constexpr int) k-blocks, which the split form always does; chunks have 16 columns then; static constexpr bool INFINITE: sums of
//     infinite elements are infinite by their signs and not NaN (split form; for the update of one small matrix it would take 1.5 us of 98).
template <class Op>
__global__ void __launch_bounds__(Op::Form::BOUND, 1) tile_kernel(const __grid_constant__ TileMaps maps, const __grid_constant__ TileLayout L,
                                                                const __grid_constant__ typename Op::Params params) {
  typedef typename Op::Form F;
  constexpr bool SPLIT = F::SPLIT, PAIR = !F::ONE;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[TILE_MAX_STAGES];
  __shared__ __align__(8) uint64_t empty_bar[TILE_MAX_STAGES];
  __shared__ __align__(8) uint64_t acc_full_bar[2];
  __shared__ __align__(8) uint64_t acc_empty_bar[2];
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s;

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
  const int first_tile = blockIdx.x / F::CTAS, every = gridDim.x / F::CTAS;
  volatile int* abort_flag = &abort_s;

  if (threadIdx.x == 0) {
    abort_s = 0;
    for (int s = 0; s < F::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full_bar[a], 1);
      mbar_init(&acc_empty_bar[a], F::CTAS * F::WARPS);  // the element warps of all
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.a) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.b) : "memory");
  }
  if (warp == 1) {
    tmem_take<PAIR>(&tmem_base_s);
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_s;
  after_previous();
  let_next_start();
  Op op(params, maps);
  const int tiles = op.tiles();

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t full0 = map_to_cta(smem_u32(full_bar), 0), empty0 = smem_u32(empty_bar), ring0 = smem_u32(smem);
      for (int t = first_tile; t < tiles && ok; t += every) {
        const Tile tile = op.tile(t);
        const int am = tile.a_mn + (int)rank * 128, bn = tile.b_mn + (int)rank * F::B_ROWS;
        for (int kb = 0; kb < tile.kblocks; ++kb) {
          if (!mbar_wait(empty0 + 8u * stage, phase ^ 1, abort_flag, &tile_report.role, 1u)) { ok = false; break; }
          const uint32_t s0 = ring0 + (uint32_t)stage * F::SLABS;
          if (rank == 0) mbar_expect_tx(smem_u32(full_bar) + 8u * stage, F::CTAS * F::SLABS);  // both CTAs' bytes
          const uint32_t full = full0 + 8u * stage;
          const int ka = tile.a_k + kb * TILE_K, kbb = tile.b_k + kb * TILE_K;
          load_slab<PAIR>(&maps.a, full, s0, L.a_form, ka, am, 2, TILE_K * 128, 6);
          const uint32_t sb = s0 + F::A_BYTES * (SPLIT ? 2 : 1);
          load_slab<PAIR>(&maps.b, full, sb, L.b_form, kbb, bn, F::B_ROWS / 64, TILE_K * 128, 6);
          if (SPLIT) {
            load_slab<PAIR>(&maps.a_lo, full, s0 + F::A_BYTES, L.a_form, ka, am, 2, TILE_K * 128, 6);
            load_slab<PAIR>(&maps.b_lo, full, sb + F::B_BYTES, L.b_form, kbb, bn, F::B_ROWS / 64, TILE_K * 128, 6);
          }
          if (++stage == F::STAGES) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      const uint64_t a_tmpl = make_smem_desc(smem_u32(smem), L.a_lbo, 1024, 2);
      const uint64_t b_tmpl = make_smem_desc(smem_u32(smem) + F::A_BYTES * (SPLIT ? 2 : 1), L.b_lbo, 1024, 2);
      const uint32_t a_step = L.a_kstep >> 4, b_step = L.b_kstep >> 4, idesc = L.idesc;
      const uint32_t full0 = smem_u32(full_bar), empty0 = smem_u32(empty_bar), acc_full0 = smem_u32(acc_full_bar);
      for (int t = first_tile; t < tiles && ok; t += every) {
        const int kblocks = op.tile(t).kblocks;
        for (int kb = 0; kb < kblocks; ++kb) {
          const bool first = kb == 0 || (Op::LONG && kb % Op::SUM == 0);
          if (first) {
            if (!mbar_wait(&acc_empty_bar[acc], acc_phase ^ 1, abort_flag, &tile_report.role, 2u)) { ok = false; break; }
            tc_fence_after();
          }
          if (!mbar_wait(full0 + 8u * stage, phase, abort_flag, &tile_report.role, 3u)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d = tmem_base + (uint32_t)acc * ACC_COLS;
          const uint32_t off = ((uint32_t)stage * F::SLABS) >> 4;
#pragma unroll
          for (int ks = 0; ks < TILE_K / 16; ++ks) {
            const uint64_t ad = a_tmpl + off + (uint64_t)(ks * a_step), bd = b_tmpl + off + (uint64_t)(ks * b_step);
            const uint32_t go = first && ks == 0 ? 0u : 1u;
            if (SPLIT && !PAIR) {
              // B's halves lie behind one another, as their results do: one MMA of twice the columns reads hi once for both. Shared memory is
              // what bounds these tiles (1024 x 1024: 185 -> 164 us per update). In a pair each CTA has half of either.
              mma_issue<false, PAIR>(d, ad, bd, idesc + ((uint32_t)(F::BN >> 3) << 17), go);
              mma_issue<false, PAIR>(d + F::BN, ad + (F::A_BYTES >> 4), bd, idesc, 1u);
              continue;
            }
            mma_issue<false, PAIR>(d, ad, bd, idesc, go);
            if (SPLIT) {
              mma_issue<false, PAIR>(d + F::BN, ad, bd + (F::B_BYTES >> 4), idesc, go);
              mma_issue<false, PAIR>(d + F::BN, ad + (F::A_BYTES >> 4), bd, idesc, 1u);
            }
          }
          tile_commit<PAIR>(empty0 + 8u * stage);
          if (++stage == F::STAGES) { stage = 0; phase ^= 1; }
          if (kb + 1 == kblocks || (Op::LONG && (kb + 1) % Op::SUM == 0)) {
            tile_commit<PAIR>(acc_full0 + 8u * acc);
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1;
          }
        }
      }
    }
  } else {
    const int q = warp & 3, part = (warp - 2) >> 2;
    constexpr int CHUNK = F::CHUNK;
    uint8_t* stage = smem + F::STAGES * F::SLABS + (warp - 2) * F::STAGE;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int t = first_tile; t < tiles && ok; t += every) {
      const Tile tile = op.tile(t);
      const int row0 = tile.m0 + (int)rank * 128 + q * 32, col0 = tile.n0 + part * F::COLS;
      const uint32_t place = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(part * F::COLS);
      op.begin(tile, row0, col0, lane);
      if constexpr (SPLIT) {
        float sum[F::COLS];
        if (tile.kblocks == 0) {
#pragma unroll
          for (int c = 0; c < F::COLS; ++c) sum[c] = 0.f;
        }
        for (int kb = 0; kb < tile.kblocks; kb += Op::SUM) {
          if (!mbar_wait(&acc_full_bar[acc], acc_phase, abort_flag, &tile_report.role, 4u)) { ok = false; break; }
          tc_fence_after();
          const uint32_t from = place + (uint32_t)acc * ACC_COLS;
          uint32_t r[F::COLS], x[F::COLS];
          tile_read(from, r);
          tile_read(from + F::BN, x);
#pragma unroll
          for (int j = 0; j < F::COLS; ++j) {
            const float main = __uint_as_float(r[j]);
            // an infinite element's low half is not a number: the high halves alone say what its sums are
            const float v = !Op::INFINITE || fabsf(main) < INFINITY ? fmaf(__uint_as_float(x[j]), 1.f / LO_UP, main) : main;
            sum[j] = kb == 0 ? v : sum[j] + v;
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_leader(map_to_cta(smem_u32(&acc_empty_bar[acc]), 0));
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1;
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < F::COLS; c += CHUNK) {
          float v[CHUNK];
#pragma unroll
          for (int j = 0; j < CHUNK; ++j) v[j] = sum[c + j];
          op.chunk(tile, row0, col0 + c, v, stage, lane);
        }
        op.end(tile, row0 + lane, part);
      } else if constexpr (Op::LONG) {
        // sums of SUM k-blocks at a time are added up in registers; the last ones go straight on, 16 columns at a time
        float sum[F::COLS];
#pragma unroll
        for (int c = 0; c < F::COLS; ++c) sum[c] = 0.f;
        for (int kb = 0; kb < tile.kblocks; kb += Op::SUM) {
          if (!mbar_wait(&acc_full_bar[acc], acc_phase, abort_flag, &tile_report.role, 4u)) { ok = false; break; }
          tc_fence_after();
          const uint32_t from = place + (uint32_t)acc * ACC_COLS;
          if (kb + Op::SUM < tile.kblocks) {
#pragma unroll
            for (int c = 0; c < F::COLS; c += 16) tile_add16(from + c, sum + c);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_leader(map_to_cta(smem_u32(&acc_empty_bar[acc]), 0));
          } else {
#pragma unroll
            for (int c = 0; c < F::COLS; c += 16) {
              tile_add16(from + c, sum + c);
              if (c + 16 == F::COLS) {  // all read: the next tile may be summed here
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_leader(map_to_cta(smem_u32(&acc_empty_bar[acc]), 0));
              }
              float v[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] = sum[c + j];
              op.chunk(tile, row0, col0 + c, v, stage, lane);
            }
          }
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1;
        }
        if (!ok) break;
        op.end(tile, row0 + lane, part);
      } else {
        const bool summed = tile.kblocks > 0;
        if (summed) {
          if (!mbar_wait(&acc_full_bar[acc], acc_phase, abort_flag, &tile_report.role, 4u)) break;
          tc_fence_after();
        }
        const uint32_t from = place + (uint32_t)acc * ACC_COLS;
#pragma unroll 1
        for (int c = 0; c < F::COLS; c += CHUNK) {
          uint32_t r[32];
          if (summed) {
            tmem_ld32(from + c, r);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = 0u;
          }
          if (summed && c + CHUNK == F::COLS) {  // all read: the next tile may be summed here
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_leader(map_to_cta(smem_u32(&acc_empty_bar[acc]), 0));
          }
          float v[CHUNK];
#pragma unroll
          for (int j = 0; j < CHUNK; ++j) v[j] = __uint_as_float(r[j]);
          op.chunk(tile, row0, col0 + c, v, stage, lane);
        }
        op.end(tile, row0 + lane, part);
        if (summed) {
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1;
        }
      }
    }
    if (Op::STORES && lane == 0) bulk_wait_all();  // the buffers must outlive the stores that read them
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (abort_s) {  // whichever role gave up: copies and MMAs in flight get a bounded time to end before their memory is given back
    if (threadIdx.x == 0) {
      atomicAdd(&tile_report.count, 1u);
      const unsigned long long t0 = globaltimer();
      while (globaltimer() - t0 < 2000000ull) __nanosleep(1000);
    }
    __syncthreads();
  }
  if (PAIR) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_give<PAIR>(tmem_base);
  }
}

__device__ __forceinline__ void split_half(float v, __half& hi, __half& lo) {
  hi = __float2half_rn(v);
  lo = __float2half_rn((v - __half2float(hi)) * LO_UP);
}

__device__ __forceinline__ void store_pair(__half* hi, __half* lo, long long at, const float4& x) {
  const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);  // two at a time
  const float2 f = __half22float2(a), g = __half22float2(b);
  const __half2 c = __floats2half2_rn((x.x - f.x) * LO_UP, (x.y - f.y) * LO_UP), d = __floats2half2_rn((x.z - g.x) * LO_UP, (x.w - g.y) * LO_UP);
  *reinterpret_cast<uint2*>(hi + at) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  *reinterpret_cast<uint2*>(lo + at) = make_uint2(*reinterpret_cast<const uint32_t*>(&c), *reinterpret_cast<const uint32_t*>(&d));
}
struct Pair4 {  // four neighbouring elements as they lie in memory
  uint2 hi, lo;
};
__device__ __forceinline__ Pair4 load_pair(const __half* hi, const __half* lo, long long at) {
  return Pair4{*reinterpret_cast<const uint2*>(hi + at), *reinterpret_cast<const uint2*>(lo + at)};
}
__device__ __forceinline__ float4 pair_value(const Pair4& p) {
  const __half2 *a = reinterpret_cast<const __half2*>(&p.hi), *b = reinterpret_cast<const __half2*>(&p.lo);
  const float2 a0 = __half22float2(a[0]), a1 = __half22float2(a[1]), b0 = __half22float2(b[0]), b1 = __half22float2(b[1]);
  return make_float4(fmaf(b0.x, 1.f / LO_UP, a0.x), fmaf(b0.y, 1.f / LO_UP, a0.y), fmaf(b1.x, 1.f / LO_UP, a1.x), fmaf(b1.y, 1.f / LO_UP, a1.y));
}

// A chunk of W columns through shared memory, so that a warp's accesses to global memory cover whole rows: W / 4 lanes take four
// neighbouring columns of a row each. Quad i of a lane is row quad_row<W>(i, lane), columns quad_col<W>(lane) and up, of the chunk; f(i,
// row, col, v) gets it. 16-byte pieces are swizzled so that there are no conflicts either way.
template <int W>
__device__ __forceinline__ int quad_row(int i, int lane) { return i * (128 / W) + lane / (W / 4); }
template <int W>
__device__ __forceinline__ int quad_col(int lane) { return lane % (W / 4) * 4; }
template <int W>
__device__ __forceinline__ int quad_slot(int row, int piece) { return row * W * 4 + ((piece ^ (W == 32 ? row & 7 : row >> 1 & 3)) << 4); }
template <int W, class Fn>
__device__ __forceinline__ void by_rows(int row0, int col0, const float (&v)[W], uint8_t* stage, int lane, Fn f) {
#pragma unroll
  for (int j = 0; j < W / 4; ++j)
    *reinterpret_cast<float4*>(stage + quad_slot<W>(lane, j)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  __syncwarp();
  const int c = quad_col<W>(lane);
#pragma unroll
  for (int i = 0; i < W / 4; ++i) {
    const int r = quad_row<W>(i, lane);
    f(i, row0 + r, col0 + c, *reinterpret_cast<const float4*>(stage + quad_slot<W>(r, c / 4)));
  }
  __syncwarp();
}
// Quads as by_rows hands them out, transposed: f(col, row, v) gets four neighbouring rows of a column. Rows of a column lie
// at r ^ 8 (c / 4), for 16 columns.
template <class Fn>
__device__ __forceinline__ void by_columns(int row0, int col0, const float4 (&x)[4], uint8_t* stage, int lane, Fn f) {
  float* t = reinterpret_cast<float*>(stage);
  const int c0 = quad_col<16>(lane), turn = (c0 >> 2) * 8;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = quad_row<16>(i, lane) ^ turn;
    t[c0 * 32 + r] = x[i].x;
    t[(c0 + 1) * 32 + r] = x[i].y;
    t[(c0 + 2) * 32 + r] = x[i].z;
    t[(c0 + 3) * 32 + r] = x[i].w;
  }
  __syncwarp();
  const int r = (lane & 7) * 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = 4 * i + (lane >> 3);
    f(col0 + c, row0 + r, *reinterpret_cast<const float4*>(t + c * 32 + (r ^ (i * 8))));
  }
  __syncwarp();
}
// 2 N columns (16 or 32) of 16-bit elements, from column `col` of the map's matrix on, into their place in a buffer of 64 columns, in
// the swizzle that TMA stores undo; with the last ones the buffer leaves. The first ones wait until the store before has
// read the buffer.
template <int N>
__device__ __forceinline__ void store_half_words(const CUtensorMap* map, const uint32_t (&w)[N], int row, int col, uint8_t* stage, int lane) {
  const int part = (col & 63) / (2 * N);
  if (part == 0) {
    if (lane == 0) bulk_wait_read<0>();
    __syncwarp();
  }
#pragma unroll
  for (int j = 0; j < N / 4; ++j)
    *reinterpret_cast<uint4*>(stage + lane * 128 + (((part * (N / 4) + j) ^ (lane & 7)) << 4)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
  if (part == 32 / N - 1) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_2d(map, stage, col & ~63, row);
      bulk_commit();
    }
  }
}

// ------------------------------------------------------------------ host side

// An operand in device memory: `mn` rows (or, with mn_contiguous, columns) by k elements of 16 bits, ld between rows.
struct TileOperand {
  const void *hi, *lo;
  long long mn, k, ld;
  bool mn_contiguous;
};

template <class F>
bool tile_maps(const TileOperand& a, const TileOperand& b, bool bf16, TileMaps* maps, TileLayout* L) {
  auto one = [](const TileOperand& o, const void* p, int rows, int* form, CUtensorMap* m) {
    if (!o.mn_contiguous) {
      *form = SLAB_K;
      return make_map(m, p, 2, o.k, o.mn, o.ld, TILE_K, rows, 0);
    }
    if (o.mn % 64 == 0 && make_map_columns(m, p, 2, o.mn, o.k, o.ld, TILE_K, rows / 64, 0)) {
      *form = SLAB_MN3;
      return true;
    }
    *form = SLAB_MN2;
    return make_map(m, p, 2, o.mn, o.k, o.ld, 64, TILE_K, 0);
  };
  bool ok = one(a, a.hi, 128, &L->a_form, &maps->a) && one(b, b.hi, F::B_ROWS, &L->b_form, &maps->b);
  if (F::SPLIT) {
    ok = ok && one(a, a.lo, 128, &L->a_form, &maps->a_lo) && one(b, b.lo, F::B_ROWS, &L->b_form, &maps->b_lo);
  } else {
    maps->a_lo = maps->a;
    maps->b_lo = maps->b;
  }
  L->a_lbo = a.mn_contiguous ? TILE_K * 128 : 16;
  L->b_lbo = b.mn_contiguous ? TILE_K * 128 : 16;
  L->a_kstep = a.mn_contiguous ? 16 * 128 : 32;
  L->b_kstep = b.mn_contiguous ? 16 * 128 : 32;
  const uint32_t fmt = bf16 ? 1u : 0u;  // bf16 : f16
  L->idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)a.mn_contiguous << 15) | ((uint32_t)b.mn_contiguous << 16) |
             ((uint32_t)(F::BN >> 3) << 17) | ((uint32_t)(F::M >> 4) << 24);
  return ok;
}

// Whether single CTAs take less time than pairs: what shared memory takes to be filled and read for a k-block of a tile, times k-blocks and
// rounds of tiles, and 3 us for a launch of clusters, all in clocks.
template <bool SPLIT>
bool single_ctas(long long rounds_one, long long kblocks_one, long long rounds_pairs, long long kblocks_pairs) {
  return rounds_one * kblocks_one * (SPLIT ? 832 : 512) <= rounds_pairs * kblocks_pairs * (SPLIT ? 960 : 512) + 6000;
}

// A row-major matrix of 16-bit elements that store_half_words writes to.
struct TileResult {
  void* p;
  long long rows, cols, ld;
};

// most_tiles: an upper bound on the tiles that the kernel will find.
template <class Op>
int tile_launch(const char* who, const TileOperand& a, const TileOperand& b, const TileResult* c, const typename Op::Params& p, bool bf16,
                long long most_tiles, int sms, Chain& chain) {
  typedef typename Op::Form F;
  if (most_tiles <= 0) return B2_OK;
  TileMaps maps;
  TileLayout L;
  bool ok = tile_maps<F>(a, b, bf16, &maps, &L);
  if (c) ok = ok && make_map(&maps.c, c->p, 2, c->cols, c->rows, c->ld, 64, 32, 0);
  else maps.c = maps.a;
  if (!ok) return call_error(B2_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed", who);
  const size_t smem = F::SMEM;
  static std::atomic<unsigned long long> raised{0};  // the kernel's shared-memory limit: one bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !(raised.load() >> dev & 1))) {
    e = cudaFuncSetAttribute(tile_kernel<Op>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess && dev < 64) raised.fetch_or(1ull << dev);
  }
  if (e != cudaSuccess) return launch_error(e, who);
  const int most = sms / F::CTAS;
  const unsigned int grid = F::CTAS * (unsigned int)(most_tiles < most ? most_tiles : most);
  chain.launch(tile_kernel<Op>, dim3(grid), F::THREADS, smem, F::ONE ? 0 : 2, maps, L, p);
  return launch_error(chain.err, who);
}

// This file's report, behind the stream's work, which is waited for.
inline cudaError_t tile_report_read(TileReport* r, cudaStream_t s) {
  cudaError_t e = cudaMemcpyFromSymbolAsync(r, tile_report, sizeof *r, 0, cudaMemcpyDeviceToHost, s);
  return e == cudaSuccess ? cudaStreamSynchronize(s) : e;
}

}  // namespace
}  // namespace b2
