// Softmax cross entropy behind a linear layer as wide as a vocabulary, with its gradients, without keeping more than 512 MB of logits and 640 MB
// of their gradients (from 327 680 rows in bf16 and 163 840 in fp32 on, 1024 columns of the latter):
//
//   x_iv = h_i . w_v      l_i = log sum_v exp(x_iv) - x_i,t_i      d_iv = exp(x_iv) / sum_u exp(x_iu) - [v = t_i]
//   dh_i = scale sum_v d_iv w_v      dw_v = scale sum_i d_iv h_i
//
// Work: 2 R V F operations for the losses and 6 R V F with gradients; 8 R V F in this form where the logits are
// computed a second time when their row's maximum and sum are known, instead of R x V of them being kept (keeps_logits).
// It is bound by the tensor cores (tile kernels of lm_tile.cuh) unless R is small, when reading w is what it takes.
//
//   1. Rows without a target are left out: the others' numbers are listed in order, their h copied one after another (fp32: as pairs,
//      and w too). So such a row costs nothing, and nothing in it (a NaN, say) reaches dw.
//   2. Logits, a tile at a time; each row's maximum and sum over a warp's columns go to a list.
//   3. The lists give each row's maximum and sum, and the loss.
//   4. Per piece of the vocabulary: d from logits that are kept or computed again to a buffer of R x piece; dh += d w; dw of the
//      piece = d' h.
// A few rows with few tiles of long sums: the logits go out in parts of the k range, and 3 and d are one kernel with a block per row.
//
// Precision: bf16 matrices are multiplied as they are, with fp32 sums, which are handed over and joined where they would be long; d is rounded
// to bf16 once, as the gradients are in the end: gradients are 1.9e-3 off in norm, 1.7e-3 of it by their own rounding. fp32 matrices are
// split into fp16 pairs behind a power of two that brings the largest element to 2^14: 22 bits of an element down to 2^-27 of
// the largest, and nothing finer than 2^-50 of it; d the same, with 1 for the largest. Infinite elements take no part in that: their
// logits are infinite by the signs, or NaN, as in bf16. Maxima, sums and the losses are fp32.
#include <type_traits>

#include "lm_tile.cuh"

namespace b2 {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// k-blocks per hand-over of the split form's sums: with 16 dw of 1024 rows is 1.1e-6 off (relative), with 8 0.8e-6, in the same time
constexpr int XENT_SUM = 8;
constexpr int D_EXP = 14;  // fp32 matrices: d is kept as 2^14 (p - [v = t])

struct Meta {
  unsigned int rows;  // with a target
  unsigned int max_h, max_w;  // bits of the largest magnitude (fp32 matrices)
};

__device__ __forceinline__ float ex2(float x) {  // 2^x, two units in the last place
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Power of two that brings a matrix whose largest finite magnitude has these bits below 2^15: its exponent, 0 for zeros.
__device__ __forceinline__ int up_exp(unsigned int max_bits) {
  return max_bits == 0 ? 0 : min(14 - ((int)(max_bits >> 23) - 127), 100);
}
__device__ __forceinline__ unsigned int finite_bits(unsigned int v) {  // of the magnitude; what is not finite stays so under any scale
  v &= 0x7FFFFFFFu;
  return v < 0x7F800000u ? v : 0u;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// ------------------------------------------------------------------ rows with a target

constexpr int FRONT_THREADS = 512;
struct Front {
  const void* targets;
  int wide, rows, share, vocab, width, pitch;
  const unsigned int* counts;  // rows with a target in each block's share, where a kernel before has counted them
  Meta* meta;
  int *row_of, *slot_of, *target;
  float* row_loss;
  const void *h, *w;
  long long ldh, ldw;
  int blocks_h, blocks_w;  // blocks on h, and behind them on w
  uint16_t *h_hi, *h_lo, *w_hi, *w_lo;
  unsigned int* most;  // fp32: each block's largest magnitude
};

__device__ __forceinline__ unsigned int block_sum(unsigned int mine, unsigned int* warp_sum) {  // over all threads; the warps' sums stay in warp_sum
  const int lane = threadIdx.x & 31;
  mine = __reduce_add_sync(0xFFFFFFFFu, mine);
  __syncthreads();
  if (lane == 0) warp_sum[threadIdx.x >> 5] = mine;
  __syncthreads();
  return __reduce_add_sync(0xFFFFFFFFu, lane < FRONT_THREADS / 32 ? warp_sum[lane] : 0u);
}
__device__ __forceinline__ unsigned int block_max(unsigned int mine, unsigned int* warp_max) {
  const int lane = threadIdx.x & 31;
  mine = __reduce_max_sync(0xFFFFFFFFu, mine);
  __syncthreads();
  if (lane == 0) warp_max[threadIdx.x >> 5] = mine;
  __syncthreads();
  return __reduce_max_sync(0xFFFFFFFFu, lane < FRONT_THREADS / 32 ? warp_max[lane] : 0u);
}
// Threads of a row of n pieces, as a shift: the power of two below, up to the whole block.
__host__ __device__ __forceinline__ int row_shift(int n) {
  int shift = 0;
  while (shift < 9 && 2 << shift <= n) ++shift;
  return shift;
}
static_assert(FRONT_THREADS == 1 << 9, "a whole block");

// An element as a pair, behind the scale. One that is too small for the high half gets the smallest number there, of its sign, and the rest in
// the low one, whose steps are the same as they would be otherwise: times an infinity it is then not 0, which would make it NaN.
__device__ __forceinline__ void split_scaled(float v, float up, __half& hi, __half& lo) {
  const float x = v * up;
  hi = __float2half_rn(x);
  if (__half2float(hi) == 0.f && v != 0.f) hi = __ushort_as_half(v < 0.f ? 0x8001 : 0x0001);
  lo = __float2half_rn((x - __half2float(hi)) * LO_UP);
}

// Rows first + k of a copy, for a block's share of the k below n: row of(k) of x, zeros behind `width` up to `pitch`, or zeros alone where
// of(k) is negative.
template <typename T, class Of>
__device__ __forceinline__ void copy_rows(const T* __restrict__ x, long long ld, int n, int block, int blocks, int width, int pitch, float up,
                                          uint16_t* __restrict__ hi, uint16_t* __restrict__ lo, long long first, Of of) {
  constexpr bool SPLIT = sizeof(T) == 4;
  const bool vec = ld % (16 / sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  const int shift = row_shift(pitch / 8), lanes = 1 << shift, at_once = FRONT_THREADS >> shift;
  for (int k = block * at_once + (threadIdx.x >> shift); k < n; k += blocks * at_once) {
    const int from = of(k);
    const T* src = x + (from < 0 ? 0 : from * ld);
    const long long to = (first + k) * pitch;
#pragma unroll 4
    for (int c = (threadIdx.x & (lanes - 1)) * 8; c < pitch; c += 8 * lanes) {
      T v[8];
      if (from >= 0 && vec && c + 8 <= width) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(v)[i] = __ldg(reinterpret_cast<const uint4*>(src + c) + i);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = from >= 0 && c + i < width ? src[c + i] : (T)0.f;
      }
      if (SPLIT) {
        __half a[8], b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) split_scaled((float)v[i], up, a[i], b[i]);
        *reinterpret_cast<uint4*>(hi + to + c) = *reinterpret_cast<const uint4*>(a);
        *reinterpret_cast<uint4*>(lo + to + c) = *reinterpret_cast<const uint4*>(b);
      } else {
        *reinterpret_cast<uint4*>(hi + to + c) = *reinterpret_cast<const uint4*>(v);
      }
    }
  }
}
// Largest finite magnitude of the same rows.
template <class Of>
__device__ __forceinline__ unsigned int max_rows(const float* __restrict__ x, long long ld, int n, int block, int blocks, int width, Of of) {
  const bool vec = width % 4 == 0 && ld % 4 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  const int per_row = vec ? width / 4 : width, shift = row_shift(per_row), lanes = 1 << shift;
  const int at_once = FRONT_THREADS >> shift;
  unsigned int most = 0;
  for (int k = block * at_once + (threadIdx.x >> shift); k < n; k += blocks * at_once) {
    const float* row = x + of(k) * ld;
#pragma unroll 4
    for (int c = threadIdx.x & (lanes - 1); c < per_row; c += lanes) {
      if (vec) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(row) + c);
        most = max(most, max(max(finite_bits(v.x), finite_bits(v.y)), max(finite_bits(v.z), finite_bits(v.w))));
      } else {
        most = max(most, finite_bits(__float_as_uint(__ldg(row + c))));
      }
    }
  }
  return most;
}

// Rows of the copy of h: whole k-blocks of the product that sums over them, which the rows behind the listed ones fill with zeros.
__device__ __forceinline__ int whole_rows(unsigned int rows) { return max(1, (int)((rows + TILE_K - 1) / TILE_K)) * TILE_K; }

// Rows with a target in each block's share of front_kernel, for calls where every block counting all rows would take long.
__global__ void __launch_bounds__(FRONT_THREADS) count_kernel(const __grid_constant__ Front p, unsigned int* __restrict__ counts) {
  __shared__ unsigned int warp_sum[32];
  let_next_start();
  const int begin = blockIdx.x * p.share, end = min(p.rows, begin + p.share);
  unsigned int mine = 0;
  for (int r = begin + threadIdx.x; r < end; r += FRONT_THREADS) mine += token_at(p.targets, p.wide, r, p.vocab) < (unsigned int)p.vocab;
  mine = block_sum(mine, warp_sum);
  if (threadIdx.x == 0) counts[blockIdx.x] = mine;
}

// Each block lists its own share of the rows, behind the rows that it counts in the shares before. bf16: it also copies their h, and
// blocks behind copy w where that is wanted. fp32: it finds their largest magnitude, and blocks behind that of w.
template <typename T>
__global__ void __launch_bounds__(FRONT_THREADS) front_kernel(const __grid_constant__ Front p) {
  constexpr bool SPLIT = sizeof(T) == 4;
  __shared__ unsigned int warp_sum[32];
  __shared__ int list[FRONT_THREADS];
  after_previous();
  let_next_start();
  const T *h = static_cast<const T*>(p.h), *w = static_cast<const T*>(p.w);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if ((int)blockIdx.x >= p.blocks_h) {
    const int block = blockIdx.x - p.blocks_h;
    auto same = [](int k) { return k; };
    if constexpr (SPLIT) {
      unsigned int most = 0;
      if (p.ldw == p.width && reinterpret_cast<uintptr_t>(w) % 16 == 0) {  // rows without gaps: one list of elements, whatever the width
        const long long all = (long long)p.vocab * p.width, step = (long long)p.blocks_w * FRONT_THREADS;
#pragma unroll 4
        for (long long i = (long long)block * FRONT_THREADS + threadIdx.x; i < all / 4; i += step) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(w) + i);
          most = max(most, max(max(finite_bits(v.x), finite_bits(v.y)), max(finite_bits(v.z), finite_bits(v.w))));
        }
        if (block == 0 && threadIdx.x < (all & 3)) most = max(most, finite_bits(__float_as_uint(__ldg(w + (all & ~3ll) + threadIdx.x))));
      } else {
        most = max_rows(w, p.ldw, p.vocab, block, p.blocks_w, p.width, same);
      }
      most = block_max(most, warp_sum);
      if (threadIdx.x == 0) p.most[blockIdx.x] = most;
    } else {
      copy_rows(w, p.ldw, p.vocab, block, p.blocks_w, p.width, p.pitch, 1.f, p.w_hi, p.w_lo, 0, same);
    }
    return;
  }
  const unsigned int vocab = p.vocab;
  const int begin = blockIdx.x * p.share, end = min(p.rows, begin + p.share);
  unsigned int before = 0, all = 0;
  if (p.counts) {
    for (int b = threadIdx.x; b < p.blocks_h; b += FRONT_THREADS) {
      const unsigned int n = p.counts[b];
      all += n;
      before += b < (int)blockIdx.x ? n : 0u;
    }
  } else {
#pragma unroll 8
    for (int r = threadIdx.x; r < p.rows; r += FRONT_THREADS) {
      const unsigned int n = token_at(p.targets, p.wide, r, vocab) < vocab;
      all += n;
      before += r < begin ? n : 0u;
    }
  }
  all = block_sum(all, warp_sum);
  unsigned int base = block_sum(before, warp_sum), most = 0;
  for (int r0 = begin; r0 < end; r0 += FRONT_THREADS) {
    const int r = r0 + threadIdx.x;
    const unsigned int t = r < end ? token_at(p.targets, p.wide, r, vocab) : vocab;
    const unsigned int have = __ballot_sync(0xFFFFFFFFu, t < vocab);
    const unsigned int n = block_sum(t < vocab ? 1u : 0u, warp_sum);
    const unsigned int at = __reduce_add_sync(0xFFFFFFFFu, lane < warp ? warp_sum[lane] : 0u) + __popc(have & ((1u << lane) - 1));
    if (t < vocab) {
      list[at] = r;
      p.row_of[base + at] = r;
      p.target[base + at] = (int)t;
      p.slot_of[r] = (int)(base + at);
    } else if (r < end) {
      p.slot_of[r] = -1;
      p.row_loss[r] = 0.f;
    }
    __syncthreads();
    auto listed = [&](int k) { return list[k]; };
    if constexpr (SPLIT) {
      most = max(most, max_rows(h, p.ldh, (int)n, 0, 1, p.width, listed));
    } else {
      copy_rows(h, p.ldh, (int)n, 0, 1, p.width, p.pitch, 1.f, p.h_hi, p.h_lo, base, listed);
    }
    base += n;
  }
  if constexpr (SPLIT) {
    most = block_max(most, warp_sum);
    if (threadIdx.x == 0) p.most[blockIdx.x] = most;
  } else {
    copy_rows(h, p.ldh, whole_rows(all) - (int)all, blockIdx.x, p.blocks_h, p.width, p.pitch, 1.f, p.h_hi, p.h_lo, all, [](int) { return -1; });
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) p.meta->rows = all;
}

// fp32: the copies of the listed rows of h and of w as pairs, behind the power of two that the largest magnitudes allow.
__global__ void __launch_bounds__(FRONT_THREADS) pairs_kernel(const __grid_constant__ Front p, int blocks_h, int blocks_w) {
  __shared__ unsigned int warp_max[32];
  after_previous();
  let_next_start();
  const bool of_h = (int)blockIdx.x < blocks_h;
  const unsigned int* from = of_h ? p.most : p.most + p.blocks_h;
  const int count = of_h ? p.blocks_h : p.blocks_w, block = of_h ? blockIdx.x : blockIdx.x - blocks_h;
  unsigned int most = 0;
  for (int i = threadIdx.x; i < count; i += FRONT_THREADS) most = max(most, from[i]);
  most = block_max(most, warp_max);
  if (block == 0 && threadIdx.x == 0) (of_h ? p.meta->max_h : p.meta->max_w) = most;
  const float up = pow2(up_exp(most));
  if (of_h) {
    const int rows = (int)p.meta->rows;
    copy_rows(static_cast<const float*>(p.h), p.ldh, whole_rows(rows), block, blocks_h, p.width, p.pitch, up, p.h_hi, p.h_lo, 0,
              [&](int k) { return k < rows ? __ldg(p.row_of + k) : -1; });
  } else {
    copy_rows(static_cast<const float*>(p.w), p.ldw, p.vocab, block, blocks_w, p.width, p.pitch, up, p.w_hi, p.w_lo, 0, [](int k) { return k; });
  }
}


// ------------------------------------------------------------------ logits

struct LogitParams {
  const Meta* meta;
  int vocab, v_begin, v_count;  // this call's piece of the vocabulary
  int kblocks;
  long long row_pitch;  // rows of the lists: parts are [warp of a tile's row][row]
  const int* target;
  float2* parts;        // maximum (times log2 e) and sum of 2^(x - maximum)
  float* target_logit;  // times log2 e
  const float2* row_stat;  // maximum and 1 / sum of whole rows
  uint16_t *d_hi, *d_lo;
  long long ld_d;
  float* x;  // logits as they are summed, where they are kept: parts x all_rows x ld_x
  long long ld_x;
  int x_parts, all_rows;
};

template <class F>
struct LogitTiles {
  typedef F Form;
  static constexpr bool SPLIT = F::SPLIT, INFINITE = true;
  static constexpr int SUM = XENT_SUM, BN = F::BN, W = F::CHUNK;
  const LogitParams& p;
  int rows, m_blocks, n_blocks, band;
  float unit;  // accumulators times this are logits times log2 e
  __device__ explicit LogitTiles(const LogitParams& q, const TileMaps&) : p(q) {
    rows = (int)p.meta->rows;
    m_blocks = max(1, (rows + F::M - 1) / F::M);
    n_blocks = (p.v_count + BN - 1) / BN;
    // all row blocks of a column block one after another, as long as the copy of h they read stays in the L2 cache
    band = m_blocks <= 64 ? m_blocks : 16;
    unit = SPLIT ? LOG2E * pow2(-up_exp(p.meta->max_h)) * pow2(-up_exp(p.meta->max_w)) : LOG2E;
  }
  __device__ int tiles() const { return m_blocks * n_blocks; }
  __device__ Tile tile(int t) const {
    const int b = t / (band * n_blocks), in = t - b * band * n_blocks;
    const int tall = min(band, m_blocks - b * band);
    Tile r;
    r.m0 = (b * band + in % tall) * F::M;
    r.n0 = in / tall * BN;
    r.a_mn = r.m0;
    r.b_mn = p.v_begin + r.n0;
    r.a_k = r.b_k = 0;
    r.kblocks = p.kblocks;
    r.z = 0;
    return r;
  }
};

// Few tiles: their sums as they are, in parts of the k range where there are more SMs than tiles.
template <class F>
struct PlainOp : LogitTiles<F> {
  typedef LogitParams Params;
  static constexpr bool LONG = true, STORES = false;
  static constexpr int SUM = F::SPLIT ? XENT_SUM : 16, W = 16;
  using LogitTiles<F>::p;
  __device__ explicit PlainOp(const LogitParams& q, const TileMaps& m) : LogitTiles<F>(q, m) {}
  __device__ int tiles() const { return LogitTiles<F>::tiles() * p.x_parts; }
  __device__ Tile tile(int t) const {
    const int whole = LogitTiles<F>::tiles(), part = t / whole, from = p.kblocks * part / p.x_parts;
    Tile r = LogitTiles<F>::tile(t - part * whole);
    r.a_k = r.b_k = from * TILE_K;
    r.kblocks = p.kblocks * (part + 1) / p.x_parts - from;
    r.z = part;
    return r;
  }
  __device__ __forceinline__ void begin(const Tile&, int, int, int) {}
  __device__ __forceinline__ void chunk(const Tile& t, int row0, int col0, float (&v)[W], uint8_t* stage, int lane) {
    by_rows(row0, col0, v, stage, lane, [&](int, int r, int c, const float4& x) {
      if (r < this->rows && c < p.vocab) *reinterpret_cast<float4*>(p.x + ((long long)t.z * p.all_rows + r) * p.ld_x + c) = x;
    });
  }
  __device__ __forceinline__ void end(const Tile&, int, int) {}
};

// Maximum and sum of exponentials of a row over the columns of one warp, and the target's logit. LONG: for more than 16 k-blocks,
// whose sums the tensor core would leave too small (bf16, width 2048: losses 1.0e-6 off, with sums of 16 added in fp32 0.5e-6, in the
// same time). RUN: all tiles have the same rows, so a warp goes on with its maximum and sum, and lists are [warp][row].
template <class F, bool LONG_, bool KEEP, bool RUN>
struct StatOp : LogitTiles<F> {
  typedef LogitParams Params;
  static constexpr bool LONG = F::SPLIT || LONG_;
  static constexpr int SUM = F::SPLIT ? XENT_SUM : 16;
  static constexpr bool STORES = false;
  using LogitTiles<F>::p;
  float top, sum;
  int target;
  __device__ explicit StatOp(const LogitParams& q, const TileMaps& m) : LogitTiles<F>(q, m) {}
  bool begun = false;
  __device__ __forceinline__ void begin(const Tile&, int row0, int, int lane) {
    if (!RUN || !begun) {
      top = -INFINITY;
      sum = 0.f;
    }
    begun = true;
    target = row0 + lane < this->rows ? __ldg(p.target + row0 + lane) : -1;
  }
  static constexpr int W = LONG ? 16 : LogitTiles<F>::W;
  __device__ __forceinline__ void chunk(const Tile&, int row0, int col0, float (&v)[W], uint8_t* stage, int lane) {
    if (col0 >= p.vocab || row0 >= this->rows) return;
    if (KEEP)
      by_rows(row0, col0, v, stage, lane, [&](int, int r, int c, const float4& x) {
        if (r < this->rows && c < p.vocab) *reinterpret_cast<float4*>(p.x + r * p.ld_x + c) = x;
      });
    if (col0 + W > p.vocab) {
#pragma unroll
      for (int j = 0; j < W; ++j)
        if (col0 + j >= p.vocab) v[j] = -INFINITY;
    }
    float most = v[0];
#pragma unroll
    for (int j = 1; j < W; ++j) most = fmaxf(most, v[j]);
    const float now = fmaxf(top, most * this->unit);
    const float base = now == -INFINITY ? 0.f : now;  // nothing but -inf so far: their exponentials are 0
    float s[4] = {sum * ex2(top - base), 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < W; ++j) s[j & 3] += ex2(fmaf(v[j], this->unit, -base));
    sum = (s[0] + s[1]) + (s[2] + s[3]);
    top = now;
    const int at = target - col0;
    if (at >= 0 && at < W) {
      float x = v[0];
#pragma unroll
      for (int j = 1; j < W; ++j) x = j == at ? v[j] : x;
      p.target_logit[row0 + lane] = x * this->unit;
    }
  }
  __device__ __forceinline__ void end(const Tile& t, int row, int part) {
    const int list = RUN ? blockIdx.x / F::CTAS : t.n0 / F::BN;
    if (row < this->rows) p.parts[(long long)(list * F::PARTS + part) * p.row_pitch + row] = make_float2(top, sum);
  }
};

// d of a piece, zeros in rows and columns that fill up tiles. What an element takes here bounds the kernel when width is small
// (1024 and less: 8 us per tile before stores went by TMA and the target's column was a branch of its own, 5.8 us
// of products), so it is one FMA, one exponential, one product and half a conversion. Sums are handed over as in StatOp, so that the
// logits are the same bits: where one pass truncates more than the other, a row's p do not add up to 1, and p - 1 of a target that is
// nearly certain is wrong by as much (width 2000, logits of 65: off by as much as itself at p = 1 - 1e-4).
template <class F, bool LONG_>
struct GradOp : LogitTiles<F> {
  typedef LogitParams Params;
  static constexpr bool LONG = F::SPLIT || LONG_;
  static constexpr int SUM = StatOp<F, LONG_, false, false>::SUM;
  static constexpr bool STORES = !F::SPLIT;
  using LogitTiles<F>::p;
  const CUtensorMap* map;
  float top, by, to;
  int target;
  bool in;
  __device__ explicit GradOp(const LogitParams& q, const TileMaps& m) : LogitTiles<F>(q, m), map(&m.c) {
    to = F::SPLIT ? (float)(1 << D_EXP) : 1.f;  // the caller's scale comes behind the products: -1 at an unlikely target is exact
  }
  __device__ __forceinline__ void begin(const Tile&, int row0, int, int lane) {
    const int row = row0 + lane;
    in = row < this->rows;
    const float2 st = in ? __ldg(p.row_stat + row) : make_float2(0.f, 0.f);
    top = st.x;
    by = st.y * to;
    target = in ? __ldg(p.target + row) - p.v_begin : -1;
  }
  static constexpr int W = LONG ? 16 : LogitTiles<F>::W;
  __device__ __forceinline__ void chunk(const Tile&, int row0, int col0, float (&v)[W], uint8_t* stage, int lane) {
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = ex2(fmaf(v[j], this->unit, -top)) * by;
    const int at = target - col0;
    if (at >= 0 && at < W) {
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] -= j == at ? to : 0.f;
    }
    if (!in || col0 + W > p.v_count) {
#pragma unroll
      for (int j = 0; j < W; ++j)
        if (!in || col0 + j >= p.v_count) v[j] = 0.f;
    }
    if constexpr (F::SPLIT) {
      by_rows(row0, col0, v, stage, lane, [&](int, int r, int c, const float4& x) {
        store_pair(reinterpret_cast<__half*>(p.d_hi), reinterpret_cast<__half*>(p.d_lo), (long long)r * p.ld_d + c, x);
      });
    } else {
      uint32_t w[W / 2];
#pragma unroll
      for (int j = 0; j < W / 2; ++j) w[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
      store_half_words(map, w, row0, col0, stage, lane);
    }
  }
  __device__ __forceinline__ void end(const Tile&, int, int) {}
};

// The same d from kept logits, eight neighbouring elements per thread, zeros up to whole k-blocks of the products that read it.
template <bool SPLIT>
__global__ void __launch_bounds__(256) kept_kernel(const LogitParams p) {
  after_previous();
  let_next_start();
  const Meta meta = *p.meta;
  const unsigned int rows = meta.rows, rows_up = whole_rows(rows);
  const unsigned int per_row = (unsigned int)((p.v_count + TILE_K - 1) / TILE_K * (TILE_K / 8)), all = rows_up * per_row;
  const float unit = SPLIT ? LOG2E * pow2(-up_exp(meta.max_h)) * pow2(-up_exp(meta.max_w)) : LOG2E, to = SPLIT ? (float)(1 << D_EXP) : 1.f;
#pragma unroll 2
  for (unsigned int i = blockIdx.x * 256 + threadIdx.x; i < all; i += gridDim.x * 256) {
    const unsigned int r = i / per_row;
    const int c = (int)(i - r * per_row) * 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (r < rows) {
      const float* from = p.x + r * p.ld_x + p.v_begin + c;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (c + 4 * j < p.v_count) *reinterpret_cast<float4*>(v + 4 * j) = *reinterpret_cast<const float4*>(from + 4 * j);
      const float2 st = __ldg(p.row_stat + r);
      const int target = __ldg(p.target + r) - p.v_begin - c;
      const float by = st.y * to;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = ex2(fmaf(v[j], unit, -st.x)) * by;
        v[j] -= j == target ? to : 0.f;
        if (c + j >= p.v_count) v[j] = 0.f;
      }
    }
    const long long at = r * p.ld_d + c;
    if (SPLIT) {
      __half hi[8], lo[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) split_half(v[j], hi[j], lo[j]);
      *reinterpret_cast<uint4*>(p.d_hi + at) = *reinterpret_cast<const uint4*>(hi);
      *reinterpret_cast<uint4*>(p.d_lo + at) = *reinterpret_cast<const uint4*>(lo);
    } else {
      *reinterpret_cast<uint4*>(p.d_hi + at) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    }
  }
}

// Loss of a row, and its d, from the parts of its logits: a block has a row, its threads four neighbouring columns at a time, and
// keeps it in registers. d has zeros up to whole k-blocks, as above.
constexpr int ROW_THREADS = 512, ROW_QUADS = 10;
template <bool SPLIT>
__global__ void __launch_bounds__(ROW_THREADS) row_kernel(const LogitParams p, const int* __restrict__ row_of, float* __restrict__ row_loss, int grads) {
  __shared__ float across[ROW_THREADS / 32];
  after_previous();
  let_next_start();
  const int lane = threadIdx.x & 31, r = blockIdx.x, at = threadIdx.x * 4;
  const Meta meta = *p.meta;
  const int rows = (int)meta.rows, whole = whole_rows(rows);
  if (r >= whole) return;
  const float unit = SPLIT ? LOG2E * pow2(-up_exp(meta.max_h)) * pow2(-up_exp(meta.max_w)) : LOG2E, to = SPLIT ? (float)(1 << D_EXP) : 1.f;
  const long long stride = (long long)p.all_rows * p.ld_x;
  const float* from = p.x + r * p.ld_x;
  auto over_all = [&](float v, auto join) {  // threads
#pragma unroll
    for (int d = 16; d; d >>= 1) v = join(v, __shfl_xor_sync(0xFFFFFFFFu, v, d));
    __syncthreads();
    if (lane == 0) across[threadIdx.x >> 5] = v;
    __syncthreads();
    v = across[lane & 15];
#pragma unroll
    for (int d = 8; d; d >>= 1) v = join(v, __shfl_xor_sync(0xFFFFFFFFu, v, d));
    return v;
  };
  static_assert(ROW_THREADS == 512, "16 warps");
  float x[ROW_QUADS][4];
  float top = -INFINITY, sum = 0.f, by = 0.f;
  int target = -1;
  if (r < rows) {
#pragma unroll
    for (int i = 0; i < ROW_QUADS; ++i) {
      const int c = at + i * ROW_THREADS * 4;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[i][j] = 0.f;
      if (c >= p.vocab) continue;
#pragma unroll 4
      for (int k = 0; k < p.x_parts; ++k) {
        const float4 y = *reinterpret_cast<const float4*>(from + k * stride + c);
        x[i][0] += y.x; x[i][1] += y.y; x[i][2] += y.z; x[i][3] += y.w;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (c + j >= p.vocab) x[i][j] = -INFINITY;
        top = fmaxf(top, x[i][j]);
      }
    }
    top = over_all(top, [](float a, float b) { return fmaxf(a, b); }) * unit;
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int i = 0; i < ROW_QUADS; ++i) {
      if (at + i * ROW_THREADS * 4 >= p.vocab) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[i][j] = ex2(fmaf(x[i][j], unit, -base));
        sum += x[i][j];
      }
    }
    sum = over_all(sum, [](float a, float b) { return a + b; });
    by = to / sum;
    target = __ldg(p.target + r);
    if (at == 0) {
      float own = 0.f;
      for (int k = 0; k < p.x_parts; ++k) own += from[k * stride + target];
      row_loss[row_of[r]] = ((top - own * unit) + log2f(sum)) * LN2;
    }
  }
  if (!grads) return;
  const int cols = (p.vocab + TILE_K - 1) / TILE_K * TILE_K;
#pragma unroll
  for (int i = 0; i < ROW_QUADS; ++i) {
    const int c = at + i * ROW_THREADS * 4;
    if (c >= cols) continue;
    float d[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) d[j] = r < rows && c + j < p.vocab ? x[i][j] * by - (c + j == target ? to : 0.f) : 0.f;
    const long long to_at = r * p.ld_d + c;
    if (SPLIT) store_pair(reinterpret_cast<__half*>(p.d_hi), reinterpret_cast<__half*>(p.d_lo), to_at, make_float4(d[0], d[1], d[2], d[3]));
    else *reinterpret_cast<uint2*>(p.d_hi + to_at) = make_uint2(pack_bf16(d[0], d[1]), pack_bf16(d[2], d[3]));
  }
}

// Whole rows' maximum and sum from the lists, and the losses. A block has 32 rows: its warps share their lists first, and then each
// joins one row's 32 shares.
__global__ void __launch_bounds__(1024) join_rows_kernel(const float2* __restrict__ parts, long long row_pitch, int count,
                                                         const Meta* __restrict__ meta, const float* __restrict__ target_logit,
                                                         const int* __restrict__ row_of, float2* __restrict__ row_stat,
                                                         float* __restrict__ row_loss) {
  __shared__ float2 part[32][33];
  after_previous();
  let_next_start();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rows = (int)meta->rows, row0 = blockIdx.x * 32;
  if (row0 >= rows) return;
  float top = -INFINITY, sum = 0.f;
  for (int k = warp; k < count; k += 8 * 32) {  // eight lists at a time, on one maximum
    float2 x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      x[u] = k + 32 * u < count && row0 + lane < rows ? __ldg(parts + (long long)(k + 32 * u) * row_pitch + row0 + lane) : make_float2(-INFINITY, 0.f);
    float now = top;
#pragma unroll
    for (int u = 0; u < 8; ++u) now = fmaxf(now, x[u].x);
    const float base = now == -INFINITY ? 0.f : now;  // nothing but -inf so far: their exponentials are 0
    sum *= ex2(top - base);
#pragma unroll
    for (int u = 0; u < 8; ++u) sum = fmaf(x[u].y, ex2(x[u].x - base), sum);
    top = now;
  }
  part[warp][lane] = make_float2(top, sum);
  __syncthreads();
  const int row = row0 + warp;
  if (row >= rows) return;
  const float2 mine = part[lane][warp];
  top = mine.x;
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
  sum = mine.y * ex2(mine.x - (top == -INFINITY ? 0.f : top));
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
  if (lane == 0) {
    row_stat[row] = make_float2(top, 1.f / sum);
    row_loss[row_of[row]] = ((top - target_logit[row]) + log2f(sum)) * LN2;
  }
}

// ------------------------------------------------------------------ gradients

// k-blocks of bf16 products after which sums are handed over and added up in fp32, where there are more than four times as many: the tensor core
// truncates at each of its additions, which leaves long sums of one sign too small (dw of 8192 rows 2e-6, of 65536 4e-4, of 2^20 6.5e-3 of
// its value, where a bf16 result is rounded by up to 4e-3).
constexpr int LONG_SUM = 128;

struct ProductParams {
  const Meta* meta;
  int v_begin, v_count;
  int width;
  float scale;
  // dh: fp32 sums over the pieces
  float *acc, *slots;
  long long ld_acc;
  int pairs, full_kblocks;  // pairs of CTAs, or single ones; full_kblocks: of a whole piece
  int first;                // first piece: written, not added to
  // dw
  void* dw;
  long long ld_dw;
  int out_bf16, vec;  // vec: rows begin on whole groups of four elements
  int by_tma;         // rows are whole 16-byte pieces, which is how TMA clips
};

// How the tiles of dh go over the pairs. There are few of them and their sums are long, so whole tiles alone would leave many
// pairs idle in the last round (232 tiles on 74 pairs: 4 rounds for 3.1). Whole tiles fill complete rounds, all pairs in step so
// that they share their slabs in the L2 cache; the k range of the `rest` tiles behind them is cut into equal parts, one per
// pair, which may cover the end of one tile and the beginning of the next. A part's sum goes to a slot of its pair, and
// spread_rows_kernel adds a tile's parts in order. Which part is whose does not depend on the piece, so the slots are added to
// from piece to piece.
// Where the rest is whole rows of tiles, `side` pairs go through the k range of a row of tiles side by side, so that they read the
// same slab of d at the same time (28 tiles, 4 in a row, 296 k-blocks, twice: 450 -> 435 us
// for the whole call).
struct HiddenSplit {
  int m_blocks, n_blocks, whole, side, rest, shares;  // rest and shares count rows of `side` tiles and of pairs
  __device__ HiddenSplit(const ProductParams& p, unsigned int rows, int bm, int bn) {
    m_blocks = max(1, (int)((rows + bm - 1) / bm));
    n_blocks = (p.width + bn - 1) / bn;
    const int tiles = m_blocks * n_blocks;
    whole = tiles / p.pairs * p.pairs;
    side = whole == 0 && n_blocks <= 8 ? n_blocks : 1;
    rest = (tiles - whole) / side;
    // no part shorter than eight k-blocks, where there is a choice
    shares = (int)min((long long)(p.pairs / side), max((long long)rest, (long long)rest * p.full_kblocks / 8));
  }
  // Part j (0, 1) of pair s: tile behind the whole ones, and its range of k in 1 / shares of a tile. False: there is none.
  __device__ bool part(int s, int j, int& tile, int& from, int& to) const {
    const int begin = s / side * rest, end = begin + rest;  // in 1 / shares of a row of tiles
    if (s / side >= shares) return false;
    const int row = begin / shares + j;
    tile = row * side + s % side;
    from = max(begin - row * shares, 0);
    to = min(end - row * shares, shares);
    return to > from;
  }
  // How many parts tile t has, and the slot of the n-th, where there are more than one.
  __device__ int parts(int t) const { return t < 0 ? 1 : ((t / side + 1) * shares - 1) / rest - t / side * shares / rest + 1; }
  __device__ int slot(int t, int n) const {
    const int share = t / side * shares / rest + n;
    return slot_of(share * side + t % side, share * rest > t / side * shares);
  }
  __device__ static int slot_of(int s, bool begun_before) { return 2 * s + (begun_before ? 0 : 1); }
};

// dh (listed rows) += d w over a piece.
template <class F, bool LONG_>
struct HiddenOp {
  typedef ProductParams Params;
  typedef F Form;
  static constexpr bool SPLIT = F::SPLIT, STORES = false, INFINITE = true;
  static constexpr bool LONG = SPLIT || LONG_;
  static constexpr int SUM = SPLIT ? XENT_SUM : LONG_SUM, BN = F::BN;
  const ProductParams& p;
  HiddenSplit split;
  int kblocks;
  float unit;
  float* to;
  long long ld;
  __device__ explicit HiddenOp(const ProductParams& q, const TileMaps&) : p(q), split(q, q.meta->rows, F::M, BN) {
    kblocks = (p.v_count + TILE_K - 1) / TILE_K;
    unit = SPLIT ? p.scale * pow2(-D_EXP) * pow2(-up_exp(p.meta->max_w)) : p.scale;
  }
  __device__ int tiles() const { return split.whole + 2 * p.pairs; }
  __device__ Tile tile(int t) const {
    Tile r;
    int at = t, from = 0, kb = kblocks;
    r.z = -1;  // straight to acc
    if (t >= split.whole) {
      const int j = (t - split.whole) / p.pairs, s = t - split.whole - j * p.pairs;
      int a, b;
      if (!split.part(s, j, at, a, b)) {
        r.z = -2;  // nothing
        r.m0 = r.n0 = r.a_mn = r.b_mn = r.a_k = r.b_k = r.kblocks = 0;
        return r;
      }
      at += split.whole;
      from = (int)((long long)kblocks * a / split.shares);
      kb = (int)((long long)kblocks * b / split.shares) - from;
      if (a > 0 || b < split.shares) r.z = HiddenSplit::slot_of(s, a > 0);
    }
    r.m0 = at / split.n_blocks * F::M;
    r.n0 = at % split.n_blocks * BN;
    r.a_mn = r.m0;
    r.b_mn = r.n0;
    r.a_k = from * TILE_K;
    r.b_k = p.v_begin + from * TILE_K;
    r.kblocks = kb;
    return r;
  }
  __device__ __forceinline__ void begin(const Tile& t, int, int, int) {
    if (t.z >= 0) {
      ld = BN;
      to = p.slots + (long long)t.z * F::M * BN - (t.m0 * ld + t.n0);
    } else {
      ld = p.ld_acc;
      to = p.acc;
    }
  }
  static constexpr int W = LONG ? 16 : F::CHUNK;
  __device__ __forceinline__ void chunk(const Tile& t, int row0, int col0, float (&v)[W], uint8_t* stage, int lane) {
    if (t.z == -2 || col0 >= p.width) return;
    float4 old[W / 4];
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const int c = col0 + quad_col<W>(lane);
      old[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (!p.first && c < p.width) old[i] = *reinterpret_cast<const float4*>(to + (row0 + quad_row<W>(i, lane)) * ld + c);
    }
    by_rows(row0, col0, v, stage, lane, [&](int i, int r, int c, const float4& x) {
      if (c < p.width)
        *reinterpret_cast<float4*>(to + r * ld + c) =
            make_float4(fmaf(x.x, unit, old[i].x), fmaf(x.y, unit, old[i].y), fmaf(x.z, unit, old[i].z), fmaf(x.w, unit, old[i].w));
    });
  }
  __device__ __forceinline__ void end(const Tile&, int, int) {}
};

// dw of a piece = d' h.
template <class F, bool LONG_>
struct WeightOp {
  typedef ProductParams Params;
  typedef F Form;
  static constexpr bool SPLIT = F::SPLIT, STORES = !SPLIT, INFINITE = true;
  static constexpr bool LONG = SPLIT || LONG_;
  static constexpr int SUM = SPLIT ? XENT_SUM : LONG_SUM, BN = F::BN;
  const ProductParams& p;
  const CUtensorMap* map;
  int m_blocks, n_blocks, kblocks;
  float unit;
  __device__ explicit WeightOp(const ProductParams& q, const TileMaps& m) : p(q), map(&m.c) {
    m_blocks = (p.v_count + F::M - 1) / F::M;
    n_blocks = (p.width + BN - 1) / BN;
    kblocks = max(1, (int)((p.meta->rows + TILE_K - 1) / TILE_K));  // without rows: zeros, as they are stored
    unit = SPLIT ? p.scale * pow2(-D_EXP) * pow2(-up_exp(p.meta->max_h)) : p.scale;
  }
  __device__ int tiles() const { return m_blocks * n_blocks; }
  __device__ Tile tile(int t) const {
    Tile r;
    r.m0 = t / n_blocks * F::M;
    r.n0 = t % n_blocks * BN;
    r.a_mn = r.m0;
    r.b_mn = r.n0;
    r.a_k = r.b_k = 0;
    r.kblocks = kblocks;
    r.z = 0;
    return r;
  }
  __device__ __forceinline__ void begin(const Tile&, int, int, int) {}
  static constexpr int W = LONG ? 16 : F::CHUNK;
  __device__ __forceinline__ void chunk(const Tile&, int row0, int col0, float (&v)[W], uint8_t* stage, int lane) {
    if constexpr (!SPLIT) {
      if (p.by_tma) {  // pieces are whole 256-row tiles but for the last one, whose rows the map ends with
        uint32_t w[W / 2];
#pragma unroll
        for (int j = 0; j < W / 2; ++j) w[j] = pack_bf16(v[2 * j] * unit, v[2 * j + 1] * unit);
        store_half_words(map, w, p.v_begin + row0, col0, stage, lane);
        return;
      }
    }
    by_rows(row0, col0, v, stage, lane, [&](int, int r, int c, const float4& x) {
      if (r >= p.v_count || c >= p.width) return;
      const long long at = (long long)(p.v_begin + r) * p.ld_dw + c;
      const float f[4] = {x.x * unit, x.y * unit, x.z * unit, x.w * unit};
      if (p.out_bf16) {
        __nv_bfloat16* to = static_cast<__nv_bfloat16*>(p.dw) + at;
        if (p.vec && c + 4 <= p.width) {
          *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (c + i < p.width) to[i] = __float2bfloat16_rn(f[i]);
        }
      } else {
        float* to = static_cast<float*>(p.dw) + at;
        if (p.vec && c + 4 <= p.width) {
          *reinterpret_cast<float4*>(to) = make_float4(f[0], f[1], f[2], f[3]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (c + i < p.width) to[i] = f[i];
        }
      }
    });
  }
  __device__ __forceinline__ void end(const Tile&, int, int) {}
};

// dh in the caller's order and type, zeros for rows without a target.
template <typename T, class F>
__global__ void __launch_bounds__(256) spread_rows_kernel(const ProductParams p, const int* __restrict__ slot_of, int rows, int vec,
                                                          T* __restrict__ dh, size_t ld) {
  constexpr int BN = F::BN;
  after_previous();
  let_next_start();
  const HiddenSplit split(p, p.meta->rows, F::M, BN);
  const int width = p.width;
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    const int slot = slot_of[r];
    T* to = dh + (size_t)r * ld;
    for (int c = threadIdx.x * 4; c < width; c += 256 * 4) {
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (slot >= 0) {
        const int t = slot / F::M * split.n_blocks + c / BN - split.whole;
        const int parts = split.parts(t);
        if (parts == 1) {
          x = *reinterpret_cast<const float4*>(p.acc + slot * p.ld_acc + c);
        } else {
          for (int n = 0; n < parts; ++n) {
            const float4 y = *reinterpret_cast<const float4*>(p.slots + ((long long)split.slot(t, n) * F::M + slot % F::M) * BN + c % BN);
            x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
          }
        }
      }
      const float f[4] = {x.x, x.y, x.z, x.w};
      if (vec && c + 4 <= width) {
        typedef Elems<T, 4 * (int)sizeof(T)> E;
        *reinterpret_cast<typename E::raw*>(to + c) = E::put(f);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (c + i < width) to[c + i] = (T)f[i];
      }
    }
  }
}

// ------------------------------------------------------------------ host side

struct Sizes {
  long long rows_up, pitch;  // rows of the copy of h (whole blocks), elements per row of the copies
  long long parts;           // lists per row
  long long piece;           // columns of d
  bool split, copy_w;
  bool one;                  // few tiles of logits: single CTAs
  bool by_rows;              // and few rows: PlainOp and row_kernel
  int x_parts;               // parts of their k range
  bool keep;                 // logits are kept
  long long ld_x;
};
constexpr int MOST_PAIRS = 74;  // 148 SMs
template <class F>
long long tiles_of(long long m, long long n) { return (m + F::M - 1) / F::M * ((n + F::BN - 1) / F::BN); }
// Where single CTAs would leave SMs idle through a long k range, it goes in parts, and row_kernel takes its time for each of a few rows
// (with gradients 1 x 3972 x 806 in fp32 84 -> 74 us, 75 x 1152 x 2411 in bf16 43 -> 38).
template <class F>
int lists_of(size_t rows, size_t vocab, int sms, int* run) {  // per row: for one block of rows (*run) a list per warp, else per tile and warp
  const long long tiles = ((long long)vocab + F::BN - 1) / F::BN, most = sms / F::CTAS;
  *run = rows <= F::M;
  return (int)(F::PARTS * (*run && tiles > most ? most : tiles));
}
template <class F>
void logit_sizes(Sizes* z, size_t rows, size_t width, size_t vocab) {  // F: single CTAs
  typedef TileForm<F::SPLIT> Pairs;
  const int sms = 2 * MOST_PAIRS;
  const long long one = tiles_of<F>(rows, vocab), pairs = tiles_of<Pairs>(rows, vocab), kblocks = (long long)(width + TILE_K - 1) / TILE_K;
  z->one = single_ctas<F::SPLIT>((one + sms - 1) / sms, kblocks, (pairs + MOST_PAIRS - 1) / MOST_PAIRS, kblocks);
  long long parts = z->one ? sms / one : 1;
  if (parts > kblocks / 4) parts = kblocks / 4;
  z->by_rows = parts > 1 && kblocks - kblocks / parts >= 8 && rows <= 4 * MOST_PAIRS && vocab <= ROW_QUADS * 4 * ROW_THREADS;
  z->x_parts = z->by_rows ? (int)parts : 1;
  int run;
  z->parts = z->by_rows ? 0 : z->one ? lists_of<F>(rows, vocab, sms, &run) : lists_of<Pairs>(rows, vocab, sms, &run);
}
// Logits that are kept cost their bytes twice, others 2 F operations each again. What stays in the L2 cache is kept (1024 x 512 x 8192 in
// fp32 140 -> 125 us, 16 x 2048 x 65536 in bf16 251 -> 217); beyond it the operations cost more with three MMAs or great widths (2048 x
// 1024 x 32768 in fp32 1 550 -> 1 340 us, 1024 x 4096 x 32768 in bf16 923 -> 800) and less with small ones (bf16: 2048 x 512 x 32768 241 -> 303,
// 2048 x 768 x 32768 387 -> 415, 2048 x 1024 x 32768 474 -> 480). 8192 x 2048 x 65536 would gain 4 % and take 2 GB.
bool keeps_logits(long long bytes, size_t width, bool split) {
  return bytes <= 64ll << 20 || (bytes <= 512ll << 20 && width >= (split ? 256 : 2048));
}
Sizes sizes_of(size_t rows, size_t width, size_t vocab, int dtype, int grads, const void* w, size_t ldw) {
  Sizes z;
  z.split = dtype == B2_DTYPE_F32;
  // TMA reads rows that begin on 16-byte boundaries
  z.copy_w = z.split || reinterpret_cast<uintptr_t>(w) % 16 != 0 || ldw % 8 != 0;
  z.rows_up = (long long)(rows + TILE_M - 1) / TILE_M * TILE_M;
  z.pitch = (long long)(width + 63) / 64 * 64;
  if (z.split) logit_sizes<TileForm<true, true>>(&z, rows, width, vocab);
  else logit_sizes<TileForm<false, true>>(&z, rows, width, vocab);
  z.piece = 0;
  z.ld_x = ((long long)vocab + 3) / 4 * 4;
  z.keep = z.by_rows || (grads && keeps_logits((long long)rows * z.ld_x * 4, width, z.split));
  if (grads) {
    // Few pieces: each has three kernels to fill and drain, which costs more than reading d from HBM (8192 x 2048 x 65536 with pieces of 160
    // MB 6.05 ms, 320 MB 5.94, 640 MB 5.86, 80 MB 6.5; 2048 x 1024 x 65536 948, 906 and 832 us). The 256-wide column blocks of a piece should go
    // evenly over 74 pairs: 37 of them do for any number of row blocks.
    const long long all = ((long long)vocab + 255) / 256 * 256, unit = 37 * 256;
    long long fit = (640ll << 20) / (z.rows_up * (z.split ? 4 : 2));
    if (fit >= unit) fit = fit / unit * unit;
    else fit = fit / 256 * 256;
    if (fit < 1024) fit = 1024;
    z.piece = all < fit ? all : fit;
  }
  return z;
}
struct Space {
  Meta* meta;
  unsigned int *counts, *most;
  int *row_of, *slot_of, *target;
  float* target_logit;
  float2 *row_stat, *parts;
  uint16_t *h_hi, *h_lo, *w_hi, *w_lo, *d_hi, *d_lo;
  float *acc, *slots, *x;
};
constexpr int FRONT_BLOCKS = 4 * MOST_PAIRS;  // on h at most: two per SM; on w twice as many
size_t space_of(const Sizes& z, size_t rows, size_t vocab, int grads, void* base, Space* s) {
  Carver c(base);
  const size_t lo = z.split ? 1 : 0;
  s->meta = c.take<Meta>(1);
  s->counts = c.take<unsigned int>(FRONT_BLOCKS);
  s->most = c.take<unsigned int>(3 * FRONT_BLOCKS);
  s->row_of = c.take<int>(z.rows_up);
  s->slot_of = c.take<int>(rows);
  s->target = c.take<int>(z.rows_up);
  s->target_logit = c.take<float>(z.rows_up);
  s->row_stat = c.take<float2>(z.rows_up);
  s->parts = c.take<float2>(z.parts * z.rows_up);
  s->h_hi = c.take<uint16_t>(z.rows_up * z.pitch);
  s->h_lo = c.take<uint16_t>(lo * z.rows_up * z.pitch);
  s->w_hi = c.take<uint16_t>(z.copy_w ? vocab * z.pitch : 0);
  s->w_lo = c.take<uint16_t>(lo * vocab * z.pitch);
  s->d_hi = c.take<uint16_t>(z.rows_up * z.piece);
  s->d_lo = c.take<uint16_t>(lo * z.rows_up * z.piece);
  s->acc = c.take<float>(grads ? z.rows_up * z.pitch : 0);
  s->slots = c.take<float>(grads ? 2ll * MOST_PAIRS * TILE_M * (z.split ? 128 : 256) : 0);
  s->x = c.take<float>(z.keep ? z.x_parts * rows * z.ld_x : 0);
  return c.used;
}

struct XentCall {
  size_t rows, width, vocab;
  int dtype;
  const void* h;
  size_t ldh;
  const void* w;
  size_t ldw;
  const void* targets;
  int wide;
  float scale;
  float* row_loss;
  void* dh;
  size_t ld_dh;
  void* dw;
  size_t ld_dw;
};

constexpr int COUNT_ROWS = 1 << 15;  // rows up to which every block counts all targets: 26.6 us against 29.6 for 32768 x 64 x 256, 41.9 against 27.9 for 65536

template <bool SPLIT>
int xent_run(const XentCall& c, const Sizes& z, const Space& s, int sms, cudaStream_t st) {
  typedef typename std::conditional<SPLIT, float, __nv_bfloat16>::type T;
  typedef TileForm<SPLIT> Pairs;
  typedef TileForm<SPLIT, true> One;
  const char* who = "b2_xent";
  const int rows = (int)c.rows, width = (int)c.width, vocab = (int)c.vocab, pitch = (int)z.pitch;
  const T *h = static_cast<const T*>(c.h), *w = static_cast<const T*>(c.w);
  Chain chain(st);
  auto blocks = [&](long long n) { return (unsigned int)(n < 8ll * sms ? n : 8ll * sms); };
  Front f{};
  f.targets = c.targets;
  f.wide = c.wide;
  f.rows = rows;
  f.vocab = vocab;
  f.width = width;
  f.pitch = pitch;
  f.meta = s.meta;
  f.row_of = s.row_of;
  f.slot_of = s.slot_of;
  f.target = s.target;
  f.row_loss = c.row_loss;
  f.h = h;
  f.w = w;
  f.ldh = (long long)c.ldh;
  f.ldw = (long long)c.ldw;
  f.h_hi = s.h_hi;
  f.h_lo = s.h_lo;
  f.w_hi = s.w_hi;
  f.w_lo = s.w_lo;
  f.most = s.most;
  auto some = [](long long n, int most) { return (int)(n < most ? n : most); };
  // a block has four rows of h at least
  f.share = (rows + FRONT_BLOCKS - 1) / FRONT_BLOCKS;
  if (f.share < 4) f.share = 4;
  f.blocks_h = (rows + f.share - 1) / f.share;
  const int at_once = FRONT_THREADS >> row_shift(pitch / 8);
  f.blocks_w = z.copy_w ? some((vocab + at_once - 1) / at_once, 2 * FRONT_BLOCKS) : 0;
  if (rows > COUNT_ROWS) {
    chain.launch(count_kernel, dim3(f.blocks_h), FRONT_THREADS, 0, 0, f, s.counts);
    f.counts = s.counts;
  }
  chain.launch(front_kernel<T>, dim3(f.blocks_h + f.blocks_w), FRONT_THREADS, 0, 0, f);
  if (SPLIT) {
    const int on_h = some((z.rows_up + at_once - 1) / at_once, FRONT_BLOCKS);
    chain.launch(pairs_kernel, dim3(on_h + f.blocks_w), FRONT_THREADS, 0, 0, f, on_h, f.blocks_w);
  }
  int rc = launch_error(chain.err, who);
  if (rc != B2_OK) return rc;

  const TileOperand h_k{s.h_hi, s.h_lo, z.rows_up, pitch, pitch, false}, h_mn{s.h_hi, s.h_lo, pitch, z.rows_up, pitch, true};
  const void* w_hi = z.copy_w ? (const void*)s.w_hi : c.w;
  const long long w_width = z.copy_w ? pitch : width, w_ld = z.copy_w ? pitch : (long long)c.ldw;
  const TileOperand w_k{w_hi, s.w_lo, vocab, w_width, w_ld, false}, w_mn{w_hi, s.w_lo, w_width, vocab, w_ld, true};
  LogitParams lp{};
  lp.meta = s.meta;
  lp.vocab = vocab;
  lp.v_count = vocab;
  lp.kblocks = (width + TILE_K - 1) / TILE_K;
  lp.row_pitch = z.rows_up;
  lp.target = s.target;
  lp.parts = s.parts;
  lp.target_logit = s.target_logit;
  lp.row_stat = s.row_stat;
  lp.d_hi = s.d_hi;
  lp.d_lo = s.d_lo;
  lp.ld_d = z.piece;
  lp.x = s.x;
  lp.ld_x = z.ld_x;
  lp.x_parts = z.x_parts;
  lp.all_rows = rows;
  const int grads = c.dh || c.dw;
  const bool sums = !SPLIT && lp.kblocks > StatOp<Pairs, true, false, false>::SUM;
  if (z.by_rows) {
    rc = tile_launch<PlainOp<One>>(who, h_k, w_k, nullptr, lp, !SPLIT, tiles_of<One>(rows, vocab) * z.x_parts, sms, chain);
    if (rc != B2_OK) return rc;
    chain.launch(row_kernel<SPLIT>, dim3((rows + TILE_K - 1) / TILE_K * TILE_K), ROW_THREADS, 0, 0, lp, s.row_of, c.row_loss, grads);
  } else {
    int run;
    const int lists = z.one ? lists_of<One>(rows, vocab, sms, &run) : lists_of<Pairs>(rows, vocab, sms, &run);
    const std::true_type yes;
    const std::false_type no;
    auto by_run = [&](auto form, auto keep, auto goes_on) {
      typedef decltype(form) F;
      constexpr bool KEEP = decltype(keep)::value, RUN = decltype(goes_on)::value;
      return sums ? tile_launch<StatOp<F, !SPLIT, KEEP, RUN>> : tile_launch<StatOp<F, false, KEEP, RUN>>;
    };
    auto by_keep = [&](auto form, auto keep) { return run ? by_run(form, keep, yes) : by_run(form, keep, no); };
    auto stat_of = [&](auto form) { return z.keep ? by_keep(form, yes) : by_keep(form, no); };
    auto stat = z.one ? stat_of(One()) : stat_of(Pairs());
    rc = stat(who, h_k, w_k, nullptr, lp, !SPLIT, z.one ? tiles_of<One>(rows, vocab) : tiles_of<Pairs>(rows, vocab), sms, chain);
    if (rc != B2_OK) return rc;
    chain.launch(join_rows_kernel, dim3((rows + 31) / 32), 1024, 0, 0, s.parts, z.rows_up, lists, s.meta, s.target_logit, s.row_of, s.row_stat,
                 c.row_loss);
  }
  rc = launch_error(chain.err, who);
  if (rc != B2_OK || !grads) return rc;

  ProductParams pp{};
  pp.meta = s.meta;
  pp.width = width;
  pp.scale = c.scale;
  pp.acc = s.acc;
  pp.slots = s.slots;
  // dh's k range is shared out evenly over CTAs or pairs, in parts of eight k-blocks at least
  const long long dh_one = tiles_of<One>(rows, width), dh_pairs = tiles_of<Pairs>(rows, width), dh_k = ((vocab < z.piece ? vocab : z.piece) + TILE_K - 1) / TILE_K;
  const int pairs = sms / 2 < MOST_PAIRS ? sms / 2 : MOST_PAIRS;
  auto share_of = [&](long long tiles, int over) {
    const long long k = (tiles * dh_k + over - 1) / over, least = dh_k < 8 ? dh_k : 8;
    return k > least ? k : least;
  };
  const bool h_one = single_ctas<SPLIT>(1, share_of(dh_one, 2 * pairs), 1, share_of(dh_pairs, pairs));
  pp.pairs = h_one ? 2 * pairs : pairs;
  // long: the k range of a tile, or of a CTA's part where all tiles are cut. No part of such a range is empty, which the long form leaves out.
  auto is_long = [](long long k) { return !SPLIT && k > 4 * LONG_SUM; };
  const long long dh_tiles = h_one ? dh_one : dh_pairs;
  const bool dh_long = is_long(dh_tiles >= pp.pairs ? dh_k : share_of(dh_tiles, pp.pairs));
  auto hidden = h_one ? (dh_long ? tile_launch<HiddenOp<One, !SPLIT>> : tile_launch<HiddenOp<One, false>>)
                      : (dh_long ? tile_launch<HiddenOp<Pairs, !SPLIT>> : tile_launch<HiddenOp<Pairs, false>>);
  pp.full_kblocks = (int)(z.piece / TILE_K);
  pp.ld_acc = pitch;
  pp.dw = c.dw;
  pp.ld_dw = (long long)c.ld_dw;
  pp.out_bf16 = !SPLIT;
  pp.vec = c.ld_dw % 4 == 0 && reinterpret_cast<uintptr_t>(c.dw) % (4 * sizeof(T)) == 0;
  const TileOperand d_k{s.d_hi, s.d_lo, z.rows_up, z.piece, z.piece, false}, d_mn{s.d_hi, s.d_lo, z.piece, z.rows_up, z.piece, true};
  pp.by_tma = !SPLIT && reinterpret_cast<uintptr_t>(c.dw) % 16 == 0 && c.ld_dw % 8 == 0 && width % 8 == 0;
  const TileResult dw_out{c.dw, vocab, width, (long long)c.ld_dw};
  const TileResult d_out{s.d_hi, z.rows_up, z.piece, z.piece};
  for (int v0 = 0; v0 < vocab; v0 += (int)z.piece) {
    const int count = vocab - v0 < z.piece ? vocab - v0 : (int)z.piece;
    lp.v_begin = pp.v_begin = v0;
    lp.v_count = pp.v_count = count;
    pp.first = v0 == 0;
    if (z.by_rows) {  // d is there
    } else if (z.keep) {
      const long long r = (rows + TILE_K - 1) / TILE_K * TILE_K, n = (count + TILE_K - 1) / TILE_K * TILE_K;
      chain.launch(kept_kernel<SPLIT>, dim3(blocks((r * n / 8 + 255) / 256)), 256, 0, 0, lp);
      rc = launch_error(chain.err, who);
    } else {
      rc = (sums ? tile_launch<GradOp<Pairs, !SPLIT>> : tile_launch<GradOp<Pairs, false>>)(who, h_k, w_k, SPLIT ? nullptr : &d_out, lp, !SPLIT, tiles_of<Pairs>(rows, count), sms, chain);
    }
    if (rc == B2_OK && c.dh) rc = hidden(who, d_k, w_mn, nullptr, pp, !SPLIT, pp.pairs, sms, chain);
    if (rc == B2_OK && c.dw) {
      const long long k = (rows + TILE_K - 1) / TILE_K;
      const bool one = single_ctas<SPLIT>((tiles_of<One>(count, width) + sms - 1) / sms, k, (tiles_of<Pairs>(count, width) + pairs - 1) / pairs, k);
      auto weight = one ? (is_long(k) ? tile_launch<WeightOp<One, !SPLIT>> : tile_launch<WeightOp<One, false>>)
                        : (is_long(k) ? tile_launch<WeightOp<Pairs, !SPLIT>> : tile_launch<WeightOp<Pairs, false>>);
      rc = weight(who, d_mn, h_mn, pp.by_tma ? &dw_out : nullptr, pp, !SPLIT, one ? tiles_of<One>(count, width) : tiles_of<Pairs>(count, width), sms, chain);
    }
    if (rc != B2_OK) return rc;
  }
  if (c.dh) {
    const int vec = c.ld_dh % 4 == 0 && reinterpret_cast<uintptr_t>(c.dh) % (4 * sizeof(T)) == 0;
    chain.launch(h_one ? spread_rows_kernel<T, One> : spread_rows_kernel<T, Pairs>, dim3(blocks(rows)), 256, 0, 0, pp, s.slot_of, rows, vec, static_cast<T*>(c.dh), c.ld_dh);
    rc = launch_error(chain.err, who);
  }
  return rc;
}

int check_sizes(const char* who, size_t rows, size_t width, size_t vocab, int dtype) {
  if (!dtype_ok(dtype)) return call_error(B2_ERR_INVALID, "%s: dtype %d", who, dtype);
  if (rows > (1u << 24)) return call_error(B2_ERR_INVALID, "%s: %zu rows, at most %u", who, rows, 1u << 24);
  if (width < 1 || width > (1u << 20)) return call_error(B2_ERR_INVALID, "%s: width %zu", who, width);
  if (vocab < 1 || vocab > (1u << 24)) return call_error(B2_ERR_INVALID, "%s: vocab %zu", who, vocab);
  if (rows * vocab > (1ull << 44)) return call_error(B2_ERR_INVALID, "%s: %zu rows x %zu columns of logits, at most 2^44", who, rows, vocab);
  return B2_OK;
}

}  // namespace

cudaError_t xent_waits_given_up(unsigned int* count, unsigned int* role, cudaStream_t s) {
  TileReport r{};
  const cudaError_t e = tile_report_read(&r, s);
  *count = r.count;
  *role = r.role;
  return e;
}

}  // namespace b2

using namespace b2;

extern "C" {

int b2_xent_workspace(size_t rows, size_t width, size_t vocab, int dtype, int grads, const void* w, size_t ldw, size_t* bytes) {
  int rc = check_sizes("b2_xent_workspace", rows, width, vocab, dtype);
  if (rc != B2_OK) return rc;
  if (!bytes) return call_error(B2_ERR_INVALID, "b2_xent_workspace: null pointer");
  Space s;
  *bytes = rows ? space_of(sizes_of(rows, width, vocab, dtype, grads, w, ldw), rows, vocab, grads, nullptr, &s) : 0;
  return B2_OK;
}

int b2_xent(size_t rows, size_t width, size_t vocab, int dtype, const void* h, size_t ldh, const void* w, size_t ldw,
            const void* targets, int token_bytes, float scale, float* row_loss, void* dh, size_t ld_dh, void* dw,
            size_t ld_dw, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_sizes("b2_xent", rows, width, vocab, dtype);
  if (rc != B2_OK) return rc;
  if (token_bytes != 4 && token_bytes != 8) return call_error(B2_ERR_INVALID, "b2_xent: token_bytes is 4 or 8, not %d", token_bytes);
  if (!w || (rows && (!h || !targets || !row_loss || !workspace))) return call_error(B2_ERR_INVALID, "b2_xent: null pointer");
  if (ldh < width || ldw < width || (dh && ld_dh < width) || (dw && ld_dw < width))
    return call_error(B2_ERR_INVALID, "b2_xent: leading dimension smaller than the width");
  const size_t e = dtype_bytes(dtype);
  if ((reinterpret_cast<size_t>(h) | reinterpret_cast<size_t>(w) | reinterpret_cast<size_t>(dh) | reinterpret_cast<size_t>(dw)) % e ||
      reinterpret_cast<size_t>(targets) % token_bytes || reinterpret_cast<size_t>(row_loss) % 4)
    return call_error(B2_ERR_INVALID, "b2_xent: a pointer is not aligned to its elements");
  if (reinterpret_cast<size_t>(workspace) % 256) return call_error(B2_ERR_INVALID, "b2_xent: the workspace is not on a 256-byte boundary");
  const int grads = dh || dw;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Sizes z{};
  Space s;
  size_t need = 0;
  if (rows) {
    z = sizes_of(rows, width, vocab, dtype, grads, w, ldw);
    need = space_of(z, rows, vocab, grads, workspace, &s);
    if (workspace_bytes < need) return call_error(B2_ERR_INVALID, "b2_xent: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  }
  int sms;
  if ((rc = lm_device(&sms)) != B2_OK) return rc;
  if (sms > 2 * MOST_PAIRS) sms = 2 * MOST_PAIRS;  // what the workspace is made for
  Extent args[] = {extent("h", h, rows, width * e, ldh * e, false), extent("w", w, vocab, width * e, ldw * e, false),
                   extent("targets", targets, 1, rows * token_bytes, rows * token_bytes, false), extent("row_loss", row_loss, 1, rows * 4, rows * 4, true),
                   extent("dh", dh, rows, width * e, ld_dh * e, true), extent("dw", dw, vocab, width * e, ld_dw * e, true),
                   extent("the workspace", workspace, 1, need, need, true)};
  if ((rc = refuse_overlap("b2_xent", args, 7)) != B2_OK) return rc;
  if (rows == 0) return dw ? launch_error(cudaMemset2DAsync(dw, ld_dw * e, 0, width * e, vocab, st), "b2_xent") : B2_OK;
  const XentCall c{rows, width, vocab, dtype, h, ldh, w, ldw, targets, token_bytes == 8, scale, row_loss, dh, ld_dh, dw, ld_dw};
  return z.split ? xent_run<true>(c, z, s, sms, st) : xent_run<false>(c, z, s, sms, st);
}

}  // extern "C"
