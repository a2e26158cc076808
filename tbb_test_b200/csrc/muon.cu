// Momentum and an orthogonalised update of matrices, by Newton-Schulz products:
//
//   m = mu m + g        u = g + mu m (Nesterov) or m        x = u / (|u|_F + eps)
//   `steps` times:  a = x x'   x = (A I + B a + C a a) x          with A, B, C = 3.4445, -4.7750, 2.0315
//   w = (1 - lr decay) w - lr scale x
//
// The polynomial A s + B s^3 + C s^5 takes every singular value s of x to between 0.7 and 1.2 in five steps, so that the
// update is x's nearest matrix with equal singular values, roughly. Small singular values grow by A each step, and with
// them every rounding error of the products before: 485 times in five steps. That is why products are of fp16 pairs
// (22 bits, lm_tile.cuh) and not of bf16: x is at most 1 in norm and a, B a + C a a stay below 4, so fixed powers of two
// bring them into fp16's range.
//
// With r the smaller and c the larger side of a matrix a step has 2 r^2 c operations for a, 2 r^3 for a a and 2 r^2 c for the
// new x, all on the tensor cores. a and a a are symmetric: only tiles on and above the diagonal are computed, which stores
// each tile twice. The smaller side is m for wide matrices and n for tall ones; tall ones are not transposed, as the
// tile kernel reads operands along either side. A I is added to the middle factor, whose tiles it only touches on the
// diagonal, so that x is read once per step. The last step's tiles update w as they are finished.
//
// Matrices of a call have one shape and go side by side, so that small ones fill the GPU together. Sides are rounded up to
// 64, a k-block, with zeros, which stay zeros.
#include <memory>
#include <new>

#include "lm_tile.cuh"
#include "wait_reports.h"

namespace b2 {
namespace {

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
// powers of two on x (norm at most 1.3), a (1.6) and the middle factor (3.5): below fp16's 65504 with room
constexpr float X_UP = 8192.f, A_UP = 16384.f, P_UP = 8192.f;
// k-blocks per hand-over of sums: 16 leaves 3e-6 of x, 8 would halve that and take 3 % longer (8 matrices of 4096 x 4096)
constexpr int MUON_SUM = 16;
constexpr int MUON_GROUP = 16;   // matrices per launch at most
constexpr int NORM_PARTS = 256;  // partial sums of a matrix's squares

struct MatrixList {
  float* w[MUON_GROUP];
  __nv_bfloat16* copy[MUON_GROUP];
  float* m[MUON_GROUP];
  const void* g[MUON_GROUP];
};
struct Elementwise {
  MatrixList list;
  int rows, cols;
  long long ld_m, ld_g;
  int rows_up, cols_up;
  float mu, eps;
  int nesterov;
  double* parts;  // matrices x NORM_PARTS
  __half *x_hi, *x_lo;
};

__device__ __forceinline__ float update_of(float g, float m, const Elementwise& p) {
  return p.nesterov ? fmaf(p.mu, m, g) : m;
}

// m = mu m + g, and the sum of u's squares: each block has its own place for it, so that the sum has one order. VEC: rows
// are whole groups of four elements on 16-byte (g: 8-byte) boundaries.
template <typename G, bool VEC>
__global__ void __launch_bounds__(256) momentum_kernel(const __grid_constant__ Elementwise p) {
  __shared__ double part[8];
  float* m = p.list.m[blockIdx.y];
  const G* g = static_cast<const G*>(p.list.g[blockIdx.y]);
  let_next_start();
  double sum = 0.0;
  constexpr int E = VEC ? 4 : 1, AHEAD = 4;
  const int per_row = p.cols / E;
  const long long all = (long long)p.rows * per_row, stride = (long long)gridDim.x * 256;
  for (long long i0 = (long long)blockIdx.x * 256 + threadIdx.x; i0 < all; i0 += stride * AHEAD) {
    typedef Elems<float, 4 * E> M;
    typedef Elems<G, (int)sizeof(G) * E> V;
    typename M::raw mr[AHEAD];
    typename V::raw gr[AHEAD];
    float* to[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const long long i = i0 + u * stride;
      to[u] = nullptr;
      if (i < all) {
        const int r = (int)(i / per_row), c = (int)(i - (long long)r * per_row) * E;
        to[u] = m + (long long)r * p.ld_m + c;
        mr[u] = *reinterpret_cast<const typename M::raw*>(to[u]);
        gr[u] = __ldg(reinterpret_cast<const typename V::raw*>(g + (long long)r * p.ld_g + c));
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (!to[u]) continue;
      float mv[E], gv[E];
      M::get(mr[u], mv);
      V::get(gr[u], gv);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        mv[e] = fmaf(p.mu, mv[e], gv[e]);
        const double x = update_of(gv[e], mv[e], p);
        sum = fma(x, x, sum);
      }
      *reinterpret_cast<typename M::raw*>(to[u]) = M::put(mv);
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < 8; ++k) sum += part[k];
    p.parts[blockIdx.y * NORM_PARTS + blockIdx.x] = sum;
  }
}

// x = u / (|u| + eps) as a pair, zeros in the rows and columns that fill up.
template <typename G, bool VEC>
__global__ void __launch_bounds__(256) normalise_kernel(const __grid_constant__ Elementwise p, int parts) {
  __shared__ double part[8];
  after_previous();
  let_next_start();
  double sum = (int)threadIdx.x < parts ? p.parts[blockIdx.y * NORM_PARTS + threadIdx.x] : 0.0;
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0.0;
  for (int k = 0; k < 8; ++k) sum += part[k];
  // A matrix of zeros stays one without an eps too; a norm whose reciprocal is no normal fp32 number takes a power of two first.
  const double norm = sqrt(sum) + (double)p.eps;
  const float first = norm < 0x1p-100 ? 0x1p100f : norm > 0x1p100 ? 0x1p-100f : 1.f, by = sum == 0.0 ? 0.f : (float)(1.0 / (norm * first));
  const float* m = p.list.m[blockIdx.y];
  const G* g = static_cast<const G*>(p.list.g[blockIdx.y]);
  const size_t base = (size_t)blockIdx.y * p.rows_up * p.cols_up;
  const int per_row = p.cols_up / 4;
  const long long all = (long long)p.rows_up * per_row, stride = (long long)gridDim.x * 256;
#pragma unroll 4
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += stride) {
    const int r = (int)(i / per_row), c = (int)(i - (long long)r * per_row) * 4;
    const float* mr = m + (long long)r * p.ld_m + c;
    const G* gr = g + (long long)r * p.ld_g + c;
    float mv[4] = {0.f, 0.f, 0.f, 0.f}, gv[4] = {0.f, 0.f, 0.f, 0.f};
    if (VEC) {
      if (r < p.rows && c < p.cols) {
        Elems<float, 16>::get(*reinterpret_cast<const uint4*>(mr), mv);
        typedef Elems<G, 4 * (int)sizeof(G)> V;
        if (p.nesterov) V::get(__ldg(reinterpret_cast<const typename V::raw*>(gr)), gv);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (r < p.rows && c + e < p.cols) {
          mv[e] = mr[e];
          if (p.nesterov) gv[e] = (float)gr[e];
        }
    }
    __half hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) split_half(update_of(gv[e], mv[e], p) * first * by * X_UP, hi[e], lo[e]);
    const size_t at = base + (size_t)r * p.cols_up + c;
    *reinterpret_cast<uint2*>(p.x_hi + at) = *reinterpret_cast<const uint2*>(hi);
    *reinterpret_cast<uint2*>(p.x_lo + at) = *reinterpret_cast<const uint2*>(lo);
  }
}

// ------------------------------------------------------------------ products

constexpr float A_UNIT = A_UP / (X_UP * X_UP);  // of sums of x x'

// Symmetric results, side x side per matrix: a = x x' (middle 0), or A I + B a + C a a from a a (middle 1).
struct SymmetricParams {
  int side, count, kblocks;
  long long a_step, b_step;  // rows (or k) between matrices in the operands
  int steps_k;               // 1: matrices lie behind one another along k
  const __half *a_hi, *a_lo;
  __half *to_hi, *to_lo;
  int parts;     // PARTS: of the k range
  float* sums;   // matrices x parts x side x side
};
enum Symmetric { WHOLE, MIDDLE_FACTOR, PARTS };
template <Symmetric KIND, bool ONE>
struct SymmetricOp {
  typedef SymmetricParams Params;
  typedef TileForm<true, ONE> Form;
  static constexpr bool MIDDLE = KIND == MIDDLE_FACTOR;
  static constexpr bool STORES = false, LONG = true, INFINITE = false;
  static constexpr int SUM = MUON_SUM;
  const SymmetricParams& p;
  int m_blocks, n_blocks, per;
  __device__ explicit SymmetricOp(const SymmetricParams& q, const TileMaps&) : p(q) {
    m_blocks = (p.side + Form::M - 1) / Form::M;
    n_blocks = (p.side + Form::BN - 1) / Form::BN;
    per = m_blocks * n_blocks - m_blocks * (m_blocks - 1);  // row block i has column blocks 2 i and up
  }
  __device__ int tiles() const { return per * p.count * (KIND == PARTS ? p.parts : 1); }
  __device__ Tile tile(int t) const {
    Tile r;
    r.z = t / per;  // PARTS: a part of a matrix
    int in = t - r.z * per, i = 0;
    while (in >= n_blocks - 2 * i) in -= n_blocks - 2 * i++;
    r.m0 = i * Form::M;
    r.n0 = (2 * i + in) * Form::BN;
    const int matrix = KIND == PARTS ? r.z / p.parts : r.z, off = matrix * (int)p.a_step;
    r.a_mn = r.m0 + (p.steps_k ? 0 : off);
    r.b_mn = r.n0 + (p.steps_k ? 0 : off);
    r.a_k = r.b_k = p.steps_k ? off : 0;
    r.kblocks = p.kblocks;
    if (KIND == PARTS) {
      const int part = r.z - matrix * p.parts, from = p.kblocks * part / p.parts;
      r.a_k = r.b_k += from * TILE_K;
      r.kblocks = p.kblocks * (part + 1) / p.parts - from;
    }
    return r;
  }
  // a is loaded while the products are summed: it is what a small matrix's middle factor would wait for otherwise (5.6 against 2.7 us
  // for the elements of a tile)
  static constexpr int QUADS = Form::COLS / 4;
  Pair4 a[QUADS];
  __device__ __forceinline__ void begin(const Tile& t, int row0, int col0, int lane) {
    if (!MIDDLE || row0 >= p.side || col0 >= p.side) return;
    const __half *hi = p.a_hi + (long long)t.z * p.side * p.side, *lo = p.a_lo + (long long)t.z * p.side * p.side;
#pragma unroll
    for (int i = 0; i < QUADS; ++i)
      a[i] = load_pair(hi, lo, (long long)(row0 + quad_row<16>(i & 3, lane)) * p.side + col0 + (i >> 2) * 16 + quad_col<16>(lane));
  }
  __device__ __forceinline__ void chunk(const Tile& t, int row0, int col0, float (&v)[16], uint8_t* stage, int lane) {
    if (row0 >= p.side || col0 >= p.side) return;  // uniform: sides are multiples of 64
    const long long base = (long long)t.z * p.side * p.side;
    if constexpr (KIND == PARTS) {
      by_rows(row0, col0, v, stage, lane, [&](int, int r, int c, const float4& y) { *reinterpret_cast<float4*>(p.sums + base + (long long)r * p.side + c) = y; });
      return;
    }
    constexpr float unit = MIDDLE ? P_UP * NS_C / (A_UP * A_UP) : A_UNIT, b = P_UP * NS_B / A_UP;
    const bool second = QUADS > 4 && (col0 - t.n0) & 16;  // of the warp's two chunks
    float4 x[4];
    by_rows(row0, col0, v, stage, lane, [&](int i, int r, int c, const float4& y) {
      x[i] = make_float4(y.x * unit, y.y * unit, y.z * unit, y.w * unit);
      if (MIDDLE) {
        const float4 old = pair_value(second ? a[QUADS - 4 + i] : a[i]);
        x[i] = make_float4(fmaf(b, old.x, x[i].x), fmaf(b, old.y, x[i].y), fmaf(b, old.z, x[i].z), fmaf(b, old.w, x[i].w));
        if (r == c) x[i].x += NS_A * P_UP;
        if (r == c + 1) x[i].y += NS_A * P_UP;
        if (r == c + 2) x[i].z += NS_A * P_UP;
        if (r == c + 3) x[i].w += NS_A * P_UP;
      }
      store_pair(p.to_hi, p.to_lo, base + (long long)r * p.side + c, x[i]);
    });
    if (t.n0 >= t.m0 + Form::M)  // on the diagonal both halves are computed
      by_columns(row0, col0, x, stage, lane, [&](int r, int c, const float4& y) { store_pair(p.to_hi, p.to_lo, base + (long long)r * p.side + c, y); });
  }
  __device__ __forceinline__ void end(const Tile&, int, int) {}
};

// a from its parts on and above the diagonal, in order, 32 x 32 elements per block; the block on the other side of the diagonal gets
// them transposed.
__global__ void __launch_bounds__(256) join_parts_kernel(const float* __restrict__ sums, int parts, int side, __half* __restrict__ hi, __half* __restrict__ lo) {
  __shared__ float turned[32][33];
  after_previous();
  let_next_start();
  const int n = side / 32, z = blockIdx.y;
  int in = blockIdx.x, i = 0;
  while (in >= n - i) in -= n - i++;
  const int r = threadIdx.x >> 3, c = (threadIdx.x & 7) * 4, j = i + in;
  const long long all = (long long)side * side;
  const float* from = sums + z * parts * all + (long long)(i * 32 + r) * side + j * 32 + c;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = 0; k < parts; ++k) {
    const float4 y = *reinterpret_cast<const float4*>(from + k * all);
    x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
  }
  x = make_float4(x.x * A_UNIT, x.y * A_UNIT, x.z * A_UNIT, x.w * A_UNIT);
  store_pair(hi, lo, z * all + (long long)(i * 32 + r) * side + j * 32 + c, x);
  if (i == j) return;  // computed on both sides of the diagonal
  turned[c][r] = x.x;
  turned[c + 1][r] = x.y;
  turned[c + 2][r] = x.z;
  turned[c + 3][r] = x.w;
  __syncthreads();
  store_pair(hi, lo, z * all + (long long)(j * 32 + r) * side + i * 32 + c, make_float4(turned[r][c], turned[r][c + 1], turned[r][c + 2], turned[r][c + 3]));
}

// The new x: middle factor times x (wide) or x times middle factor (tall); the last one updates w instead.
struct NextParams {
  MatrixList list;
  int rows, cols, rows_up, cols_up, count, kblocks, wide;
  __half *to_hi, *to_lo;
  long long ld_w, ld_copy;
  float keep, step;  // w = keep w - step x
  int vec_w, vec_copy;
};
template <bool LAST, bool ONE>
struct NextOp {
  typedef NextParams Params;
  typedef TileForm<true, ONE> Form;
  static constexpr bool STORES = false, LONG = true, INFINITE = false;
  static constexpr int SUM = MUON_SUM;
  const NextParams& p;
  int m_blocks, n_blocks;
  __device__ explicit NextOp(const NextParams& q, const TileMaps&) : p(q) {
    m_blocks = (p.rows_up + Form::M - 1) / Form::M;
    n_blocks = (p.cols_up + Form::BN - 1) / Form::BN;
  }
  __device__ int tiles() const { return m_blocks * n_blocks * p.count; }
  __device__ Tile tile(int t) const {
    Tile r;
    const int per = m_blocks * n_blocks;
    r.z = t / per;
    const int in = t - r.z * per;
    // bands of eight row blocks: what the pairs work on at a time is about square
    const int b = in / (8 * n_blocks), at = in - b * 8 * n_blocks, tall = min(8, m_blocks - 8 * b);
    r.m0 = (8 * b + at % tall) * Form::M;
    r.n0 = at / tall * Form::BN;
    r.a_mn = r.m0 + r.z * p.rows_up;
    r.a_k = 0;
    r.b_mn = r.n0 + (p.wide ? 0 : r.z * p.cols_up);
    r.b_k = p.wide ? r.z * p.rows_up : 0;
    r.kblocks = p.kblocks;
    return r;
  }
  static constexpr int QUADS = Form::COLS / 4;
  float4 old[QUADS];  // of w, loaded while the last step's products are summed
  __device__ __forceinline__ void begin(const Tile& t, int row0, int col0, int lane) {
    if (!LAST) return;
    const float* w = p.list.w[t.z];
#pragma unroll
    for (int i = 0; i < QUADS; ++i) {
      const int r = row0 + quad_row<16>(i & 3, lane), c = col0 + (i >> 2) * 16 + quad_col<16>(lane);
      old[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r >= p.rows || c >= p.cols) continue;
      const float* from = w + (long long)r * p.ld_w + c;
      if (p.vec_w && c + 4 <= p.cols) {
        old[i] = *reinterpret_cast<const float4*>(from);
      } else {
        old[i].x = from[0];
        if (c + 1 < p.cols) old[i].y = from[1];
        if (c + 2 < p.cols) old[i].z = from[2];
        if (c + 3 < p.cols) old[i].w = from[3];
      }
    }
  }
  __device__ __forceinline__ void chunk(const Tile& t, int row0, int col0, float (&v)[16], uint8_t* stage, int lane) {
    if (row0 >= p.rows_up || col0 >= p.cols_up) return;
    if (!LAST) {
      const long long base = (long long)t.z * p.rows_up * p.cols_up;
      constexpr float unit = 1.f / P_UP;
      by_rows(row0, col0, v, stage, lane, [&](int, int r, int c, const float4& x) {
        store_pair(p.to_hi, p.to_lo, base + (long long)r * p.cols_up + c, make_float4(x.x * unit, x.y * unit, x.z * unit, x.w * unit));
      });
      return;
    }
    const float unit = p.step / (X_UP * P_UP);
    const bool second = QUADS > 4 && (col0 - t.n0) & 16;  // of the warp's two chunks
    float* w = p.list.w[t.z];
    __nv_bfloat16* copy = p.list.copy[t.z];
    by_rows(row0, col0, v, stage, lane, [&](int i, int r, int c, const float4& x) {
      if (r >= p.rows || c >= p.cols) return;
      const float4 o = second ? old[QUADS - 4 + i] : old[i];
      const float f[4] = {fmaf(p.keep, o.x, -x.x * unit), fmaf(p.keep, o.y, -x.y * unit), fmaf(p.keep, o.z, -x.z * unit), fmaf(p.keep, o.w, -x.w * unit)};
      float* to = w + (long long)r * p.ld_w + c;
      const bool whole = c + 4 <= p.cols;
      if (p.vec_w && whole) {
        *reinterpret_cast<float4*>(to) = make_float4(f[0], f[1], f[2], f[3]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (c + k < p.cols) to[k] = f[k];
      }
      if (!copy) return;
      __nv_bfloat16* out = copy + (long long)r * p.ld_copy + c;
      if (p.vec_copy && whole) {
        *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]));
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (c + k < p.cols) out[k] = __float2bfloat16_rn(f[k]);
      }
    });
  }
  __device__ __forceinline__ void end(const Tile&, int, int) {}
};

// ------------------------------------------------------------------ host side

struct MuonSizes {
  int rows_up, cols_up, side, group;
  int most_parts;  // of a, over all matrices of a group
};
constexpr int MOST_SMS = 148;
long long symmetric_tiles(int side, int bm) {
  const long long m = (side + bm - 1) / bm, n = (side + bm / 2 - 1) / (bm / 2);
  return m * n - m * (m - 1);
}
// A product x x' of few tiles and a long k range goes in parts, as many as there are SMs for and of four k-blocks at least. In clocks: 832 per
// k-block, 4500 for the kernel that joins them, 1 per 250 elements of every part. 4000 x 256 189 -> 123 us per update, 512 x 8192 370 -> 236,
// 64 x 2048 115 -> 86; 1024 x 1024 stays whole (164 us, 172 in two parts).
int parts_of(int count, int side, int kblocks, int sms) {
  long long most = sms / (symmetric_tiles(side, 128) * count);
  if (most > kblocks / 4) most = kblocks / 4;
  long long parts = 1, least = 832ll * kblocks - 4500;
  for (int n = 2; n <= most; ++n) {
    const long long clocks = 832ll * ((kblocks + n - 1) / n) + (long long)n * count * side * side / 250;
    if (clocks < least) {
      least = clocks;
      parts = n;
    }
  }
  return (int)parts;
}
MuonSizes muon_sizes(int count, int rows, int cols) {
  MuonSizes z;
  z.rows_up = (rows + TILE_K - 1) / TILE_K * TILE_K;
  z.cols_up = (cols + TILE_K - 1) / TILE_K * TILE_K;
  z.side = rows <= cols ? z.rows_up : z.cols_up;
  // as many side by side as give every pair of SMs several tiles of the smallest product
  const long long blocks = (z.side + 127) / 128, per = (blocks * blocks / 2 + blocks) / 2 + 1;
  long long group = (4 * 74 + per - 1) / per;
  if (group > MUON_GROUP) group = MUON_GROUP;
  z.group = count < group ? count : (int)group;
  const int long_side = rows <= cols ? z.cols_up : z.rows_up;
  z.most_parts = 0;
  for (int n = 1; n <= z.group; ++n) {
    const int parts = parts_of(n, z.side, long_side / TILE_K, MOST_SMS);
    if (parts > 1 && parts * n > z.most_parts) z.most_parts = parts * n;
  }
  return z;
}
struct MuonSpace {
  double* parts;
  float* sums;
  __half *x_hi[2], *x_lo[2], *a_hi, *a_lo, *p_hi, *p_lo;
};
size_t muon_space(const MuonSizes& z, void* base, MuonSpace* s) {
  Carver c(base);
  const size_t x = (size_t)z.group * z.rows_up * z.cols_up, a = (size_t)z.group * z.side * z.side;
  s->parts = c.take<double>((size_t)z.group * NORM_PARTS);
  for (int i = 0; i < 2; ++i) {
    s->x_hi[i] = c.take<__half>(x);
    s->x_lo[i] = c.take<__half>(x);
  }
  s->a_hi = c.take<__half>(a);
  s->a_lo = c.take<__half>(a);
  s->p_hi = c.take<__half>(a);
  s->p_lo = c.take<__half>(a);
  s->sums = c.take<float>((size_t)z.most_parts * z.side * z.side);
  return c.used;
}

int muon_group(const MatrixList& list, int count, int rows, int cols, int grad_dtype, size_t ld_w, size_t ld_copy, size_t ld_m,
               size_t ld_g, const b2_muon_options& o, const MuonSizes& z, const MuonSpace& s, int sms, cudaStream_t st) {
  const char* who = "b2_muon";
  Elementwise e{};
  e.list = list;
  e.rows = rows;
  e.cols = cols;
  e.ld_m = (long long)ld_m;
  e.ld_g = (long long)ld_g;
  e.rows_up = z.rows_up;
  e.cols_up = z.cols_up;
  e.mu = o.momentum;
  e.eps = o.eps;
  e.nesterov = o.nesterov;
  e.parts = s.parts;
  e.x_hi = s.x_hi[0];
  e.x_lo = s.x_lo[0];
  bool vec = cols % 4 == 0 && ld_m % 4 == 0 && ld_g % 4 == 0;
  for (int i = 0; i < count; ++i)
    if (reinterpret_cast<uintptr_t>(list.m[i]) % 16 || reinterpret_cast<uintptr_t>(list.g[i]) % (4 * dtype_bytes(grad_dtype))) vec = false;
  auto blocks = [&](long long threads, int most) {  // of a matrix: eight per SM over all of them
    long long n = (threads + 255) / 256, fair = (8 * sms + count - 1) / count;
    if (n > fair) n = fair;
    return (int)(n > most ? most : n);
  };
  const int parts = blocks((long long)rows * cols / (vec ? 16 : 4) + 1, NORM_PARTS);
  const dim3 grid(parts, count), grid2(blocks((long long)z.rows_up * z.cols_up / 8, 1 << 20), count);
  Chain chain(st);
  auto start = [&](auto momentum, auto normalise) {
    chain.launch(momentum, grid, 256, 0, 0, e);
    chain.launch(normalise, grid2, 256, 0, 0, e, parts);
  };
  if (grad_dtype == B2_DTYPE_BF16) {
    if (vec) start(momentum_kernel<__nv_bfloat16, true>, normalise_kernel<__nv_bfloat16, true>);
    else start(momentum_kernel<__nv_bfloat16, false>, normalise_kernel<__nv_bfloat16, false>);
  } else {
    if (vec) start(momentum_kernel<float, true>, normalise_kernel<float, true>);
    else start(momentum_kernel<float, false>, normalise_kernel<float, false>);
  }
  int rc = launch_error(chain.err, who);
  const bool wide = rows <= cols;
  const long long x_rows = (long long)z.rows_up * count, a_rows = (long long)z.side * count;
  // Tiles of a symmetric and of a full product, in tiles of bm rows
  auto symmetric = [&](int bm) { return symmetric_tiles(z.side, bm) * count; };
  auto full = [&](int bm) { return (long long)((z.rows_up + bm - 1) / bm) * ((z.cols_up + bm / 2 - 1) / (bm / 2)) * count; };
  auto one_is_less = [&](long long one, long long pairs, int kblocks) {
    return single_ctas<true>((one + sms - 1) / sms, kblocks, (pairs + sms / 2 - 1) / (sms / 2), kblocks);
  };
  const int k_a = (wide ? z.cols_up : z.rows_up) / TILE_K, k_b = z.side / TILE_K;
  const bool a_one = one_is_less(symmetric(128), symmetric(256), k_a), p_one = one_is_less(symmetric(128), symmetric(256), k_b),
             full_one = one_is_less(full(128), full(256), k_b);
  const int a_parts = parts_of(count, z.side, k_a, sms < MOST_SMS ? sms : MOST_SMS);
  const long long a_tiles = symmetric(a_one ? 128 : 256), p_tiles = symmetric(p_one ? 128 : 256), tiles = full(full_one ? 128 : 256);
  const TileOperand a_op{s.a_hi, s.a_lo, a_rows, z.side, z.side, false}, p_op{s.p_hi, s.p_lo, a_rows, z.side, z.side, false};
  int at = 0;
  for (int k = 0; k < o.steps && rc == B2_OK; ++k, at ^= 1) {
    const TileOperand x_k{s.x_hi[at], s.x_lo[at], x_rows, z.cols_up, z.cols_up, false};
    const TileOperand x_mn{s.x_hi[at], s.x_lo[at], z.cols_up, x_rows, z.cols_up, true};
    SymmetricParams q{};
    q.side = z.side;
    q.count = count;
    q.kblocks = k_a;
    q.a_step = z.rows_up;
    q.steps_k = !wide;
    q.to_hi = s.a_hi;
    q.to_lo = s.a_lo;
    const TileOperand& x = wide ? x_k : x_mn;
    if (a_parts > 1) {
      q.parts = a_parts;
      q.sums = s.sums;
      rc = tile_launch<SymmetricOp<PARTS, true>>(who, x, x, nullptr, q, false, symmetric(128) * a_parts, sms, chain);
      const int n = z.side / 32;
      chain.launch(join_parts_kernel, dim3(n * (n + 1) / 2, count), 256, 0, 0, s.sums, a_parts, z.side, s.a_hi, s.a_lo);
      if (rc == B2_OK) rc = launch_error(chain.err, who);
    } else {
      rc = (a_one ? tile_launch<SymmetricOp<WHOLE, true>> : tile_launch<SymmetricOp<WHOLE, false>>)(who, x, x, nullptr, q, false, a_tiles, sms, chain);
    }
    if (rc != B2_OK) return rc;
    q.kblocks = k_b;
    q.a_step = z.side;
    q.steps_k = 0;
    q.a_hi = s.a_hi;
    q.a_lo = s.a_lo;
    q.to_hi = s.p_hi;
    q.to_lo = s.p_lo;
    rc = (p_one ? tile_launch<SymmetricOp<MIDDLE_FACTOR, true>> : tile_launch<SymmetricOp<MIDDLE_FACTOR, false>>)(who, a_op, a_op, nullptr, q, false, p_tiles, sms, chain);
    if (rc != B2_OK) return rc;
    NextParams n{};
    n.list = list;
    n.rows = rows;
    n.cols = cols;
    n.rows_up = z.rows_up;
    n.cols_up = z.cols_up;
    n.count = count;
    n.kblocks = k_b;
    n.wide = wide;
    n.to_hi = s.x_hi[at ^ 1];
    n.to_lo = s.x_lo[at ^ 1];
    n.ld_w = (long long)ld_w;
    n.ld_copy = (long long)ld_copy;
    n.keep = (float)(1.0 - (double)o.lr * o.weight_decay);
    n.step = (float)((double)o.lr * o.scale);
    n.vec_w = ld_w % 4 == 0;
    n.vec_copy = ld_copy % 4 == 0;
    for (int i = 0; i < count; ++i) {
      if (reinterpret_cast<uintptr_t>(list.w[i]) % 16) n.vec_w = 0;
      if (reinterpret_cast<uintptr_t>(list.copy[i]) % 8) n.vec_copy = 0;
    }
    const TileOperand &ao = wide ? p_op : x_k, &bo = wide ? x_mn : p_op;
    auto next = k + 1 < o.steps ? (full_one ? tile_launch<NextOp<false, true>> : tile_launch<NextOp<false, false>>)
                                : (full_one ? tile_launch<NextOp<true, true>> : tile_launch<NextOp<true, false>>);
    rc = next(who, ao, bo, nullptr, n, false, tiles, sms, chain);
  }
  return rc;
}

// The matrices of a call may lie in one another's gaps, but share nothing, gradients among themselves excepted.
int check_overlap(const char* who, int count, int rows, int cols, int grad_dtype, float* const* w, size_t ld_w, void* const* copy, size_t ld_copy,
                  float* const* momentum, size_t ld_m, const void* const* grad, size_t ld_g, void* workspace, size_t need) {
  constexpr int FEW = 4 * MUON_GROUP + 1;
  Extent few[FEW], *x = few;
  std::unique_ptr<Extent[]> many;
  if (4ll * count + 1 > FEW) {
    many.reset(new (std::nothrow) Extent[4 * (size_t)count + 1]);
    if (!many) return call_error(B2_ERR_STATE, "%s: no host memory for a list of %d matrices", who, count);
    x = many.get();
  }
  const size_t n = rows, c = cols, g = dtype_bytes(grad_dtype);
  int used = 0;
  for (int i = 0; i < count; ++i) {
    x[used++] = extent("w", w[i], n, c * 4, ld_w * 4, true);
    x[used++] = extent("momentum", momentum[i], n, c * 4, ld_m * 4, true);
    x[used++] = extent("grad", grad[i], n, c * g, ld_g * g, false);
    if (copy) x[used++] = extent("copy", copy[i], n, c * 2, ld_copy * 2, true);
  }
  x[used++] = extent("the workspace", workspace, 1, need, need, true);
  return refuse_overlap(who, x, used);
}

int check_muon(const char* who, int count, int rows, int cols) {
  if (count < 0 || count > 1 << 24 || rows < 1 || cols < 1 || rows > 65536 || cols > 65536)
    return call_error(B2_ERR_INVALID, "%s: %d matrices of %d x %d (sides of 1 to 65536)", who, count, rows, cols);
  return B2_OK;
}

}  // namespace

}  // namespace b2

using namespace b2;

extern "C" {

int b2_muon_options_default(b2_muon_options* o) {
  if (!o) return call_error(B2_ERR_INVALID, "b2_muon_options_default: null pointer");
  *o = b2_muon_options{0.02f, 0.95f, 0.f, 1.f, 1e-7f, 1, 5};
  return B2_OK;
}

int b2_muon_workspace(int count, int rows, int cols, size_t* bytes) {
  int rc = check_muon("b2_muon_workspace", count, rows, cols);
  if (rc != B2_OK) return rc;
  if (!bytes) return call_error(B2_ERR_INVALID, "b2_muon_workspace: null pointer");
  MuonSpace s;
  *bytes = muon_space(muon_sizes(count, rows, cols), nullptr, &s);
  return B2_OK;
}

int b2_muon(int count, int rows, int cols, int grad_dtype, float* const* w, size_t ld_w, void* const* copy, size_t ld_copy,
            float* const* momentum, size_t ld_m, const void* const* grad, size_t ld_g, const b2_muon_options* options,
            void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "b2_muon";
  int rc = check_muon(who, count, rows, cols);
  if (rc != B2_OK) return rc;
  if (!dtype_ok(grad_dtype)) return call_error(B2_ERR_INVALID, "%s: dtype %d", who, grad_dtype);
  if (!options || (count && (!w || !momentum || !grad || !workspace))) return call_error(B2_ERR_INVALID, "%s: null pointer", who);
  const size_t c = (size_t)cols;
  if (ld_w < c || ld_m < c || ld_g < c || (copy && ld_copy < c)) return call_error(B2_ERR_INVALID, "%s: leading dimension smaller than the width", who);
  if (options->steps < 1 || options->steps > 100) return call_error(B2_ERR_INVALID, "%s: %d steps (1 to 100)", who, options->steps);
  if (!(options->eps >= 0.f)) return call_error(B2_ERR_INVALID, "%s: eps is negative or not a number", who);
  for (int i = 0; i < count; ++i) {
    if (!w[i] || !momentum[i] || !grad[i] || (copy && !copy[i])) return call_error(B2_ERR_INVALID, "%s: null pointer of matrix %d", who, i);
    if ((reinterpret_cast<uintptr_t>(w[i]) | reinterpret_cast<uintptr_t>(momentum[i])) % 4 ||
        reinterpret_cast<uintptr_t>(grad[i]) % dtype_bytes(grad_dtype) || (copy && reinterpret_cast<uintptr_t>(copy[i]) % 2))
      return call_error(B2_ERR_INVALID, "%s: a pointer of matrix %d is not aligned to its elements", who, i);
  }
  if (reinterpret_cast<size_t>(workspace) % 256) return call_error(B2_ERR_INVALID, "%s: the workspace is not on a 256-byte boundary", who);
  if (count == 0) return B2_OK;
  const MuonSizes z = muon_sizes(count, rows, cols);
  MuonSpace s;
  const size_t need = muon_space(z, workspace, &s);
  if (workspace_bytes < need) return call_error(B2_ERR_INVALID, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, need);
  int sms;
  if ((rc = lm_device(&sms)) != B2_OK) return rc;
  rc = check_overlap(who, count, rows, cols, grad_dtype, w, ld_w, copy, ld_copy, momentum, ld_m, grad, ld_g, workspace, need);
  for (int i = 0; i < count && rc == B2_OK; i += z.group) {
    const int n = count - i < z.group ? count - i : z.group;
    MatrixList list{};
    for (int k = 0; k < n; ++k) {
      list.w[k] = w[i + k];
      list.copy[k] = copy ? static_cast<__nv_bfloat16*>(copy[i + k]) : nullptr;
      list.m[k] = momentum[i + k];
      list.g[k] = grad[i + k];
    }
    rc = muon_group(list, n, rows, cols, grad_dtype, ld_w, ld_copy, ld_m, ld_g, *options, z, s, sms, static_cast<cudaStream_t>(stream));
  }
  return rc;
}

int b2_lm_sync(void* stream) {
  static WaitReports reports;
  int sms, dev = 0, rc = lm_device(&sms);
  if (rc != B2_OK) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  unsigned int xent = 0, role = 0;
  unsigned long long id = 0;  // of a stream that is gone no other one gets it, unlike its address
  TileReport own{};
  cudaError_t e = xent_waits_given_up(&xent, &role, st);
  if (e == cudaSuccess) e = tile_report_read(&own, st);
  if (e == cudaSuccess) e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaStreamGetId(st, &id);
  if (e != cudaSuccess) return launch_error(e, "b2_lm_sync");
  bool news = true;
  try {
    news = reports.news(dev, id, xent + own.count);
  } catch (...) {  // no memory to note what was told: it is told again
    news = xent + own.count != 0;
  }
  if (news) return call_error(B2_ERR_TIMEOUT, "a tile kernel gave up waiting on a pipeline barrier (role %u)", role ? role : own.role);
  return B2_OK;
}

}  // extern "C"
