// Root-mean-square norm of rows with the residual stream's addition, and its gradients:
//
//   t = x + residual (rounded)     r = 1 / sqrt(mean(t^2) + eps)     out = t r w       or in e4m3 with scales
//   g = dy w     dx = r (g - t r^2 mean(g t)) + dtotal               dw = sum over rows of dy t r
//
// Both are bound by HBM: every matrix is read or written once. A row is held in registers by a group of threads, from 1 to a block of
// 1024, each with K vectors at distances of the group, so that the row's sum of squares is one reduction between the load and the store.
// The gradient needs no statistics of the forward pass: mean(t^2) and mean(g t) are reduced together.
//
// Measured on one B200 (a copy reaches 6.56 TB/s): 65536 x 1024 bf16 with residual and fp32 weight 85 us, 6.3 TB/s; its gradients 101 us, 5.3 TB/s (63 % of issue slots;
// two kernels); 8192 x 4096 bf16 with residual to e4m3 47 us, 5.0 TB/s (73 % of issue slots: the largest magnitude, the quotient mended and rounded per element); one row of
// 4096 2.5 us.
#include <cuda_fp8.h>

#include "lm.cuh"

namespace b2 {
namespace {

constexpr float E4M3_MAX = 448.f;
constexpr float LEAST_SCALE = 1.17549435e-38f;  // 2^-126: the least whose reciprocal fp32 has
constexpr size_t SCALE_BLOCK = 128;
constexpr int NORM_THREADS = 256, ROW_MOST_THREADS = 1024;

struct NormArgs {
  const char *x, *residual, *weight;
  char *total, *out;
  float* scales;
  size_t ld_x, ld_residual, ld_total, ld_out, ld_scales;  // bytes; ld_scales in elements
  size_t rows;
  int width, weight_f32, block;
  float eps;
  double inverse_width;
};

// 1 / sqrt(mean + eps), and whether products with it have to be taken in fp64: outside this range r or t r leaves fp32's. The approximate root's reciprocal and a step of
// Newton's are as near as a rounded root and a rounded quotient, in a quarter of the instructions.
struct Rms {
  double wide;
  float r;
  bool far;
  __device__ __forceinline__ Rms(double mean, float eps) {
    const double m = mean + (double)eps;
    far = !(m > 1e-36 && m < 1e36);
    const float f = (float)m, x = rsqrtf(f);
    r = fmaf(0.5f * x, fmaf(-f * x, x, 1.f), x);
    wide = 0.0;
    if (far) wide = 1.0 / sqrt(m);
  }
  __device__ __forceinline__ float times(float t) const { return far ? (float)(t * wide) : t * r; }
};

// N consecutive weights from column `col`.
template <int N>
__device__ __forceinline__ void load_weight(const char* w, int f32, int col, float (&o)[N]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = 1.f;
  } else if (f32) {
    constexpr int B = N * 4 < 16 ? N * 4 : 16;
    const typename Raw<B>::type* p = reinterpret_cast<const typename Raw<B>::type*>(w + (size_t)col * 4);
#pragma unroll
    for (int j = 0; j < N * 4 / B; ++j) {
      float f[B / 4];
      Elems<float, B>::get(__ldg(p + j), f);
#pragma unroll
      for (int i = 0; i < B / 4; ++i) o[j * (B / 4) + i] = f[i];
    }
  } else {
    typedef Elems<__nv_bfloat16, N * 2> E;
    E::get(__ldg(reinterpret_cast<const typename E::raw*>(w + (size_t)col * 2)), o);
  }
}

// Sums (or, with MAX, the largest) over the row's group of 1 << g_log2 neighbouring threads, the same bits in all of them. Groups of more than a
// warp exchange through `slots` (one double per warp and value, not used again before another barrier).
template <int COUNT>
__device__ __forceinline__ void row_sums(double (&s)[COUNT], int g_log2, double* slots) {
  const int g = 1 << g_log2, lanes = g < 32 ? g : 32;
  for (int o = lanes >> 1; o; o >>= 1)
#pragma unroll
    for (int k = 0; k < COUNT; ++k) s[k] += __shfl_xor_sync(0xFFFFFFFFu, s[k], o);
  if (g <= 32) return;
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int k = 0; k < COUNT; ++k) slots[warp * COUNT + k] = s[k];
  __syncthreads();
  const int warps = g >> 5, first = warp & ~(warps - 1);
#pragma unroll
  for (int k = 0; k < COUNT; ++k) s[k] = 0.0;
  for (int i = 0; i < warps; ++i)
#pragma unroll
    for (int k = 0; k < COUNT; ++k) s[k] += slots[(first + i) * COUNT + k];
}

// The largest |value| of a row's group, or of 1 << l neighbouring threads of a warp.
__device__ __forceinline__ float lanes_max(float m, int lanes) {
  for (int o = lanes >> 1; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  return m;
}

// largest / 448: the product with 1 / 448, mended by a step of Newton's (which would make NaN of infinity)
__device__ __forceinline__ float scale_of(float largest) {
  const float q = largest * (1.f / E4M3_MAX), s = fmaf(fmaf(-q, E4M3_MAX, largest), 1.f / E4M3_MAX, q);
  return fmaxf(largest < INFINITY ? s : largest, LEAST_SCALE);
}

// y / scale as e4m3: fp32's quotient rounded once more, which is off by more than half a step of e4m3 only within 2^-24 of a tie. The quotient is the product with
// the reciprocal, mended by one step of Newton's, which a scale of infinity would make NaN of 0.
struct Scaled {
  float scale, inverse;
  __device__ __forceinline__ explicit Scaled(float s) : scale(s < INFINITY ? s : 0.f) { asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(s)); }
  __device__ __forceinline__ float of(float y) const {
    const float q = y * inverse;
    return fmaf(fmaf(-q, scale, y), inverse, q);
  }
};
template <int N>
__device__ __forceinline__ void store_e4m3(char* at, const float (&y)[N], const Scaled& s) {
  if constexpr (N == 1) {
    *reinterpret_cast<unsigned char*>(at) = __nv_cvt_float_to_fp8(s.of(y[0]), __NV_SATFINITE, __NV_E4M3);
  } else {
    unsigned short b[N / 2];
#pragma unroll
    for (int i = 0; i < N; i += 2) b[i / 2] = __nv_cvt_float2_to_fp8x2(make_float2(s.of(y[i]), s.of(y[i + 1])), __NV_SATFINITE, __NV_E4M3);
    typename Raw<N>::type r;
    memcpy(&r, b, N);
    *reinterpret_cast<typename Raw<N>::type*>(at) = r;
  }
}

template <typename T, int VB, int K, bool E4M3>
__global__ void __launch_bounds__(ROW_MOST_THREADS) norm_kernel(const NormArgs a, int g_log2) {
  typedef Elems<T, VB> E;
  typedef typename E::raw raw;
  constexpr int N = E::N;
  __shared__ double slots[ROW_MOST_THREADS / 32];
  extern __shared__ unsigned int block_max[];  // E4M3 with a scale per 128 columns that more than a warp shares: bits of the largest |out|, by row and block
  const int g = 1 << g_log2, in_row = threadIdx.x & (g - 1), sub = threadIdx.x >> g_log2;
  const size_t row = (size_t)blockIdx.x * (blockDim.x >> g_log2) + sub;
  const bool active = row < a.rows;
  const int vecs = a.width / N;
  raw v[K];
  {
    const raw* x = reinterpret_cast<const raw*>(a.x + row * a.ld_x);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      memset(&v[k], 0, sizeof(raw));
      if (active && in_row + (k << g_log2) < vecs) v[k] = __ldg(x + in_row + (k << g_log2));
    }
  }
  if (a.residual) {
    const raw* s = reinterpret_cast<const raw*>(a.residual + row * a.ld_residual);
    raw w[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      memset(&w[k], 0, sizeof(raw));
      if (active && in_row + (k << g_log2) < vecs) w[k] = __ldg(s + in_row + (k << g_log2));
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float p[N], q[N];
      E::get(v[k], p);
      E::get(w[k], q);
#pragma unroll
      for (int i = 0; i < N; ++i) p[i] += q[i];
      v[k] = E::put(p);
    }
    if (a.total && active) {
      raw* t = reinterpret_cast<raw*>(a.total + row * a.ld_total);
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (in_row + (k << g_log2) < vecs) t[in_row + (k << g_log2)] = v[k];
    }
  }
  double s[1] = {0.0};
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float f[N];
    E::get(v[k], f);
    add_squares(f, s[0]);
  }
  row_sums(s, g_log2, slots);
  const Rms rms(s[0] * a.inverse_width, a.eps);
  if constexpr (!E4M3) {
    if (!active) return;
    raw* out = reinterpret_cast<raw*>(a.out + row * a.ld_out);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = in_row + (k << g_log2);
      if (c >= vecs) break;
      float f[N], w[N];
      E::get(v[k], f);
      load_weight(a.weight, a.weight_f32, c * N, w);
      if (!rms.far) {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = f[i] * rms.r * w[i];
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = rms.times(f[i]) * w[i];
      }
      out[c] = E::put(f);
    }
  } else {
    const int blocks = (a.width + (int)SCALE_BLOCK - 1) / (int)SCALE_BLOCK;
    constexpr bool IN_WARP = N >= 4;  // 128 columns are the vectors of 32 lanes at most
    float y[K][N], largest[K], whole = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = in_row + (k << g_log2);
      float w[N];
      E::get(v[k], y[k]);
      largest[k] = 0.f;
      if (c < vecs) {
        load_weight(a.weight, a.weight_f32, c * N, w);
        if (!rms.far) {
#pragma unroll
          for (int i = 0; i < N; ++i) y[k][i] = y[k][i] * rms.r * w[i];
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) y[k][i] = rms.times(y[k][i]) * w[i];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) largest[k] = fmaxf(largest[k], fabsf(y[k][i]));
      }
      whole = fmaxf(whole, largest[k]);
    }
    float* scales = a.scales + row * a.ld_scales;
    if (!a.block) {
      whole = lanes_max(whole, g < 32 ? g : 32);
      if (g > 32) {
        float* most = reinterpret_cast<float*>(slots);
        __syncthreads();  // slots are still being read as sums
        const int warp = threadIdx.x >> 5, warps = g >> 5, first = warp & ~(warps - 1);
        if ((threadIdx.x & 31) == 0) most[warp] = whole;
        __syncthreads();
        for (int i = 0; i < warps; ++i) whole = fmaxf(whole, most[first + i]);
      }
      if (active && in_row == 0) scales[0] = scale_of(whole);
#pragma unroll
      for (int k = 0; k < K; ++k) largest[k] = whole;
    } else if constexpr (IN_WARP) {
      constexpr int LANES = (int)SCALE_BLOCK / N;  // the group has as many threads at least
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = in_row + (k << g_log2);
        largest[k] = lanes_max(largest[k], LANES);
        if (active && c < vecs && in_row % LANES == 0) scales[c * N / SCALE_BLOCK] = scale_of(largest[k]);
      }
    } else {
      const int rows_here = blockDim.x >> g_log2;
      for (int i = threadIdx.x; i < rows_here * blocks; i += blockDim.x) block_max[i] = 0;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = in_row + (k << g_log2);
        if (c < vecs) atomicMax(block_max + sub * blocks + c * N / SCALE_BLOCK, __float_as_uint(largest[k]));  // bits of positive floats are in their order
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = in_row + (k << g_log2);
        if (c < vecs) largest[k] = __uint_as_float(block_max[sub * blocks + c * N / SCALE_BLOCK]);
        if (active && c < vecs && c * N % SCALE_BLOCK == 0) scales[c * N / SCALE_BLOCK] = scale_of(largest[k]);
      }
    }
    if (!active) return;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = in_row + (k << g_log2);
      if (c < vecs) store_e4m3(a.out + row * a.ld_out + (size_t)c * N, y[k], Scaled(scale_of(largest[k])));
    }
  }
}

// ------------------------------------------------------------------ rows that registers do not hold: a block per row, read again for each pass

__device__ __forceinline__ float block_max_of(float m, float* slots) {
  m = lanes_max(m, 32);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = m;
  __syncthreads();
  for (int i = 0; i < (int)blockDim.x >> 5; ++i) m = fmaxf(m, slots[i]);
  return m;
}

template <typename T>
struct LongRow {
  const T *x, *residual;
  const char* weight;
  int weight_f32;
  __device__ __forceinline__ float sum(int c) const {
    const float f = (float)x[c];
    return residual ? (float)(T)(f + (float)residual[c]) : f;
  }
  __device__ __forceinline__ float scale(int c) const {
    float w[1];
    load_weight(weight, weight_f32, c, w);
    return w[0];
  }
};

template <typename T, bool E4M3>
__global__ void __launch_bounds__(ROW_MOST_THREADS) norm_long_kernel(const NormArgs a) {
  __shared__ double slots[ROW_MOST_THREADS / 32];
  __shared__ float most[ROW_MOST_THREADS / 32];
  const size_t row = blockIdx.x;
  const LongRow<T> in{reinterpret_cast<const T*>(a.x + row * a.ld_x), a.residual ? reinterpret_cast<const T*>(a.residual + row * a.ld_residual) : nullptr,
                      a.weight, a.weight_f32};
  T* total = a.total ? reinterpret_cast<T*>(a.total + row * a.ld_total) : nullptr;
  double s[1] = {0.0};
  for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
    const float f[1] = {in.sum(c)};
    if (total) total[c] = (T)f[0];
    add_squares(f, s[0]);
  }
  row_sums(s, 10, slots);
  const Rms rms(s[0] * a.inverse_width, a.eps);
  if constexpr (!E4M3) {
    T* out = reinterpret_cast<T*>(a.out + row * a.ld_out);
    for (int c = threadIdx.x; c < a.width; c += blockDim.x) out[c] = (T)(rms.times(in.sum(c)) * in.scale(c));
  } else {
    char* out = a.out + row * a.ld_out;
    float* scales = a.scales + row * a.ld_scales;
    const int lane = threadIdx.x & 31;
    float whole = 0.f;
    if (!a.block) {
      for (int c = threadIdx.x; c < a.width; c += blockDim.x) whole = fmaxf(whole, fabsf(rms.times(in.sum(c)) * in.scale(c)));
      whole = block_max_of(whole, most);
      if (threadIdx.x == 0) scales[0] = scale_of(whole);
    }
    constexpr int PER_LANE = (int)SCALE_BLOCK / 32;
    for (int b = threadIdx.x >> 5; b * (int)SCALE_BLOCK < a.width; b += (int)blockDim.x >> 5) {
      float y[PER_LANE], largest = 0.f;
#pragma unroll
      for (int i = 0; i < PER_LANE; ++i) {
        const int c = b * (int)SCALE_BLOCK + i * 32 + lane;
        y[i] = c < a.width ? rms.times(in.sum(c)) * in.scale(c) : 0.f;
        largest = fmaxf(largest, fabsf(y[i]));
      }
      largest = a.block ? lanes_max(largest, 32) : whole;
      if (a.block && lane == 0) scales[b] = scale_of(largest);
      const Scaled scaled(scale_of(largest));
#pragma unroll
      for (int i = 0; i < PER_LANE; ++i) {
        const int c = b * (int)SCALE_BLOCK + i * 32 + lane;
        const float f[1] = {y[i]};
        if (c < a.width) store_e4m3(out + c, f, scaled);
      }
    }
  }
}

// ------------------------------------------------------------------ gradients

struct NormGradArgs {
  const char *dy, *total, *dtotal, *weight;
  char* dx;
  float* partial;  // by block, a row of `width` each; null: the weight's gradient is not wanted
  size_t ld_dy, ld_total, ld_dtotal, ld_dx;
  size_t rows;
  int width, weight_f32;
  float eps;
  double inverse_width;
};

// sum += f * h, as add_squares() does.
template <int N>
__device__ __forceinline__ void add_products(const float (&f)[N], const float (&h)[N], double& sum) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) s = fmaf(f[i], h[i], s);
  if (safe_sum(s)) {
    sum += (double)s;
  } else {
    unsigned int any = 0;  // rows without a gradient are common
#pragma unroll
    for (int i = 0; i < N; ++i) any |= __float_as_uint(f[i]) << 1;
    if (any) {
#pragma unroll
      for (int i = 0; i < N; ++i) sum = fma((double)f[i], (double)h[i], sum);
    }
  }
}

// One row's numbers: n = t r and dx = r (g - n c) + dtotal with c = r mean(g t).
struct GradRow {
  Rms rms;
  float c;
  __device__ __forceinline__ GradRow(const double (&s)[2], double inverse_width, float eps)
      : rms(s[0] * inverse_width, eps), c((float)((rms.far ? rms.wide : (double)rms.r) * (s[1] * inverse_width))) {}
  __device__ __forceinline__ float dx(float g, float n, float more) const { return rms.times(g - n * c) + more; }
};

// A block's groups take rows at distances of the grid, the next one's loads on their way while one is worked on; weights and the sums for the weight's gradient
// stay in registers. K as small as a block of 256 threads allows: 8 elements per thread have room for three blocks per SM, 16 for two, and 32 for two without loads ahead.
template <int K, int N, int MOST>
constexpr int GRAD_PER_SM = MOST > NORM_THREADS ? 1 : K * N <= 8 ? 3 : 2;

template <typename T, int VB, int K, int MOST>
__global__ void __launch_bounds__(MOST, (GRAD_PER_SM<K, VB / (int)sizeof(T), MOST>)) norm_grad_kernel(const NormGradArgs a, int g_log2) {
  typedef Elems<T, VB> E;
  typedef typename E::raw raw;
  constexpr int N = E::N;
  constexpr bool AHEAD = MOST <= NORM_THREADS && K * N <= 16;
  __shared__ double slots[2][2 * MOST / 32];
  extern __shared__ float sums[];  // a row of partial sums
  let_next_start();
  const int g = 1 << g_log2, in_row = threadIdx.x & (g - 1), sub = threadIdx.x >> g_log2, rows_here = blockDim.x >> g_log2;
  const int vecs = a.width / N;
  float dw[K][N], w[K][N];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = in_row + (k << g_log2);
#pragma unroll
    for (int i = 0; i < N; ++i) dw[k][i] = w[k][i] = 0.f;
    if (AHEAD && c < vecs) load_weight(a.weight, a.weight_f32, c * N, w[k]);
  }
  struct Row {
    raw t[K], d[K], m[K];
  };
  auto load = [&](Row& v, size_t row) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = in_row + (k << g_log2);
      memset(&v.t[k], 0, sizeof(raw));
      memset(&v.d[k], 0, sizeof(raw));
      memset(&v.m[k], 0, sizeof(raw));
      if (row < a.rows && c < vecs) {
        v.t[k] = __ldg(reinterpret_cast<const raw*>(a.total + row * a.ld_total) + c);
        v.d[k] = __ldg(reinterpret_cast<const raw*>(a.dy + row * a.ld_dy) + c);
        if (a.dtotal) v.m[k] = __ldg(reinterpret_cast<const raw*>(a.dtotal + row * a.ld_dtotal) + c);
      }
    }
  };
  int turn = 0;
  const size_t step = (size_t)gridDim.x * rows_here;
  Row now, next;
  if (AHEAD) load(now, (size_t)blockIdx.x * rows_here + sub);
  for (size_t row0 = (size_t)blockIdx.x * rows_here; row0 < a.rows; row0 += step, turn ^= 1) {
    const size_t row = row0 + sub;
    if (AHEAD) load(next, row + step);
    else load(now, row);
    double s[2] = {0.0, 0.0};
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = in_row + (k << g_log2);
      float f[N], h[N];
      E::get(now.t[k], f);
      E::get(now.d[k], h);
      if (c < vecs) {
        if (!AHEAD) load_weight(a.weight, a.weight_f32, c * N, w[k]);
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] *= w[k][i];
        add_squares(f, s[0]);
        add_products(h, f, s[1]);
      }
    }
    row_sums(s, g_log2, slots[turn]);
    const GradRow r(s, a.inverse_width, a.eps);
    if (row < a.rows) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = in_row + (k << g_log2);
        if (c >= vecs) break;
        float f[N], h[N], o[N];
        E::get(now.t[k], f);
        E::get(now.d[k], h);
        E::get(now.m[k], o);
        if (!AHEAD) load_weight(a.weight, a.weight_f32, c * N, w[k]);
        if (!r.rms.far) {
          const float rr = r.rms.r;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float n = f[i] * rr;
            dw[k][i] = fmaf(h[i], n, dw[k][i]);
            o[i] = fmaf(rr, h[i] * w[k][i] - n * r.c, o[i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float n = r.rms.times(f[i]);
            dw[k][i] = fmaf(h[i], n, dw[k][i]);
            o[i] = r.dx(h[i] * w[k][i], n, o[i]);
          }
        }
        reinterpret_cast<raw*>(a.dx + row * a.ld_dx)[c] = E::put(o);
      }
    }
    if (AHEAD) now = next;
  }
  after_previous();
  if (!a.partial) return;
  // the block's groups add theirs in turn
  for (int i = 0; i < rows_here; ++i) {
    if (sub == i)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = in_row + (k << g_log2);
        if (c >= vecs) break;
#pragma unroll
        for (int j = 0; j < N; ++j) sums[c * N + j] = i ? sums[c * N + j] + dw[k][j] : dw[k][j];
      }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < a.width; c += blockDim.x) a.partial[(size_t)blockIdx.x * a.width + c] = sums[c];
}

// dweight[c] = sum of `count` partial sums: 32 columns per block, a warp for every 32nd partial sum, and the warps' sums in order.
constexpr int JOIN_WARPS = 32;
__global__ void __launch_bounds__(JOIN_WARPS * 32) norm_join_kernel(const float* __restrict__ partial, int count, int width, void* dweight, int f32) {
  __shared__ float part[JOIN_WARPS][33];
  after_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < width) {
#pragma unroll 8
    for (int i = warp; i < count; i += JOIN_WARPS) s += partial[(size_t)i * width + c];
  }
  part[warp][lane] = s;
  __syncthreads();
  // a warp per column of the first
  s = part[lane][warp];
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  const int mine = blockIdx.x * 32 + warp;
  if (lane || mine >= width) return;
  if (f32) static_cast<float*>(dweight)[mine] = s;
  else static_cast<__nv_bfloat16*>(dweight)[mine] = (__nv_bfloat16)s;
}

// Long rows: dx by a block per row, which leaves r; then sums by columns over slices of rows.
template <typename T>
__global__ void __launch_bounds__(ROW_MOST_THREADS) norm_grad_long_kernel(const NormGradArgs a, double* rms_of) {
  __shared__ double slots[2 * ROW_MOST_THREADS / 32];
  let_next_start();
  const size_t row = blockIdx.x;
  const LongRow<T> in{reinterpret_cast<const T*>(a.total + row * a.ld_total), nullptr, a.weight, a.weight_f32};
  const T* dy = reinterpret_cast<const T*>(a.dy + row * a.ld_dy);
  const T* more = a.dtotal ? reinterpret_cast<const T*>(a.dtotal + row * a.ld_dtotal) : nullptr;
  T* dx = reinterpret_cast<T*>(a.dx + row * a.ld_dx);
  double s[2] = {0.0, 0.0};
  for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
    const float f[1] = {in.sum(c)}, h[1] = {(float)dy[c] * in.scale(c)};
    add_squares(f, s[0]);
    add_products(h, f, s[1]);
  }
  row_sums(s, 10, slots);
  const GradRow r(s, a.inverse_width, a.eps);
  if (threadIdx.x == 0 && rms_of) rms_of[row] = r.rms.far ? -r.rms.wide : (double)r.rms.r;
  for (int c = threadIdx.x; c < a.width; c += blockDim.x)
    dx[c] = (T)r.dx((float)dy[c] * in.scale(c), r.rms.times(in.sum(c)), more ? (float)more[c] : 0.f);
  after_previous();
}

template <typename T>
__global__ void __launch_bounds__(NORM_THREADS) norm_columns_kernel(const NormGradArgs a, const double* rms_of) {
  let_next_start();
  after_previous();
  const int c = blockIdx.x * NORM_THREADS + threadIdx.x;
  if (c >= a.width) return;
  float s = 0.f;
  for (size_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float f = (float)reinterpret_cast<const T*>(a.total + row * a.ld_total)[c], h = (float)reinterpret_cast<const T*>(a.dy + row * a.ld_dy)[c];
    const double r = rms_of[row];
    s = fmaf(h, r < 0.0 ? (float)(f * -r) : f * (float)r, s);
  }
  a.partial[(size_t)blockIdx.y * a.width + c] = s;
}

// ------------------------------------------------------------------ which form

// Threads per row (a power of two) and vectors per thread; k = 0: the row is too long for registers.
struct RowForm {
  int g_log2, k, threads;
  int g() const { return 1 << g_log2; }
};
// most_k: vectors that a thread may hold; the fewest threads that hold a row leave the most loads in flight and the fewest threads to reduce over (65536 x 1024 bf16 with 4, 2
// and 1 vectors 85, 86 and 94 us; 8192 x 4096 to e4m3 47, 52 and 57). few: rows times threads below this leave the GPU partly idle, so that more threads share a row (1 x
// 4096 bf16 2.5 us for 3.3, 600 x 1024 2.9 for 3.7).
RowForm row_form(size_t rows, int vecs, int most_k, int least_g, int most_g, size_t few) {
  RowForm f{0, 0, 0};
  while (f.g() < least_g || (f.g() < most_g && (size_t)f.g() * most_k < (size_t)vecs)) ++f.g_log2;
  if ((size_t)f.g() * most_k < (size_t)vecs) return f;
  while (f.g() < most_g && f.g() < vecs && rows * f.g() < few) ++f.g_log2;
  f.k = 1;
  while ((size_t)f.g() * f.k < (size_t)vecs) f.k *= 2;
  f.threads = f.g() > NORM_THREADS ? f.g() : NORM_THREADS;
  return f;
}

// The widest vector of the matrices' elements that also fits the weight's address.
int norm_vector(size_t e, size_t bits, const void* weight, size_t weight_e) {
  int vb = vector_bytes(e, bits);
  const size_t w = reinterpret_cast<size_t>(weight);
  while (vb > (int)e) {
    const size_t need = vb / e * weight_e;
    if (w % (need < 16 ? need : 16) == 0) break;
    vb >>= 1;
  }
  return vb;
}

template <typename T, int VB, bool E4M3>
void norm_launch(const NormArgs& a, int sms, Chain& chain) {
  constexpr int N = VB / (int)sizeof(T), MOST_K = N >= 8 ? 4 : 8;
  const int least_g = E4M3 && a.block && N >= 4 ? (int)SCALE_BLOCK / N : 1;
  const RowForm f = row_form(a.rows, a.width / N, MOST_K, least_g, ROW_MOST_THREADS, (size_t)sms * 1024);
  if (!f.k) {
    chain.launch(norm_long_kernel<T, E4M3>, dim3((unsigned int)a.rows), ROW_MOST_THREADS, 0, 0, a);
    return;
  }
  const size_t here = f.threads >> f.g_log2;
  const dim3 grid((unsigned int)((a.rows + here - 1) / here));
  const size_t smem = E4M3 && a.block && N < 4 ? here * ((a.width + SCALE_BLOCK - 1) / SCALE_BLOCK) * 4 : 0;
  if (f.k == 1) chain.launch(norm_kernel<T, VB, 1, E4M3>, grid, f.threads, smem, 0, a, f.g_log2);
  else if (f.k == 2) chain.launch(norm_kernel<T, VB, 2, E4M3>, grid, f.threads, smem, 0, a, f.g_log2);
  else if (f.k == 4) chain.launch(norm_kernel<T, VB, 4, E4M3>, grid, f.threads, smem, 0, a, f.g_log2);
  else if constexpr (MOST_K == 8) chain.launch(norm_kernel<T, VB, 8, E4M3>, grid, f.threads, smem, 0, a, f.g_log2);
}

template <typename T, bool E4M3>
void norm_by_vector(const NormArgs& a, int vb, int sms, Chain& chain) {
  if (vb == 16) norm_launch<T, 16, E4M3>(a, sms, chain);
  else if (vb == 8) norm_launch<T, 8, E4M3>(a, sms, chain);
  else if (vb == 4) norm_launch<T, 4, E4M3>(a, sms, chain);
  else if constexpr (sizeof(T) == 2) norm_launch<T, 2, E4M3>(a, sms, chain);
}

// Blocks of the gradient's kernels, as for 148 SMs at most, so that the workspace does not depend on the device, and slices of rows where a row takes more than a
// block's registers (from 4097 columns on, by alignment).
constexpr int SMS_MOST = 148, COLUMN_SLICES = 64;
constexpr size_t GRAD_LEAST_LONG = 4097, GRAD_WIDTH_MOST = (size_t)ROW_MOST_THREADS * 16;
constexpr size_t ROWS_MOST = (size_t)1 << 31, WIDTH_MOST = (size_t)1 << 20;

size_t grad_space(size_t rows, size_t width, void* base, float** partial, double** rms_of) {
  Carver c(base);
  const size_t per_sm = width <= NORM_THREADS * 8 ? 3 : 2;
  const size_t blocks = width <= NORM_THREADS * 32 ? SMS_MOST * per_sm : width <= GRAD_WIDTH_MOST ? SMS_MOST : COLUMN_SLICES;
  *partial = c.take<float>((blocks > COLUMN_SLICES ? blocks : COLUMN_SLICES) * width);
  *rms_of = c.take<double>(width >= GRAD_LEAST_LONG ? rows : 0);
  return c.used;
}

template <typename T, int VB, int K, int MOST>
int grad_rows(const NormGradArgs& a, const RowForm& f, int sms, Chain& chain) {
  constexpr int PER_SM = GRAD_PER_SM<K, VB / (int)sizeof(T), MOST>;
  const size_t here = f.threads >> f.g_log2, blocks = (a.rows + here - 1) / here, most = (size_t)(sms < SMS_MOST ? sms : SMS_MOST) * PER_SM;
  const int parts = (int)(blocks < most ? blocks : most);
  const size_t smem = a.partial ? (size_t)a.width * 4 : 0;
  if (smem > 40 * 1024) chain.err = with_shared<norm_grad_kernel<T, VB, K, MOST>>((int)GRAD_WIDTH_MOST * 4);
  chain.launch(norm_grad_kernel<T, VB, K, MOST>, dim3(parts), f.threads, smem, 0, a, f.g_log2);
  return parts;
}

template <typename T, int VB>
void norm_grad_launch(const NormGradArgs& a, double* rms_of, void* dweight, int sms, Chain& chain) {
  constexpr int N = VB / (int)sizeof(T), MOST_K = N >= 8 ? 4 : 8;
  // two vectors per thread share the row's reduction and leave registers for the next row's loads (65536 x 1024 bf16 101 us, with one 118, with four and no loads ahead 217);
  // 1024 threads have 64 registers each: half as many elements. 256 threads with more than two vectors have MOST_K, and 1024 threads half of that: rows that fewer hold go to fewer threads
  RowForm f = row_form(1, a.width / N, 2, 1, NORM_THREADS, 0);
  if (!f.k) f = row_form(1, a.width / N, MOST_K, 1, NORM_THREADS, 0);
  if (!f.k) f = row_form(1, a.width / N, MOST_K / 2, 1, ROW_MOST_THREADS, 0);
  int parts = 0;
  if (f.k && f.threads > NORM_THREADS) {
    parts = grad_rows<T, VB, MOST_K / 2, ROW_MOST_THREADS>(a, f, sms, chain);
  } else if (f.k) {
    if (f.k == 1) parts = grad_rows<T, VB, 1, NORM_THREADS>(a, f, sms, chain);
    else if (f.k == 2) parts = grad_rows<T, VB, 2, NORM_THREADS>(a, f, sms, chain);
    else parts = grad_rows<T, VB, MOST_K, NORM_THREADS>(a, f, sms, chain);
  } else {
    parts = a.rows < COLUMN_SLICES ? (int)a.rows : COLUMN_SLICES;
    chain.launch(norm_grad_long_kernel<T>, dim3((unsigned int)a.rows), ROW_MOST_THREADS, 0, 0, a, rms_of);
    if (a.partial)
      chain.launch(norm_columns_kernel<T>, dim3((unsigned int)((a.width + NORM_THREADS - 1) / NORM_THREADS), parts), NORM_THREADS, 0, 0, a, rms_of);
  }
  if (a.partial)
    chain.launch(norm_join_kernel, dim3((unsigned int)((a.width + 31) / 32)), JOIN_WARPS * 32, 0, 0, a.partial, parts, a.width, dweight, a.weight_f32);
}

int check_norm(const char* who, size_t rows, size_t width, int dtype, const void* weight, int weight_dtype, float eps) {
  if (!dtype_ok(dtype)) return call_error(B2_ERR_INVALID, "%s: dtype %d", who, dtype);
  if (weight && weight_dtype != dtype && weight_dtype != B2_DTYPE_F32) return call_error(B2_ERR_INVALID, "%s: weight_dtype %d", who, weight_dtype);
  if (rows >= ROWS_MOST || width == 0 || width > WIDTH_MOST) return call_error(B2_ERR_INVALID, "%s: %zu rows of %zu (below 2^31, 1 to 2^20)", who, rows, width);
  if (!(eps >= 0.f) || eps > 3.4e38f) return call_error(B2_ERR_INVALID, "%s: eps is negative or not finite", who);
  return B2_OK;
}

size_t address(const void* p) { return reinterpret_cast<size_t>(p); }

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

int b2_norm(size_t rows, size_t width, int dtype, const void* x, size_t ld_x, const void* residual, size_t ld_residual, const void* weight,
            int weight_dtype, float eps, void* total, size_t ld_total, int out_dtype, void* out, size_t ld_out, float* scales, size_t ld_scales,
            size_t block, void* stream) {
  const char* who = "b2_norm";
  int rc = check_norm(who, rows, width, dtype, weight, weight_dtype, eps);
  if (rc != B2_OK) return rc;
  const bool e4m3 = out_dtype == B2_DTYPE_E4M3;
  if (!e4m3 && out_dtype != dtype) return call_error(B2_ERR_INVALID, "%s: out_dtype %d", who, out_dtype);
  if (e4m3 && block != 0 && block != SCALE_BLOCK) return call_error(B2_ERR_INVALID, "%s: block %zu (0 or 128)", who, block);
  if (total && !residual) return call_error(B2_ERR_INVALID, "%s: total without residual", who);
  if (rows && (!x || !out || (e4m3 && !scales))) return call_error(B2_ERR_INVALID, "%s: null pointer", who);
  const size_t e = dtype_bytes(dtype), oe = e4m3 ? 1 : e, blocks = block ? (width + block - 1) / block : 1, we = dtype_bytes(weight_dtype);
  if (ld_x < width || (residual && ld_residual < width) || (total && ld_total < width) || ld_out < width || (e4m3 && ld_scales < blocks))
    return call_error(B2_ERR_INVALID, "%s: leading dimension smaller than the width", who);
  if ((address(x) | address(residual) | address(total)) % e || address(out) % oe || (weight && address(weight) % we) || (e4m3 && address(scales) % 4))
    return call_error(B2_ERR_INVALID, "%s: a pointer is not aligned to its elements", who);
  int sms;
  if ((rc = lm_device(&sms)) != B2_OK) return rc;
  Extent args[] = {extent("x", x, rows, width * e, ld_x * e, false), extent("residual", residual, rows, width * e, ld_residual * e, false),
                   extent("weight", weight, 1, width * we, width * we, false), extent("total", total, rows, width * e, ld_total * e, true),
                   extent("out", out, rows, width * oe, ld_out * oe, true),
                   extent("scales", e4m3 ? scales : nullptr, rows, blocks * 4, ld_scales * 4, true)};
  if ((rc = refuse_overlap(who, args, 6)) != B2_OK) return rc;
  if (!rows) return B2_OK;
  NormArgs a{};
  a.x = static_cast<const char*>(x);
  a.residual = static_cast<const char*>(residual);
  a.weight = static_cast<const char*>(weight);
  a.total = static_cast<char*>(total);
  a.out = static_cast<char*>(out);
  a.scales = scales;
  a.ld_x = ld_x * e;
  a.ld_residual = ld_residual * e;
  a.ld_total = ld_total * e;
  a.ld_out = ld_out * oe;
  a.ld_scales = ld_scales;
  a.rows = rows;
  a.width = (int)width;
  a.weight_f32 = weight_dtype == B2_DTYPE_F32;
  a.block = (int)block;
  a.eps = eps;
  a.inverse_width = 1.0 / (double)width;
  size_t bits = address(x) | a.ld_x | width * e;
  if (residual) bits |= address(residual) | a.ld_residual;
  if (total) bits |= address(total) | a.ld_total;
  bits |= e4m3 ? (address(out) | ld_out) * e : address(out) | a.ld_out;
  const int vb = norm_vector(e, bits, weight, we);
  Chain chain(static_cast<cudaStream_t>(stream));
  if (dtype == B2_DTYPE_BF16) {
    if (e4m3) norm_by_vector<__nv_bfloat16, true>(a, vb, sms, chain);
    else norm_by_vector<__nv_bfloat16, false>(a, vb, sms, chain);
  } else {
    if (e4m3) norm_by_vector<float, true>(a, vb, sms, chain);
    else norm_by_vector<float, false>(a, vb, sms, chain);
  }
  return launch_error(chain.err, who);
}

int b2_norm_grad_workspace(size_t rows, size_t width, int dtype, size_t* bytes) {
  const int rc = check_norm("b2_norm_grad_workspace", rows, width, dtype, nullptr, dtype, 0.f);
  if (rc != B2_OK) return rc;
  if (!bytes) return call_error(B2_ERR_INVALID, "b2_norm_grad_workspace: null pointer");
  float* partial;
  double* rms_of;
  *bytes = grad_space(rows, width, nullptr, &partial, &rms_of);
  return B2_OK;
}

int b2_norm_grad(size_t rows, size_t width, int dtype, const void* dy, size_t ld_dy, const void* total, size_t ld_total, const void* dtotal,
                 size_t ld_dtotal, const void* weight, int weight_dtype, float eps, void* dx, size_t ld_dx, void* dweight, void* workspace,
                 size_t workspace_bytes, void* stream) {
  const char* who = "b2_norm_grad";
  int rc = check_norm(who, rows, width, dtype, weight, weight_dtype, eps);
  if (rc != B2_OK) return rc;
  if (dweight && !weight) return call_error(B2_ERR_INVALID, "%s: dweight without weight", who);
  if ((rows && (!dy || !total || !dx)) || !workspace) return call_error(B2_ERR_INVALID, "%s: null pointer", who);
  const size_t e = dtype_bytes(dtype), we = dtype_bytes(weight_dtype);
  if (ld_dy < width || ld_total < width || (dtotal && ld_dtotal < width) || ld_dx < width)
    return call_error(B2_ERR_INVALID, "%s: leading dimension smaller than the width", who);
  if ((address(dy) | address(total) | address(dtotal) | address(dx)) % e || (weight && (address(weight) | address(dweight)) % we))
    return call_error(B2_ERR_INVALID, "%s: a pointer is not aligned to its elements", who);
  if (address(workspace) % 256) return call_error(B2_ERR_INVALID, "%s: the workspace is not on a 256-byte boundary", who);
  float* partial;
  double* rms_of;
  const size_t need = grad_space(rows, width, workspace, &partial, &rms_of);
  if (workspace_bytes < need) return call_error(B2_ERR_INVALID, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, need);
  int sms;
  if ((rc = lm_device(&sms)) != B2_OK) return rc;
  Extent args[] = {extent("dy", dy, rows, width * e, ld_dy * e, false), extent("total", total, rows, width * e, ld_total * e, false),
                   extent("dtotal", dtotal, rows, width * e, ld_dtotal * e, false), extent("weight", weight, 1, width * we, width * we, false),
                   extent("dx", dx, rows, width * e, ld_dx * e, true), extent("dweight", dweight, 1, width * we, width * we, true),
                   extent("the workspace", workspace, 1, need, need, true)};
  if ((rc = refuse_overlap(who, args, 7)) != B2_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!rows) return dweight ? launch_error(cudaMemsetAsync(dweight, 0, width * we, s), who) : B2_OK;
  NormGradArgs a{};
  a.dy = static_cast<const char*>(dy);
  a.total = static_cast<const char*>(total);
  a.dtotal = static_cast<const char*>(dtotal);
  a.weight = static_cast<const char*>(weight);
  a.dx = static_cast<char*>(dx);
  a.partial = dweight ? partial : nullptr;
  a.ld_dy = ld_dy * e;
  a.ld_total = ld_total * e;
  a.ld_dtotal = ld_dtotal * e;
  a.ld_dx = ld_dx * e;
  a.rows = rows;
  a.width = (int)width;
  a.weight_f32 = weight_dtype == B2_DTYPE_F32;
  a.eps = eps;
  a.inverse_width = 1.0 / (double)width;
  size_t bits = address(dy) | a.ld_dy | address(total) | a.ld_total | address(dx) | a.ld_dx | width * e;
  if (dtotal) bits |= address(dtotal) | a.ld_dtotal;
  const int vb = norm_vector(e, bits, weight, we);
  Chain chain(s);
  if (dtype == B2_DTYPE_BF16) {
    if (vb == 16) norm_grad_launch<__nv_bfloat16, 16>(a, rms_of, dweight, sms, chain);
    else if (vb == 8) norm_grad_launch<__nv_bfloat16, 8>(a, rms_of, dweight, sms, chain);
    else if (vb == 4) norm_grad_launch<__nv_bfloat16, 4>(a, rms_of, dweight, sms, chain);
    else norm_grad_launch<__nv_bfloat16, 2>(a, rms_of, dweight, sms, chain);
  } else {
    if (vb == 16) norm_grad_launch<float, 16>(a, rms_of, dweight, sms, chain);
    else if (vb == 8) norm_grad_launch<float, 8>(a, rms_of, dweight, sms, chain);
    else norm_grad_launch<float, 4>(a, rms_of, dweight, sms, chain);
  }
  return launch_error(chain.err, who);
}

}  // extern "C"
