// A token per row of logits from a given uniform number, with temperature, top-k, top-p and min-p:
//
//   w[v] = exp((x[v] - max) / T)      kept = a prefix of the tokens in falling order of x, equal ones by number
//   token = first v by number with  sum of kept w up to v  >  u * sum of all kept w
//
// Bound by reading the logits once. Two kernels:
//
//   sample_tiles_kernel   a warp per tile of 1024 logits: their maximum, their weight relative to it, and for top-k each lane's maximum
//   sample_kernel         a block per row. From the tiles' numbers come the row's maximum and weight. Without a limit the tile in which the running
//                         weight crosses u's share is read once more. Otherwise a floor below which no token is kept comes from the lanes' maxima (top-k: as many
//                         lanes as top_k reach it), the row's weight (top-p: tokens of less than (1 - p) / vocab of it are never needed,
//                         and a part of a long row says how many more are not, which the weight of the gathered ones has to confirm) or the least
//                         weight (min-p), and the tokens above it, mostly few, are gathered in shared memory from the tiles that have any; where there is no room for
//                         them, passes read the row again.
//
// Up to 512 gathered tokens are put in order one by one. With more nothing is sorted: top-k and top-p are a logit (the last one kept) and how many of the
// tokens that have exactly this one are kept, found by counting tokens in bins: first bins of equal width in max - x, then of equal width in the logit's bits
// inside the bin in which the limit must lie, until a bin has few enough tokens to put them in order, or a single logit. For top-k counts say which bin. For top-p
// they only give an estimate, since a bin's weights differ; the weight above and up to the bin is then summed exactly, so that a wrong estimate is
// found and the search goes on beside it.
//
// The token has to be the exact formula's. With a vocabulary of 10^5 a step of the running sum may be 10^-5 of it, and what the sum is off, times the number
// of steps, is the probability that another token comes out: sums in fp32 would be wrong in some of a thousand rows. So a weight is computed to 5e-12 and summed in
// fp64, some 30 instructions; but where all tokens of a row count (no limit, or top-p's whole weight), first in fp32, 8 instructions, with a bound of the
// error: only where target and step are nearer than that, the row is summed once more in fp64.
//
// Measured on one B200 (a copy reaches 6.56 TB/s): 1024 rows of 65536 bf16 without a limit and with log probabilities 66 us, of which the tiles take 40 (75 % of issue slots: 14
// instructions per logit; 3.4 TB/s), the rows that fp32 leaves open, some 4 %, 20, and the largest tokens' tiles in fp64 4; 256 rows of 65536 with top-p 0.94 over a flat distribution
// (11 000 of the tokens kept) 122 to 132 us on several machines: a block per row and 16 warps per SM, two rounds of 85 000 clocks, of which 26 000 gather tokens, 25 000 find the limit,
// 10 000 sum up and 17 000 estimate and confirm; one row of 32768 with top-k 50 16 to 18 us: latency of one block.
#include <math.h>

#include "lm.cuh"

namespace b2 {
namespace {

constexpr int SAMPLE_THREADS = 512, SAMPLE_WARPS = SAMPLE_THREADS / 32;
constexpr int TILE_THREADS = 256, TILE = 1024, PER_LANE = TILE / 32;
constexpr int BINS = 1024, BINS_PER_THREAD = BINS / SAMPLE_THREADS;
constexpr int LIST = SAMPLE_THREADS;  // tokens that are put in order one by one
constexpr int STEPS = 16;             // 2^(n / 16) for n = 0 to 15 lie in different banks of shared memory
constexpr double REACH = 40.0;        // in units of T: what weighs less than e^-40 of the largest weighs nothing where top-p's limit is looked for

struct TileStat {
  double weight;  // of its tokens relative to 2^rint(largest * c), see FastWeights; negative: not to be had in fp32
  float largest, none;
};

// What weights in fp32 need of a temperature: c = log2(e) / T in two parts, 80 T.
struct TemperatureScale {
  float c, c_low, reach;
  bool usable;
};
__host__ __device__ inline TemperatureScale scale_of_temperature(float t) {
  const double exact = 1.4426950408889634 / (double)t;
  TemperatureScale s;
  s.usable = t > 1e-25f && t < 1e25f;
  s.c = s.usable ? (float)exact : 0.f;
  s.c_low = s.usable ? (float)(exact - (double)s.c) : 0.f;
  s.reach = 80.f * t;
  return s;
}

struct SampleArgs {
  const char* logits;
  size_t ld;  // bytes
  unsigned int vocab, tiles;
  const float* u;
  float temperature, top_p, min_p;
  int top_k;
  TemperatureScale scale;  // of the temperature for all rows
  const float *row_temperature, *row_top_p, *row_min_p;
  const int* row_top_k;
  void* tokens;
  int wide;
  float* logprob;
  TileStat* stats;    // rows x tiles
  float* lane_most;   // rows x tiles x 32, or null where no row has a top_k
  unsigned int* open;        // rows whose token fp32 leaves open
  unsigned int* open_count;
};

// What one row asks for.
struct SampleRow {
  float t, top_p, min_p;
  int top_k;
  TemperatureScale scale;
  bool by_k, by_p, by_m, greedy, whole;  // whole: the row's whole weight is needed
  __device__ __forceinline__ SampleRow(const SampleArgs& a, size_t r) {
    t = a.row_temperature ? a.row_temperature[r] : a.temperature;
    top_p = a.row_top_p ? a.row_top_p[r] : a.top_p;
    min_p = a.row_min_p ? a.row_min_p[r] : a.min_p;
    top_k = a.row_top_k ? a.row_top_k[r] : a.top_k;
    greedy = !(t > 0.f) || top_k == 1 || top_p <= 0.f || min_p > 1.f;
    t = fminf(t, 3.4028235e38f);
    scale = a.row_temperature ? scale_of_temperature(t) : a.scale;
    by_k = top_k > 0 && (unsigned int)top_k < a.vocab;
    by_p = top_p < 1.f;
    by_m = min_p > 0.f;
    whole = !greedy && !by_k && (by_p || !by_m);
  }
};

// A row's tokens by place: place = number + shift, so that vectors of 16 bytes of the row begin at multiples of their length. What is not in the row, or not a
// number, is -inf.
template <typename T>
struct RowView {
  const T* row;
  unsigned int shift, end;  // end: the place behind the last one
  __device__ __forceinline__ RowView(const SampleArgs& a, size_t r) {
    row = reinterpret_cast<const T*>(a.logits + r * a.ld);
    shift = (unsigned int)(reinterpret_cast<size_t>(row) & 15) / sizeof(T);
    end = a.vocab + shift;
  }
  // 16 bytes from place i on as they are, what is not in the row as -inf
  __device__ __forceinline__ uint4 load_vector(unsigned int i) const {
    constexpr int N = 16 / (int)sizeof(T);
    if (i >= shift && i + N <= end) return __ldg(reinterpret_cast<const uint4*>(row + (i - shift)));
    float f[N];
    load(i, f);
    return Elems<T, 16>::put(f);
  }
  // M neighbours from place i on, a multiple of M
  template <int M>
  __device__ __forceinline__ void load(unsigned int i, float (&f)[M]) const {
    if (i >= shift && i + M <= end) {
      Elems<T, M * (int)sizeof(T)>::get(__ldg(reinterpret_cast<const typename Raw<M * (int)sizeof(T)>::type*>(row + (i - shift))), f);
#pragma unroll
      for (int j = 0; j < M; ++j) f[j] = fmaxf(f[j], -INFINITY);
    } else {
#pragma unroll
      for (int j = 0; j < M; ++j) f[j] = i + j >= shift && i + j < end ? fmaxf((float)row[i + j - shift], -INFINITY) : -INFINITY;
    }
  }
};

// Logits as unsigned numbers in the same order; -0 is +0, so that no token has the key below +0's.
__device__ __forceinline__ unsigned int key_of(float f) {
  const unsigned int b = __float_as_uint(f + 0.f);
  return b ^ (b >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned int key) { return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xFFFFFFFFu)); }

// 2^(s / 16) - 1 for |s| <= 1/2, off by at most 5.1e-12, and exactly 0 at 0: s q(s), where q interpolates (2^(s / 16) - 1) / s at the four Chebyshev nodes of the range.
__device__ __forceinline__ double small_power(double s) {
  double q = fma(1.4676329855091502e-07, s, 1.3551125679403628e-05);
  q = fma(q, s, 0.0009383847927372583);
  q = fma(q, s, 0.043321698775062194);
  return q * s;
}

// fp32 to fp64 by integer instructions, of which an SM has eight times as many per clock as conversions: exact for normal numbers; what is smaller comes out
// as something below 2^-125, infinities as 2^128.
__device__ __forceinline__ double widened(float f) {
  const unsigned int b = __float_as_uint(f);
  return __hiloint2double((b & 0x80000000u) | (((b & 0x7FFFFFFFu) >> 3) + 0x38000000u), b << 29);
}

// An upper edge: compared as a logit, -0 would let +0 in.
__device__ __forceinline__ unsigned int without_minus_zero(unsigned int key) { return key == 0x7FFFFFFFu ? key - 1 : key; }

// The row's largest logit and temperature.
struct Weights {
  float top;
  double wide_top, inv_t, steps;     // steps: 16 log2(e) / T
  double reach;                      // -693 T: weights of 2^-1000
  const double* powers;              // in shared memory
  float least;                       // logits below it weigh nothing: less than 2^-1000, -inf. Rounded up: one below top + reach is outside of sixteenths()'s range
  float half_top, per_bin;           // per_bin: bins for each 2 of the logit
  bool plain;                        // what widened() makes of small numbers and infinities does not matter

  __device__ __forceinline__ void set(float largest, float t) {
    top = largest;
    plain = (t > 1e-25f && t < 1e25f) || top == INFINITY;
    wide_top = plain ? widened(top) : (double)top;
    inv_t = 1.0 / (double)t;
    reach = -693.0 * (double)t;
    steps = STEPS * 1.4426950408889634 * inv_t;
    least = top == INFINITY ? top : __double2float_ru(fmax((double)top + reach, -3.4028234663852886e38));
    half_top = 0.5f * top;
  }
  // Bins that reach `span` below the top, in units of T; the last one has all that is lower.
  __device__ __forceinline__ void set_bins(double span) { per_bin = (float)fmin(2 * (BINS - 1) / span * inv_t, 1e38); }
  __device__ __forceinline__ double exponent(float f) const { return f == top ? 0.0 : ((double)f - (double)top) * inv_t; }
  // 2^(x / 16) = 2^((n + s) / 16), n an integer, for x = d * by of -16000 at least
  __device__ __forceinline__ double sixteenths(double d, double by) const {
    const double t = fma(d, by, 6755399441055744.0);  // 1.5 * 2^52: the sum's low bits are n
    const double s = fma(d, by, 6755399441055744.0 - t);
    const int n = __double2loint(t);
    const double base = powers[n & (STEPS - 1)], x = fma(base, small_power(s), base);
    return __hiloint2double(__double2hiint(x) + ((n & ~(STEPS - 1)) << 16), __double2loint(x));
  }
  // The weight of a logit d <= 0 above the top, for d of -693 T at least
  __device__ __forceinline__ double power(double d) const { return sixteenths(d, steps); }
  __device__ __forceinline__ double of(float f) const {
    const float g = fmaxf(f, least);
    const double x = power((plain ? widened(g) : (double)g) - wide_top);
    return f < least ? 0.0 : x;
  }
  // The nearest whole number of bins below the top; falls with f in steps, whatever fp32 rounds.
  __device__ __forceinline__ unsigned int bin(float f) const {
    const float b = f == top ? 0.f : fminf(fmaf(-0.5f, f, half_top) * per_bin, (float)(BINS - 1));
    return __float_as_uint(b + 8388608.f) & (2 * BINS - 1);  // 2^23: the sum's low bits
  }
  // Below the top, in units of the logit: where bins of numbers up to b end at the latest, and those from b on begin at the earliest. Rounded differences and products move a
  // token by less than 1e-3 of a bin.
  __device__ __forceinline__ double bin_end(unsigned int b) const { return (b + 0.501) * 2.0 / (double)per_bin; }
  __device__ __forceinline__ double bin_begin(unsigned int b) const { return b ? (b - 0.501) * 2.0 / (double)per_bin : 0.0; }
};

// Weights in fp32 up to a factor that all of them share: 2^(x c - N) with c = log2(e) / T and N = rint(largest c), by the nearest integer n of x c and 2^(x c - n).
// A sum of eight is off by at most 3.5e-7 of itself: 1.5e-7 for ex2.approx (the most over all numbers in +-0.51), 2e-8 for its argument, 2^-24 for each of
// three additions. Two such sums are compared: SLACK is twice that and a third more. (tests/test_sample_gpu.py compares log probabilities with this bound over powers in +-1/2.)
constexpr double SLACK = 9.5367431640625e-7;          // 2^-20
constexpr double SLACK_OF_ONE = 4.76837158203125e-7;  // 2^-21: such a sum against an exact one
// Whether the token whose own weight lies between `before` and `before + weight` is the one at `goal` for sure, all relative to its tile's unit. Logits of less than 80 T below a
// tile's largest, -inf among them, and places that are not in the row weigh some 2^-115 each in fp32 instead of less or nothing, below 2^-104 per tile: goals above
// 2^-80 have a slack of more than that (2^-100), and the smaller ones, which take a u of less than 1e-23, are left open.
__device__ __forceinline__ bool for_sure(double before, double weight, double goal) {
  return goal > 8.271806125530277e-25 && goal - before > SLACK * goal && before + weight - goal > SLACK * goal;
}
__device__ __forceinline__ float2 fma_pair(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)), "l"(reinterpret_cast<const unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 add_pair(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)));
  return d;
}

struct FastWeights {
  TemperatureScale t;
  float n, magic, least;  // n: N
  bool usable;            // x c is exact enough and all of it in range
  __device__ __forceinline__ void set(float largest, const TemperatureScale& scale) {
    t = scale;
    n = rintf(largest * t.c);
    magic = 12582912.f - n;  // 1.5 * 2^23: the sum's low bits are n of x c less N
    least = largest - t.reach;
    usable = t.usable && fabsf(n) < 131072.f;  // x c_low is below 2^-7: r stays in +-0.51
  }
  __device__ __forceinline__ float of(float f) const {
    f = fmaxf(f, least);
    const float m = fmaf(f, t.c, magic);
    return finish(fmaf(f, t.c_low, fmaf(f, t.c, magic - m)), m);
  }
  static __device__ __forceinline__ float finish(float r, float m) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(r));
    return __uint_as_float(__float_as_uint(y) + (__float_as_uint(m) << 23));
  }
  // The same two at a time, the same bits.
  __device__ __forceinline__ float2 of_pair(float f, float g) const {
    const float2 x = make_float2(fmaxf(f, least), fmaxf(g, least)), c = make_float2(t.c, t.c), low = make_float2(t.c_low, t.c_low), base = make_float2(magic, magic);
    const float2 m = fma_pair(x, c, base), r = fma_pair(x, low, fma_pair(x, c, fma_pair(m, make_float2(-1.f, -1.f), base)));
    return make_float2(finish(r.x, m.x), finish(r.y, m.y));
  }
  // What weights relative to another largest logit are to be multiplied by: a power of two.
  __device__ __forceinline__ double unit(float other) const { return __hiloint2double((1023 + (int)fmaxf(rintf(other * t.c) - n, -1000.f)) << 20, 0); }
  // To weights relative to the largest logit itself.
  __device__ __forceinline__ double to_top(const Weights& w) const { return w.sixteenths((double)n - (double)w.top * 1.4426950408889634 * w.inv_t, STEPS); }
  template <int M>
  __device__ __forceinline__ double sum(const float (&f)[M]) const {
    float2 x[M / 2];
#pragma unroll
    for (int j = 0; j < M / 2; ++j) x[j] = of_pair(f[2 * j], f[2 * j + 1]);
#pragma unroll
    for (int o = 1; o < M / 2; o *= 2)
#pragma unroll
      for (int j = 0; j + o < M / 2; j += 2 * o) x[j] = add_pair(x[j], x[j + o]);
    return (double)(x[0].x + x[0].y);
  }
};

// The largest of 16 bytes of logits; NaN is none.
template <typename T>
__device__ __forceinline__ float largest_of(const uint4& v) {
  if constexpr (sizeof(T) == 2) {
    const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
    return fmaxf(fmaxf(__low2float(m), __high2float(m)), -INFINITY);
  } else {
    const float* p = reinterpret_cast<const float*>(&v);
    return fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), -INFINITY);
  }
}

// A warp per tile.
template <typename T>
__global__ void __launch_bounds__(TILE_THREADS) sample_tiles_kernel(const SampleArgs a, unsigned long long all) {
  constexpr int N = 16 / (int)sizeof(T), VECS = PER_LANE / N;
  let_next_start();
  const unsigned long long tile = ((unsigned long long)blockIdx.x * TILE_THREADS + threadIdx.x) >> 5;
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.open_count = 0;
  if (tile >= all) return;
  const size_t r = all >> 32 ? tile / a.tiles : (unsigned int)tile / a.tiles;
  const unsigned int lane = threadIdx.x & 31, first = (unsigned int)(tile - r * a.tiles) * TILE + lane * N;
  const RowView<T> row(a, r);
  uint4 v[VECS];
#pragma unroll
  for (int k = 0; k < VECS; ++k) v[k] = row.load_vector(first + k * 32 * N);
  float most = largest_of<T>(v[0]);
#pragma unroll
  for (int k = 1; k < VECS; ++k) most = fmaxf(most, largest_of<T>(v[k]));
  if (a.lane_most) a.lane_most[tile * 32 + lane] = most;
  for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
  const SampleRow ask(a, r);
  double sum = 0.0;
  if (ask.whole && most > -INFINITY) {
    FastWeights w;
    w.set(most, ask.scale);
    if (w.usable) {
#pragma unroll
      for (int k = 0; k < VECS; ++k) {
        float f[N];
        Elems<T, 16>::get(v[k], f);
        sum += w.sum(f);
      }
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    } else {
      sum = -1.0;
    }
  }
  if (lane == 0) a.stats[tile] = TileStat{sum, most, 0.f};
}

// Tokens that the shared memory of a block holds of one warp's tiles.
template <typename T> constexpr unsigned int SEGMENT = sizeof(T) == 2 ? 1280 : 896;
constexpr unsigned int SEGMENT_TILES = 64;  // of one warp at most: offsets in 16 bits

template <typename T>
struct SampleShared {
  unsigned int bins[3][BINS];  // the first ones, and two that take turns
  unsigned long long list[LIST], ordered[LIST], own[LIST];
  double sums[4][SAMPLE_WARPS];
  double powers[STEPS];
  unsigned int counts[SAMPLE_WARPS], found[4], listed;
  alignas(16) T values[SAMPLE_WARPS * SEGMENT<T>];           // gathered tokens by warp, in their order
  unsigned short offsets[SAMPLE_WARPS * SEGMENT<T>];         // of their places to the warp's first
};

// What is kept: logits above `value`, and the first `ties` of `equal` tokens that have it.
struct Cut {
  float value;
  unsigned int ties, equal;
};

__device__ __forceinline__ double warp_sum(double s) {
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  return s;
}
__device__ __forceinline__ float warp_max(float m) {
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  return m;
}
__device__ __forceinline__ double target_of(double u, double total) { return u >= 0.0 ? u * total : u < 0.0 ? 0.0 : INFINITY; }  // NaN: the end

// One warp's: the number of the first token of a tile that has this logit.
template <typename T>
__device__ __forceinline__ unsigned int first_of(const RowView<T>& row, unsigned int tile, float logit, int lane) {
  constexpr int N = 16 / (int)sizeof(T);
  unsigned int at = 0xFFFFFFFFu;
  for (unsigned int i = tile * TILE + lane * N; i < (tile + 1) * TILE; i += 32 * N) {
    float f[N];
    row.load(i, f);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (f[j] == logit) at = min(at, i + j);
  }
  return __reduce_min_sync(0xFFFFFFFFu, at) - row.shift;
}

// One warp's: the first token of places [from, to) with which `start` and the weight exceed the target, its weight, and in `start` what lies before it; without one the
// last token with any weight. weights(i, f, x): a lane's K logits from place i on and their weights, 0 for what is not kept.
template <int K, class V, class Of>
__device__ __forceinline__ bool walk(int lane, unsigned int from, unsigned int to, double& start, double target, unsigned int& place, float& logit, double& weight, Of weights) {
  for (unsigned int i = from + lane * K; i - lane * K < to; i += 32 * K) {
    float f[K];
    V x[K];
    weights(i, f, x);
    double mine = 0.0;
#pragma unroll
    for (int j = 0; j < K; ++j) mine += (double)x[j];
    double run = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const double below = __shfl_up_sync(0xFFFFFFFFu, run, o);
      if (lane >= o) run += below;
    }
    const unsigned int past = __ballot_sync(0xFFFFFFFFu, mine > 0.0 && start + run > target);
    const unsigned int any = __ballot_sync(0xFFFFFFFFu, mine > 0.0);
    if (any) {
      // in these vectors, or so far the last token with any weight
      const int who = past ? __ffs(past) - 1 : 31 - __clz(any);
      unsigned int at = 0;
      float l = 0.f;
      double s = start + (run - mine), before = s, own = 0.0;
      bool done = false;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        if (x[j] > (V)0 && !done) {
          at = i + j;
          l = f[j];
          before = s;
          own = (double)x[j];
          s += own;
          done = past && s > target;
        }
      }
      place = __shfl_sync(0xFFFFFFFFu, at, who);
      logit = __shfl_sync(0xFFFFFFFFu, l, who);
      weight = __shfl_sync(0xFFFFFFFFu, own, who);
      before = __shfl_sync(0xFFFFFFFFu, before, who);
      if (past) {
        start = before;
        return true;
      }
    }
    start += __shfl_sync(0xFFFFFFFFu, run, 31);
  }
  return false;
}

// PART: where the row need not be read a second time to see how far down top-p can reach, see estimated.
template <typename T, bool PART>
struct Sampler {
  static constexpr int M = 16 / (int)sizeof(T);  // neighbours that a lane takes at a time, of the gathered tokens or of the row
  const SampleArgs& a;
  SampleShared<T>& sh;
  size_t r;
  RowView<T> row;
  int lane, warp;
  Weights w;
  bool stored;                // places are those of the gathered tokens, otherwise the row's
  unsigned int begin, end;    // the warp's places
  float floor;                // of those that count

  // M tokens from place i on; what does not count as -inf.
  __device__ __forceinline__ void fetch(unsigned int i, float (&f)[M]) const {
    if (stored) {
      Elems<T, 16>::get(*reinterpret_cast<const uint4*>(sh.values + i), f);
    } else {
      row.load(i, f);
#pragma unroll
      for (int j = 0; j < M; ++j) f[j] = f[j] >= floor ? f[j] : -INFINITY;
    }
  }
  __device__ __forceinline__ unsigned int number_of(unsigned int place) const {
    return (stored ? first_tile(place / SEGMENT<T>) * TILE + sh.offsets[place] : place) - row.shift;
  }
  // Warps take neighbouring tiles.
  __device__ __forceinline__ unsigned int first_tile(unsigned int of_warp) const { return (unsigned int)((unsigned long long)a.tiles * of_warp / SAMPLE_WARPS); }
  // body(place of the first, logits) for the warp's tokens.
  template <class Body>
  __device__ __forceinline__ void each(Body body) const {
    for (unsigned int i = begin + lane * M; i - lane * M < end; i += 32 * M) {
      float f[M];
      fetch(i, f);
      body(i, f);
    }
  }
  // The weight of those that `counts` says, without a branch: the computations go side by side.
  template <int K, class Counts>
  __device__ __forceinline__ double weigh(const float (&f)[K], Counts counts) const {
    double x[K];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      x[j] = w.of(f[j]);
      x[j] = counts(f[j]) ? x[j] : 0.0;
    }
#pragma unroll
    for (int o = 1; o < K; o *= 2)
#pragma unroll
      for (int j = 0; j + o < K; j += 2 * o) x[j] += x[j + o];
    return x[0];
  }
  // Sums over the block of one value per thread, the same bits in all; the warps' own stay in sh.sums[k].
  __device__ __forceinline__ double block_sum(double s, int k) {
    s = warp_sum(s);
    __syncthreads();
    if (lane == 0) sh.sums[k][warp] = s;
    __syncthreads();
    return warps_sum(k);
  }
  __device__ __forceinline__ double warps_sum(int k) const { return warp_sum(lane < SAMPLE_WARPS ? sh.sums[k][lane] : 0.0); }
  // Inclusive scan over the block's threads.
  template <typename V>
  __device__ __forceinline__ V scan(V v, V* sums) {
    for (int o = 1; o < 32; o <<= 1) {
      const V below = __shfl_up_sync(0xFFFFFFFFu, v, o);
      if (lane >= o) v += below;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = v;
    __syncthreads();
    V before = lane < SAMPLE_WARPS ? sums[lane] : (V)0;
    for (int o = 1; o < SAMPLE_WARPS; o <<= 1) {
      const V below = __shfl_up_sync(0xFFFFFFFFu, before, o);
      if (lane >= o) before += below;
    }
    before = __shfl_sync(0xFFFFFFFFu, before, warp ? warp - 1 : 0);
    return warp ? before + v : v;
  }
  // Four of them at a time.
  __device__ __forceinline__ void scan4(double (&v)[4]) {
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const double below = __shfl_up_sync(0xFFFFFFFFu, v[k], o);
        if (lane >= o) v[k] += below;
      }
    __syncthreads();
    if (lane == 31)
#pragma unroll
      for (int k = 0; k < 4; ++k) sh.sums[k][warp] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      double before = lane < warp ? sh.sums[k][lane] : 0.0;
      for (int o = SAMPLE_WARPS / 2; o; o >>= 1) before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
      v[k] += __shfl_sync(0xFFFFFFFFu, before, 0);
    }
  }
  __device__ __forceinline__ unsigned int lanes_before(unsigned int v) const {
    unsigned int upto = v;
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned int below = __shfl_up_sync(0xFFFFFFFFu, upto, o);
      if (lane >= o) upto += below;
    }
    return upto - v;
  }

  // Largest key whose first bin is at least b, and smallest whose first bin is at most b.
  __device__ __forceinline__ unsigned int edge(unsigned int b, bool upper) const {
    // 32 places of the range at a time: how many of them lie on the lower side
    unsigned int lo = key_of(-INFINITY), span = key_of(w.top) - lo;  // the edge lies in [lo, lo + span]
    while (span) {
      const unsigned int step = span / 32 + 1, at = lo + (lane + 1) * step;  // candidates lo + step, ...; beyond lo + span counts as the upper side
      const bool inside = (lane + 1) * (unsigned long long)step <= span;
      bool low = false;  // whether the answer is at `at` or above
      if (inside) low = upper ? w.bin(value_of(at)) >= b : w.bin(value_of(at - 1)) > b;
      const unsigned int n = __popc(__ballot_sync(0xFFFFFFFFu, low));
      const unsigned int gone = n * step;
      lo += gone;
      span = span - gone < step - 1 ? span - gone : step - 1;
    }
    return lo;
  }

  // The first bin up to which the bins hold `count` (BINS where none does), with what is below it and in it in sh.found[1] and [2].
  __device__ __forceinline__ unsigned int reaches(int buffer, unsigned int count) {
    unsigned int own[BINS_PER_THREAD], mine = 0;
#pragma unroll
    for (int k = 0; k < BINS_PER_THREAD; ++k) mine += own[k] = sh.bins[buffer][threadIdx.x * BINS_PER_THREAD + k];
    unsigned int upto = scan(mine, sh.counts) - mine;
    if (threadIdx.x == 0) sh.found[0] = BINS;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < BINS_PER_THREAD; ++k) {
      if (upto < count && count <= upto + own[k]) {
        sh.found[0] = threadIdx.x * BINS_PER_THREAD + k;
        sh.found[1] = upto;
        sh.found[2] = own[k];
      }
      upto += own[k];
    }
    __syncthreads();
    return sh.found[0];
  }

  // Lowest and highest key of bin b of a window.
  __device__ __forceinline__ unsigned int edge_of(bool first, unsigned int lo, unsigned int hi, unsigned int shift, unsigned int b, bool upper) const {
    if (first) return edge(b, upper);
    if (upper) return hi - (b << shift);
    const unsigned int down = ((b + 1) << shift) - 1;
    return hi - lo > down ? hi - down : lo;
  }
  // What a limit is reached at: a share of a mass that may be off by `slack` of it. heavy: the part of the mass from `floor` on in fp64, 0 where it is not known.
  struct Target {
    double share, heavy, low, at, high;
    __device__ __forceinline__ Target(double share, double mass, double slack, double heavy = 0.0) : share(share), heavy(heavy), at(share * mass) {
      low = at * (1.0 - slack);
      high = at * (1.0 + slack);
    }
    // Whether a sum's side depends on what the mass is off.
    __device__ __forceinline__ bool open(double sum) const { return sum >= low && sum < high; }
  };
  // A nearer target, while sums and lists stay as they are. Some 7 % of rows with a flat distribution need it. The light tokens anew in fp32, and what these are off is less by
  // their share of the mass; only what that leaves open takes the row in fp64 (20 000 clocks more).
  __device__ __noinline__ void settle(Target& target) {
    if (PART && target.heavy > 0.0) {
      const SampleRow ask(a, r);
      FastWeights fast;
      fast.set(w.top, ask.scale);
      if (fast.usable) {
        double s = 0.0;
        each_of_row(-INFINITY, [&](unsigned int, const float (&f)[M]) {
          float light[M];
#pragma unroll
          for (int j = 0; j < M; ++j) light[j] = f[j] < floor ? f[j] : -INFINITY;
          s += fast.sum(light);
        });
        s = block_sum(s, 1) * fast.to_top(w);
        const double mass = target.heavy + s;
        target = Target(target.share, mass, SLACK_OF_ONE * s / mass + 1e-14);  // and what fp64 sums are off
        return;
      }
    }
    target = Target(target.share, whole_weight(), 0.0);
  }
  // Bins of a window in which the running weight, `mass` above it, reaches the target: at the earliest, by estimate, at the latest; false where it does not before the
  // tokens that weigh nothing. Weights of a bin's tokens are between those of its ends.
  // In mid and count: the estimates up to the ends of the thread's bins, and their tokens; in before: those of earlier threads' bins.
  __device__ __forceinline__ bool bracket(int buffer, bool first, unsigned int lo, unsigned int hi, unsigned int shift, double mass, const Target& target, unsigned int& b1, unsigned int& m, unsigned int& b2, double (&mid)[BINS_PER_THREAD],
                                          unsigned int (&count)[BINS_PER_THREAD], unsigned int& before) {
    unsigned int mine = 0;
    double low[BINS_PER_THREAD], high[BINS_PER_THREAD];
    double sum_low = 0.0, sum_mid = 0.0, sum_high = 0.0;
#pragma unroll
    for (int k = 0; k < BINS_PER_THREAD; ++k) {
      const unsigned int b = threadIdx.x * BINS_PER_THREAD + k;
      count[k] = first && b == BINS - 1 ? 0 : sh.bins[buffer][b];
      mine += count[k];
      double wl = 0.0, wh = 0.0;
      if (count[k]) {
        if (first) {
          wl = -w.bin_end(b) >= w.reach ? w.power(-w.bin_end(b)) : 0.0;
          wh = w.power(fmax(-w.bin_begin(b), w.reach));
        } else {
          wl = w.of(value_of(edge_of(false, lo, hi, shift, b, false)));
          wh = w.of(value_of(edge_of(false, lo, hi, shift, b, true)));
        }
      }
      low[k] = sum_low += wl * count[k];
      high[k] = sum_high += wh * count[k];
      mid[k] = sum_mid += 0.5 * (wl + wh) * count[k];
    }
    double upto4[4] = {sum_low, sum_mid, sum_high, (double)mine};
    scan4(upto4);
    const double before_low = upto4[0] - sum_low, before_mid = upto4[1] - sum_mid, before_high = upto4[2] - sum_high;
    unsigned int upto = (unsigned int)upto4[3] - mine;
    if (threadIdx.x == 0) sh.found[0] = 0;
    __syncthreads();
    // bins with tokens only: the first ones whose running weight reaches the target
    b1 = m = b2 = 0;
#pragma unroll
    for (int k = 0; k < BINS_PER_THREAD; ++k) {
      upto += count[k];
      if (count[k]) atomicMax(&sh.found[0], (unsigned int)(threadIdx.x * BINS_PER_THREAD + k));
      b1 += __syncthreads_count(upto == 0 || mass + before_high + high[k] < target.low);
      mid[k] += mass + before_mid;
      m += __syncthreads_count(upto == 0 || mid[k] < target.at);
      b2 += __syncthreads_count(upto == 0 || mass + before_low + low[k] < target.high);
    }
    if (first && b1 >= BINS) return false;
    const unsigned int last = sh.found[0];
    if (b2 > last) b2 = last;
    if (b1 > b2) b1 = b2;
    m = m < b1 ? b1 : m > b2 ? b2 : m;
#pragma unroll
    for (int k = BINS_PER_THREAD - 1; k >= 0; --k) {
      if (threadIdx.x * BINS_PER_THREAD + k == b2) sh.found[3] = upto;  // tokens up to this bin's end
      upto -= count[k];
    }
    before = upto;
    return true;
  }

  // find()'s part in the first bins for weights, while bins have few tokens: exact sums up to the ends of some bins around the estimated one say whether the limit is in them,
  // and what all estimates are off by there, so that the next ones are hardly ever wrong. Where the weight of all counted tokens is known, the first one is
  // corrected, too: what it is off comes from the heavy tokens. Without it half of the rows needed a second pass. False: bin m has too many tokens.
  static constexpr unsigned int BESIDE = 48;
  __device__ __forceinline__ bool by_bins(Target& target, unsigned int b1, unsigned int& m, unsigned int b2, const double (&mid)[BINS_PER_THREAD],
                                          const unsigned int (&count)[BINS_PER_THREAD], unsigned int before, Cut& cut) {
    bool corrected = PART && target.heavy > 0.0;
    double off = 0.0;
    if (corrected) {
      if (threadIdx.x == SAMPLE_THREADS - 1) sh.sums[3][0] = mid[BINS_PER_THREAD - 1];
      __syncthreads();
      off = target.heavy - sh.sums[3][0];
    }
    for (;;) {
      __syncthreads();
      if (corrected) {
        // the first bin with tokens from b1 on that reaches the target, or the last one with tokens up to b2
        if (threadIdx.x == 0) {
          sh.found[0] = BINS;
          sh.found[1] = 0;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < BINS_PER_THREAD; ++k) {
          const unsigned int b = threadIdx.x * BINS_PER_THREAD + k;
          if (count[k] && b >= b1 && b <= b2) {
            if (mid[k] + off >= target.at) atomicMin(&sh.found[0], b);
            atomicMax(&sh.found[1], b);
          }
        }
        __syncthreads();
        m = sh.found[0] < BINS ? sh.found[0] : sh.found[1];
        __syncthreads();
      }
      unsigned int upto = before;
#pragma unroll
      for (int k = 0; k < BINS_PER_THREAD; ++k) {
        if (threadIdx.x * BINS_PER_THREAD + k == m) {
          sh.listed = 0;
          sh.found[0] = sh.found[1] = m;
          sh.found[2] = upto;
          sh.found[3] = upto + count[k];
        }
        upto += count[k];
      }
      __syncthreads();
      const unsigned int before_m = sh.found[2], upto_m = sh.found[3];
      if (upto_m - before_m > LIST) return false;
      if (upto_m - before_m + 2 * BESIDE <= LIST) {
        upto = before;
#pragma unroll
        for (int k = 0; k < BINS_PER_THREAD; ++k) {
          const unsigned int b = threadIdx.x * BINS_PER_THREAD + k;
          if (b >= b1 && b < m && before_m - upto <= BESIDE) atomicMin(&sh.found[0], b);
          upto += count[k];
          if (b > m && b <= b2 && upto - upto_m <= BESIDE) atomicMax(&sh.found[1], b);
        }
        __syncthreads();
      }
      const unsigned int from = sh.found[0], to = sh.found[1];
#pragma unroll
      for (int k = 0; k < BINS_PER_THREAD; ++k)
        if (threadIdx.x * BINS_PER_THREAD + k == to) sh.sums[3][0] = mid[k];
      double s1 = 0.0, s2 = 0.0;  // the weight above these bins, and up to their end
      each([&](unsigned int i, const float (&f)[M]) {
        double x[M];
#pragma unroll
        for (int j = 0; j < M; ++j) x[j] = w.of(f[j]);
#pragma unroll
        for (int j = 0; j < M; ++j) {
          const unsigned int b = w.bin(f[j]);
          s2 += b <= to ? x[j] : 0.0;
          s1 += b < from ? x[j] : 0.0;
          if (b >= from && b <= to) append(f[j], i + j);
        }
      });
      s1 = block_sum(s1, 0);
      s2 = block_sum(s2, 1);
      while (target.open(s1) || target.open(s2)) settle(target);
      const bool left = s1 >= target.at && from > b1, right = s2 < target.at && to < b2;
      if (!left && !right) {
        order_list<false>(sh.listed, 0, target, s1, cut);
        return true;
      }
      if (left) b2 = from - 1;
      else b1 = to + 1;
      off = s2 - sh.sums[3][0];
      corrected = true;
    }
  }

  // The cut at which `target` tokens (BY_COUNT) or `target` weight is reached. The first bins have been counted.
  // False: there are not so many tokens; the weight is not reached before the tokens that weigh nothing.
  template <bool BY_COUNT>
  __device__ __noinline__ bool find(Target target, Cut& cut) {
    unsigned int lo = 0, hi = key_of(w.top), shift = 0;  // the window's keys
    unsigned int goal = BY_COUNT ? (unsigned int)target.at : 0;
    double mass = 0.0;  // weight above the window
    bool first = true;
    int buffer = 0;
    for (;;) {
      __syncthreads();  // all have counted
      const unsigned int next = buffer == 1 ? 2 : 1;
      auto edge_of = [&](unsigned int b, bool upper) { return this->edge_of(first, lo, hi, shift, b, upper); };
      unsigned int b1 = 0, b2 = 0, m = 0, above = 0;
      if constexpr (BY_COUNT) {
        m = reaches(buffer, goal);
        if (m >= BINS) return false;  // no more tokens than that
        above = sh.found[1];
        if (first && sh.found[2] <= LIST) {
          const unsigned int n = sh.found[2];
          if (threadIdx.x == 0) sh.listed = 0;
          __syncthreads();
          each([&](unsigned int i, const float (&f)[M]) {
#pragma unroll
            for (int j = 0; j < M; ++j)
              if (f[j] > -INFINITY && w.bin(f[j]) == m) append(f[j], i + j);
          });
          order_list<true>(n, goal - above, target, 0.0, cut);
          return true;
        }
      } else {
        double mid[BINS_PER_THREAD];
        unsigned int count[BINS_PER_THREAD], before;
        if (!bracket(buffer, first, lo, hi, shift, mass, target, b1, m, b2, mid, count, before)) return false;
        if (first && by_bins(target, b1, m, b2, mid, count, before, cut)) return true;
        __syncthreads();
        if (threadIdx.x == 0) sh.found[2] = sh.bins[buffer][m];
      }
      for (int i = threadIdx.x; i < BINS; i += SAMPLE_THREADS) sh.bins[next][i] = 0;
      if (threadIdx.x == 0) sh.listed = 0;
      __syncthreads();
      // the last one of the first bins has no lower end
      const unsigned int n = sh.found[2], key_lo = max(edge_of(m, false), key_of(-3.4028234663852886e38f)), key_hi = without_minus_zero(edge_of(m, true));
      if constexpr (BY_COUNT) goal -= above;  // of the bin's
      const bool one = key_lo == key_hi, listed = !one && n <= LIST;
      unsigned int new_shift = 0;
      while ((key_hi - key_lo) >> new_shift >= BINS) ++new_shift;
      double s1 = 0.0, s2 = 0.0;  // the weight above the bin, and up to its end
      const float least_in = value_of(key_lo), most_in = value_of(key_hi);
      if (!BY_COUNT || !one)
        each([&](unsigned int i, const float (&f)[M]) {
#pragma unroll
          for (int j = 0; j < M; ++j)
            if (!one && f[j] >= least_in && f[j] <= most_in) {
              if (listed) append(f[j], i + j);
              else atomicAdd(&sh.bins[next][(key_hi - key_of(f[j])) >> new_shift], 1u);
            }
          if constexpr (!BY_COUNT) {
            double x[M];
#pragma unroll
            for (int j = 0; j < M; ++j) x[j] = w.of(f[j]);
#pragma unroll
            for (int j = 0; j < M; ++j) {
              s2 += f[j] >= least_in ? x[j] : 0.0;
              s1 += f[j] > most_in ? x[j] : 0.0;
            }
          }
        });
      if constexpr (!BY_COUNT) {
        s1 = block_sum(s1, 0);
        s2 = block_sum(s2, 1);
        while (target.open(s1) || target.open(s2)) settle(target);
        const bool left = s1 >= target.at && m > b1, right = s2 < target.at && m < b2;
        if (left || right) {
          // the estimate was beside it: the bins between, counted anew
          const unsigned int old_lo = edge_of(b2, false), old_hi = edge_of(b1, true);
          lo = left ? key_hi + 1 : old_lo;
          hi = without_minus_zero(left ? old_hi : key_lo - 1);
          shift = 0;
          while ((hi - lo) >> shift >= BINS) ++shift;
          for (int i = threadIdx.x; i < BINS; i += SAMPLE_THREADS) sh.bins[next][i] = 0;
          __syncthreads();
          const float above_this = value_of(hi);
          double heavier = 0.0;
          each([&](unsigned int, const float (&f)[M]) {
            heavier += weigh(f, [&](float g) { return g > above_this; });
#pragma unroll
            for (int j = 0; j < M; ++j) {
              const unsigned int key = key_of(f[j]);
              if (key >= lo && key <= hi) atomicAdd(&sh.bins[next][(hi - key) >> shift], 1u);
            }
          });
          mass = block_sum(heavier, 0);
          first = false;
          buffer = next;
          continue;
        }
      }
      if (one) {
        cut.value = value_of(key_lo);
        cut.equal = n;
        if constexpr (BY_COUNT) {
          cut.ties = goal;
        } else {
          const double each_one = w.of(cut.value);
          while (ceil((target.low - s1) / each_one) != ceil((target.high - s1) / each_one)) settle(target);
          const double more = ceil((target.at - s1) / each_one);
          cut.ties = more < 1.0 ? 1u : more > (double)n ? n : (unsigned int)more;
        }
        return true;
      }
      if (listed) {
        order_list<BY_COUNT>(n, goal, target, s1, cut);
        return true;
      }
      lo = key_lo;
      hi = key_hi;
      shift = new_shift;
      mass = s1;
      first = false;
      buffer = next;
    }
  }

  // A token into the list.
  __device__ __forceinline__ void append(float f, unsigned int place) {
    sh.list[atomicAdd(&sh.listed, 1u) % LIST] = (unsigned long long)~key_of(f) << 32 | place;
  }
  // The n listed tokens in `ordered`: by falling logit, equal ones by place.
  __device__ __forceinline__ void order(unsigned int n) {
    __syncthreads();
    const unsigned int t = threadIdx.x;
    if (t < n) {
      const unsigned long long mine = sh.list[t];
      unsigned int place = 0;
#pragma unroll 8
      for (unsigned int j = 0; j < n; ++j) place += sh.list[j] < mine;
      sh.ordered[place] = mine;
    }
    __syncthreads();
  }
  // The cut among the n listed tokens: after `count` of them, or where `before` and their weight reach the target.
  template <bool BY_COUNT>
  __device__ __forceinline__ void order_list(unsigned int n, unsigned int count, Target& target, double before, Cut& cut) {
    order(n);
    const unsigned int t = threadIdx.x;
    const unsigned int key = t < n ? ~(unsigned int)(sh.ordered[t] >> 32) : 0;
    unsigned int keep = count;
    if constexpr (!BY_COUNT) {
      const double x = t < n ? w.of(value_of(key)) : 0.0;
      const double at = before + (scan(x, sh.sums[0]) - x);
      while (__syncthreads_or(t < n && target.open(at))) settle(target);
      keep = __syncthreads_count(t < n && at < target.at);
      if (keep == 0) keep = 1;
    }
    const unsigned int last = ~(unsigned int)(sh.ordered[keep - 1] >> 32);
    cut.value = value_of(last);
    cut.ties = __syncthreads_count(t < keep && key == last);
    cut.equal = __syncthreads_count(t < n && key == last);
  }

  // One thread's.
  __device__ __forceinline__ void write(long long token, float lp) {
    if (a.wide) static_cast<long long*>(a.tokens)[r] = token;
    else static_cast<int*>(a.tokens)[r] = (int)token;
    if (a.logprob) a.logprob[r] = lp;
  }
  __device__ __forceinline__ void write(unsigned int token, float logit, double total) { write(token, (float)(w.exponent(logit) - log(total))); }

  // The row's whole weight in fp64.
  __device__ __forceinline__ double whole_weight() {
    double s = 0.0;
    each_of_row(-INFINITY, [&](unsigned int, const float (&f)[M]) { s += weigh(f, [](float g) { return g >= -INFINITY; }); });  // not NaN
    return block_sum(s, 1);
  }

  // The token from the n listed ones, which hold all that are kept. mass: of all tokens that top_p counts, where it is not that of the first top_k; it may be
  // off by SLACK_OF_ONE. confirm: false where the listed tokens do not reach top_p's share for sure.
  __device__ __forceinline__ bool choose(unsigned int n, const SampleRow& ask, double mass, double u, bool confirm) {
    order(n);
    const unsigned int t = threadIdx.x, number = t < n ? (unsigned int)sh.ordered[t] : 0xFFFFFFFFu;
    const float logit = t < n ? value_of(~(unsigned int)(sh.ordered[t] >> 32)) : -INFINITY;
    double x = t < n && (!ask.by_k || t < (unsigned int)ask.top_k) ? w.of(logit) : 0.0;
    if (ask.by_p) {
      const double before = scan(x, sh.sums[0]) - x, p = ask.top_p;
      if (PART && confirm && warps_sum(0) < p * mass * (1.0 + SLACK)) return false;
      if (ask.by_k) mass = warps_sum(0);
      else if (__syncthreads_or(t < n && before >= p * mass * (1.0 - SLACK_OF_ONE) && before < p * mass * (1.0 + SLACK_OF_ONE))) mass = whole_weight();
      if (t > 0 && !(before < p * mass)) x = 0.0;
    }
    if (ask.by_m && t > 0 && !(x >= (double)ask.min_p)) x = 0.0;
    // kept tokens by number
    sh.own[t] = (unsigned long long)number << 32 | t;
    const unsigned int kept = __syncthreads_count(x > 0.0);  // a prefix
    double* sums = reinterpret_cast<double*>(sh.list);
    if (t < kept) {
      const unsigned long long mine = sh.own[t];
      unsigned int place = 0;
#pragma unroll 8
      for (unsigned int j = 0; j < kept; ++j) place += sh.own[j] < mine;
      sums[place] = x;
      sh.ordered[place] = (unsigned long long)__float_as_uint(logit) << 32 | number;
    }
    __syncthreads();
    const double upto = scan(t < kept ? sums[t] : 0.0, sh.sums[0]), total = warps_sum(0);
    const double target = target_of(u, total);
    unsigned int at = __syncthreads_count(t < kept && !(upto > target));
    if (at >= kept) at = kept - 1;
    if (t == 0) write((unsigned int)sh.ordered[at], __uint_as_float((unsigned int)(sh.ordered[at] >> 32)), total);
    return true;
  }

  // From the tiles' weights, relative to 2^n: their sum, and without a limit (choose) the token. False where fp32 leaves it open.
  __device__ __forceinline__ bool from_tiles(const SampleRow& ask, bool token, double u, double& total) {
    const TileStat* stats = a.stats + r * a.tiles;
    FastWeights top;
    top.set(w.top, ask.scale);
    // a thread's tiles are neighbours
    const unsigned int each_has = (a.tiles + SAMPLE_THREADS - 1) / SAMPLE_THREADS, t0 = min(threadIdx.x * each_has, a.tiles), t1 = min(t0 + each_has, a.tiles);
    double sum = 0.0;
    bool usable = top.usable;
    for (unsigned int k = t0; k < t1; ++k) {
      const TileStat s = stats[k];
      if (s.weight < 0.0) usable = false;
      if (s.weight > 0.0) sum += s.weight * top.unit(s.largest);
    }
    if (!__syncthreads_and(usable)) return false;
    const double upto = scan(sum, sh.sums[0]);
    total = warps_sum(0);
    const double to_top = top.to_top(w);
    if (!token) {
      total *= to_top;
      return true;
    }
    const double target = target_of(u, total);
    // the thread, the tile, and the warp of that thread goes through the tile
    if (threadIdx.x == 0) sh.found[0] = 0, sh.found[1] = SAMPLE_THREADS;
    __syncthreads();
    if (sum > 0.0 && upto > target && upto - sum <= target) atomicMin(&sh.found[1], threadIdx.x);
    __syncthreads();
    const unsigned int owner = sh.found[1];
    if (owner >> 5 == (unsigned int)warp && owner < SAMPLE_THREADS) {
      const int from = owner & 31;
      double start = __shfl_sync(0xFFFFFFFFu, upto - sum, from), weight = 0.0;
      const unsigned int k0 = __shfl_sync(0xFFFFFFFFu, t0, from), k1 = __shfl_sync(0xFFFFFFFFu, t1, from);
      for (unsigned int k = k0; k < k1; ++k) {
        const TileStat s = stats[k];
        if (!(s.weight > 0.0)) continue;
        const double scale = top.unit(s.largest);
        if (k + 1 < k1 && start + s.weight * scale <= target) {
          start += s.weight * scale;
          continue;
        }
        constexpr int N = 16 / (int)sizeof(T);
        FastWeights tile;
        tile.set(s.largest, ask.scale);
        unsigned int place = 0;
        float logit = w.top;
        double before = start / scale;  // an exact quotient by a power of two
        const double goal = target / scale;
        const bool found = walk<N, float>(lane, k * TILE, k * TILE + TILE, before, goal, place, logit, weight, [&](unsigned int i, float (&f)[N], float (&x)[N]) {
          row.load(i, f);
#pragma unroll
          for (int j = 0; j < N; ++j) x[j] = tile.of(f[j]);
        });
        if (found && for_sure(before, weight, goal) && lane == 0) {
          write(place - row.shift, logit, total * to_top);
          sh.found[0] = 1;
        }
        break;
      }
    }
    __syncthreads();
    return sh.found[0];
  }

  // body(place of the first, logits) for the row's tokens, M neighbours per lane and four such vectors at a time, by all warps. Vectors of tiles that have nothing of at
  // least `least` are left out. EVERY one of so many warps' vectors.
  template <unsigned int EVERY = 1, class Body>
  __device__ __forceinline__ void each_of_row(float least, Body body) const {
    constexpr unsigned int PER_TILE = PER_LANE / M;
    const TileStat* stats = a.stats + r * a.tiles;
    for (unsigned int q = warp * EVERY; q < a.tiles * PER_TILE; q += 4 * SAMPLE_WARPS * EVERY) {
      uint4 v[4];
      bool some[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned int at = q + k * SAMPLE_WARPS * EVERY;
        some[k] = at < a.tiles * PER_TILE && stats[at / PER_TILE].largest >= least;
        if (some[k]) v[k] = row.load_vector(at * (32 * M) + lane * M);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (some[k]) {
          float f[M];
          Elems<T, 16>::get(v[k], f);
          body((q + k * SAMPLE_WARPS * EVERY) * (32 * M) + lane * M, f);
        }
    }
  }

  // top-p from a part of the row: an estimate of how far down the limit can be, which the weight of the tokens above it has to confirm. What is left out,
  // (1 - p) of the weight, is mostly many light tokens, so that a part tells its weight well; of sampled tokens of at most weight w its variance is at most STRIDE w times it,
  // and four deviations are kept as a distance. 8000 clocks where counting the whole row took 29 000; 256 rows of 65536 with top-p 0.9, by their spread: 2.5 139 -> 118 us,
  // 4 110 -> 91, 6 65 -> 53; at 2, with more tokens kept than shared memory holds, 159 -> 164.
  static constexpr unsigned int STRIDE = 8;
  __device__ __forceinline__ bool estimated(double lowest, double left_out, double t, double& from, unsigned int& expected) {
    lowest -= 10.0 * t;  // what is lighter yet weighs e^-10 of what may be left out
    w.set_bins(fmin(REACH, -lowest * w.inv_t * 1.01 + 1e-6));
    for (int i = threadIdx.x; i < BINS; i += SAMPLE_THREADS) sh.bins[0][i] = 0;
    __syncthreads();
    const float least = fmaxf((float)((double)w.top + lowest), -3.4028235e38f);
    each_of_row<STRIDE>(least, [&](unsigned int, const float (&f)[M]) {
#pragma unroll
      for (int j = 0; j < M; ++j)
        if (f[j] >= least) atomicAdd(&sh.bins[0][w.bin(f[j])], 1u);
    });
    __syncthreads();
    double heaviest[BINS_PER_THREAD], upto[BINS_PER_THREAD], mine = 0.0;
    unsigned int count = 0;
#pragma unroll
    for (int k = 0; k < BINS_PER_THREAD; ++k) {
      const unsigned int b = threadIdx.x * BINS_PER_THREAD + k, n = sh.bins[0][b];
      heaviest[k] = w.power(fmax(-w.bin_begin(b), w.reach));
      upto[k] = mine += heaviest[k] * n * STRIDE;
      count += n;
    }
    const double before = scan(mine, sh.sums[0]) - mine, all_bins = warps_sum(0);
    unsigned int bin = 0;  // the first one behind which little enough is
#pragma unroll
    for (int k = 0; k < BINS_PER_THREAD; ++k) {
      const double behind = fmax(all_bins - before - upto[k], 0.0);
      bin += __syncthreads_count(behind + 4.0 * sqrt(behind * heaviest[k] * STRIDE) > left_out);
    }
    scan(threadIdx.x * BINS_PER_THREAD <= bin ? count : 0u, sh.counts);
    const unsigned int kept = __reduce_add_sync(0xFFFFFFFFu, lane < SAMPLE_WARPS ? sh.counts[lane] : 0u);
    __syncthreads();
    from = -w.bin_end(bin);
    expected = STRIDE * (unsigned int)(kept + 3.f * sqrtf((float)kept) + 1.f);
    return bin < BINS - 1;
  }
  // top-p: the tokens from `lowest` on are counted in bins, which say how far down the limit can be at most, and how many tokens there are up to there.
  __device__ __forceinline__ double narrowed(double lowest, const Target& target, unsigned int& expected) {
    w.set_bins(fmin(REACH, -lowest * w.inv_t * 1.01 + 1e-6));
    for (int i = threadIdx.x; i < 3 * BINS; i += SAMPLE_THREADS) sh.bins[0][i] = 0;
    __syncthreads();
    const float least = fmaxf((float)((double)w.top + lowest), -3.4028235e38f);
    unsigned int* bins = sh.bins[warp % 3];  // three sets: fewer warps meet at one bin
    each_of_row(least, [&](unsigned int, const float (&f)[M]) {
#pragma unroll
      for (int j = 0; j < M; ++j)
        if (f[j] >= least) atomicAdd(bins + w.bin(f[j]), 1u);
    });
    __syncthreads();
    for (int i = threadIdx.x; i < BINS; i += SAMPLE_THREADS) sh.bins[0][i] += sh.bins[1][i] + sh.bins[2][i];
    __syncthreads();
    unsigned int b1, m, b2, count[BINS_PER_THREAD], before;
    double mid[BINS_PER_THREAD];
    if (!bracket(0, true, 0, 0, 0, 0.0, target, b1, m, b2, mid, count, before)) return lowest;
    __syncthreads();
    expected = sh.found[3];
    return fmax(lowest, -w.bin_end(b2));
  }

  // The tokens of at least `floor` where few are expected, listed with their numbers for places: how many there are, or some number above LIST where there are more.
  __device__ __forceinline__ unsigned int gather_few() {
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    each_of_row(floor, [&](unsigned int i, const float (&f)[M]) {
      if (*(volatile unsigned int*)&sh.listed > LIST) return;
#pragma unroll
      for (int j = 0; j < M; ++j)
        if (f[j] >= floor) {
          const unsigned int at = atomicAdd(&sh.listed, 1u);
          if (at < LIST) sh.list[at] = (unsigned long long)~key_of(f[j]) << 32 | (i + j - row.shift);
        }
    });
    __syncthreads();
    return sh.listed;
  }

  // The tokens of at least `floor`: how many there are. Each warp's go to its segment of shared memory, in their order and with -inf behind them, where there is room.
  __device__ __forceinline__ unsigned int gather() {
    const TileStat* stats = a.stats + r * a.tiles;
    constexpr unsigned int SEG = SEGMENT<T>;
    T* to = sh.values + warp * SEG;
    unsigned short* offsets = sh.offsets + warp * SEG;
    unsigned int own = 0;
    const unsigned int t0 = first_tile(warp), t1 = first_tile(warp + 1), lower = (1u << lane) - 1;
    uint4 v[PER_LANE / M], next[PER_LANE / M];
    auto load = [&](unsigned int k) {
      return k < t1 && stats[k].largest >= floor;
    };
    auto vectors = [&](unsigned int k) {
#pragma unroll
      for (int q = 0; q < PER_LANE / M; ++q) next[q] = row.load_vector(k * TILE + (q * 32 + lane) * M);
    };
    bool some = load(t0);
    if (some) vectors(t0);
    for (unsigned int k = t0; k < t1; ++k) {
      const bool now = some;
#pragma unroll
      for (int q = 0; q < PER_LANE / M; ++q) v[q] = next[q];
      some = load(k + 1);
      if (some) vectors(k + 1);
      if (!now) continue;
#pragma unroll
      for (int q = 0; q < PER_LANE / M; ++q) {
        float f[M];
        unsigned int mine = 0;
        Elems<T, 16>::get(v[q], f);
#pragma unroll
        for (int j = 0; j < M; ++j) mine += f[j] >= floor;
        // how many the lanes before have, by the bits of their numbers
        unsigned int before = 0, all = 0;
#pragma unroll
        for (int b = 0; (1 << b) <= M; ++b) {
          const unsigned int have = __ballot_sync(0xFFFFFFFFu, mine >> b & 1);
          before += __popc(have & lower) << b;
          all += __popc(have) << b;
        }
        if (mine) {
          unsigned int at = own + before;
          const unsigned int offset = (k - t0) * TILE + (q * 32 + lane) * M;
#pragma unroll
          for (int j = 0; j < M; ++j) {
            const bool keep = f[j] >= floor;
            if (keep && at < SEG) {
              to[at] = (T)f[j];
              offsets[at] = (unsigned short)(offset + j);
            }
            at += keep;
          }
        }
        own += all;
      }
    }
    const unsigned int whole = min((own + 32 * M - 1) / (32 * M) * (32 * M), SEG);
    for (unsigned int i = own + lane; i < whole; i += 32) to[i] = (T)-INFINITY;
    if (lane == 0) sh.counts[warp] = own;
    begin = warp * SEG;
    end = begin + whole;
    stored = __syncthreads_and(own <= SEG && t1 - t0 <= SEGMENT_TILES);
    return __reduce_add_sync(0xFFFFFFFFu, lane < SAMPLE_WARPS ? sh.counts[lane] : 0u);
  }
  // They are counted in the first bins. WEIGHED: returns their weight.
  template <bool WEIGHED>
  __device__ __forceinline__ double counted(double lowest) {
    w.set_bins(fmin(REACH, -lowest * w.inv_t * 1.01 + 1e-6));
    __syncthreads();
    for (int i = threadIdx.x; i < BINS; i += SAMPLE_THREADS) sh.bins[0][i] = 0;
    __syncthreads();
    double s = 0.0;
    each([&](unsigned int, const float (&f)[M]) {
      if constexpr (WEIGHED) s += weigh(f, [](float g) { return g > -INFINITY; });
#pragma unroll
      for (int j = 0; j < M; ++j)
        if (f[j] > -INFINITY) atomicAdd(&sh.bins[0][w.bin(f[j])], 1u);
    });
    if constexpr (WEIGHED) s = block_sum(s, 0);
    return s;
  }
  // The gathered tokens as a list.
  __device__ __forceinline__ void list_all() {
    const unsigned int own = sh.counts[warp], before = __reduce_add_sync(0xFFFFFFFFu, lane < warp ? sh.counts[lane] : 0u);
    for (unsigned int i = lane; i < own; i += 32)
      sh.list[before + i] = (unsigned long long)~key_of((float)sh.values[begin + i]) << 32 | number_of(begin + i);
  }

  // The token by sums over the kept ones in fp64, by places.
  __device__ __forceinline__ void by_sums(const Cut& cut, double least, double u) {
    unsigned int ties = 0;  // of this warp's at the cut
    if (cut.ties) {
      ties = 0xFFFFFFFFu;
      if (cut.ties < cut.equal) {
        unsigned int mine = 0;
        each([&](unsigned int, const float (&f)[M]) {
#pragma unroll
          for (int j = 0; j < M; ++j) mine += f[j] == cut.value;
        });
        mine = __reduce_add_sync(0xFFFFFFFFu, mine);
        const unsigned int before = __shfl_sync(0xFFFFFFFFu, scan(lane == 0 ? mine : 0u, sh.counts), 0) - mine;
        ties = before >= cut.ties ? 0 : cut.ties - before;
        if (ties >= mine) ties = 0xFFFFFFFFu;  // all of them
      }
    }
    const bool in_part = ties && ties != 0xFFFFFFFFu;
    unsigned int seen = 0;  // tokens at the cut in the warp's vectors before
    auto kept = [&](unsigned int i, float (&f)[M], double (&x)[M]) {
      unsigned int order = 0;
      fetch(i, f);
      if (in_part) {
        unsigned int mine = 0;
#pragma unroll
        for (int j = 0; j < M; ++j) mine += f[j] == cut.value;
        order = lanes_before(mine);
        const unsigned int all = __shfl_sync(0xFFFFFFFFu, order + mine, 31);
        order += seen;
        seen += all;
      }
#pragma unroll
      for (int j = 0; j < M; ++j) x[j] = w.of(f[j]);
#pragma unroll
      for (int j = 0; j < M; ++j) {
        const bool equal = f[j] == cut.value && ties, keep = (f[j] > cut.value || (equal && order < ties)) && x[j] >= least;
        order += equal;
        x[j] = keep ? x[j] : 0.0;
      }
    };
    double sum = 0.0;
    for (unsigned int i = begin + lane * M; i - lane * M < end; i += 32 * M) {
      float f[M];
      double x[M];
      kept(i, f, x);
#pragma unroll
      for (int j = 0; j < M; ++j) sum += x[j];
    }
    const double total = block_sum(sum, 1), target = target_of(u, total);
    // the warp in which it is crossed, or the last one with any weight
    double start = 0.0, upto = 0.0, weight;
    int where = 0;
    for (int i = 0; i < SAMPLE_WARPS; ++i) {
      const double s = sh.sums[1][i];
      if (s > 0.0) {
        where = i;
        start = upto;
        upto += s;
        if (upto > target) break;
      }
    }
    if (where != warp) return;
    unsigned int place = 0;
    float logit = w.top;
    seen = 0;
    walk<M, double>(lane, begin, end, start, target, place, logit, weight, kept);
    if (lane == 0) write(number_of(place), logit, total);
  }

  // The warps' shares of `all` places.
  __device__ __forceinline__ void share(unsigned int all) {
    constexpr unsigned int PIECE = 32 * M;
    const unsigned int pieces = (all + PIECE - 1) / PIECE;
    begin = pieces * warp / SAMPLE_WARPS * PIECE;
    end = pieces * (warp + 1) / SAMPLE_WARPS * PIECE;
  }

  __device__ __forceinline__ void run() {
    const SampleRow ask(a, r);
    const TileStat* stats = a.stats + r * a.tiles;
    const double u = a.u[r];
    w.powers = sh.powers;
    float top = -INFINITY;
    for (unsigned int k = threadIdx.x; k < a.tiles; k += SAMPLE_THREADS) top = fmaxf(top, stats[k].largest);
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    if (lane == 0) sh.sums[0][warp] = top;
    __syncthreads();
    for (int i = 0; i < SAMPLE_WARPS; ++i) top = fmaxf(top, (float)sh.sums[0][i]);
    if (!(top > -INFINITY)) {
      if (threadIdx.x == 0) write(-1, 0.f);
      return;
    }
    if (ask.greedy) {
      // the first tile that has the largest, and in it the first place
      unsigned int tile = 0xFFFFFFFFu, at;
      for (unsigned int k = threadIdx.x; k < a.tiles; k += SAMPLE_THREADS)
        if (stats[k].largest == top) {
          tile = k;
          break;
        }
      tile = __reduce_min_sync(0xFFFFFFFFu, tile);
      if (lane == 0) sh.counts[warp] = tile;
      __syncthreads();
      for (int i = 0; i < SAMPLE_WARPS; ++i) tile = min(tile, sh.counts[i]);
      if (warp) return;
      at = first_of(row, tile, top, lane);
      if (lane == 0) write(at, 0.f);
      return;
    }
    w.set(top, ask.t);
    stored = false;
    floor = -3.4028234663852886e38f;
    Cut cut{-INFINITY, 0, 0};
    double all = 0.0, slack = SLACK_OF_ONE;
    if (!ask.by_k && !ask.by_p && !ask.by_m) {
      if (!a.logprob && from_tiles(ask, true, u, all)) return;  // a logarithm near 0 needs more than fp32 sums
      share(row.end);
      by_sums(cut, 0.0, u);
      return;
    }
    // what is certainly not kept
    double lowest = -INFINITY;  // of logits, as a difference to the largest
    unsigned int expected = 0xFFFFFFFFu;  // tokens that will be gathered
    bool part = false, narrow = false;    // from what a part of the row says, to be confirmed, and from all of it
    double from = 0.0, whole = 0.0;       // whole: the gathered tokens' weight, where it is known
    if (ask.by_k) {
      // as many lanes as top_k have a logit in the bins up to this one
      for (int i = threadIdx.x; i < BINS; i += SAMPLE_THREADS) sh.bins[0][i] = 0;
      __syncthreads();
      w.set_bins(REACH);
      const float* most = a.lane_most + r * a.tiles * 32;
      for (unsigned int i = threadIdx.x; i < a.tiles * 32; i += SAMPLE_THREADS)
        if (most[i] > -INFINITY) atomicAdd(&sh.bins[0][w.bin(most[i])], 1u);
      __syncthreads();
      const unsigned int bin = reaches(0, ask.top_k);
      if (bin < BINS - 1) {
        lowest = -w.bin_end(bin);
        expected = ask.top_k;  // and some
      }
    } else if (ask.by_p) {
      if (!from_tiles(ask, false, u, all)) {
        all = whole_weight();
        slack = 0.0;
      }
      // logf is off by 1e-5 at most here, and the sum by less
      lowest = (double)(logf((float)((1.0 - (double)ask.top_p) * all) / (float)a.vocab) - 1e-3f) * (double)ask.t;
      if constexpr (PART) part = top < INFINITY && estimated(lowest, (1.0 - (double)ask.top_p) * all, (double)ask.t, from, expected) && from > lowest;
      narrow = !part;
    }
    const double lightest = ask.by_m && !(ask.by_k && ask.by_p) ? (double)(logf(ask.min_p) - 1e-3f) * (double)ask.t : -INFINITY;  // top_p counts all of the first top_k
    unsigned int n;
    for (;;) {
      if (narrow) lowest = narrowed(lowest, Target(ask.top_p, all, SLACK), expected);
      // rounded to fp32 it is no more than any logit that it is no more than
      floor = top == INFINITY ? top : (float)fmax((double)top + fmax(part ? from : lowest, lightest), -3.4028234663852886e38);
      if (expected <= LIST) {
        n = gather_few();
        if (n <= LIST) {
          if (choose(n, ask, all, u, part && lightest < from)) return;
          part = false;
          narrow = true;
          continue;
        }
      }
      n = gather();
      if constexpr (!PART) break;
      if (!part || lightest >= from) break;
      if (!stored) share(row.end);
      whole = counted<true>(from);
      if (whole >= (double)ask.top_p * all * (1.0 + SLACK)) break;
      whole = 0.0;
      part = false;
      narrow = true;
    }
    if (part) lowest = from;
    lowest = fmax(lowest, lightest);
    if (stored && n <= LIST) {
      list_all();
      choose(n, ask, all, u, false);
      return;
    }
    if (!stored) share(row.end);
    if (ask.by_k || ask.by_p) {
      if (whole == 0.0) counted<false>(lowest);
      if (ask.by_k) {
        find<true>(Target(1.0, ask.top_k, 0.0), cut);
        if (ask.by_p) {
          double s = 0.0;
          each([&](unsigned int, const float (&f)[M]) { s += weigh(f, [&](float g) { return g > cut.value; }); });
          all = block_sum(s, 0);
          if (cut.ties) all += cut.ties * w.of(cut.value);
          slack = 0.0;
        }
      }
      if (ask.by_p) {
        Cut c;
        const bool found = find<false>(Target(ask.top_p, all, slack, whole), c);
        if (found && (c.value > cut.value || (c.value == cut.value && c.ties < cut.ties))) cut = c;
      }
    }
    by_sums(cut, ask.by_m ? (double)ask.min_p : 0.0, u);
  }
};

// ------------------------------------------------------------------ calls without a limit: a warp per row (1024 rows of 65536 62 us, by a block per row 130)

constexpr int WHOLE_THREADS = 128;

// EXACT = false: every row, by its tiles' weights in fp32; rows that these leave open are listed. EXACT = true: the listed ones, by weights in fp64.
template <typename T, bool EXACT>
__global__ void __launch_bounds__(WHOLE_THREADS) sample_whole_kernel(const SampleArgs a, size_t rows) {
  constexpr int N = 16 / (int)sizeof(T);
  __shared__ double powers[STEPS];
  let_next_start();
  if (threadIdx.x < STEPS) powers[threadIdx.x] = exp2(threadIdx.x / (double)STEPS);
  __syncthreads();
  after_previous();
  const int lane = threadIdx.x & 31;
  const size_t count = EXACT ? *a.open_count : rows;
  for (size_t at = ((size_t)blockIdx.x * WHOLE_THREADS + threadIdx.x) >> 5; at < count; at += (size_t)gridDim.x * WHOLE_THREADS / 32) {
    const size_t r = EXACT ? a.open[at] : at;
    const SampleRow ask(a, r);
    const RowView<T> row(a, r);
    const TileStat* stats = a.stats + r * a.tiles;
    auto write = [&](long long token, float lp) {
      if (lane) return;
      if (a.wide) static_cast<long long*>(a.tokens)[r] = token;
      else static_cast<int*>(a.tokens)[r] = (int)token;
      if (a.logprob) a.logprob[r] = lp;
    };
    // a lane's tiles are neighbours
    const unsigned int each_has = (a.tiles + 31) / 32, t0 = min(lane * each_has, a.tiles), t1 = min(t0 + each_has, a.tiles);
    float top = -INFINITY;
    unsigned int first = 0xFFFFFFFFu;
    for (unsigned int k = t0; k < t1; ++k)
      if (stats[k].largest > top) {
        top = stats[k].largest;
        first = k;
      }
    const float own = top;
    top = warp_max(top);
    if (!(top > -INFINITY)) {
      write(-1, 0.f);
      continue;
    }
    if (ask.greedy) {
      first = __reduce_min_sync(0xFFFFFFFFu, own == top ? first : 0xFFFFFFFFu);
      write(first_of(row, first, top, lane), 0.f);
      continue;
    }
    Weights w;
    w.powers = powers;
    w.set(top, ask.t);
    FastWeights fast;
    fast.set(top, ask.scale);
    auto weight_of = [&](unsigned int k) {
      const TileStat s = stats[k];
      return EXACT ? s.weight : s.weight > 0.0 ? s.weight * fast.unit(s.largest) : 0.0;
    };
    double sum = 0.0;
    bool usable = EXACT || fast.usable;
    for (unsigned int k = t0; k < t1; ++k) {
      usable = usable && (EXACT || stats[k].weight >= 0.0);
      sum += weight_of(k);
    }
    usable = __all_sync(0xFFFFFFFFu, usable);
    double upto = sum;
    for (int o = 1; o < 32; o <<= 1) {
      const double below = __shfl_up_sync(0xFFFFFFFFu, upto, o);
      if (lane >= o) upto += below;
    }
    const double total = __shfl_sync(0xFFFFFFFFu, upto, 31), target = target_of(a.u[r], total);
    // the lane's tiles, then the tile, in which it is crossed; the last one with any weight
    const unsigned int any = __ballot_sync(0xFFFFFFFFu, sum > 0.0), past = __ballot_sync(0xFFFFFFFFu, sum > 0.0 && upto > target);
    const int from = past ? __ffs(past) - 1 : 31 - __clz(any);
    double start = __shfl_sync(0xFFFFFFFFu, upto - sum, from);
    unsigned int tile = 0;
    {
      const unsigned int k0 = __shfl_sync(0xFFFFFFFFu, t0, from), k1 = __shfl_sync(0xFFFFFFFFu, t1, from);
      double before = start;
      for (unsigned int k = k0; k < k1; ++k) {
        const double x = weight_of(k);
        if (!(x > 0.0)) continue;
        tile = k;
        start = before;
        before += x;
        if (before > target) break;
      }
    }
    unsigned int place = 0;
    float logit = top;
    double weight = 0.0;
    uint4 v[PER_LANE / N];  // the tile, its loads side by side
#pragma unroll
    for (int k = 0; k < PER_LANE / N; ++k) v[k] = row.load_vector(tile * TILE + (k * 32 + lane) * N);
    auto logits = [&](unsigned int i, float (&f)[N]) {
#pragma unroll
      for (int k = 0; k < PER_LANE / N; ++k)
        if ((i - tile * TILE) / (32 * N) == k) Elems<T, 16>::get(v[k], f);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = fmaxf(f[j], -INFINITY);
    };
    if constexpr (EXACT) {
      walk<N, double>(lane, tile * TILE, tile * TILE + TILE, start, target, place, logit, weight, [&](unsigned int i, float (&f)[N], double (&x)[N]) {
        logits(i, f);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = w.of(f[j]);
      });
      write(place - row.shift, (float)(w.exponent(logit) - log(total)));
    } else {
      bool sure = false;
      if (usable) {
        FastWeights own_unit;
        own_unit.set(stats[tile].largest, ask.scale);
        const double unit = fast.unit(stats[tile].largest), goal = target / unit;  // exact quotients by a power of two
        double before = start / unit;
        const bool found = walk<N, float>(lane, tile * TILE, tile * TILE + TILE, before, goal, place, logit, weight, [&](unsigned int i, float (&f)[N], float (&x)[N]) {
          logits(i, f);
#pragma unroll
          for (int j = 0; j < N; ++j) x[j] = own_unit.of(f[j]);
        });
        sure = found && for_sure(before, weight, goal);
      }
      double all = total * fast.to_top(w);
      if (a.logprob && usable) {
        // the largest token's tile in fp64: where it has most of the weight the logarithm is near 0, and what fp32 is off would be much of it
        const unsigned int most = __reduce_min_sync(0xFFFFFFFFu, own == top ? first : 0xFFFFFFFFu);
        double exact = 0.0;
#pragma unroll
        for (int k = 0; k < PER_LANE / N; ++k) {
          float f[N];
          Elems<T, 16>::get(row.load_vector(most * TILE + (k * 32 + lane) * N), f);
#pragma unroll
          for (int j = 0; j < N; ++j) exact += w.of(fmaxf(f[j], -INFINITY));
        }
        for (int o = 16; o; o >>= 1) exact += __shfl_xor_sync(0xFFFFFFFFu, exact, o);
        all += exact - stats[most].weight * fast.unit(stats[most].largest) * fast.to_top(w);
      }
      if (sure) write(place - row.shift, (float)(w.exponent(logit) - log(all)));
      else if (lane == 0) a.open[atomicAdd(a.open_count, 1u)] = (unsigned int)r;
    }
  }
}

// Weights of the listed rows' tiles in fp64, relative to the row's largest logit: a warp per tile.
template <typename T>
__global__ void __launch_bounds__(TILE_THREADS) sample_exact_kernel(const SampleArgs a) {
  constexpr int N = 16 / (int)sizeof(T);
  __shared__ double powers[STEPS];
  let_next_start();
  if (threadIdx.x < STEPS) powers[threadIdx.x] = exp2(threadIdx.x / (double)STEPS);
  __syncthreads();
  after_previous();
  const int lane = threadIdx.x & 31;
  const unsigned long long all = (unsigned long long)*a.open_count * a.tiles;
  for (unsigned long long at = ((unsigned long long)blockIdx.x * TILE_THREADS + threadIdx.x) >> 5; at < all; at += (unsigned long long)gridDim.x * TILE_THREADS / 32) {
    const size_t r = a.open[at / a.tiles];
    const unsigned int k = (unsigned int)(at % a.tiles);
    TileStat* stats = a.stats + r * a.tiles;
    float top = -INFINITY;
    for (unsigned int i = lane; i < a.tiles; i += 32) top = fmaxf(top, stats[i].largest);
    top = warp_max(top);
    Weights w;
    w.powers = powers;
    w.set(top, SampleRow(a, r).t);
    const RowView<T> row(a, r);
    double sum = 0.0;
    for (unsigned int i = k * TILE + lane * N; i < (k + 1) * TILE; i += 32 * N) {
      float f[N];
      row.load(i, f);
      double x[N];
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = w.of(f[j]);
#pragma unroll
      for (int o = 1; o < N; o *= 2)
#pragma unroll
        for (int j = 0; j + o < N; j += 2 * o) x[j] += x[j + o];
      sum += x[0];
    }
    sum = warp_sum(sum);
    if (lane == 0) stats[k].weight = sum;
  }
}

template <typename T, bool PART>
__global__ void __launch_bounds__(SAMPLE_THREADS) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) unsigned char shared[];
  SampleShared<T>& sh = *reinterpret_cast<SampleShared<T>*>(shared);
  if (threadIdx.x < STEPS) sh.powers[threadIdx.x] = exp2(threadIdx.x / (double)STEPS);
  after_previous();
  Sampler<T, PART> s{a, sh, blockIdx.x, RowView<T>(a, blockIdx.x), (int)threadIdx.x & 31, (int)threadIdx.x >> 5};
  s.run();
}

constexpr size_t SAMPLE_ROWS_MOST = 1 << 24, SAMPLE_VOCAB_MOST = 1 << 24;

size_t sample_space(size_t rows, size_t vocab, void* base, SampleArgs* a) {
  Carver c(base);
  a->tiles = (unsigned int)((vocab + 7 + TILE - 1) / TILE);  // with up to 7 places before the first token
  a->stats = c.take<TileStat>(rows * a->tiles);
  a->lane_most = c.take<float>(rows * a->tiles * 32);
  a->open_count = c.take<unsigned int>(1);
  a->open = c.take<unsigned int>(rows);
  return c.used;
}

// Rows of at least so many tiles are estimated from a part: 256 rows with top-p 0.99, 32768 with a spread of 4 104 -> 82 us, 24576 92 -> 78; but 16384 with a spread of 2
// and top-p 0.9 76 -> 87, 8192 66 -> 71.
constexpr unsigned int PART_TILES = 32;

template <typename T>
cudaError_t sample_rows(const SampleArgs& a, size_t rows, bool limits, int sms, cudaStream_t s) {
  const unsigned long long all = (unsigned long long)rows * a.tiles;
  Chain chain(s);
  if (!limits) {
    const unsigned int per_block = WHOLE_THREADS / 32, blocks = (unsigned int)((rows + per_block - 1) / per_block), some = (unsigned int)sms * 4;
    chain.launch(sample_tiles_kernel<T>, dim3((unsigned int)((all * 32 + TILE_THREADS - 1) / TILE_THREADS)), TILE_THREADS, 0, 0, a, all);
    chain.launch(sample_whole_kernel<T, false>, dim3(blocks), WHOLE_THREADS, 0, 0, a, rows);
    chain.launch(sample_exact_kernel<T>, dim3(all * 32 / TILE_THREADS + 1 < some ? (unsigned int)(all * 32 / TILE_THREADS + 1) : some), TILE_THREADS, 0, 0, a);
    chain.launch(sample_whole_kernel<T, true>, dim3(blocks < some ? blocks : some), WHOLE_THREADS, 0, 0, a, rows);
    return chain.err;
  }
  const bool part = !a.lane_most && (a.row_top_p || a.top_p < 1.f) && a.tiles >= PART_TILES;
  const auto kernel = part ? sample_kernel<T, true> : sample_kernel<T, false>;
  chain.err = part ? with_shared<sample_kernel<T, true>>((int)sizeof(SampleShared<T>)) : with_shared<sample_kernel<T, false>>((int)sizeof(SampleShared<T>));
  chain.launch(sample_tiles_kernel<T>, dim3((unsigned int)((all * 32 + TILE_THREADS - 1) / TILE_THREADS)), TILE_THREADS, 0, 0, a, all);
  chain.launch(kernel, dim3((unsigned int)rows), SAMPLE_THREADS, sizeof(SampleShared<T>), 0, a);
  return chain.err;
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

int b2_sample_options_default(b2_sample_options* o) {
  if (!o) return call_error(B2_ERR_INVALID, "b2_sample_options_default: null pointer");
  *o = b2_sample_options{1.f, 0, 1.f, 0.f, nullptr, nullptr, nullptr, nullptr};
  return B2_OK;
}

int b2_sample_workspace(size_t rows, size_t vocab, size_t* bytes) {
  if (rows > SAMPLE_ROWS_MOST || vocab == 0 || vocab > SAMPLE_VOCAB_MOST)
    return call_error(B2_ERR_INVALID, "b2_sample_workspace: %zu rows of %zu (2^24 at most, 1 to 2^24)", rows, vocab);
  if (!bytes) return call_error(B2_ERR_INVALID, "b2_sample_workspace: null pointer");
  SampleArgs a{};
  *bytes = sample_space(rows, vocab, nullptr, &a);
  return B2_OK;
}

int b2_sample(size_t rows, size_t vocab, int dtype, const void* logits, size_t ld, const float* u, const b2_sample_options* o, void* tokens,
              int token_bytes, float* logprob, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "b2_sample";
  if (!dtype_ok(dtype)) return call_error(B2_ERR_INVALID, "%s: dtype %d", who, dtype);
  if (rows > SAMPLE_ROWS_MOST || vocab == 0 || vocab > SAMPLE_VOCAB_MOST)
    return call_error(B2_ERR_INVALID, "%s: %zu rows of %zu (2^24 at most, 1 to 2^24)", who, rows, vocab);
  if (token_bytes != 4 && token_bytes != 8) return call_error(B2_ERR_INVALID, "%s: tokens of %d bytes", who, token_bytes);
  if (!o || (rows && (!logits || !u || !tokens || !workspace))) return call_error(B2_ERR_INVALID, "%s: null pointer", who);
  const size_t e = dtype_bytes(dtype);
  if (ld < vocab) return call_error(B2_ERR_INVALID, "%s: leading dimension smaller than the width", who);
  if (reinterpret_cast<size_t>(logits) % e || reinterpret_cast<size_t>(tokens) % token_bytes ||
      (reinterpret_cast<size_t>(u) | reinterpret_cast<size_t>(logprob) | reinterpret_cast<size_t>(o->row_temperature) | reinterpret_cast<size_t>(o->row_top_k) |
       reinterpret_cast<size_t>(o->row_top_p) | reinterpret_cast<size_t>(o->row_min_p)) % 4)
    return call_error(B2_ERR_INVALID, "%s: a pointer is not aligned to its elements", who);
  if (o->temperature != o->temperature || o->top_p != o->top_p || o->min_p != o->min_p) return call_error(B2_ERR_INVALID, "%s: an option is not a number", who);
  if (reinterpret_cast<size_t>(workspace) % 256) return call_error(B2_ERR_INVALID, "%s: the workspace is not on a 256-byte boundary", who);
  SampleArgs a{};
  const size_t need = sample_space(rows, vocab, workspace, &a);
  if (rows && workspace_bytes < need) return call_error(B2_ERR_INVALID, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, need);
  int sms, rc;
  if ((rc = lm_device(&sms)) != B2_OK) return rc;
  auto vector = [&](const char* name, const void* p, size_t bytes, bool written) { return extent(name, p, 1, rows * bytes, rows * bytes, written); };
  Extent args[] = {extent("logits", logits, rows, vocab * e, ld * e, false), vector("u", u, 4, false), vector("row_temperature", o->row_temperature, 4, false),
                   vector("row_top_k", o->row_top_k, 4, false), vector("row_top_p", o->row_top_p, 4, false), vector("row_min_p", o->row_min_p, 4, false),
                   vector("tokens", tokens, token_bytes, true), vector("logprob", logprob, 4, true),
                   extent("the workspace", workspace, 1, rows ? need : 0, need, true)};
  if ((rc = refuse_overlap(who, args, 9)) != B2_OK) return rc;
  if (!rows) return B2_OK;
  a.logits = static_cast<const char*>(logits);
  a.ld = ld * e;
  a.vocab = (unsigned int)vocab;
  a.u = u;
  a.temperature = o->temperature;
  a.scale = scale_of_temperature(o->temperature < 3.4028235e38f ? o->temperature : 3.4028235e38f);
  a.top_p = o->top_p;
  a.min_p = o->min_p;
  a.top_k = o->top_k;
  a.row_temperature = o->row_temperature;
  a.row_top_k = o->row_top_k;
  a.row_top_p = o->row_top_p;
  a.row_min_p = o->row_min_p;
  a.tokens = tokens;
  a.wide = token_bytes == 8;
  a.logprob = logprob;
  if (!o->row_top_k && !(o->top_k > 0 && (size_t)o->top_k < vocab)) a.lane_most = nullptr;
  const bool greedy = (!o->row_temperature && !(o->temperature > 0.f)) || (!o->row_top_k && o->top_k == 1) || (!o->row_top_p && o->top_p <= 0.f) || (!o->row_min_p && o->min_p > 1.f);
  const bool limits = !greedy && (a.lane_most || o->row_top_p || o->top_p < 1.f || o->row_min_p || o->min_p > 0.f);
  const cudaError_t err = dtype == B2_DTYPE_BF16 ? sample_rows<__nv_bfloat16>(a, rows, limits, sms, static_cast<cudaStream_t>(stream))
                                                 : sample_rows<float>(a, rows, limits, sms, static_cast<cudaStream_t>(stream));
  return launch_error(err, who);
}

}  // extern "C"
