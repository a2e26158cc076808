// A token per row of logits from a given uniform number, with temperature, top-k, top-p and min-p:
//
//   w[v] = exp((x[v] - max) / T)      kept = a prefix of the tokens in falling order of x, equal ones by number
//   token = first v by number with  sum of kept w up to v  >  u * sum of all kept w
//
// A cluster of 1, 2, 4 or 8 blocks takes a row, each block a part of it by number and each warp a part of that. Nothing is sorted: top-k and top-p
// are a logit (the last one kept) and how many of the tokens that have exactly this one are kept, found by counting tokens in bins:
// first bins of equal width in (max - x) / T, then of equal width in the logit's bits inside the bin in which the limit must lie, until a bin has few
// enough tokens to put them in order one by one, or a single logit. For top-k counts say which bin. For top-p they only give an estimate, since a bin's
// weights differ; the weight above and up to the bin is then summed exactly, so that a wrong estimate is found and the search goes on beside it.
// Then every warp sums its kept weights, and the one in which the running sum crosses the target goes through its part once more.
//
// Sums are in fp64: with a vocabulary of 10^5 a step of the running sum may be 10^-5 of it, and what the sum is off, times the number of steps, is the
// probability that another token comes out.
#include <cooperative_groups.h>
#include <math.h>

#include "lm.cuh"

namespace cg = cooperative_groups;

namespace b2 {
namespace {

constexpr int SAMPLE_THREADS = 512, SAMPLE_WARPS = SAMPLE_THREADS / 32;
constexpr int BINS = 1024, BINS_PER_THREAD = BINS / SAMPLE_THREADS;
constexpr float REACH = 40.f;  // of the first bins, in units of T: the last bin has all tokens of less than e^-40 of the largest weight
constexpr int LIST = SAMPLE_THREADS;  // tokens that are put in order one by one
constexpr int MOST_CLUSTER = 8;
constexpr int STEPS = 16;  // 2^(n / 16) for n = 0 to 15 lie in different banks of shared memory

struct SampleArgs {
  const char* logits;
  size_t ld;  // bytes
  unsigned int vocab, part;  // part: tokens per block, whole tiles for each warp
  int vec;                   // rows begin on 16-byte boundaries
  const float* u;
  float temperature, top_p, min_p;
  int top_k;
  const float *row_temperature, *row_top_p, *row_min_p;
  const int* row_top_k;
  void* tokens;
  int wide;
  float* logprob;
};

struct SampleShared {
  unsigned int bins[3][BINS];  // the first ones, and two that take turns
  unsigned long long gathered[LIST], own[LIST], ordered[LIST];
  unsigned int gathered_n[2];  // by search
  double slots[2][MOST_CLUSTER][2];
  double warp_sums[2][SAMPLE_WARPS];
  unsigned int warp_counts[SAMPLE_WARPS];
  unsigned int found[4];
  double powers[STEPS];
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
  const double* powers;              // in shared memory
  float least;                       // logits below it weigh nothing: less than 2^-1000, -inf
  float half_top, per_bin;           // per_bin: bins for each 2 of the logit
  bool plain;                        // what widened() makes of small numbers and infinities does not matter

  __device__ __forceinline__ void set(float largest, float t) {
    top = largest;
    plain = (t > 1e-25f && t < 1e25f) || top == INFINITY;
    wide_top = plain ? widened(top) : (double)top;
    inv_t = 1.0 / (double)t;
    steps = STEPS * 1.4426950408889634 * inv_t;
    least = top == INFINITY ? top : (float)fmax((double)top - 693.0 * (double)t, -3.4028234663852886e38);
    half_top = 0.5f * top;
    per_bin = (float)fmin(2 * (BINS - 1) / REACH * inv_t, 1e38);
  }
  __device__ __forceinline__ double exponent(float f) const { return f == top ? 0.0 : ((double)f - (double)top) * inv_t; }
  // The weight: 2^((n + s) / 16), n an integer
  __device__ __forceinline__ double of(float f) const {
    const float g = fmaxf(f, least);
    const double d = (plain ? widened(g) : (double)g) - wide_top;
    const double t = fma(d, steps, 6755399441055744.0);  // 1.5 * 2^52: the sum's low bits are n
    const double s = fma(d, steps, 6755399441055744.0 - t);
    const int n = __double2loint(t);
    const double base = powers[n & (STEPS - 1)], w = fma(base, small_power(s), base);
    const unsigned int hi = __double2hiint(w) + ((n & ~(STEPS - 1)) << 16);
    return __hiloint2double(f < least ? 0 : hi, f < least ? 0 : __double2loint(w));
  }
  // 0 at the top; falls with f in steps, whatever fp32 rounds
  __device__ __forceinline__ unsigned int bin(float f) const {
    const unsigned int b = f == top ? 0u : __float2uint_rz(fmaf(-0.5f, f, half_top) * per_bin);
    return b < BINS ? b : BINS - 1;
  }
};

// What is kept: logits above `value`, and the first `ties` of `equal` tokens that have it.
struct Cut {
  float value;
  unsigned int ties, equal;
};

template <typename T, bool HELD>
struct Sampler {
  static constexpr int N = 16 / (int)sizeof(T), TILE = 32 * N;
  const SampleArgs& a;
  SampleShared& sh;
  cg::cluster_group cluster;
  const T* row;           // the whole row
  const uint4* held;      // this block's part in shared memory
  unsigned int part0, w0, w1;  // tokens: the block's first one, the warp's first one and the end of its tiles
  int lane, warp, ranks, rank, turn;
  Weights w;

  __device__ __forceinline__ void everyone() {
    if (ranks > 1) cluster.sync();
    else __syncthreads();
  }
  // N tokens from number i on, NaN and what is behind the row as -inf.
  __device__ __forceinline__ void load(unsigned int i, float (&f)[N]) const {
    if (a.vec && i + N <= a.vocab) {
      Elems<T, 16>::get(__ldg(reinterpret_cast<const uint4*>(row + i)), f);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = fmaxf(f[j], -INFINITY);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = i + j < a.vocab ? fmaxf((float)row[i + j], -INFINITY) : -INFINITY;
    }
  }
  __device__ __forceinline__ void fetch(unsigned int i, float (&f)[N]) const {
    if constexpr (HELD) Elems<T, 16>::get(held[(i - part0) / N], f);
    else load(i, f);
  }
  // body(number, logit) for the warp's tokens, lane by lane N neighbours at a time.
  template <class Body>
  __device__ __forceinline__ void each(Body body) const {
    for (unsigned int i = w0 + lane * N; i < w1; i += TILE) {
      float f[N];
      fetch(i, f);
#pragma unroll
      for (int j = 0; j < N; ++j) body(i + j, f[j]);
    }
  }

  // body(number of the first, logits) for the warp's tokens, N neighbours at a time.
  template <class Body>
  __device__ __forceinline__ void each_vector(Body body) const {
    for (unsigned int i = w0 + lane * N; i < w1; i += TILE) {
      float f[N];
      fetch(i, f);
      body(i, f);
    }
  }
  // The sum of the weights that `counts` says, without a branch: the N computations go side by side.
  template <class Counts>
  __device__ __forceinline__ double weigh(const float (&f)[N], Counts counts) const {
    double x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      x[j] = w.of(f[j]);
      x[j] = counts(f[j]) ? x[j] : 0.0;
    }
#pragma unroll
    for (int o = 1; o < N; o *= 2)
#pragma unroll
      for (int j = 0; j + o < N; j += 2 * o) x[j] += x[j + o];
    return x[0];
  }

  // Sums over the cluster of two values per thread, the same bits everywhere.
  __device__ __forceinline__ void sum2(double& x, double& y) {
    for (int o = 16; o; o >>= 1) {
      x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
      y += __shfl_xor_sync(0xFFFFFFFFu, y, o);
    }
    if (lane == 0) {
      sh.warp_sums[0][warp] = x;
      sh.warp_sums[1][warp] = y;
    }
    __syncthreads();
    x = y = 0.0;
    for (int i = 0; i < SAMPLE_WARPS; ++i) {
      x += sh.warp_sums[0][i];
      y += sh.warp_sums[1][i];
    }
    exchange(x, y);
  }
  // x and y: the block's, in all of its threads; sums over the blocks in their order.
  __device__ __forceinline__ void exchange(double& x, double& y) {
    give(x, y);
    x = y = 0.0;
    for (int i = 0; i < ranks; ++i) {
      x += taken(i, 0);
      y += taken(i, 1);
    }
  }
  // Every block's pair into every block's slots. The other set of slots is written next time: who gets there has seen that all blocks are past reading this one.
  __device__ __forceinline__ void give(double x, double y) {
    turn ^= 1;
    if ((int)threadIdx.x < ranks) {
      double* s = ranks > 1 ? cluster.map_shared_rank(&sh.slots[turn][rank][0], threadIdx.x) : &sh.slots[turn][0][0];
      s[0] = x;
      s[1] = y;
    }
    everyone();
  }
  __device__ __forceinline__ double taken(int r, int k) const { return sh.slots[turn][r][k]; }

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
    for (int i = 0; i < warp; ++i) v += sums[i];
    return v;
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

  // The cut at which `target` tokens (BY_COUNT) or `target` weight is reached. The first bins have been counted. search: 0 or 1, a list's counter of its own.
  // NONE: it is not reached before the tokens that weigh nothing. GATHERED: no cut, but a list of `gathered` tokens from the first one on in which it lies.
  enum Found { NONE, CUT, GATHERED };
  template <bool BY_COUNT>
  __device__ Found find(double target, int search, Cut& cut, unsigned int& gathered) {
    unsigned int lo = 0, hi = key_of(w.top), shift = 0;  // the window's keys
    const unsigned int goal = BY_COUNT ? (unsigned int)target : 0;
    unsigned int above = 0;  // tokens above the window
    double mass = 0.0;       // weight above the window
    bool first = true;
    int buffer = 0;
    for (;;) {
      if (!first) everyone();  // all blocks have counted
      unsigned int count[BINS_PER_THREAD];
#pragma unroll
      for (int k = 0; k < BINS_PER_THREAD; ++k) {
        count[k] = 0;
        for (int r = 0; r < ranks; ++r)
          count[k] += *(ranks > 1 ? cluster.map_shared_rank(&sh.bins[buffer][threadIdx.x * BINS_PER_THREAD + k], r) : &sh.bins[buffer][threadIdx.x * BINS_PER_THREAD + k]);
      }
      const unsigned int next = buffer == 1 ? 2 : 1;
      for (int i = threadIdx.x; i < BINS; i += SAMPLE_THREADS) sh.bins[next][i] = 0;
      auto edge_of = [&](unsigned int b, bool upper) -> unsigned int {
        if (first) return edge(b, upper);
        if (upper) return hi - (b << shift);
        const unsigned int down = ((b + 1) << shift) - 1;
        return hi - lo > down ? hi - down : lo;
      };
      unsigned int b1 = 0, b2 = 0, m = 0;
      if constexpr (BY_COUNT) {
        unsigned int mine = 0;
#pragma unroll
        for (int k = 0; k < BINS_PER_THREAD; ++k) mine += count[k];
        unsigned int upto = scan(mine, sh.warp_counts) - mine;
        if (threadIdx.x == 0) sh.found[0] = BINS;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < BINS_PER_THREAD; ++k) {
          if (above + upto < goal && goal <= above + upto + count[k]) {
            sh.found[0] = threadIdx.x * BINS_PER_THREAD + k;
            sh.found[1] = upto;
            sh.found[2] = count[k];
          }
          upto += count[k];
        }
        __syncthreads();
        m = sh.found[0];
        if (first && m >= BINS - 1) return NONE;
        b2 = m;
      } else {
        // the running weight at the bins' ends, by the lightest, the heaviest and a middle token of each
        double low[BINS_PER_THREAD], mid[BINS_PER_THREAD], high[BINS_PER_THREAD];
        double sum_low = 0.0, sum_mid = 0.0, sum_high = 0.0;
#pragma unroll
        for (int k = 0; k < BINS_PER_THREAD; ++k) {
          const unsigned int b = threadIdx.x * BINS_PER_THREAD + k;
          double wl = 0.0, wh = 0.0;
          if (count[k]) {
            if (first) {
              const double width = 2.0 * w.inv_t / (double)w.per_bin;  // rounded differences and products move a token by less than 1e-3 of a bin
              wl = exp(-width * (b + 1.001));
              wh = exp(-width * (b > 0 ? b - 0.001 : 0.0));
            } else {
              wl = w.of(value_of(edge_of(b, false)));
              wh = w.of(value_of(edge_of(b, true)));
            }
          }
          low[k] = sum_low += wl * count[k];
          high[k] = sum_high += wh * count[k];
          mid[k] = sum_mid += 0.5 * (wl + wh) * count[k];
        }
        const double before_low = scan(sum_low, sh.warp_sums[0]) - sum_low, before_high = scan(sum_high, sh.warp_sums[0]) - sum_high,
                     before_mid = scan(sum_mid, sh.warp_sums[0]) - sum_mid;
        unsigned int mine = 0;
#pragma unroll
        for (int k = 0; k < BINS_PER_THREAD; ++k) mine += count[k];
        unsigned int upto = scan(mine, sh.warp_counts) - mine;
        if (threadIdx.x == 0) sh.found[0] = 0;
        __syncthreads();
        // bins with tokens only: the first ones whose running weight reaches the target
#pragma unroll
        for (int k = 0; k < BINS_PER_THREAD; ++k) {
          upto += count[k];
          if (count[k]) atomicMax(&sh.found[0], (unsigned int)(threadIdx.x * BINS_PER_THREAD + k));
          b1 += __syncthreads_count(upto == 0 || mass + before_high + high[k] < target);
          m += __syncthreads_count(upto == 0 || mass + before_mid + mid[k] < target);
          b2 += __syncthreads_count(upto == 0 || mass + before_low + low[k] < target);
        }
        if (first && b1 >= BINS) return NONE;
        const unsigned int last = sh.found[0];
        if (b2 > last) b2 = last;
        if (b1 > b2) b1 = b2;
        m = m < b1 ? b1 : m > b2 ? b2 : m;
#pragma unroll
        for (int k = 0; k < BINS_PER_THREAD; ++k) {
          if (threadIdx.x * BINS_PER_THREAD + k == m) sh.found[2] = count[k];
          if (threadIdx.x * BINS_PER_THREAD + k == b2) sh.found[3] = upto - (k + 1 < BINS_PER_THREAD ? count[BINS_PER_THREAD - 1] : 0);
        }
        __syncthreads();
      }
      if (first) {
        const unsigned int all = BY_COUNT ? sh.found[1] + sh.found[2] : sh.found[3];
        if (all <= LIST) {
          each([&](unsigned int i, float f) {
            if (w.bin(f) <= b2) append(search, f, i);
          });
          everyone();
          gathered = all;
          return GATHERED;
        }
      }
      const unsigned int n = sh.found[2], key_lo = edge_of(m, false), key_hi = without_minus_zero(edge_of(m, true));
      if constexpr (BY_COUNT) above += sh.found[1];
      const bool one = key_lo == key_hi, listed = !one && n <= LIST;
      const unsigned int width = key_hi - key_lo;
      unsigned int new_shift = 0;
      while (width >> new_shift >= BINS) ++new_shift;
      __syncthreads();  // the bins are zeroed, sh.found is read
      double s1 = 0.0, s2 = 0.0;
      if (!BY_COUNT || !one) {
        const float least_in = value_of(key_lo), most_in = value_of(key_hi);
        if (!one)
          each([&](unsigned int i, float f) {
            if (!(f >= least_in && f <= most_in)) return;
            if (listed) append(search, f, i);
            else atomicAdd(&sh.bins[next][(key_hi - key_of(f)) >> new_shift], 1u);
          });
        if constexpr (!BY_COUNT)
          each_vector([&](unsigned int, const float (&f)[N]) {
            double x[N];
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = w.of(f[j]);
#pragma unroll
            for (int j = 0; j < N; ++j) {
              s2 += f[j] >= least_in ? x[j] : 0.0;
              s1 += f[j] > most_in ? x[j] : 0.0;
            }
          });
        if constexpr (!BY_COUNT) sum2(s1, s2);
        else everyone();
      }
      if constexpr (!BY_COUNT) {
        const bool left = s1 >= target && m > b1, right = s2 < target && m < b2;
        if (left || right) {
          // the estimate was beside it: the bins between, counted anew
          const unsigned int old_lo = edge_of(b2, false), old_hi = edge_of(b1, true);
          lo = left ? key_hi + 1 : old_lo;
          hi = without_minus_zero(left ? old_hi : key_lo - 1);
          mass = left ? 0.0 : s2;
          shift = 0;
          while ((hi - lo) >> shift >= BINS) ++shift;
          if (listed && threadIdx.x == 0 && rank == 0) sh.gathered_n[search] = 0;
          for (int i = threadIdx.x; i < BINS; i += SAMPLE_THREADS) sh.bins[next][i] = 0;
          double above_window = 0.0, none = 0.0;
          __syncthreads();
          each([&](unsigned int i, float f) {
            const unsigned int key = key_of(f);
            if (key >= lo && key <= hi) atomicAdd(&sh.bins[next][(hi - key) >> shift], 1u);
          });
          if (left) {
            const float above_this = value_of(hi);
            each_vector([&](unsigned int, const float (&f)[N]) { above_window += weigh(f, [&](float g) { return g > above_this; }); });
            sum2(above_window, none);
            mass = above_window;
          }
          first = false;
          buffer = next;
          continue;
        }
      }
      if (one) {
        cut.value = value_of(key_lo);
        cut.equal = n;
        if constexpr (BY_COUNT) {
          cut.ties = goal - above;
        } else {
          const double more = ceil((target - s1) / w.of(cut.value));
          cut.ties = more < 1.0 ? 1u : more > (double)n ? n : (unsigned int)more;
        }
        return CUT;
      }
      if (listed) {
        order_list(n, BY_COUNT ? (double)(goal - above) : target, s1, BY_COUNT, cut);
        return CUT;
      }
      lo = key_lo;
      hi = key_hi;
      shift = new_shift;
      mass = s1;
      first = false;
      buffer = next;
    }
  }

  // A token into the first block's list.
  __device__ __forceinline__ void append(int search, float f, unsigned int i) {
    unsigned int* counter = ranks > 1 ? cluster.map_shared_rank(&sh.gathered_n[search], 0) : &sh.gathered_n[search];
    unsigned long long* list = ranks > 1 ? cluster.map_shared_rank(sh.gathered, 0) : sh.gathered;
    list[atomicAdd(counter, 1u) % LIST] = (unsigned long long)~key_of(f) << 32 | i;
  }
  // The n gathered tokens in `ordered`: by falling logit, equal ones by number.
  __device__ __forceinline__ void order(unsigned int n) {
    const unsigned long long* list = ranks > 1 ? cluster.map_shared_rank(sh.gathered, 0) : sh.gathered;
    const unsigned int t = threadIdx.x;
    unsigned long long mine = ~0ull;
    if (t < n) sh.own[t] = mine = list[t];
    __syncthreads();
    if (t < n) {
      unsigned int place = 0;
      for (unsigned int j = 0; j < n; ++j) place += sh.own[j] < mine;
      sh.ordered[place] = mine;
    }
    __syncthreads();
  }
  // The token from n gathered ones that hold all that are kept, by the first block. mass: of all tokens that top_p counts, where it is not that of the first top_k.
  __device__ __forceinline__ void choose(unsigned int r, unsigned int n, unsigned int top_k, bool by_k, double mass, bool by_p, double top_p, double least, double u) {
    order(n);
    const unsigned int t = threadIdx.x, number = t < n ? (unsigned int)sh.ordered[t] : 0xFFFFFFFFu;
    const float logit = t < n ? value_of(~(unsigned int)(sh.ordered[t] >> 32)) : -INFINITY;
    double x = t < n && (!by_k || t < top_k) ? w.of(logit) : 0.0;
    if (by_p) {
      const double upto = scan(x, sh.warp_sums[0]);
      if (by_k) {
        mass = 0.0;
        for (int i = 0; i < SAMPLE_WARPS; ++i) mass += sh.warp_sums[0][i];
      }
      if (t > 0 && !(upto - x < top_p * mass)) x = 0.0;
    }
    if (t > 0 && !(x >= least)) x = 0.0;
    // kept tokens by number
    __syncthreads();
    sh.own[t] = (unsigned long long)number << 32 | t;
    const unsigned int kept = __syncthreads_count(x > 0.0);  // a prefix
    double* sums = reinterpret_cast<double*>(sh.gathered);
    if (t < kept) {
      unsigned int place = 0;
      for (unsigned int j = 0; j < kept; ++j) place += sh.own[j] < sh.own[t];
      sums[place] = x;
      sh.ordered[place] = (unsigned long long)__float_as_uint(logit) << 32 | number;
    }
    __syncthreads();
    const double upto = scan(t < kept ? sums[t] : 0.0, sh.warp_sums[0]);
    double total = 0.0;
    for (int i = 0; i < SAMPLE_WARPS; ++i) total += sh.warp_sums[0][i];
    const double target = target_of(u, total);
    unsigned int at = __syncthreads_count(t < kept && !(upto > target));
    if (at >= kept) at = kept - 1;
    if (t == 0) write(r, (unsigned int)sh.ordered[at], (float)(w.exponent(__uint_as_float((unsigned int)(sh.ordered[at] >> 32))) - log(total)));
  }
  __device__ __forceinline__ static double target_of(double u, double total) { return u >= 0.0 ? u * total : u < 0.0 ? 0.0 : INFINITY; }  // NaN: the end

  // The cut among the n gathered tokens.
  __device__ __forceinline__ void order_list(unsigned int n, double target, double before, bool by_count, Cut& cut) {
    order(n);
    const unsigned int t = threadIdx.x;
    const unsigned int key = t < n ? ~(unsigned int)(sh.ordered[t] >> 32) : 0;
    unsigned int keep;
    if (by_count) {
      keep = (unsigned int)target;
    } else {
      const double x = t < n ? w.of(value_of(key)) : 0.0;
      const double upto = scan(x, sh.warp_sums[0]);
      keep = __syncthreads_count(t < n && before + (upto - x) < target);
      if (keep == 0) keep = 1;
    }
    const unsigned int last = ~(unsigned int)(sh.ordered[keep - 1] >> 32);
    cut.value = value_of(last);
    cut.ties = __syncthreads_count(t < keep && key == last);
    cut.equal = __syncthreads_count(t < n && key == last);
  }

  __device__ __forceinline__ void write(unsigned int r, long long token, float lp) {
    if (a.wide) static_cast<long long*>(a.tokens)[r] = token;
    else static_cast<int*>(a.tokens)[r] = (int)token;
    if (a.logprob) a.logprob[r] = lp;
  }

  __device__ void run(unsigned int r) {
    float t = a.row_temperature ? a.row_temperature[r] : a.temperature, top_p = a.row_top_p ? a.row_top_p[r] : a.top_p,
          min_p = a.row_min_p ? a.row_min_p[r] : a.min_p;
    const int top_k = a.row_top_k ? a.row_top_k[r] : a.top_k;
    const double u = a.u[r];
    // the part into shared memory, and the largest logit
    float top = -INFINITY;
    for (unsigned int i = w0 + lane * N; i < w1; i += TILE * 4) {
      float f[4][N];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k * TILE < w1) load(i + k * TILE, f[k]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (i + k * TILE >= w1) break;
        if constexpr (HELD) const_cast<uint4*>(held)[(i + k * TILE - part0) / N] = Elems<T, 16>::put(f[k]);
#pragma unroll
        for (int j = 0; j < N; ++j) top = fmaxf(top, f[k][j]);
      }
    }
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    if (lane == 0) sh.warp_sums[0][warp] = top;
    for (int i = threadIdx.x; i < BINS; i += SAMPLE_THREADS) sh.bins[0][i] = 0;
    if (threadIdx.x < 2) sh.gathered_n[threadIdx.x] = 0;
    if (threadIdx.x < STEPS) sh.powers[threadIdx.x] = exp2(threadIdx.x / (double)STEPS);
    w.powers = sh.powers;
    __syncthreads();
    for (int i = 0; i < SAMPLE_WARPS; ++i) top = fmaxf(top, (float)sh.warp_sums[0][i]);
    give(top, 0.0);
    for (int i = 0; i < ranks; ++i) top = fmaxf(top, (float)taken(i, 0));
    if (!(top > -INFINITY)) {
      if (rank == 0 && threadIdx.x == 0) write(r, -1, 0.f);
      return;
    }
    if (!(t > 0.f) || top_k == 1 || top_p <= 0.f || min_p > 1.f) {
      unsigned int at = 0xFFFFFFFFu;
      each([&](unsigned int i, float f) {
        if (f == top && i < at) at = i;
      });
      at = __reduce_min_sync(0xFFFFFFFFu, at);
      if (lane == 0) sh.warp_counts[warp] = at;
      __syncthreads();
      for (int i = 0; i < SAMPLE_WARPS; ++i) at = min(at, sh.warp_counts[i]);
      give(at, 0.0);
      for (int i = 0; i < ranks; ++i) at = min(at, (unsigned int)taken(i, 0));
      if (rank == 0 && threadIdx.x == 0) write(r, at, 0.f);
      return;
    }
    t = fminf(t, 3.4028235e38f);
    w.set(top, t);
    Cut cut{-INFINITY, 0, 0};
    const bool by_k = top_k > 0 && (unsigned int)top_k < a.vocab, by_p = top_p < 1.f;
    if (by_k || by_p) {
      double all = 0.0, none = 0.0;
      each([&](unsigned int, float f) {
        const unsigned int b = w.bin(f);
        if (b < BINS - 1) atomicAdd(&sh.bins[0][b], 1u);
      });
      if (!by_k)
        each_vector([&](unsigned int, const float (&f)[N]) { all += weigh(f, [](float) { return true; }); });
      sum2(all, none);  // of all blocks: the bins are counted
      unsigned int n = 0;
      if (by_k) {
        if (find<true>(top_k, 0, cut, n) == GATHERED) {
          if (rank == 0) choose(r, n, top_k, true, 0.0, by_p, top_p, min_p, u);
          return;
        }
        if (by_p) {
          all = none = 0.0;
          each_vector([&](unsigned int, const float (&f)[N]) { all += weigh(f, [&](float g) { return g > cut.value; }); });
          sum2(all, none);
          if (cut.ties) all += cut.ties * w.of(cut.value);
        }
      }
      if (by_p) {
        Cut c;
        const Found found = find<false>((double)top_p * all, 1, c, n);
        if (found == GATHERED) {
          if (rank == 0) choose(r, n, 0, false, all, true, top_p, min_p, u);
          return;
        }
        if (found == CUT && (c.value > cut.value || (c.value == cut.value && c.ties < cut.ties))) cut = c;
      }
    }
    // tokens at the cut: how many of them in blocks and warps before this one
    unsigned int ties = 0;  // of this warp's
    const bool some = cut.ties < cut.equal;
    if (cut.ties) {
      ties = 0xFFFFFFFFu;
      if (some) {
        unsigned int mine = 0;
        each([&](unsigned int i, float f) { mine += f == cut.value; });
        mine = __reduce_add_sync(0xFFFFFFFFu, mine);
        __syncthreads();
        if (lane == 0) sh.warp_counts[warp] = mine;
        __syncthreads();
        unsigned int block = 0, before = 0;
        for (int i = 0; i < SAMPLE_WARPS; ++i) {
          if (i < warp) before += sh.warp_counts[i];
          block += sh.warp_counts[i];
        }
        give(block, 0.0);
        for (int i = 0; i < rank; ++i) before += (unsigned int)taken(i, 0);
        ties = before >= cut.ties ? 0 : cut.ties - before;
        if (ties >= mine) ties = 0xFFFFFFFFu;  // all of them
      }
    }
    const bool in_part = ties && ties != 0xFFFFFFFFu;
    const double least = min_p > 0.f ? min_p : 0.0;
    // weights of a lane's N tokens of the tile at i, 0 for what is not kept. seen: tokens at the cut in the warp's tiles before.
    auto kept = [&](unsigned int i, unsigned int& seen, float (&f)[N], double (&x)[N]) {
      unsigned int order = 0;
      if (i < w1) {
        fetch(i, f);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = -INFINITY;
      }
      if (in_part) {
        unsigned int mine = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) mine += f[j] == cut.value;
        order = mine;
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned int below = __shfl_up_sync(0xFFFFFFFFu, order, o);
          if (lane >= o) order += below;
        }
        const unsigned int tile = __shfl_sync(0xFFFFFFFFu, order, 31);
        order += seen - mine;
        seen += tile;
      }
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = w.of(f[j]);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const bool equal = f[j] == cut.value && ties, keep = (f[j] > cut.value || (equal && order < ties)) && x[j] >= least;
        order += equal;
        x[j] = keep ? x[j] : 0.0;
      }
    };
    double sum = 0.0;
    unsigned int seen = 0;
    for (unsigned int i = w0 + lane * N; i - lane * N < w1; i += TILE) {
      float f[N];
      double x[N];
      kept(i, seen, f, x);
#pragma unroll
      for (int j = 0; j < N; ++j) sum += x[j];
    }
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    __syncthreads();
    if (lane == 0) sh.warp_sums[1][warp] = sum;
    __syncthreads();
    double block = 0.0;
    for (int i = 0; i < SAMPLE_WARPS; ++i) block += sh.warp_sums[1][i];
    give(block, 0.0);
    double total = 0.0;
    for (int i = 0; i < ranks; ++i) total += taken(i, 0);
    // which block, and which warp of it; the last one with any weight where rounding, or u, leaves none
    const double target = target_of(u, total);
    int where = -1;
    double upto = 0.0, start = 0.0;
    bool crossed = false;
    for (int i = 0; i < ranks && !crossed; ++i) {
      const double s = taken(i, 0);
      if (s > 0.0) {
        where = i;
        start = upto;
        upto += s;
        crossed = upto > target;
      }
    }
    if (where != rank) return;
    int in_warp = -1;
    upto = start;
    bool here = false;
    for (int i = 0; i < SAMPLE_WARPS && !here; ++i) {
      const double s = sh.warp_sums[1][i];
      if (s > 0.0) {
        in_warp = i;
        start = upto;
        upto += s;
        here = upto > target;
      }
    }
    if (in_warp != warp) return;
    unsigned int token = 0xFFFFFFFFu;
    float logit = 0.f;
    seen = 0;
    for (unsigned int i = w0 + lane * N; i - lane * N < w1; i += TILE) {
      float f[N];
      double x[N];
      kept(i, seen, f, x);
      double mine = 0.0;
#pragma unroll
      for (int j = 0; j < N; ++j) mine += x[j];
      double run = mine;
      for (int o = 1; o < 32; o <<= 1) {
        const double below = __shfl_up_sync(0xFFFFFFFFu, run, o);
        if (lane >= o) run += below;
      }
      const unsigned int past = __ballot_sync(0xFFFFFFFFu, mine > 0.0 && start + run > target);
      const unsigned int any = __ballot_sync(0xFFFFFFFFu, mine > 0.0);
      if (any) {
        // in this tile, or so far the last token with any weight
        const int who = past ? __ffs(past) - 1 : 31 - __clz(any);
        unsigned int at = 0;
        float l = 0.f;
        double s = start + (run - mine);
        bool done = false;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          if (x[j] > 0.0 && !done) {
            at = i + j;
            l = f[j];
            s += x[j];
            done = past && s > target;
          }
        }
        token = __shfl_sync(0xFFFFFFFFu, at, who);
        logit = __shfl_sync(0xFFFFFFFFu, l, who);
      }
      if (past) break;
      start += __shfl_sync(0xFFFFFFFFu, run, 31);
    }
    if (lane == 0) write(r, token, (float)(w.exponent(logit) - log(total)));
  }
};

template <typename T, bool HELD>
__global__ void __launch_bounds__(SAMPLE_THREADS, 2) sample_kernel(const SampleArgs a) {
  __shared__ SampleShared sh;
  extern __shared__ uint4 held[];
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const unsigned int r = blockIdx.x / ranks;
  const unsigned int part0 = rank * a.part, per_warp = a.part / SAMPLE_WARPS;
  Sampler<T, HELD> s{a, sh, cluster, reinterpret_cast<const T*>(a.logits + r * a.ld), held, part0};
  s.warp = threadIdx.x >> 5;
  s.lane = threadIdx.x & 31;
  s.w0 = part0 + s.warp * per_warp;
  s.w1 = s.w0 + per_warp;
  if (s.w1 > a.vocab) s.w1 = s.w0 >= a.vocab ? s.w0 : s.w0 + (a.vocab - s.w0 + s.TILE - 1) / s.TILE * s.TILE;
  s.ranks = ranks;
  s.rank = rank;
  s.turn = 0;
  s.run(r);
  if (ranks > 1) cluster.sync();  // the others may still read this block's shared memory
}

constexpr size_t HELD_MOST = 200 * 1024;  // of a block's part in shared memory
constexpr size_t SAMPLE_ROWS_MOST = 1 << 24, SAMPLE_VOCAB_MOST = 1 << 24;

template <typename T, bool HELD>
cudaError_t sample_launch(SampleArgs a, size_t rows, int ranks, cudaStream_t s) {
  const size_t smem = HELD ? (size_t)a.part * sizeof(T) : 0;
  cudaError_t e = cudaSuccess;
  if (HELD) e = cudaFuncSetAttribute(sample_kernel<T, HELD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)HELD_MOST);
  Chain chain(s);
  chain.err = e;
  chain.launch(sample_kernel<T, HELD>, dim3((unsigned int)(rows * ranks)), SAMPLE_THREADS, smem, ranks > 1 ? ranks : 0, a);
  return chain.err;
}

template <typename T>
cudaError_t sample_rows(SampleArgs a, size_t rows, int sms, cudaStream_t s) {
  constexpr unsigned int WHOLE = SAMPLE_WARPS * 32 * (16 / (int)sizeof(T));  // tokens of one tile for each warp
  auto part = [&](int ranks) {
    const size_t share = (a.vocab + (size_t)ranks - 1) / ranks;
    return (unsigned int)((share + WHOLE - 1) / WHOLE * WHOLE);
  };
  // more blocks per row while that takes less shared memory or more SMs, and each warp keeps a tile
  int ranks = 1;
  while (ranks < MOST_CLUSTER && part(ranks) > WHOLE && ((size_t)part(ranks) * sizeof(T) > 64 * 1024 || rows * ranks < (size_t)sms * 2)) ranks *= 2;
  a.part = part(ranks);
  if ((size_t)a.part * sizeof(T) <= HELD_MOST) return sample_launch<T, true>(a, rows, ranks, s);
  return sample_launch<T, false>(a, rows, ranks, s);
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

int b2_sample(size_t rows, size_t vocab, int dtype, const void* logits, size_t ld, const float* u, const b2_sample_options* o, void* tokens,
              int token_bytes, float* logprob, void* stream) {
  const char* who = "b2_sample";
  if (!dtype_ok(dtype)) return call_error(B2_ERR_INVALID, "%s: dtype %d", who, dtype);
  if (rows > SAMPLE_ROWS_MOST || vocab == 0 || vocab > SAMPLE_VOCAB_MOST)
    return call_error(B2_ERR_INVALID, "%s: %zu rows of %zu (2^24 at most, 1 to 2^24)", who, rows, vocab);
  if (token_bytes != 4 && token_bytes != 8) return call_error(B2_ERR_INVALID, "%s: tokens of %d bytes", who, token_bytes);
  if (!o || (rows && (!logits || !u || !tokens))) return call_error(B2_ERR_INVALID, "%s: null pointer", who);
  const size_t e = dtype_bytes(dtype);
  if (ld < vocab) return call_error(B2_ERR_INVALID, "%s: leading dimension smaller than the width", who);
  if (reinterpret_cast<size_t>(logits) % e || reinterpret_cast<size_t>(tokens) % token_bytes ||
      (reinterpret_cast<size_t>(u) | reinterpret_cast<size_t>(logprob) | reinterpret_cast<size_t>(o->row_temperature) | reinterpret_cast<size_t>(o->row_top_k) |
       reinterpret_cast<size_t>(o->row_top_p) | reinterpret_cast<size_t>(o->row_min_p)) % 4)
    return call_error(B2_ERR_INVALID, "%s: a pointer is not aligned to its elements", who);
  if (o->temperature != o->temperature || o->top_p != o->top_p || o->min_p != o->min_p) return call_error(B2_ERR_INVALID, "%s: an option is not a number", who);
  int sms, rc;
  if ((rc = lm_device(&sms)) != B2_OK) return rc;
  auto vector = [&](const char* name, const void* p, size_t bytes, bool written) { return extent(name, p, 1, rows * bytes, rows * bytes, written); };
  Extent args[] = {extent("logits", logits, rows, vocab * e, ld * e, false), vector("u", u, 4, false), vector("row_temperature", o->row_temperature, 4, false),
                   vector("row_top_k", o->row_top_k, 4, false), vector("row_top_p", o->row_top_p, 4, false), vector("row_min_p", o->row_min_p, 4, false),
                   vector("tokens", tokens, token_bytes, true), vector("logprob", logprob, 4, true)};
  if ((rc = refuse_overlap(who, args, 8)) != B2_OK) return rc;
  if (!rows) return B2_OK;
  SampleArgs a{};
  a.logits = static_cast<const char*>(logits);
  a.ld = ld * e;
  a.vocab = (unsigned int)vocab;
  a.vec = reinterpret_cast<size_t>(logits) % 16 == 0 && (ld * e % 16 == 0 || rows == 1);
  a.u = u;
  a.temperature = o->temperature;
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
  const cudaError_t err = dtype == B2_DTYPE_BF16 ? sample_rows<__nv_bfloat16>(a, rows, sms, static_cast<cudaStream_t>(stream))
                                                 : sample_rows<float>(a, rows, sms, static_cast<cudaStream_t>(stream));
  return launch_error(err, who);
}

}  // extern "C"
