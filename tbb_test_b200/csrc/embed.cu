// Rows of a table by token number, scaled, and the table's gradient:
//
//   out[i]   = scale * table[t_i]                     (zeros where t_i is outside [0, vocab))
//   dtable[v] = scale * sum over i with t_i = v of dout[i]
//
// Both are bound by HBM: the forward pass reads and writes n rows, the gradient reads n rows and writes vocab rows.
//
// The gradient sorts (token, position) pairs and adds each token's rows in the order of their positions, in fp32, so
// that its bits do not depend on the order in which blocks run; no float is added by an atomic. The sorted list is cut
// into chunks of equal length, one group of threads per chunk and slice of columns, so that a token that makes up
// a tenth of a batch takes no longer than many rare ones. A run of one token inside a chunk is finished there. One that
// crosses chunk borders leaves a partial sum per chunk, and a second kernel adds these in order. The rows of tokens that do
// not occur are zeroed meanwhile.
#include "lm.cuh"

namespace b2 {
namespace {

constexpr int EMBED_THREADS = 256;

template <typename T, int VB, int U>
__global__ void __launch_bounds__(EMBED_THREADS) embed_kernel(const void* __restrict__ tokens, int wide, size_t n,
                                                              const char* __restrict__ table, unsigned int vocab,
                                                              int vecs, size_t ld_table, float scale,
                                                              char* __restrict__ out, size_t ld_out, int tpr_log2) {
  typedef Elems<T, VB> E;
  typedef typename E::raw raw;
  const int col0 = threadIdx.x & ((1 << tpr_log2) - 1), sub = threadIdx.x >> tpr_log2;
  const int group = EMBED_THREADS >> tpr_log2;
  const size_t row0 = (size_t)blockIdx.x * group * U + sub;
  unsigned int t[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const size_t r = row0 + (size_t)u * group;
    t[u] = r < n ? token_at(tokens, wide, r, vocab) : vocab;
  }
  for (int c = col0; c < vecs; c += 1 << tpr_log2) {
    raw v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // U loads in flight
      memset(&v[u], 0, sizeof(raw));
      if (t[u] < vocab) v[u] = __ldg(reinterpret_cast<const raw*>(table + t[u] * ld_table) + c);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const size_t r = row0 + (size_t)u * group;
      if (r >= n) continue;
      float f[E::N];
      E::get(v[u], f);
#pragma unroll
      for (int i = 0; i < E::N; ++i) f[i] = t[u] < vocab ? f[i] * scale : 0.f;
      reinterpret_cast<raw*>(out + r * ld_out)[c] = E::put(f);
    }
  }
}

// ------------------------------------------------------------------ sorting (token, position)

// Short lists: an element's place is the number of elements that sort before it. Every block holds all keys in shared
// memory and each warp counts for four elements at once.
constexpr int RANK_MOST = 8192;
constexpr int RANK_THREADS = 256, RANK_PER_WARP = 4;
__global__ void __launch_bounds__(RANK_THREADS) rank_sort_kernel(const void* __restrict__ tokens, int wide, int n,
                                                                 unsigned int vocab, unsigned int* __restrict__ keys,
                                                                 unsigned int* __restrict__ pos, unsigned int* joins) {
  extern __shared__ unsigned int key_s[];
  let_next_start();
  if (blockIdx.x == 0 && threadIdx.x == 0) *joins = 0;
  for (int i = threadIdx.x; i < n; i += RANK_THREADS) key_s[i] = token_at(tokens, wide, i, vocab);
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const int i0 = (blockIdx.x * (RANK_THREADS / 32) + (threadIdx.x >> 5)) * RANK_PER_WARP;
  unsigned int key[RANK_PER_WARP], before[RANK_PER_WARP];
#pragma unroll
  for (int u = 0; u < RANK_PER_WARP; ++u) {
    key[u] = i0 + u < n ? key_s[i0 + u] : 0u;
    before[u] = 0;
  }
  for (int j = lane; j < n; j += 32) {
    const unsigned int k = key_s[j];
#pragma unroll
    for (int u = 0; u < RANK_PER_WARP; ++u) before[u] += k < key[u] + (j < i0 + u ? 1u : 0u);  // equal keys: by position
  }
#pragma unroll
  for (int u = 0; u < RANK_PER_WARP; ++u) {
    const unsigned int r = __reduce_add_sync(0xFFFFFFFFu, before[u]);
    if (lane == 0 && i0 + u < n) {
      keys[r] = key[u];
      pos[r] = i0 + u;
    }
  }
}

// Longer ones: a stable radix sort, lowest digit first, of at most RADIX_TILES tiles of consecutive elements, so that a
// block finds its digits' first places by reading all tiles' counts itself instead of after a third launch per digit.
// A block places RADIX_THREADS * ROUNDS elements at a time: 2 rounds where that gives 64 tiles of few steps, 8 for long lists,
// whose steps then cost less each.
constexpr int RADIX_THREADS = 512, RADIX_WARPS = RADIX_THREADS / 32;
constexpr int RADIX_TILES = 64, RADIX_MOST_BITS = 10;
constexpr int radix_rounds(size_t n) { return n <= (1u << 18) ? 2 : 8; }

// First index whose key is >= `key`.
__device__ __forceinline__ unsigned int lower_bound(const unsigned int* keys, unsigned int n, unsigned int key) {
  unsigned int lo = 0, hi = n;
  while (lo < hi) {
    const unsigned int mid = (lo + hi) >> 1;
    if (__ldg(keys + mid) < key) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// Rows of the gradient whose token does not occur: zeros. A warp takes FILL_ROWS of them.
constexpr int FILL_ROWS = 8;
struct Fill {
  const unsigned char* present;  // by token, or null: looked up in the sorted keys
  const unsigned int* keys;
  unsigned int n, vocab;
  char* dtable;
  size_t ld;  // bytes
  int vb, vecs;
};
__device__ __forceinline__ void fill_rows(const Fill& p, unsigned int warp, int lane) {
  const unsigned int v0 = warp * FILL_ROWS, v = v0 + lane;
  bool absent = false;
  if (lane < FILL_ROWS && v < p.vocab) {
    if (p.present) {
      absent = !p.present[v];
    } else {
      const unsigned int at = lower_bound(p.keys, p.n, v);
      absent = at == p.n || __ldg(p.keys + at) != v;
    }
  }
  for (unsigned int rows = __ballot_sync(0xFFFFFFFFu, absent); rows; rows &= rows - 1) {
    char* row = p.dtable + (size_t)(v0 + __ffs(rows) - 1) * p.ld;
    if (p.vb == 16) {
      for (int c = lane; c < p.vecs; c += 32) reinterpret_cast<uint4*>(row)[c] = make_uint4(0, 0, 0, 0);
    } else if (p.vb == 8) {
      for (int c = lane; c < p.vecs; c += 32) reinterpret_cast<uint2*>(row)[c] = make_uint2(0, 0);
    } else if (p.vb == 4) {
      for (int c = lane; c < p.vecs; c += 32) reinterpret_cast<unsigned int*>(row)[c] = 0;
    } else {
      for (int c = lane; c < p.vecs; c += 32) reinterpret_cast<unsigned short*>(row)[c] = 0;
    }
  }
}

struct RadixPass {
  const void* tokens;  // first pass: keys come from here and positions are their index
  int wide;
  unsigned int vocab;
  const unsigned int *keys, *pos;
  unsigned int *keys_out, *pos_out;
  unsigned int* counts;       // tiles x bins
  unsigned char* present;     // first pass: set for every token that occurs
  unsigned int* next_counts;  // the same of the next digit, counted where this one's elements go; zeroed by the first kernel
  unsigned int n, tile;  // elements, elements per tile (a multiple of a block's step)
  int tiles, shift, bits;
};
__device__ __forceinline__ unsigned int radix_key(const RadixPass& p, unsigned int i) {
  return p.tokens ? token_at(p.tokens, p.wide, i, p.vocab) : p.keys[i];
}

// Counts of the first digit, and zeros for what the kernels behind it count and mark.
__global__ void __launch_bounds__(RADIX_THREADS) radix_count_kernel(const RadixPass p, unsigned int* other_counts, int others,
                                                                    unsigned char* present, unsigned int* joins) {
  __shared__ unsigned int count[1 << RADIX_MOST_BITS];
  const int bins = 1 << p.bits;
  let_next_start();
  for (int b = threadIdx.x; b < bins; b += RADIX_THREADS) count[b] = 0;
  for (int b = blockIdx.x * RADIX_THREADS + threadIdx.x; b < others; b += gridDim.x * RADIX_THREADS) other_counts[b] = 0;
  for (size_t v = ((size_t)blockIdx.x * RADIX_THREADS + threadIdx.x) * 16; v < p.vocab; v += (size_t)gridDim.x * RADIX_THREADS * 16)
    *reinterpret_cast<uint4*>(present + v) = make_uint4(0, 0, 0, 0);  // the array is whole 16-byte pieces
  if (blockIdx.x == 0 && threadIdx.x == 0) *joins = 0;
  __syncthreads();
  const unsigned int begin = blockIdx.x * p.tile, end = min(p.n, begin + p.tile);
  for (unsigned int i = begin + threadIdx.x; i < end; i += RADIX_THREADS)
    atomicAdd(&count[(radix_key(p, i) >> p.shift) & (bins - 1)], 1u);
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += RADIX_THREADS) p.counts[(size_t)blockIdx.x * bins + b] = count[b];
}

// Blocks behind the tiles' zero rows meanwhile (last pass; the sort keeps 64 SMs busy at most).
template <int RADIX_ROUNDS>
__global__ void __launch_bounds__(RADIX_THREADS) radix_place_kernel(const RadixPass p, const Fill fill) {
  constexpr int RADIX_STEP = RADIX_THREADS * RADIX_ROUNDS;
  __shared__ unsigned int next[1 << RADIX_MOST_BITS];  // where this tile's next element of a digit goes
  __shared__ unsigned short seen[RADIX_WARPS][1 << RADIX_MOST_BITS];
  __shared__ unsigned int warp_sum[RADIX_WARPS];
  const int bins = 1 << p.bits, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  after_previous();
  let_next_start();
  if (blockIdx.x >= p.tiles) {
    fill_rows(fill, (blockIdx.x - p.tiles) * RADIX_WARPS + warp, lane);
    return;
  }
  // exclusive sum over digits of all tiles' counts, plus the counts of the tiles before this one
  unsigned int running = 0;
  for (int b0 = 0; b0 < bins; b0 += RADIX_THREADS) {
    const int b = b0 + threadIdx.x;
    unsigned int total = 0, before = 0;
    if (b < bins)
#pragma unroll 32
      for (int t = 0; t < p.tiles; ++t) {
        const unsigned int c = p.counts[(size_t)t * bins + b];
        total += c;
        before += t < (int)blockIdx.x ? c : 0u;
      }
    unsigned int scan = total;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const unsigned int up = __shfl_up_sync(0xFFFFFFFFu, scan, d);
      if (lane >= d) scan += up;
    }
    if (lane == 31) warp_sum[warp] = scan;
    __syncthreads();
    unsigned int base = running, all = 0;
    for (int w = 0; w < RADIX_WARPS; ++w) {
      base += w < warp ? warp_sum[w] : 0u;
      all += warp_sum[w];
    }
    if (b < bins) next[b] = base + scan - total + before;
    running += all;
    __syncthreads();
  }
  const unsigned int begin = blockIdx.x * p.tile, end = min(p.n, begin + p.tile);
  for (unsigned int step = begin; step < end; step += RADIX_STEP) {
    for (int i = threadIdx.x; i < RADIX_WARPS * bins; i += RADIX_THREADS) seen[i >> p.bits][i & (bins - 1)] = 0;
    __syncthreads();
    // a warp places its share of consecutive elements 32 at a time: equal digits of a round keep the order of the lanes
    unsigned int key[RADIX_ROUNDS], pos[RADIX_ROUNDS], place[RADIX_ROUNDS];
    const unsigned int first = step + warp * 32 * RADIX_ROUNDS + lane;
#pragma unroll
    for (int r = 0; r < RADIX_ROUNDS; ++r) {
      const unsigned int i = first + r * 32;
      key[r] = i < end ? radix_key(p, i) : 0u;
      pos[r] = i < end ? (p.tokens ? i : p.pos[i]) : 0u;
    }
#pragma unroll
    for (int r = 0; r < RADIX_ROUNDS; ++r) {
      const bool in = first + r * 32 < end;
      const unsigned int digit = (key[r] >> p.shift) & (bins - 1);
      const unsigned int same = __match_any_sync(0xFFFFFFFFu, in ? digit : 0xFFFFFFFFu);
      const unsigned int old = in ? seen[warp][digit] : 0u;
      place[r] = old + __popc(same & ((1u << lane) - 1));
      __syncwarp();
      if (in && lane == __ffs(same) - 1) seen[warp][digit] = (unsigned short)(old + __popc(same));
      __syncwarp();
    }
    __syncthreads();
    unsigned int moved[(1 << RADIX_MOST_BITS) / RADIX_THREADS];
#pragma unroll
    for (int k = 0; k < (1 << RADIX_MOST_BITS) / RADIX_THREADS; ++k) {
      const int b = k * RADIX_THREADS + threadIdx.x;
      moved[k] = 0;
      if (b < bins)
        for (int w = 0; w < RADIX_WARPS; ++w) {
          const unsigned int c = seen[w][b];
          seen[w][b] = (unsigned short)moved[k];
          moved[k] += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RADIX_ROUNDS; ++r)
      if (first + r * 32 < end) {
        const unsigned int digit = (key[r] >> p.shift) & (bins - 1);
        const unsigned int to = next[digit] + seen[warp][digit] + place[r];
        p.keys_out[to] = key[r];
        p.pos_out[to] = pos[r];
        if (p.present && key[r] < p.vocab) p.present[key[r]] = 1;
        if (p.next_counts)  // whole numbers: the order of the additions does not matter
          atomicAdd(p.next_counts + ((size_t)(to / p.tile) << p.bits) + ((key[r] >> (p.shift + p.bits)) & (bins - 1)), 1u);
      }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < (1 << RADIX_MOST_BITS) / RADIX_THREADS; ++k) {
      const int b = k * RADIX_THREADS + threadIdx.x;
      if (b < bins) next[b] += moved[k];
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ sums of runs

struct RunSum {
  const unsigned int *keys, *pos;  // sorted; positions without a token carry key = vocab and stand last
  unsigned int n, vocab, chunk;    // chunk: sorted elements per chunk
  unsigned int chunks;
  const char* dout;
  size_t ld_dout;  // bytes
  char* dtable;
  size_t ld_dtable;
  float *head, *tail;  // chunks x pitch partial sums: of the run that came from the chunk before, and of the one that goes on
  size_t pitch;        // floats per partial row
  unsigned int* joins;  // how many runs go on behind the chunk they begin in
  uint2* join_runs;     // their chunks and tokens, in any order
  float scale;
  int vecs, slices, tpr_log2;
  unsigned int fill_blocks;  // of the second kernel
};

constexpr int RUN_THREADS = 128, RUN_AHEAD = 8;
template <typename T, int VB>
__global__ void __launch_bounds__(RUN_THREADS) run_sum_kernel(const RunSum p) {
  typedef Elems<T, VB> E;
  typedef typename E::raw raw;
  const int lane = threadIdx.x & 31;
  after_previous();
  let_next_start();
  // A unit is a chunk and a slice of columns, worked on by 2^tpr_log2 >= 8 threads. Keys and positions of the next `span` elements
  // come with one load by the unit's threads and are handed round by shuffles.
  const int tpr = 1 << p.tpr_log2, span = min(tpr, 32), in_span = lane & (span - 1);
  const unsigned int unit = blockIdx.x * (RUN_THREADS >> p.tpr_log2) + (threadIdx.x >> p.tpr_log2);
  const unsigned int chunk = unit / p.slices;
  const int col = (int)(unit - chunk * p.slices) * tpr + (threadIdx.x & (tpr - 1));
  const unsigned int begin = chunk * p.chunk, end = chunk < p.chunks ? min(p.n, begin + p.chunk) : begin;
  const bool works = col < p.vecs;
  unsigned int cur = begin < end ? __ldg(p.keys + begin) : p.vocab;
  bool from_before = begin > 0 && begin < end && __ldg(p.keys + begin - 1) == cur;
  float acc[E::N];
#pragma unroll
  for (int j = 0; j < E::N; ++j) acc[j] = 0.f;
  auto finish = [&](bool goes_on) {
    if (!works) return;
    if (from_before || goes_on) {
      float* to = (from_before ? p.head : p.tail) + (size_t)chunk * p.pitch + (size_t)col * E::N;
#pragma unroll
      for (int j = 0; j < E::N; ++j) to[j] = acc[j];
      if (goes_on && !from_before && col == 0) p.join_runs[atomicAdd(p.joins, 1u)] = make_uint2(chunk, cur);
    } else {
#pragma unroll
      for (int j = 0; j < E::N; ++j) acc[j] *= p.scale;
      reinterpret_cast<raw*>(p.dtable + (size_t)cur * p.ld_dtable)[col] = E::put(acc);
    }
  };
  unsigned int next_key = p.vocab, next_pos = 0;
  auto fetch = [&](unsigned int i) {
    next_key = i < end ? __ldg(p.keys + i) : p.vocab;
    next_pos = i < end ? __ldg(p.pos + i) : 0u;
  };
  fetch(begin + in_span);
  for (unsigned int i = 0; i < p.chunk; i += span) {
    const unsigned int span_key = next_key, span_pos = next_pos;
    fetch(begin + i + span + in_span);
    for (int k0 = 0; k0 < span; k0 += RUN_AHEAD) {
      unsigned int key[RUN_AHEAD];
      raw v[RUN_AHEAD];
#pragma unroll
      for (int u = 0; u < RUN_AHEAD; ++u) {
        key[u] = __shfl_sync(0xFFFFFFFFu, span_key, k0 + u, span);
        const unsigned int pos = __shfl_sync(0xFFFFFFFFu, span_pos, k0 + u, span);
        memset(&v[u], 0, sizeof(raw));
        if (works && key[u] < p.vocab) v[u] = __ldg(reinterpret_cast<const raw*>(p.dout + (size_t)pos * p.ld_dout) + col);
      }
#pragma unroll
      for (int u = 0; u < RUN_AHEAD; ++u) {
        if (key[u] != cur && begin + i + k0 + u < end) {
          if (cur < p.vocab) finish(false);
          cur = key[u];
          from_before = false;
#pragma unroll
          for (int j = 0; j < E::N; ++j) acc[j] = 0.f;
        }
        float f[E::N];
        E::get(v[u], f);  // zeros behind the last element and in place of padding
#pragma unroll
        for (int j = 0; j < E::N; ++j) acc[j] += f[j];
      }
    }
  }
  if (cur < p.vocab) finish(end < p.n && __ldg(p.keys + end) == cur);
}

// The same for rows of 32 and more 16-byte pieces, which go through shared memory: a thread copies its own piece of the next 16 rows
// there without holding registers for them and refills a place when it has added it; seven blocks keep up to 220 KB in flight per SM.
// Where runs begin comes as a mask per 32 elements, so that a row takes about 25 instructions per warp and not 74, which is
// what bounded this kernel (65536 rows of 2 KB: 50 us and DRAM 43 % busy with eight rows ahead in registers, 39 us
// this way, while 92 MB of zero rows go from L2 to DRAM).
constexpr int SPAN = 32, RING = 16, RING_GROUP = 4, RING_GROUPS = RING / RING_GROUP;
template <typename T>
__global__ void __launch_bounds__(RUN_THREADS) run_sum_ring_kernel(const RunSum p) {
  typedef Elems<T, 16> E;
  extern __shared__ uint4 ring_s[];  // place k of this thread at k * RUN_THREADS
  uint4* ring = ring_s + threadIdx.x;
  const int lane = threadIdx.x & 31, tpr = 1 << p.tpr_log2;  // 32 and more: a warp is of one unit
  after_previous();
  let_next_start();
  const unsigned int unit = blockIdx.x * (RUN_THREADS >> p.tpr_log2) + (threadIdx.x >> p.tpr_log2);
  const unsigned int chunk = unit / p.slices;
  const int col = (int)(unit - chunk * p.slices) * tpr + (threadIdx.x & (tpr - 1));
  if (chunk >= p.chunks) return;
  const unsigned int begin = chunk * p.chunk, end = min(p.n, begin + p.chunk);
  const bool works = col < p.vecs;
  const char* from = p.dout + (size_t)col * 16;
  unsigned int cur = __ldg(p.keys + begin);
  bool from_before = begin > 0 && __ldg(p.keys + begin - 1) == cur;
  float acc[E::N];
#pragma unroll
  for (int j = 0; j < E::N; ++j) acc[j] = 0.f;
  auto finish = [&](bool goes_on) {
    if (!works) return;
    if (from_before || goes_on) {
      float4* to = reinterpret_cast<float4*>((from_before ? p.head : p.tail) + (size_t)chunk * p.pitch + (size_t)col * E::N);
#pragma unroll
      for (int j = 0; j < E::N / 4; ++j) to[j] = make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]);
      if (goes_on && !from_before && col == 0) p.join_runs[atomicAdd(p.joins, 1u)] = make_uint2(chunk, cur);
    } else {
#pragma unroll
      for (int j = 0; j < E::N; ++j) acc[j] *= p.scale;
      reinterpret_cast<uint4*>(p.dtable + (size_t)cur * p.ld_dtable)[col] = E::put(acc);
    }
  };
  // Keys and positions of 32 elements, one per lane; behind the last element key = vocab. Three spans of them: the one that is added,
  // the one whose rows are copied meanwhile, and the one whose keys are on their way.
  unsigned int key[3], pos[3];
  auto fetch = [&](unsigned int i, unsigned int& k, unsigned int& at) {
    k = i < end ? __ldg(p.keys + i) : p.vocab;
    at = i < end ? __ldg(p.pos + i) : 0u;
  };
  auto count = [&](unsigned int k) { return __popc(__ballot_sync(0xFFFFFFFFu, k < p.vocab)); };  // they stand first
  auto copy_group = [&](int g, unsigned int at, int have) {  // group g of a span
#pragma unroll
    for (int u = 0; u < RING_GROUP; ++u) {
      const int e = g * RING_GROUP + u;
      const unsigned int row = __shfl_sync(0xFFFFFFFFu, at, e);
      if (works && e < have)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned int)__cvta_generic_to_shared(ring + e % RING * RUN_THREADS)),
                     "l"(from + (size_t)row * p.ld_dout)
                     : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  fetch(begin + lane, key[0], pos[0]);
  fetch(begin + SPAN + lane, key[1], pos[1]);
  int have = count(key[0]);
#pragma unroll
  for (int g = 0; g < RING_GROUPS; ++g) copy_group(g, pos[0], have);
  unsigned int before = cur;  // the key in front of the span
  for (unsigned int i = begin; i < end && have > 0; i += SPAN) {
    fetch(i + 2 * SPAN + lane, key[2], pos[2]);
    // bit e: a run begins at element e of the span
    const unsigned int up = __shfl_up_sync(0xFFFFFFFFu, key[0], 1);
    const unsigned int starts = __ballot_sync(0xFFFFFFFFu, key[0] != (lane ? up : before));
    before = __shfl_sync(0xFFFFFFFFu, key[0], 31);
    const int next_have = count(key[1]);
#pragma unroll 1
    for (int g = 0; g < SPAN / RING_GROUP; ++g) {
      asm volatile("cp.async.wait_group %0;" ::"n"(RING_GROUPS - 1) : "memory");
#pragma unroll
      for (int u = 0; u < RING_GROUP; ++u) {
        const int e = g * RING_GROUP + u;
        if (e >= have) break;
        if (starts >> e & 1) {
          finish(false);
          cur = __shfl_sync(0xFFFFFFFFu, key[0], e);
          from_before = false;
#pragma unroll
          for (int j = 0; j < E::N; ++j) acc[j] = 0.f;
        }
        float f[E::N];
        E::get(ring[e % RING * RUN_THREADS], f);
#pragma unroll
        for (int j = 0; j < E::N; ++j) acc[j] += f[j];
      }
      const bool same = g + RING_GROUPS < SPAN / RING_GROUP;  // the group that takes the places just read
      copy_group((g + RING_GROUPS) % (SPAN / RING_GROUP), same ? pos[0] : pos[1], same ? have : next_have);
    }
    have = next_have;
    key[0] = key[1];
    pos[0] = pos[1];
    key[1] = key[2];
    pos[1] = pos[2];
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (cur < p.vocab) finish(end < p.n && __ldg(p.keys + end) == cur);
}

// Runs that cross chunk borders: the tail of the chunk a run begins in and the heads of the chunks behind it, JOIN_PARTS
// contiguous shares of them side by side, which are then added in order. A block takes 128 columns of a run at a time. Short
// lists, whose sort has no room for it, leave zeroing rows to the blocks before these; it needs no sums, so these blocks
// wait for the kernel before only when they are done: it has waited for the sorted list before this one starts.
constexpr int JOIN_PARTS = 4, JOIN_THREADS = 32 * JOIN_PARTS;
template <typename T>
__global__ void __launch_bounds__(JOIN_THREADS) run_join_kernel(const RunSum p, const Fill fill, int width) {
  __shared__ float4 part[JOIN_PARTS][32];
  const int lane = threadIdx.x & 31, share = threadIdx.x >> 5;
  let_next_start();
  if (blockIdx.x < p.fill_blocks) {
    fill_rows(fill, blockIdx.x * JOIN_PARTS + share, lane);
    after_previous();  // up to eight tokens have no runs to join: then these blocks' end is the call's, and has to be behind the sums
    return;
  }
  after_previous();
  const unsigned int slices = (width + 127) / 128;
  const size_t items = (size_t)*p.joins * slices;
  for (size_t item = blockIdx.x - p.fill_blocks; item < items; item += gridDim.x - p.fill_blocks) {
    const uint2 run = p.join_runs[item / slices];
    const unsigned int chunk = run.x, key = run.y;
    // the run's last chunk: chunks whose first element has the key
    unsigned int last = chunk;
    for (;;) {
      const size_t at = (size_t)(last + 1 + lane) * p.chunk;
      const unsigned int same = __ballot_sync(0xFFFFFFFFu, at < p.n && __ldg(p.keys + at) == key);
      last += same == 0xFFFFFFFFu ? 32 : __ffs(~same) - 1;
      if (same != 0xFFFFFFFFu) break;
    }
    const unsigned int count = last - chunk + 1;
    const unsigned int from = (unsigned int)((size_t)count * share / JOIN_PARTS), to = (unsigned int)((size_t)count * (share + 1) / JOIN_PARTS);
    const int c = (int)(item % slices) * 128 + lane * 4;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < width)
#pragma unroll 8
      for (unsigned int k = from; k < to; ++k) {
        const float4 x = *reinterpret_cast<const float4*>((k == 0 ? p.tail : p.head) + (size_t)(chunk + k) * p.pitch + c);
        sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
      }
    part[share][lane] = sum;
    __syncthreads();
    if (share == 0 && c < width) {
      for (int s = 1; s < JOIN_PARTS; ++s) {
        const float4 x = part[s][lane];
        sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
      }
      const float f[4] = {sum.x, sum.y, sum.z, sum.w};
      T* row = reinterpret_cast<T*>(p.dtable + (size_t)key * p.ld_dtable) + c;
      for (int i = 0; i < 4; ++i)
        if (c + i < width) row[i] = (T)(f[i] * p.scale);
    }
    __syncthreads();
  }
}

int log2_ceil(size_t v) {
  int b = 0;
  while (((size_t)1 << b) < v) ++b;
  return b;
}

struct GradPlan {
  int passes, bits, tiles;
  unsigned int tile, chunk, chunks;
  size_t pitch;
};
GradPlan grad_plan(size_t n, size_t vocab, size_t width) {
  GradPlan g{};
  if (n > RANK_MOST) {
    const int bits = log2_ceil(vocab + 1);
    g.passes = (bits + RADIX_MOST_BITS - 1) / RADIX_MOST_BITS;
    g.bits = (bits + g.passes - 1) / g.passes;
    const size_t step = (size_t)RADIX_THREADS * radix_rounds(n), steps = (n + step - 1) / step;
    g.tile = (unsigned int)((steps + RADIX_TILES - 1) / RADIX_TILES * step);
    g.tiles = (int)((n + g.tile - 1) / g.tile);
  }
  // about eight groups per SM where there are enough elements, and no less than eight elements in a row
  g.chunk = 8;
  while (g.chunk < 512 && n / g.chunk > 148 * 8) g.chunk *= 2;
  g.chunks = (unsigned int)((n + g.chunk - 1) / g.chunk);
  g.pitch = (width + 3) / 4 * 4;
  return g;
}
struct GradSpace {
  unsigned int *keys[2], *pos[2], *counts, *joins;
  unsigned char* present;
  uint2* join_runs;
  float *head, *tail;
};
size_t grad_space(const GradPlan& g, size_t n, size_t vocab, void* base, GradSpace* s) {
  Carver c(base);
  const int buffers = g.passes ? 2 : 1;
  for (int i = 0; i < buffers; ++i) {
    s->keys[i] = c.take<unsigned int>(n);
    s->pos[i] = c.take<unsigned int>(n);
  }
  s->counts = c.take<unsigned int>(((size_t)g.passes * g.tiles) << g.bits);
  s->present = c.take<unsigned char>(g.passes ? vocab : 0);
  s->joins = c.take<unsigned int>(1);
  s->join_runs = c.take<uint2>(g.chunks);
  s->head = c.take<float>(g.chunks * g.pitch);
  s->tail = c.take<float>(g.chunks * g.pitch);
  return c.used;
}

int check_table(const char* who, size_t n, int token_bytes, int dtype, size_t vocab, size_t width, size_t ld_rows,
                size_t ld_table) {
  if (token_bytes != 4 && token_bytes != 8) return call_error(B2_ERR_INVALID, "%s: token_bytes is 4 or 8, not %d", who, token_bytes);
  if (!dtype_ok(dtype)) return call_error(B2_ERR_INVALID, "%s: dtype %d", who, dtype);
  if (width < 1 || width > 0x7FFFFFFFu / 4) return call_error(B2_ERR_INVALID, "%s: width %zu", who, width);
  if (vocab < 1 || vocab >= 0x7FFFFFFFu) return call_error(B2_ERR_INVALID, "%s: vocab %zu", who, vocab);
  if (n >= 0x7FFFFFFFu) return call_error(B2_ERR_INVALID, "%s: %zu tokens", who, n);
  if (ld_rows < width || ld_table < width) return call_error(B2_ERR_INVALID, "%s: leading dimension smaller than the width", who);
  return B2_OK;
}

template <typename T, int VB>
cudaError_t embed_launch(const void* tokens, int wide, size_t n, const void* table, size_t vocab, size_t width,
                         size_t ld_table, float scale, void* out, size_t ld_out, int sms, cudaStream_t s) {
  const int vecs = (int)(width * sizeof(T) / VB);
  int tpr = log2_ceil(vecs);
  if (tpr > 8) tpr = 8;
  const size_t group = EMBED_THREADS >> tpr;
  // four rows per thread keep enough loads in flight; with few rows one, which spreads them over more SMs
  const bool many = n > group * 4 * (size_t)sms * 4;
  const size_t rows = group * (many ? 4 : 1);
  const size_t lt = ld_table * sizeof(T), lo = ld_out * sizeof(T);
  const unsigned int grid = (unsigned int)((n + rows - 1) / rows);
  if (many)
    embed_kernel<T, VB, 4><<<grid, EMBED_THREADS, 0, s>>>(tokens, wide, n, (const char*)table, (unsigned int)vocab, vecs, lt, scale, (char*)out, lo, tpr);
  else
    embed_kernel<T, VB, 1><<<grid, EMBED_THREADS, 0, s>>>(tokens, wide, n, (const char*)table, (unsigned int)vocab, vecs, lt, scale, (char*)out, lo, tpr);
  return cudaGetLastError();
}

template <typename T, int VB>
void run_launch(RunSum p, const Fill& fill, bool filled, size_t width, Chain& chain) {
  p.vecs = (int)(width * sizeof(T) / VB);
  p.tpr_log2 = log2_ceil(p.vecs);
  if (p.tpr_log2 > 7) p.tpr_log2 = 7;
  if (p.tpr_log2 < 3) p.tpr_log2 = 3;
  p.slices = (p.vecs + (1 << p.tpr_log2) - 1) >> p.tpr_log2;
  const size_t units = (size_t)p.chunks * p.slices, per_block = RUN_THREADS >> p.tpr_log2;
  const dim3 grid((unsigned int)((units + per_block - 1) / per_block));
  if (VB == 16 && p.tpr_log2 >= 5) {
    const size_t smem = (size_t)RING * RUN_THREADS * 16;
    if (chain.err == cudaSuccess)
      chain.err = cudaFuncSetAttribute(run_sum_ring_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    chain.launch(run_sum_ring_kernel<T>, grid, RUN_THREADS, smem, 0, p);
  } else {
    chain.launch(run_sum_kernel<T, VB>, grid, RUN_THREADS, 0, 0, p);
  }
  const size_t most = (size_t)(p.chunks - 1) * ((width + 127) / 128);
  const unsigned int per_fill = JOIN_PARTS * FILL_ROWS;
  p.fill_blocks = filled ? 0 : (p.vocab + per_fill - 1) / per_fill;
  const unsigned int join_blocks = (unsigned int)(most < 148 * 16 ? most : 148 * 16);
  if (p.fill_blocks + join_blocks) chain.launch(run_join_kernel<T>, dim3(p.fill_blocks + join_blocks), JOIN_THREADS, 0, 0, p, fill, (int)width);
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

int b2_embed(const void* tokens, int token_bytes, size_t n, const void* table, int dtype, size_t vocab, size_t width,
             size_t ld_table, float scale, void* out, size_t ld_out, void* stream) {
  int rc = check_table("b2_embed", n, token_bytes, dtype, vocab, width, ld_out, ld_table);
  if (rc != B2_OK) return rc;
  if (n == 0) return B2_OK;
  if (!tokens || !table || !out) return call_error(B2_ERR_INVALID, "b2_embed: null pointer");
  int sms;
  if ((rc = lm_device(&sms)) != B2_OK) return rc;
  const size_t e = dtype_bytes(dtype);
  if ((reinterpret_cast<size_t>(table) | reinterpret_cast<size_t>(out)) % e || reinterpret_cast<size_t>(tokens) % token_bytes)
    return call_error(B2_ERR_INVALID, "b2_embed: a pointer is not aligned to its elements");
  Extent args[] = {extent("tokens", tokens, 1, n * token_bytes, n * token_bytes, false), extent("table", table, vocab, width * e, ld_table * e, false),
                   extent("out", out, n, width * e, ld_out * e, true)};
  if ((rc = refuse_overlap("b2_embed", args, 3)) != B2_OK) return rc;
  const int vb = vector_bytes(e, reinterpret_cast<size_t>(table) | reinterpret_cast<size_t>(out) | width * e | ld_table * e | ld_out * e);
  const int wide = token_bytes == 8;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t err;
#define B2_EMBED(T, VB) err = embed_launch<T, VB>(tokens, wide, n, table, vocab, width, ld_table, scale, out, ld_out, sms, s)
  if (dtype == B2_DTYPE_BF16) {
    if (vb == 16) B2_EMBED(__nv_bfloat16, 16);
    else if (vb == 8) B2_EMBED(__nv_bfloat16, 8);
    else if (vb == 4) B2_EMBED(__nv_bfloat16, 4);
    else B2_EMBED(__nv_bfloat16, 2);
  } else {
    if (vb == 16) B2_EMBED(float, 16);
    else if (vb == 8) B2_EMBED(float, 8);
    else B2_EMBED(float, 4);
  }
#undef B2_EMBED
  return launch_error(err, "b2_embed");
}

int b2_embed_grad_workspace(size_t n, size_t vocab, size_t width, size_t* bytes) {
  int rc = check_table("b2_embed_grad_workspace", n, 4, B2_DTYPE_F32, vocab, width, width, width);
  if (rc != B2_OK) return rc;
  if (!bytes) return call_error(B2_ERR_INVALID, "b2_embed_grad_workspace: null pointer");
  GradSpace s;
  *bytes = grad_space(grad_plan(n, vocab, width), n, vocab, nullptr, &s);
  return B2_OK;
}

int b2_embed_grad(const void* tokens, int token_bytes, size_t n, const void* dout, int dtype, size_t ld_dout,
                  size_t vocab, size_t width, float scale, void* dtable, size_t ld_dtable, void* workspace,
                  size_t workspace_bytes, void* stream) {
  int rc = check_table("b2_embed_grad", n, token_bytes, dtype, vocab, width, ld_dout, ld_dtable);
  if (rc != B2_OK) return rc;
  if (!dtable || (n && (!tokens || !dout || !workspace))) return call_error(B2_ERR_INVALID, "b2_embed_grad: null pointer");
  const size_t e = dtype_bytes(dtype);
  if ((reinterpret_cast<size_t>(dout) | reinterpret_cast<size_t>(dtable)) % e || reinterpret_cast<size_t>(tokens) % token_bytes)
    return call_error(B2_ERR_INVALID, "b2_embed_grad: a pointer is not aligned to its elements");
  if (reinterpret_cast<size_t>(workspace) % 256) return call_error(B2_ERR_INVALID, "b2_embed_grad: the workspace is not on a 256-byte boundary");
  const GradPlan g = grad_plan(n, vocab, width);
  GradSpace w;
  const size_t need = grad_space(g, n, vocab, workspace, &w);
  if (n && workspace_bytes < need) return call_error(B2_ERR_INVALID, "b2_embed_grad: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  int sms;
  if ((rc = lm_device(&sms)) != B2_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Extent args[] = {extent("tokens", tokens, 1, n * token_bytes, n * token_bytes, false), extent("dout", dout, n, width * e, ld_dout * e, false),
                   extent("dtable", dtable, vocab, width * e, ld_dtable * e, true), extent("the workspace", workspace, 1, n ? need : 0, need, true)};
  if ((rc = refuse_overlap("b2_embed_grad", args, 4)) != B2_OK) return rc;
  if (n == 0)
    return launch_error(cudaMemset2DAsync(dtable, ld_dtable * e, 0, width * e, vocab, s), "b2_embed_grad");
  const int wide = token_bytes == 8;
  Chain chain(s);
  const int vb = vector_bytes(e, reinterpret_cast<size_t>(dout) | reinterpret_cast<size_t>(dtable) | width * e | ld_dout * e | ld_dtable * e);
  Fill fill{g.passes ? w.present : nullptr, nullptr, (unsigned int)n, (unsigned int)vocab, static_cast<char*>(dtable), ld_dtable * e, vb, (int)(width * e / vb)};
  int sorted = 0;
  if (g.passes == 0) {
    const int per_block = RANK_THREADS / 32 * RANK_PER_WARP;
    chain.launch(rank_sort_kernel, dim3((unsigned int)((n + per_block - 1) / per_block)), RANK_THREADS, n * 4, 0, tokens, wide, (int)n,
                 (unsigned int)vocab, w.keys[0], w.pos[0], w.joins);
  } else {
    RadixPass p{};
    p.wide = wide;
    p.vocab = (unsigned int)vocab;
    p.n = (unsigned int)n;
    p.tile = g.tile;
    p.tiles = g.tiles;
    p.bits = g.bits;
    for (int i = 0; i < g.passes; ++i) {
      p.tokens = i == 0 ? tokens : nullptr;
      p.keys = w.keys[sorted];
      p.pos = w.pos[sorted];
      if (i > 0) sorted ^= 1;
      p.keys_out = w.keys[sorted];
      p.pos_out = w.pos[sorted];
      p.shift = i * g.bits;
      const size_t bins = (size_t)g.tiles << g.bits;
      p.counts = w.counts + i * bins;
      p.present = i == 0 ? w.present : nullptr;
      p.next_counts = i + 1 < g.passes ? p.counts + bins : nullptr;
      if (i == 0)
        chain.launch(radix_count_kernel, dim3(g.tiles), RADIX_THREADS, 0, 0, p, p.counts + bins, (int)((g.passes - 1) * bins), w.present,
                     w.joins);
      // the first pass marks the tokens that occur, so that the last of several can zero the other rows
      const unsigned int per_fill = RADIX_WARPS * FILL_ROWS;
      const dim3 grid(g.tiles + (i > 0 && i + 1 == g.passes ? (unsigned int)((vocab + per_fill - 1) / per_fill) : 0));
      if (radix_rounds(n) == 2) chain.launch(radix_place_kernel<2>, grid, RADIX_THREADS, 0, 0, p, fill);
      else chain.launch(radix_place_kernel<8>, grid, RADIX_THREADS, 0, 0, p, fill);
    }
  }
  RunSum r{};
  r.keys = w.keys[sorted];
  r.pos = w.pos[sorted];
  r.n = (unsigned int)n;
  r.vocab = (unsigned int)vocab;
  r.chunk = g.chunk;
  r.chunks = g.chunks;
  r.dout = static_cast<const char*>(dout);
  r.ld_dout = ld_dout * e;
  r.dtable = static_cast<char*>(dtable);
  r.ld_dtable = ld_dtable * e;
  r.head = w.head;
  r.tail = w.tail;
  r.pitch = g.pitch;
  r.joins = w.joins;
  r.join_runs = w.join_runs;
  fill.keys = r.keys;
  const bool filled = g.passes > 1;
  r.scale = scale;
  if (dtype == B2_DTYPE_BF16) {
    if (vb == 16) run_launch<__nv_bfloat16, 16>(r, fill, filled, width, chain);
    else if (vb == 8) run_launch<__nv_bfloat16, 8>(r, fill, filled, width, chain);
    else if (vb == 4) run_launch<__nv_bfloat16, 4>(r, fill, filled, width, chain);
    else run_launch<__nv_bfloat16, 2>(r, fill, filled, width, chain);
  } else {
    if (vb == 16) run_launch<float, 16>(r, fill, filled, width, chain);
    else if (vb == 8) run_launch<float, 8>(r, fill, filled, width, chain);
    else run_launch<float, 4>(r, fill, filled, width, chain);
  }
  return launch_error(chain.err, "b2_embed_grad");
}

}  // extern "C"
