// The global norm of a list of tensors, and the tensors scaled so that it is at most max_norm:
//
//   norm = sqrt(sum over all elements of x^2)     out = x * (norm > max_norm ? max_norm / norm : 1)
//
// Bound by HBM: everything is read for the norm, and where something is to be written, read again and written. The second pass goes through
// each block's part from the end to the beginning, so that it finds what the first pass read last in the L2 cache.
//
// Elements of all tensors are cut into units of UNIT_BYTES, and every block takes an equal share of neighbouring units, whichever tensors they
// lie in (a binary search over the first units of the tensors, which are kernel parameters), and leaves one fp64 sum; each block of the second
// kernel adds all blocks' sums in the same order, so that equal inputs give equal bits.
//
// Measured on one B200 (a copy reaches 6.56 TB/s): 8 x 4096 x 4096 bf16 within the limit 46 us, 5.8 TB/s; scaled into other tensors 138 us for three passes of 268 MB (5.8
// TB/s, some of the second from the L2 cache; forwards instead of backwards 141, and 55 for 49.5 us with three matrices). 5 x 1024 x 1024 fp32 scaled 18 us: two
// kernels of 7 and 8 us, of which each is 3 us of launch, reduction and end.
#include <math.h>

#include <algorithm>
#include <exception>
#include <memory>

#include "lm.cuh"

namespace b2 {
namespace {

constexpr int CLIP_THREADS = 512;
constexpr int UNIT_BYTES = 8192;  // of bf16 or fp32 elements
constexpr int BACK_UNITS = 4;     // the second pass goes back by so many at a time: 2048 vectors, four per thread
constexpr int CLIP_BLOCKS = 148 * 2;

struct ClipTensor {
  const char* x;
  char* out;
  unsigned long long size, cols, ld_x, ld_out;  // elements
  unsigned int f32, gaps;                       // gaps: rows with gaps between them; otherwise one piece of `size` elements
};
// Kernel parameters: up to MOST tensors. Two sizes, because a launch takes longer with more of them (28 KB of the 32 KB that there are): 5 tensors take 7.1 us of the
// caller's time for 8.5.
template <int MOST>
struct ClipList {
  ClipTensor t[MOST];
  unsigned int first[MOST + 1];  // unit
  int count;
};
constexpr int LIST_SHORT = 40, LIST_MOST = 480;
static_assert(sizeof(ClipList<LIST_MOST>) < 32000, "kernel parameters have 32764 bytes");

// Part of a tensor: elements [from, from + n).
struct ClipPart {
  int tensor;
  unsigned long long from, n;
};
__host__ __device__ inline unsigned int unit_elements(unsigned int f32) { return f32 ? UNIT_BYTES / 4 : UNIT_BYTES / 2; }

template <class List>
__device__ __forceinline__ int tensor_of(const List& list, unsigned int unit) {
  int lo = 0, hi = list.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (list.first[mid] <= unit) lo = mid;
    else hi = mid;
  }
  return lo;
}
// The part of tensor k in units [u0, u1), of which the first one or the last one lies in it.
template <class List>
__device__ __forceinline__ ClipPart part_of(const List& list, int k, unsigned int u0, unsigned int u1) {
  const ClipTensor& t = list.t[k];
  if (u0 < list.first[k]) u0 = list.first[k];
  if (u1 > list.first[k + 1]) u1 = list.first[k + 1];
  const unsigned long long e = unit_elements(t.f32), from = (u0 - list.first[k]) * e, to = (u1 - list.first[k]) * e;
  return ClipPart{k, from, (to < t.size ? to : t.size) - from};
}
// This block's share of the units.
template <class List>
__device__ __forceinline__ void share(const List& list, unsigned int& u0, unsigned int& u1) {
  const unsigned long long units = list.first[list.count];
  u0 = (unsigned int)(units * blockIdx.x / gridDim.x);
  u1 = (unsigned int)(units * (blockIdx.x + 1) / gridDim.x);
}

__device__ __forceinline__ double block_sum(double s, double* slots) {
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
  for (int i = 0; i < CLIP_THREADS / 32; ++i) s += slots[i];
  return s;
}

// Elements [0, n) of a dense piece at x: ahead of the first 16-byte boundary, behind the last one, and the vectors between.
template <typename T>
__device__ __forceinline__ double squares_dense(const T* x, unsigned long long n) {
  typedef Elems<T, 16> E;
  constexpr int U = 4;
  double sum = 0.0;
  int head = (int)((16 - (reinterpret_cast<size_t>(x) & 15)) & 15) / (int)sizeof(T);
  if ((unsigned long long)head > n) head = (int)n;
  const unsigned long long vecs = (n - head) / E::N;
  const int tail = (int)(n - head - vecs * E::N);
  const uint4* v = reinterpret_cast<const uint4*>(x + head);
  for (unsigned long long i = threadIdx.x; i < vecs; i += CLIP_THREADS * U) {
    uint4 r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      r[u] = make_uint4(0, 0, 0, 0);
      if (i + u * CLIP_THREADS < vecs) r[u] = __ldg(v + i + u * CLIP_THREADS);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[E::N];
      E::get(r[u], f);
      add_squares(f, sum);
    }
  }
  const int odd = (int)threadIdx.x;
  if (odd < head + tail) {
    const float f[1] = {(float)x[odd < head ? odd : n - tail + odd - head]};
    add_squares(f, sum);
  }
  return sum;
}

// Elements [from, from + n) of a matrix with gaps between its rows.
template <typename T>
__device__ __forceinline__ double squares_rows(const ClipTensor& t, unsigned long long from, unsigned long long n) {
  const T* x = reinterpret_cast<const T*>(t.x);
  double sum = 0.0;
  for (unsigned long long i = threadIdx.x; i < n; i += CLIP_THREADS) {
    const unsigned long long at = from + i, row = at / t.cols;
    const float f[1] = {(float)x[row * t.ld_x + (at - row * t.cols)]};
    add_squares(f, sum);
  }
  return sum;
}

template <class List>
__global__ void __launch_bounds__(CLIP_THREADS, 2) clip_norm_kernel(const __grid_constant__ List list, double* __restrict__ partial) {
  __shared__ double slots[CLIP_THREADS / 32];
  let_next_start();
  unsigned int u, end;
  share(list, u, end);
  double sum = 0.0;
  for (int k = tensor_of(list, u); u < end; u = list.first[++k]) {
    const ClipTensor& t = list.t[k];
    const ClipPart p = part_of(list, k, u, end);
    if (t.gaps) sum += t.f32 ? squares_rows<float>(t, p.from, p.n) : squares_rows<__nv_bfloat16>(t, p.from, p.n);
    else if (t.f32) sum += squares_dense(reinterpret_cast<const float*>(t.x) + p.from, p.n);
    else sum += squares_dense(reinterpret_cast<const __nv_bfloat16*>(t.x) + p.from, p.n);
  }
  sum = block_sum(sum, slots);
  after_previous();
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

template <typename T, int VB>
__device__ __forceinline__ void scale_vectors(const T* x, T* out, int vecs, float factor) {
  typedef Elems<T, VB> E;
  typedef typename E::raw raw;
  constexpr int U = 4;
  const raw* v = reinterpret_cast<const raw*>(x);
  raw* o = reinterpret_cast<raw*>(out);
  for (int i = threadIdx.x; i < vecs; i += CLIP_THREADS * U) {
    raw r[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * CLIP_THREADS < vecs) r[u] = v[i + u * CLIP_THREADS];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * CLIP_THREADS >= vecs) break;
      float f[E::N];
      E::get(r[u], f);
#pragma unroll
      for (int j = 0; j < E::N; ++j) f[j] *= factor;
      o[i + u * CLIP_THREADS] = E::put(f);
    }
  }
}

template <typename T, int VB>
__device__ __forceinline__ void scale_from(const T* x, T* out, int n, int head, float factor) {
  constexpr int N = VB / (int)sizeof(T);
  if (head > n) head = n;
  const int vecs = (n - head) / N, tail = n - head - vecs * N;
  scale_vectors<T, VB>(x + head, out + head, vecs, factor);
  const int odd = (int)threadIdx.x;
  if (odd < head + tail) {
    const int i = odd < head ? odd : n - tail + odd - head;
    out[i] = (T)((float)x[i] * factor);
  }
}

// The widest vectors that both sides have boundaries of at the same elements.
template <typename T>
__device__ __forceinline__ void scale_dense(const T* x, T* out, int n, float factor) {
  const size_t a = reinterpret_cast<size_t>(x), b = reinterpret_cast<size_t>(out);
  const int apart = (int)((a ^ b) & 15);
  auto head = [&](int vb) { return (int)((vb - (a & (vb - 1))) & (vb - 1)) / (int)sizeof(T); };
  if (apart == 0) scale_from<T, 16>(x, out, n, head(16), factor);
  else if (apart % 8 == 0) scale_from<T, 8>(x, out, n, head(8), factor);
  else if (apart % 4 == 0) scale_from<T, 4>(x, out, n, head(4), factor);
  else scale_from<T, sizeof(T)>(x, out, n, 0, factor);
}

// Of a matrix with gaps between its rows; with a factor in fp64 of any tensor. N: what counts n elements.
template <typename T, typename N, typename F>
__device__ __forceinline__ void scale_rows(const ClipTensor& t, unsigned long long from, N n, F factor) {
  for (N i = threadIdx.x; i < n; i += CLIP_THREADS) {
    const unsigned long long at = from + i, row = at / t.cols, col = at - row * t.cols;
    reinterpret_cast<T*>(t.out)[row * t.ld_out + col] = (T)(float)((F)(float)reinterpret_cast<const T*>(t.x)[row * t.ld_x + col] * factor);
  }
}

// in_place: nothing is written where nothing is over the limit. norm: of the first launch of a call only.
template <class List>
__global__ void __launch_bounds__(CLIP_THREADS, 2) clip_scale_kernel(const __grid_constant__ List list, const double* __restrict__ partial, int partials,
                                                                     float max_norm, int in_place, float* norm_out) {
  __shared__ double slots[CLIP_THREADS / 32];
  let_next_start();
  after_previous();
  double sum = 0.0;
  for (int i = threadIdx.x; i < partials; i += CLIP_THREADS) sum += partial[i];
  const double norm = sqrt(block_sum(sum, slots));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const bool over = norm > (double)max_norm && (float)norm < INFINITY;  // a norm that is reported as infinite, or none, leaves the tensors as they are
  if (in_place && !over) return;
  const double exact = over ? (double)max_norm / norm : 1.0;
  const float factor = (float)exact;
  const bool far = exact > 0.0 && exact < 1.1754943508222875e-38;  // fp32 has no such factor, or not with all of its bits
  unsigned int begin, u;
  share(list, begin, u);
  if (far) {  // rare: one element at a time, in a loop of its own, which the other one is no slower for (with a branch to it there, 5 x 1024 x 1024 fp32 took 20.7 us for 18.0)
    for (int k; begin < u; begin = list.first[k + 1]) {
      k = tensor_of(list, begin);
      const ClipTensor& t = list.t[k];
      const ClipPart p = part_of(list, k, begin, u);
      if (t.f32) scale_rows<float>(t, p.from, p.n, exact);
      else scale_rows<__nv_bfloat16>(t, p.from, p.n, exact);
    }
    return;
  }
  while (u > begin) {
    const int k = tensor_of(list, u - 1);
    unsigned int from = u - begin > BACK_UNITS ? u - BACK_UNITS : begin;
    if (from < list.first[k]) from = list.first[k];
    const ClipTensor& t = list.t[k];
    const ClipPart p = part_of(list, k, from, u);
    const int n = (int)p.n;
    if (t.gaps) {
      if (t.f32) scale_rows<float>(t, p.from, n, factor);
      else scale_rows<__nv_bfloat16>(t, p.from, n, factor);
    } else if (t.f32) {
      scale_dense(reinterpret_cast<const float*>(t.x) + p.from, reinterpret_cast<float*>(t.out) + p.from, n, factor);
    } else {
      scale_dense(reinterpret_cast<const __nv_bfloat16*>(t.x) + p.from, reinterpret_cast<__nv_bfloat16*>(t.out) + p.from, n, factor);
    }
    u = from;
  }
}

size_t clip_space(size_t count, int most, void* base, double** partial) {
  Carver c(base);
  *partial = c.take<double>((count + most - 1) / most * CLIP_BLOCKS);
  return c.used;
}

constexpr size_t TENSORS_MOST = 1 << 20;
constexpr unsigned long long ELEMENTS_MOST = 1ull << 42;  // of all tensors: unit numbers have 32 bits

template <int MOST>
cudaError_t clip_launch(const std::vector<ClipTensor>& tensors, bool in_place, float max_norm, float* norm, double* partial, int sms, cudaStream_t stream) {
  typedef ClipList<MOST> List;
  const size_t launches = tensors.empty() ? 1 : (tensors.size() + MOST - 1) / MOST;
  const std::unique_ptr<List[]> lists(new List[launches]);
  std::vector<int> blocks(launches);
  int partials = 0;
  Chain chain(stream);
  for (size_t i = 0; i < launches; ++i) {
    List& l = lists[i];
    l.count = 0;
    unsigned int units = 0;
    for (size_t k = i * MOST; k < tensors.size() && l.count < MOST; ++k) {
      const ClipTensor& t = tensors[k];
      l.first[l.count] = units;
      l.t[l.count++] = t;
      units += (unsigned int)((t.size + unit_elements(t.f32) - 1) / unit_elements(t.f32));
    }
    l.first[l.count] = units;
    const int most = sms * 2 < CLIP_BLOCKS ? sms * 2 : CLIP_BLOCKS;
    blocks[i] = units == 0 ? 1 : units < (unsigned int)most ? (int)units : most;
    double* sums = partial + partials;
    chain.launch_at(clip_norm_kernel<List>, dim3(blocks[i]), CLIP_THREADS, &l, &sums);
    partials += blocks[i];
  }
  const bool limited = max_norm < INFINITY;
  int place = in_place;
  for (size_t i = 0; i < (limited ? launches : 1); ++i) {
    float* to = i == 0 ? norm : nullptr;
    const double* sums = partial;
    chain.launch_at(clip_scale_kernel<List>, dim3(limited ? blocks[i] : 1), CLIP_THREADS, &lists[i], &sums, &partials, &max_norm, &place, &to);
  }
  return chain.err;
}

struct ClipCall {
  size_t count;
  const void* const* x;
  void* const* out;
  const size_t* elements;
  const int* dtypes;
  const size_t *widths, *ld_x, *ld_out;
};

int clip_tensors(const char* who, const ClipCall& c, float max_norm, float* norm, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  const bool limited = max_norm < INFINITY;
  const size_t count = c.count;
  bool in_place = true;
  std::vector<Extent> args, outputs;
  std::vector<ClipTensor> tensors;
  args.reserve(2 * count + 2);
  outputs.reserve(c.out ? count + 2 : 2);
  tensors.reserve(count);
  unsigned long long all = 0;
  for (size_t i = 0; i < count; ++i) {
    const int dtype = c.dtypes[i];
    if (!dtype_ok(dtype)) return call_error(B2_ERR_INVALID, "%s: dtype %d of tensor %zu", who, dtype, i);
    const size_t e = dtype_bytes(dtype), size = c.elements[i];
    if (size == 0) continue;
    const void* x = c.x[i];
    void* out = c.out ? c.out[i] : const_cast<void*>(x);
    if (!x || !out) return call_error(B2_ERR_INVALID, "%s: null pointer of tensor %zu", who, i);
    if (size > ELEMENTS_MOST || (all += size) > ELEMENTS_MOST) return call_error(B2_ERR_INVALID, "%s: more than 2^42 elements up to tensor %zu", who, i);
    size_t width = size, ld_x = size, ld_out = size;
    if (c.widths && c.widths[i] != size) {
      width = c.widths[i];
      ld_x = c.ld_x[i];
      ld_out = c.out ? c.ld_out[i] : ld_x;
      if (width == 0 || size % width) return call_error(B2_ERR_INVALID, "%s: %zu elements of tensor %zu are not whole rows of %zu", who, size, i, width);
      if (ld_x < width || ld_out < width) return call_error(B2_ERR_INVALID, "%s: leading dimension of tensor %zu smaller than its width", who, i);
    }
    if ((reinterpret_cast<size_t>(x) | reinterpret_cast<size_t>(out)) % e)
      return call_error(B2_ERR_INVALID, "%s: a pointer of tensor %zu is not aligned to its elements", who, i);
    const bool here = out == x && ld_out == ld_x;
    args.push_back(extent("a tensor", x, size / width, width * e, ld_x * e, limited && here));
    if (!here) {
      outputs.push_back(extent("an output", out, size / width, width * e, ld_out * e, true));
      in_place = false;
    }
    tensors.push_back(ClipTensor{static_cast<const char*>(x), static_cast<char*>(out), size, width, ld_x, ld_out, dtype == B2_DTYPE_F32,
                                 ld_x != width || ld_out != width});
  }
  if (!limited && c.out) return call_error(B2_ERR_INVALID, "%s: outputs without a limit", who);
  const int most = count <= LIST_SHORT ? LIST_SHORT : LIST_MOST;
  double* partial;
  const size_t need = clip_space(count ? count : 1, most, workspace, &partial);
  if (workspace_bytes < need) return call_error(B2_ERR_INVALID, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, need);
  int sms, rc;
  if ((rc = lm_device(&sms)) != B2_OK) return rc;
  // tensors and outputs mostly come in the order in which they lie in memory: hundreds are sorted in no time then
  const size_t inputs = args.size();
  for (std::vector<Extent>* v : {&args, &outputs})
    if (!std::is_sorted(v->begin(), v->end(), begins_before)) std::sort(v->begin(), v->end(), begins_before);
  Extent more[] = {extent("norm", norm, 1, 4, 4, true), extent("the workspace", workspace, 1, need, need, true)};
  for (const Extent& x : more) outputs.insert(std::upper_bound(outputs.begin(), outputs.end(), x, begins_before), x);
  args.insert(args.end(), outputs.begin(), outputs.end());
  std::inplace_merge(args.begin(), args.begin() + inputs, args.end(), begins_before);
  const Extent *one, *other;
  if (first_overlap(args.data(), (int)args.size(), &one, &other)) return call_error(B2_ERR_INVALID, "%s: %s and %s overlap", who, one->name, other->name);
  const cudaError_t e = most == LIST_SHORT ? clip_launch<LIST_SHORT>(tensors, in_place, max_norm, norm, partial, sms, stream)
                                           : clip_launch<LIST_MOST>(tensors, in_place, max_norm, norm, partial, sms, stream);
  return launch_error(e, who);
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

int b2_clip_workspace(size_t count, size_t* bytes) {
  if (count > TENSORS_MOST) return call_error(B2_ERR_INVALID, "b2_clip_workspace: %zu tensors (2^20 at most)", count);
  if (!bytes) return call_error(B2_ERR_INVALID, "b2_clip_workspace: null pointer");
  double* partial;
  *bytes = clip_space(count ? count : 1, count <= LIST_SHORT ? LIST_SHORT : LIST_MOST, nullptr, &partial);
  return B2_OK;
}

int b2_clip(size_t count, const void* const* x, void* const* out, const size_t* elements, const int* dtypes, const size_t* widths, const size_t* ld_x,
            const size_t* ld_out, float max_norm, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "b2_clip";
  if (count > TENSORS_MOST) return call_error(B2_ERR_INVALID, "%s: %zu tensors (2^20 at most)", who, count);
  if (!(max_norm >= 0.f)) return call_error(B2_ERR_INVALID, "%s: max_norm is negative or not a number", who);
  if ((count && (!x || !elements || !dtypes || (widths && (!ld_x || (out && !ld_out))))) || !norm || !workspace) return call_error(B2_ERR_INVALID, "%s: null pointer", who);
  if (reinterpret_cast<size_t>(norm) % 4) return call_error(B2_ERR_INVALID, "%s: norm is not aligned", who);
  if (reinterpret_cast<size_t>(workspace) % 256) return call_error(B2_ERR_INVALID, "%s: the workspace is not on a 256-byte boundary", who);
  try {
    return clip_tensors(who, ClipCall{count, x, out, elements, dtypes, widths, ld_x, ld_out}, max_norm, norm, workspace, workspace_bytes,
                        static_cast<cudaStream_t>(stream));
  } catch (const std::exception&) {
    return call_error(B2_ERR_INVALID, "%s: no host memory for the list", who);
  }
}

}  // extern "C"
