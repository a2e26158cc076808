// What the operators around a language model's layers share (embed.cu, xent.cu, muon.cu): error texts, element
// vectors, and workspaces cut into pieces.
#pragma once

#include <stddef.h>

#include <atomic>
#include <type_traits>

#include "../../include/b200mlp.h"
#include "common.cuh"
#include "overlap.h"

namespace b2 {

// Records the text b2_last_error(NULL) returns on this thread and gives back `code` (engine.cu).
int call_error(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

// B2_OK where the calling thread's device can run this library's kernels; *sms = its multiprocessors.
int lm_device(int* sms);

// The report of xent.cu's tile kernels (lm_tile.cuh): CTAs in which a wait gave up, and the first one's role. Waits for the stream.
cudaError_t xent_waits_given_up(unsigned int* count, unsigned int* role, cudaStream_t s);

namespace {

inline int launch_error(cudaError_t e, const char* what) {
  return e == cudaSuccess ? B2_OK : call_error(B2_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}
inline size_t dtype_bytes(int dtype) { return dtype == B2_DTYPE_BF16 ? 2 : 4; }
inline bool dtype_ok(int dtype) { return dtype == B2_DTYPE_F32 || dtype == B2_DTYPE_BF16; }

// Refuses a call whose arguments x[0..n) overlap where one of them is written.
inline int refuse_overlap(const char* who, Extent* x, int n) {
  const Extent *a, *b;
  return any_overlap(x, n, &a, &b) ? call_error(B2_ERR_INVALID, "%s: %s and %s overlap", who, a->name, b->name) : B2_OK;
}

// Pieces of a caller's workspace, each on a 256-byte boundary. With a null base it only adds up sizes.
struct Carver {
  char* base;
  size_t used;
  explicit Carver(void* p) : base(static_cast<char*>(p)), used(0) {}
  template <typename T>
  T* take(size_t count) {
    T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += (count * sizeof(T) + 255) / 256 * 256;
    return p;
  }
};

// The kernels of a call follow one another by programmatic dependent launch: a kernel may be set up while the one before it
// ends, and waits in after_previous() until that one's results are there. `first` kernels of a call are launched in the
// ordinary way, behind whatever the caller's stream holds. Every kernel but the first calls after_previous() in all its blocks before it
// reads or writes anything that the kernel before writes or reads, and in any case before a block ends: only then is the end of a
// kernel, which the next one and whatever follows the call wait for, behind the ends of all kernels before it.
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

struct Chain {
  cudaStream_t stream;
  bool first;
  cudaError_t err;
  explicit Chain(cudaStream_t s) : stream(s), first(true), err(cudaSuccess) {}
  // cluster: CTAs per cluster, 0 for none
  template <typename... P, typename... A>
  void launch(void (*kernel)(P...), dim3 grid, unsigned int threads, size_t smem, int cluster, A&&... args) {
    Config c(grid, threads, smem, stream, cluster, !first);
    if (err == cudaSuccess) err = cudaLaunchKernelEx(&c.cfg, kernel, static_cast<P>(args)...);
    first = false;
  }
  // Arguments where they lie: large ones are copied once only, by the launch.
  template <typename... P>
  void launch_at(void (*kernel)(P...), dim3 grid, unsigned int threads, typename std::remove_const<P>::type*... args) {
    Config c(grid, threads, 0, stream, 0, !first);
    void* p[] = {args...};
    if (err == cudaSuccess) err = cudaLaunchKernelExC(&c.cfg, reinterpret_cast<const void*>(kernel), p);
    first = false;
  }

 private:
  struct Config {
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    Config(dim3 grid, unsigned int threads, size_t smem, cudaStream_t stream, int cluster, bool behind) : cfg() {
      cfg.gridDim = grid;
      cfg.blockDim = dim3(threads);
      cfg.dynamicSmemBytes = smem;
      cfg.stream = stream;
      int n = 0;
      if (cluster) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster;
        attr[n].val.clusterDim.y = 1;
        attr[n].val.clusterDim.z = 1;
        ++n;
      }
      if (behind) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
      }
      cfg.attrs = attr;
      cfg.numAttrs = n;
    }
  };
};

// Lets blocks of a kernel have `bytes` of dynamic shared memory on the current device; a caller asks for the most that any launch of the kernel needs. Once per device:
// it takes as long as a launch.
template <auto kernel>
cudaError_t with_shared(int bytes) {
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1))) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return e;
}

// The widest vector (16, 8 or 4 bytes, or one element) that divides every one of the given addresses and byte counts.
inline int vector_bytes(size_t elem, size_t bits) {
  for (int v = 16; v > (int)elem; v >>= 1)
    if (bits % v == 0) return v;
  return (int)elem;
}

template <int BYTES> struct Raw;
template <> struct Raw<16> { typedef uint4 type; };
template <> struct Raw<8> { typedef uint2 type; };
template <> struct Raw<4> { typedef unsigned int type; };
template <> struct Raw<2> { typedef unsigned short type; };

// BYTES bytes of elements of type T as floats, and back (rounded to nearest).
template <typename T, int BYTES>
struct Elems {
  static constexpr int N = BYTES / (int)sizeof(T);
  typedef typename Raw<BYTES>::type raw;
  static __device__ __forceinline__ void get(const raw& r, float (&f)[N]) {
    if constexpr (sizeof(T) == 2 && N > 1) {  // a bf16 is the upper half of its fp32: one instruction each
      const unsigned int* t = reinterpret_cast<const unsigned int*>(&r);
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        f[i] = __uint_as_float(t[i / 2] << 16);
        f[i + 1] = __uint_as_float(t[i / 2] & 0xFFFF0000u);
      }
    } else {
      const T* t = reinterpret_cast<const T*>(&r);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = (float)t[i];
    }
  }
  static __device__ __forceinline__ raw put(const float (&f)[N]) {
    raw r;
    if constexpr (sizeof(T) == 2 && N > 1) {  // rounded two at a time
      __nv_bfloat162* t = reinterpret_cast<__nv_bfloat162*>(&r);
#pragma unroll
      for (int i = 0; i < N; i += 2) t[i / 2] = __floats2bfloat162_rn(f[i], f[i + 1]);
    } else {
      T* t = reinterpret_cast<T*>(&r);
#pragma unroll
      for (int i = 0; i < N; ++i) t[i] = (T)f[i];
    }
    return r;
  }
};

// Sums over the whole range of fp32: up to N terms are added in fp32 and such sums in fp64; where fp32 has no product, or not with all of its bits, products are
// taken in fp64 as well.
__device__ __forceinline__ bool safe_sum(float s) { return fabsf(s) > 1e-25f && fabsf(s) < 1e38f; }
template <int N>
__device__ __forceinline__ void add_squares(const float (&f)[N], double& sum) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) s = fmaf(f[i], f[i], s);
  if (safe_sum(s)) {
    sum += (double)s;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) sum = fma((double)f[i], (double)f[i], sum);
  }
}

// Token number i of a list of 32- or 64-bit ones; anything outside [0, vocab) becomes vocab.
__device__ __forceinline__ unsigned int token_at(const void* tokens, int wide, size_t i, unsigned int vocab) {
  const long long t = wide ? __ldg(static_cast<const long long*>(tokens) + i) : (long long)__ldg(static_cast<const int*>(tokens) + i);
  return t >= 0 && t < (long long)vocab ? (unsigned int)t : vocab;
}

}  // namespace
}  // namespace b2
