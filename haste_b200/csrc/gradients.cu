// The global norm of many tensors, sqrt(sum of squares), and clipping: out = gradient min(1, max_norm / (norm + 1e-6)).
//
// Two operations an element: HBM bounds it, one reading for the norm, and a reading (from L2 what fits) and a writing
// where anything is scaled.  Tensors lie anywhere, so a launch takes a table of them by value, and no call copies
// anything to the device: it may be captured.
#include <algorithm>
#include <cmath>

#include "state_space.cuh"

namespace hb {
namespace clip {
namespace {

using namespace ss;

constexpr int THREADS = 256, LOADS = 8;           // 16-byte words of a thread and chunk
constexpr int WORDS = THREADS * LOADS;            // 32 KB of gradients a chunk
constexpr int PER_SM = 4;                         // blocks, each of which leaves one partial sum a launch

struct Entry {
  const void* data;
  void* out;       // null: nothing to write
  long long numel;
  int first;       // chunk of the launch
  signed char dtype, out_dtype, pad, wide;  // pad: elements in front of the first in its 16-byte word; wide: out takes words too
};
template <int N>
struct Table {
  int count, chunks, from;  // from: the launch's first partial
  Entry e[N];
};

struct Finish {
  const double* parts;
  int count;
  float* norm;
  float max_norm;
};

__device__ __forceinline__ double block_sum(double v, double* shared) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < THREADS / 32; ++i) v += shared[i];
  return v;
}

template <int N>
__device__ __forceinline__ const Entry& entry_of(const Table<N>& t, int chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.e[mid].first <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return t.e[lo];
}

// A thread's whole words of a chunk, and the first and the last word of a tensor, which may be its neighbours' too.
template <typename T, int B = 16>  // of B bytes
struct Words {
  static constexpr int V = B / sizeof(T), N = LOADS * 16 / B;
  Raw<T, V> w[N];
  long long first, end;  // element, counted from the start of the tensor's first word, of the thread's first word; the tensor's end
  int pad;
  __device__ __forceinline__ Words(const Entry& e, int chunk)
      : first(((long long)(chunk - e.first) * (THREADS * N) + threadIdx.x) * V), end(e.pad + e.numel), pad(e.pad) {
    const T* base = static_cast<const T*>(e.data) - pad;
#pragma unroll
    for (int k = 0; k < N; ++k) w[k] = load_if<T, V>(whole(k), base + at(k));
  }
  __device__ __forceinline__ long long at(int k) const { return first + (long long)k * THREADS * V; }
  __device__ __forceinline__ bool whole(int k) const { return at(k) >= pad && at(k) + V <= end; }
  // f(element) for those in words that are not whole
  template <typename F>
  __device__ __forceinline__ void edges(const F& f) const {
    if (whole(0) && whole(N - 1)) return;
#pragma unroll 1
    for (int k = 0; k < N; ++k)
      if (!whole(k))
        for (long long i = max(at(k), (long long)pad); i < min(at(k) + V, end); ++i) f(i);
  }
};

// The squares of a thread's whole words in 64 bits.  (A function of its own, which reads them again: what both sums
// share would be kept in 64 registers.)
template <typename T>
__device__ __noinline__ double wide_squares(const T* base, long long first, long long pad, long long end) {
  constexpr int V = 16 / sizeof(T);
  double sum = 0;
#pragma unroll 1
  for (int k = 0; k < LOADS; ++k) {
    const long long i = first + (long long)k * THREADS * V;
    if (i < pad || i + V > end) continue;
    float v[V];
    load<T, V>(base + i, v);
#pragma unroll
    for (int j = 0; j < V; ++j) sum = fma((double)v[j], (double)v[j], sum);
  }
  return sum;
}

// A thread's squares are added in float32, and once more in 64 bits where that over- or underflows.  Sums of threads
// are 64 bits, in a fixed order.  (Words of zeros have no squares that underflow.)
template <typename T>
__device__ __forceinline__ double squares(const Entry& e, int chunk) {
  const Words<T> words(e, chunk);
  constexpr int V = Words<T>::V;
  float s[4] = {};
  uint32_t bits = 0;
#pragma unroll
  for (int k = 0; k < LOADS; ++k) {
    float v[V];
#pragma unroll
    for (uint32_t w : words.w[k].w) bits |= w;
    unpack<T, V>(words.w[k], v);
#pragma unroll
    for (int j = 0; j < V; ++j) s[j % 4] = fmaf(v[j], v[j], s[j % 4]);
  }
  double sum = (s[0] + s[1]) + (s[2] + s[3]);
  const T* base = static_cast<const T*>(e.data) - e.pad;
  constexpr uint32_t SIGNS = sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
  if (!(sum > 1e-20 && sum < 1e30) && (bits & ~SIGNS)) sum = wide_squares<T>(base, words.first, e.pad, words.end);
  words.edges([&](long long i) {
    const double v = ld(base + i);
    sum = fma(v, v, sum);
  });
  return sum;
}

template <int N>
__global__ void __launch_bounds__(THREADS, PER_SM) norm_kernel(const __grid_constant__ Table<N> t, double* parts) {
  __shared__ double shared[THREADS / 32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  double sum = 0;
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const Entry& e = entry_of(t, c);
    if (e.dtype == HASTE_B200_F32) sum += squares<float>(e, c);
    else if (e.dtype == HASTE_B200_BF16) sum += squares<__nv_bfloat16>(e, c);
    else sum += squares<__half>(e, c);
  }
  sum = block_sum(sum, shared);
  if (threadIdx.x == 0) parts[t.from + blockIdx.x] = sum;
}

// The norm, from the partial sums of all launches, which every block adds for itself.
__device__ __forceinline__ double norm_of(const Finish& f, double* shared) {
  double v = 0;
  for (int i = threadIdx.x; i < f.count; i += THREADS) v += f.parts[i];
  return sqrt(block_sum(v, shared));
}
__global__ void __launch_bounds__(THREADS) finish_kernel(const Finish f) {
  __shared__ double shared[THREADS / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const double norm = norm_of(f, shared);
  if (threadIdx.x == 0) *f.norm = (float)norm;
}

template <typename T, typename O>
__device__ __forceinline__ void scale(const Entry& e, int chunk, float factor) {
  // (Words that make 16 bytes at most on either side, so that a warp's stores leave no gaps: bf16 into float32, 402 MB, two
  // stores of 16 bytes a word 250 us.)
  constexpr int B = sizeof(O) > sizeof(T) ? 8 : 16;
  const Words<T, B> words(e, chunk);
  constexpr int V = Words<T, B>::V;
  O* base = static_cast<O*>(e.out) - e.pad;
#pragma unroll
  for (int k = 0; k < Words<T, B>::N; ++k) {
    if (!words.whole(k)) continue;
    O* to = base + words.at(k);
    float v[V];
    unpack<T, V>(words.w[k], v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] *= factor;
    if (e.wide) {
      store<O, V>(to, v);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) st(to + j, v[j]);
    }
  }
  words.edges([&](long long i) { st(base + i, ld(static_cast<const T*>(e.data) - e.pad + i) * factor); });
}
template <typename T>
__device__ __forceinline__ void scale_to(const Entry& e, int chunk, float factor) {
  if (e.out_dtype == HASTE_B200_F32) scale<T, float>(e, chunk, factor);
  else if (e.out_dtype == HASTE_B200_BF16) scale<T, __nv_bfloat16>(e, chunk, factor);
  else scale<T, __half>(e, chunk, factor);
}

// The last chunks first: those are what the norm's launch has left in L2.  Gradients that stay as they are and where
// they are cost no more than the sum of the partials.
template <int N>
__global__ void __launch_bounds__(THREADS, 3) clip_kernel(const __grid_constant__ Table<N> t, const Finish f) {
  __shared__ double shared[THREADS / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");  // (this launch may have overtaken the norm's)
  const double norm = norm_of(f, shared);
  if (blockIdx.x == 0 && threadIdx.x == 0 && t.from == 0) *f.norm = (float)norm;
  const double ratio = f.max_norm / (norm + 1e-6);
  const float factor = ratio > 1. || isinf(f.max_norm) ? 1.f : (float)ratio;  // (a NaN stays)
  for (int c = t.chunks - 1 - blockIdx.x; c >= 0; c -= gridDim.x) {
    const Entry& e = entry_of(t, c);
    if (factor == 1.f && e.out == e.data) continue;
    if (e.dtype == HASTE_B200_F32) scale_to<float>(e, c, factor);
    else if (e.dtype == HASTE_B200_BF16) scale_to<__nv_bfloat16>(e, c, factor);
    else scale_to<__half>(e, c, factor);
  }
}

int size_of(int dtype) { return dtype == HASTE_B200_F32 ? 4 : 2; }
Entry entry(const haste_b200_gradient& g) {
  const int e = size_of(g.dtype), o = size_of(g.out_dtype);
  Entry r{g.data, g.out, g.numel, 0, (signed char)g.dtype, (signed char)g.out_dtype, 0, 0};
  r.pad = (signed char)(reinterpret_cast<uintptr_t>(g.data) % 16 / e);
  const int V = (o > e ? 8 : 16) / e, bytes = V * o;
  r.wide = (reinterpret_cast<uintptr_t>(g.out) - (uintptr_t)(r.pad * o)) % bytes == 0;
  return r;
}
long long chunks_of(const haste_b200_gradient& g) {
  const int V = 16 / size_of(g.dtype);
  const long long n = reinterpret_cast<uintptr_t>(g.data) % 16 / size_of(g.dtype) + g.numel;
  return (n + (long long)V * WORDS - 1) / ((long long)V * WORDS);
}

// A launch that may begin while the one in front of it ends; it waits for that itself.
template <typename K, typename... A>
int launch_behind(K kernel, int blocks, cudaStream_t s, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  HB_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, args...));
  count_launch(1);
  return HASTE_B200_OK;
}

constexpr int FEW = 60, MANY = 960;  // entries of a launch's table: 2 KB of arguments, or 31 KB
int blocks_of(long long chunks) { return (int)std::min(chunks, (long long)PER_SM * sm_count()); }

template <int N>
int launch_table(const haste_b200_gradient* g, int n, int from, int chunks, double* parts, const Finish* f, cudaStream_t s) {
  Table<N> t;
  t.count = 0;
  t.chunks = 0;
  t.from = from;
  for (int i = 0; i < n; ++i) {
    if (g[i].numel == 0) continue;
    Entry e = entry(g[i]);
    e.first = t.chunks;
    t.chunks += (int)chunks_of(g[i]);
    t.e[t.count++] = e;
  }
  // (Of several tables only the first comes close behind: what a launch waits for is the one in front of it, and all norms'
  // have ended when that one's does, since none of them begins early.)
  if (f && from == 0) return launch_behind(clip_kernel<N>, blocks_of(chunks), s, t, *f);
  if (f) clip_kernel<N><<<blocks_of(chunks), THREADS, 0, s>>>(t, *f);
  else norm_kernel<N><<<blocks_of(chunks), THREADS, 0, s>>>(t, parts);
  HB_LAUNCH_OK();
  count_launch(1);
  return HASTE_B200_OK;
}

// Runs over the launches that `count` gradients take: up to MANY of them each.
template <typename F>
int each_launch(const haste_b200_gradient* g, int count, const F& f) {
  for (int i = 0; i < count;) {
    long long chunks = 0;
    int n = 0, used = 0;
    for (; i + n < count && used < MANY; ++n) {
      if (g[i + n].numel == 0) continue;
      const long long c = chunks_of(g[i + n]);
      if (chunks + c > (1 << 30) && used) break;
      chunks += c;
      ++used;
    }
    if (chunks) HB_TRY(f(g + i, n, used, (int)chunks));
    i += n;
  }
  return HASTE_B200_OK;
}
int parts_of(const haste_b200_gradient* g, int count) {
  int parts = 0;
  each_launch(g, count, [&](const haste_b200_gradient*, int, int, int chunks) {
    parts += blocks_of(chunks);
    return HASTE_B200_OK;
  });
  return parts;
}

int check(const haste_b200_gradient* g, int count, bool writes, const float* norm, const float* scratch) {
  HB_REQUIRE(count >= 0 && (g || count == 0), "gradients");
  HB_REQUIRE(norm && (scratch || count == 0) && aligned(scratch, 8), "null pointer");
  for (int i = 0; i < count; ++i) {
    HB_REQUIRE(storage_dtype(g[i].dtype), "dtype");
    HB_REQUIRE(g[i].numel >= 0 && g[i].numel < (1LL << 42), "numel");
    HB_REQUIRE(g[i].data || g[i].numel == 0, "null pointer");
    HB_REQUIRE(aligned(g[i].data, size_of(g[i].dtype)), "misaligned gradient");
    if (!writes) continue;
    HB_REQUIRE(storage_dtype(g[i].out_dtype), "out_dtype");
    HB_REQUIRE(g[i].out || g[i].numel == 0, "null pointer");
    HB_REQUIRE(aligned(g[i].out, size_of(g[i].out_dtype)), "misaligned output");
    HB_REQUIRE(g[i].out != g[i].data || g[i].out_dtype == g[i].dtype || g[i].numel == 0, "in place a gradient keeps its own type");
  }
  return HASTE_B200_OK;
}

int run(const haste_b200_gradient* g, int count, const float* max_norm, float* norm, float* scratch, cudaStream_t s) {
  HB_TRY(check(g, count, max_norm != nullptr, norm, scratch));
  if (max_norm) HB_REQUIRE(*max_norm >= 0, "max_norm");
  ProfScope p(PH_OTHER, s);
  double* parts = reinterpret_cast<double*>(scratch);
  int from = 0;
  HB_TRY(each_launch(g, count, [&](const haste_b200_gradient* some, int n, int used, int chunks) {
    const int at = from;
    from += blocks_of(chunks);
    return used <= FEW ? launch_table<FEW>(some, n, at, chunks, parts, nullptr, s)
                       : launch_table<MANY>(some, n, at, chunks, parts, nullptr, s);
  }));
  const Finish f{parts, from, norm, max_norm ? *max_norm : 0.f};
  if (!max_norm || from == 0) {
    return launch_behind(finish_kernel, 1, s, f);
  }
  from = 0;
  return each_launch(g, count, [&](const haste_b200_gradient* some, int n, int used, int chunks) {
    const int at = from;
    from += blocks_of(chunks);
    return used <= FEW ? launch_table<FEW>(some, n, at, chunks, parts, &f, s)
                       : launch_table<MANY>(some, n, at, chunks, parts, &f, s);
  });
}

}  // namespace
}  // namespace clip

int grad_norm(const haste_b200_gradient* g, int count, float* norm, float* scratch, cudaStream_t s) {
  return clip::run(g, count, nullptr, norm, scratch, s);
}
int clip_gradients(const haste_b200_gradient* g, int count, float max_norm, float* norm, float* scratch, cudaStream_t s) {
  return clip::run(g, count, &max_norm, norm, scratch, s);
}
long long grad_norm_scratch(const haste_b200_gradient* g, int count) {
  for (int i = 0; i < count; ++i)
    if (!ss::storage_dtype(g[i].dtype) || g[i].numel < 0 || g[i].numel >= (1LL << 42)) return 0;
  return 2LL * std::max(1, clip::parts_of(g, count));
}

}  // namespace hb
