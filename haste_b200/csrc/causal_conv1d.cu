// Short causal depthwise convolution along time with bias and SiLU, forward and backward.
//
//   p_t = bias + sum_k w_k x_{t-(W-1)+k},  y_t = silu(p_t)
//
// A stream over x and y (backward: x and dy in, dx out): 2 W + 5 operations a value against 4 to 8
// bytes, so HBM bounds it.  A thread owns V neighbouring channels and walks a chunk of steps with
// the last W - 1 inputs in registers; the next group of steps is loaded while one is computed, and two
// channels go to an instruction.  fp32 T=400 N=64 D=1024: forward 39 us, 5.3 TB/s (0.82 of the measured
// copy), backward 63 us, 5.0 TB/s with its sums.  16-bit sequences move half the bytes for the same
// instructions, which then share the bound: bf16 T=4000 N=8 D=2048 56 us, 4.7 TB/s (48 without SiLU).
#include <algorithm>

#include "state_space.cuh"

namespace hb {
namespace {

using namespace ss;

// Steps of one group in the forward pass: 64 bytes where a thread has four channels.  The next group is under way
// while one is computed.
template <typename T>
constexpr int GROUP = sizeof(T) == 4 ? 4 : 8;

template <typename T>
struct ConvArgs {
  int T_, N, D, chunk, dtiles;
  bool param_f32, silu;
  Seq<const T> x, dy;
  Seq<T> y, dx;
  const void *w, *b;
  const T* state;
  T* final_state;
  const long long* lengths;
  const T* dfinal;
  T* dstate;
  float* part;
  int items, parts;
};

// The input at a step of the row, the initial state's rows before it (step >= -(W-1)).
template <typename T, int V, int W>
__device__ __forceinline__ void input_at(const ConvArgs<T>& a, int t, int len, int n, int d, float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = 0.f;
  if (t >= 0) {
    if (t < len) load<T, V>(a.x.at(t, n) + d, v);
  } else if (a.state) {
    load<T, V>(a.state + ((long long)n * (W - 1) + t + W - 1) * a.D + d, v);
  }
}

// Two neighbouring channels to an instruction; V of them are (V + 1) / 2 pairs, one channel a pair with nothing.
template <int V>
__device__ __forceinline__ void pairs(const float (&v)[V], float2 (&p)[(V + 1) / 2]) {
#pragma unroll
  for (int i = 0; i < (V + 1) / 2; ++i) p[i] = make_float2(v[2 * i], 2 * i + 1 < V ? v[2 * i + 1 < V ? 2 * i + 1 : 0] : 0.f);
}
template <int V>
__device__ __forceinline__ void single(const float2 (&p)[(V + 1) / 2], float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = i % 2 ? p[i / 2].y : p[i / 2].x;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 sigmoid(float2 v) { return make_float2(ss::sigmoid(v.x), ss::sigmoid(v.y)); }

// The taps of V neighbouring channels, W packs as they lie in memory, and their bias.
template <typename T, int V, int W>
__device__ __forceinline__ void parameters(const ConvArgs<T>& a, int d, float2 (&w)[W][(V + 1) / 2], float2 (&b)[(V + 1) / 2]) {
  float flat[W * V], row[V];
#pragma unroll
  for (int k = 0; k < W; ++k) {
    if (a.param_f32) load<float, V>(static_cast<const float*>(a.w) + (long long)d * W + k * V, row);
    else load<T, V>(static_cast<const T*>(a.w) + (long long)d * W + k * V, row);
#pragma unroll
    for (int i = 0; i < V; ++i) flat[k * V + i] = row[i];
  }
#pragma unroll
  for (int k = 0; k < W; ++k) {
#pragma unroll
    for (int i = 0; i < V; ++i) row[i] = flat[i * W + k];
    pairs<V>(row, w[k]);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) row[i] = a.b ? ldp<T>(a.b, a.param_f32, d + i) : 0.f;
  pairs<V>(row, b);
}

// bias + sum_k w_k x_k of a window
template <int P, int W>
__device__ __forceinline__ void convolve(const float2 (&w)[W][P], const float2 (&b)[P], const float2 (&x)[W][P], float2 (&p)[P]) {
#pragma unroll
  for (int i = 0; i < P; ++i) {
    p[i] = b[i];
#pragma unroll
    for (int k = 0; k < W; ++k) p[i] = __ffma2_rn(w[k][i], x[k][i], p[i]);
  }
}

// (Five resident blocks, which the launch counts on.  Left alone, four channels of 16 bits and four taps take
// 128 registers, and four blocks fit: bf16 1000 x 64 x 1024 72 us, with five 65; 400 x 64 x 1024 36 and 32.
// Forced elsewhere it costs: fp32 300 x 64 x 1024 34 and 36, three taps 11 and 13.  0: no wish.)
template <typename T, int V, int W>
__global__ void __launch_bounds__(128, sizeof(T) == 2 && V == 4 && W == 4 ? 5 : 0) conv_fwd(ConvArgs<T> a) {
  constexpr int G = GROUP<T>, P = (V + 1) / 2;
  const int d = ((blockIdx.x % a.dtiles) * blockDim.x + threadIdx.x) * V;
  const int item = blockIdx.x / a.dtiles, n = item % a.N, c = item / a.N;
  if (d >= a.D) return;
  const int len = row_length(a.lengths, n, a.T_);
  const int t0 = c * a.chunk, t1 = min(a.T_, t0 + a.chunk), live = min(t1, len);
  Raw<T, V> in[G];
  const T* px = a.x.at(t0, n) + d;
  auto fetch = [&](int t, Raw<T, V> (&to)[G]) {
#pragma unroll
    for (int u = 0; u < G; ++u) to[u] = load_if<T, V>(t + u < live, px + (long long)u * a.x.t);
    px += (long long)G * a.x.t;
  };
  fetch(t0, in);
  float2 w[W][P], b[P], xs[W][P];  // xs: the window, its last row the step at hand
  float row[V];
  parameters<T, V, W>(a, d, w, b);
#pragma unroll
  for (int k = 0; k < W - 1; ++k) {
    input_at<T, V, W>(a, t0 - (W - 1) + k, len, n, d, row);
    pairs<V>(row, xs[k + 1]);
  }
  T* py = a.y.at(t0, n) + d;
  for (int t = t0; t < t1; t += G) {
    Raw<T, V> next[G];
    fetch(t + G, next);
    float2 y[G][P];
#pragma unroll
    for (int u = 0; u < G; ++u) {
#pragma unroll
      for (int k = 0; k < W - 1; ++k)
#pragma unroll
        for (int i = 0; i < P; ++i) xs[k][i] = xs[k + 1][i];
      unpack<T, V>(in[u], row);
      pairs<V>(row, xs[W - 1]);
      convolve<P, W>(w, b, xs, y[u]);
    }
    // (all sigmoids of the group together: each is a chain of two slow instructions)
    if (a.silu)
#pragma unroll
      for (int u = 0; u < G; ++u)
#pragma unroll
        for (int i = 0; i < P; ++i) y[u][i] = __fmul2_rn(y[u][i], sigmoid(y[u][i]));
#pragma unroll
    for (int u = 0; u < G; ++u) {
      if (t + u >= len)
#pragma unroll
        for (int i = 0; i < P; ++i) y[u][i] = both(0.f);
      single<V>(y[u], row);
      if (t + u < t1) store<T, V>(py + (long long)u * a.y.t, row);
    }
    py += (long long)G * a.y.t;
#pragma unroll
    for (int u = 0; u < G; ++u) in[u] = next[u];
  }
  // The last W - 1 inputs of the row.  Row k comes from row k + len of the state at the earliest, so
  // in ascending order the two may be one buffer; what this thread has read above is in registers,
  // and no other thread reads these channels' state (a chunk is longer than W - 1 steps).
  if (c == 0 && a.final_state) {
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      input_at<T, V, W>(a, len - (W - 1) + k, len, n, d, row);
      store<T, V>(a.final_state + ((long long)n * (W - 1) + k) * a.D + d, row);
    }
  }
}

// dx_t = sum_k w_k dp_{t+(W-1)-k} with dp = dy silu'(p): a thread walks its chunk and W - 1 steps
// beyond it, recomputes p, and emits dx W - 1 steps behind.  dw and db are summed in registers over
// the chunks that a block takes in turn; its partial rows are added in a fixed order afterwards.
template <typename T, int V, int W>
__global__ void __launch_bounds__(128) conv_bwd(ConvArgs<T> a) {
  constexpr int G = 4, P = (V + 1) / 2;
  const int d = ((blockIdx.x % a.dtiles) * blockDim.x + threadIdx.x) * V;
  const int part = blockIdx.x / a.dtiles;
  if (d >= a.D) return;
  float2 w[W][P], b[P], dw[W][P], db[P];
  float row[V];
  parameters<T, V, W>(a, d, w, b);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    db[i] = both(0.f);
#pragma unroll
    for (int k = 0; k < W; ++k) dw[k][i] = both(0.f);
  }
  for (int item = part; item < a.items; item += a.parts) {
    const int n = item % a.N, c = item / a.N;
    const int len = row_length(a.lengths, n, a.T_);
    const int t0 = c * a.chunk, t1 = min(a.T_, t0 + a.chunk), end = t1 + W - 1, live = min(end, len);
    Raw<T, V> in[G], gr[G];
    const T *px = a.x.at(t0, n) + d, *pg = a.dy.at(t0, n) + d;
    auto fetch = [&](int t, Raw<T, V> (&x)[G], Raw<T, V> (&g)[G]) {
#pragma unroll
      for (int u = 0; u < G; ++u) {
        x[u] = load_if<T, V>(t + u < live, px + (long long)u * a.x.t);
        g[u] = load_if<T, V>(t + u < live, pg + (long long)u * a.dy.t);
      }
      px += (long long)G * a.x.t;
      pg += (long long)G * a.dy.t;
    };
    fetch(t0, in, gr);
    float2 xs[W][P], dp[W][P];
#pragma unroll
    for (int k = 0; k < W; ++k)
#pragma unroll
      for (int i = 0; i < P; ++i) dp[k][i] = both(0.f);
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      input_at<T, V, W>(a, t0 - (W - 1) + k, len, n, d, row);
      if (len == 0)  // (the state of a row without steps meets no tap, and may be no number)
#pragma unroll
        for (int i = 0; i < V; ++i) row[i] = 0.f;
      pairs<V>(row, xs[k + 1]);
    }
    for (int t = t0; t < end; t += G) {
      Raw<T, V> xn[G], gn[G];
      fetch(t + G, xn, gn);
#pragma unroll
      for (int u = 0; u < G; ++u) {
        const int te = t + u - (W - 1);  // the step whose dx is complete now
        float2 dx[P], g[P];
#pragma unroll
        for (int k = 0; k < W - 1; ++k)
#pragma unroll
          for (int i = 0; i < P; ++i) {
            xs[k][i] = xs[k + 1][i];
            dp[k][i] = dp[k + 1][i];
          }
        unpack<T, V>(in[u], row);
        pairs<V>(row, xs[W - 1]);
        unpack<T, V>(gr[u], row);
        pairs<V>(row, g);
        if (a.silu) {
          float2 p[P];
          convolve<P, W>(w, b, xs, p);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const float2 s = sigmoid(p[i]), rest = __ffma2_rn(s, both(-1.f), both(1.f));
            g[i] = __fmul2_rn(g[i], __ffma2_rn(__fmul2_rn(p[i], s), rest, s));
          }
          if (t + u >= len)  // (the incoming gradient counts for nothing, whatever p is)
#pragma unroll
            for (int i = 0; i < P; ++i) g[i] = both(0.f);
        } else if (t + u >= len) {  // (an infinite last input meets no step behind it; with SiLU its own step's g is no number)
#pragma unroll
          for (int k = 0; k < W; ++k)
#pragma unroll
            for (int i = 0; i < P; ++i) xs[k][i] = both(0.f);
        }
#pragma unroll
        for (int i = 0; i < P; ++i) {
          dp[W - 1][i] = g[i];
          dx[i] = __fmul2_rn(w[0][i], g[i]);
#pragma unroll
          for (int k = 1; k < W; ++k) dx[i] = __ffma2_rn(w[k][i], dp[W - 1 - k][i], dx[i]);
        }
        if (t + u < t1)
#pragma unroll
          for (int i = 0; i < P; ++i) {
            db[i] = __fadd2_rn(db[i], g[i]);
#pragma unroll
            for (int k = 0; k < W; ++k) dw[k][i] = __ffma2_rn(g[i], xs[k][i], dw[k][i]);
          }
        const bool before = te < 0;  // a row of the initial state
        if (t + u >= end || (before ? c != 0 : te < t0)) continue;
        single<V>(dx, row);
        if (a.dfinal && te >= len - (W - 1) && te < len) {
          float f[V];
          load<T, V>(a.dfinal + ((long long)n * (W - 1) + te - len + W - 1) * a.D + d, f);
#pragma unroll
          for (int i = 0; i < V; ++i) row[i] += f[i];
        }
        if (!before) {
          if (a.dx.p) store<T, V>(a.dx.at(te, n) + d, row);
        } else if (a.dstate) {
          store<T, V>(a.dstate + ((long long)n * (W - 1) + te + W - 1) * a.D + d, row);
        }
      }
#pragma unroll
      for (int u = 0; u < G; ++u) {
        in[u] = xn[u];
        gr[u] = gn[u];
      }
    }
  }
  // partial row of this block: [D][W] of dw, then [D] of db
  float* sums = a.part + (long long)part * a.D * (W + 1);
#pragma unroll
  for (int k = 0; k < W; ++k) {  // in memory order
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int at = k * V + i;
      row[i] = at / W % 2 ? dw[at % W][at / W / 2].y : dw[at % W][at / W / 2].x;
    }
    store<float, V>(sums + (long long)d * W + k * V, row);
  }
  single<V>(db, row);
  store<float, V>(sums + (long long)a.D * W + d, row);
}

int check(const haste_b200_causal_conv1d& a, bool backward) {
  HB_REQUIRE(storage_dtype(a.dtype), "dtype");
  HB_REQUIRE(a.param_dtype == HASTE_B200_F32 || a.param_dtype == a.dtype, "param_dtype");
  HB_REQUIRE(a.T >= 0 && a.T <= (1 << 30) && a.N >= 0 && a.D >= 0, "T,N,D");
  HB_REQUIRE(a.W >= 2 && a.W <= 4, "W must be 2, 3 or 4");
  HB_REQUIRE((long long)a.D * (a.W + 1) < (1LL << 31), "D");
  for (const haste_b200_sequence* q : {&a.x, &a.y, &a.dy, &a.dx})
    HB_REQUIRE(strides_fit(a.T, *q), "a step's stride must be below 2^31 elements");
  if (a.N == 0 || a.D == 0) return HASTE_B200_OK;
  HB_REQUIRE(a.weight, "null pointer");
  HB_REQUIRE(a.T == 0 || (a.x.data && (backward ? a.dy.data != nullptr : a.y.data != nullptr)), "null pointer");
  HB_REQUIRE(!backward || (a.dweight && a.scratch), "null pointer");
  HB_REQUIRE(!backward || aligned(a.scratch, 16), "scratch must be aligned to 16 bytes");
  return HASTE_B200_OK;
}

// Channels per thread: four, less where a width, a stride or a start forbids it.  (Eight 16-bit channels take
// 150 registers for their windows and taps, and too few threads are resident to fill the memory pipes.)
int width(const haste_b200_causal_conv1d& a, bool backward) {
  const int e = (int)dtype_size(a.dtype), f = (int)dtype_size(a.param_dtype);
  for (int v = 4; v > 1; v /= 2) {
    bool ok = a.D % v == 0 && aligned(a.weight, v * f) && aligned(a.x, e, v * e) && aligned(a.state, v * e) && aligned(a.final_state, v * e);
    ok &= backward ? aligned(a.dy, e, v * e) && aligned(a.dx, e, v * e) && aligned(a.dfinal_state, v * e) &&
                         aligned(a.dstate, v * e)
                   : aligned(a.y, e, v * e);
    if (ok) return v;
  }
  return 1;
}

struct Shape {
  int threads, dtiles, chunk, chunks, parts;
  Shape(const haste_b200_causal_conv1d& a, int v, bool backward) {
    const int lanes = ceil_div(a.D, v);
    threads = std::min(128, ceil_div(lanes, 32) * 32);
    dtiles = ceil_div(lanes, threads);
    // One wave: as many chunks as the resident blocks, of about 16 steps at least.  A chunk reads W - 1 steps twice.
    // fp32 T=400 N=64 D=1024, us forward / backward: chunks of 64 steps, 1.2 / 2 waves, 47 / 69; one wave 39 / 63.
    // (Blocks of 256 or 512 threads: 52 / 95, 54 / 200.)  How many blocks of 128 threads an SM holds follows from
    // the registers; with five and three for every variant, against these (us forward / backward): bf16, two taps,
    // 128 x 128 x 2048 34 / 70 and 34 / 56; bf16, three taps, 1000 x 64 x 1024 70 / 107 and 60 / 103; fp32, single
    // channels, three taps, 400 x 40 x 1001 47 / 95 and 36 / 75.
    const bool half = dtype_size(a.dtype) == 2;
    const int resident = backward ? (v < 4 ? (!half && v == 2 && a.W == 4 ? 4 : 5) : a.W == 2 || (half && a.W == 3) ? 4 : 3)
                                  : (v < 4 ? (half ? 5 : 9) : half && a.W < 4 ? 4 : 5);
    const int per = std::max(1, resident * sm_count() / dtiles);
    chunks = std::max(1, std::min(per / a.N, ceil_div(a.T, 16)));
    chunk = std::max(4, ceil_div(ceil_div(a.T, chunks), 4) * 4);
    chunks = std::max(1, ceil_div(a.T, chunk));
    // rows of partial sums in the backward pass; a block takes as many items as the next one
    const long long rounds = (items(a.N) + per - 1) / per;
    parts = (int)((items(a.N) + rounds - 1) / rounds);
  }
  long long items(int N) const { return (long long)chunks * N; }
};

template <typename T>
ConvArgs<T> pack(const haste_b200_causal_conv1d& a, const Shape& s) {
  ConvArgs<T> k;
  k.T_ = a.T; k.N = a.N; k.D = a.D; k.chunk = s.chunk; k.dtiles = s.dtiles;
  k.param_f32 = a.param_dtype == HASTE_B200_F32;
  k.silu = a.silu != 0;
  k.x = Seq<const T>(a.x); k.y = Seq<T>(a.y); k.dy = Seq<const T>(a.dy); k.dx = Seq<T>(a.dx);
  k.w = a.weight; k.b = a.bias;
  k.state = static_cast<const T*>(a.state);
  k.final_state = static_cast<T*>(a.final_state);
  k.lengths = a.lengths;
  k.dfinal = static_cast<const T*>(a.dfinal_state);
  k.dstate = static_cast<T*>(a.dstate);
  k.part = a.scratch;
  k.items = (int)s.items(a.N);
  k.parts = s.parts;
  return k;
}

template <typename T, int V, int W>
int launch(const haste_b200_causal_conv1d& a, bool backward, cudaStream_t st) {
  const Shape s(a, V, backward);
  HB_REQUIRE(s.items(a.N) * s.dtiles < (1LL << 31), "T*N too large");
  const ConvArgs<T> k = pack<T>(a, s);
  if (backward) {
    conv_bwd<T, V, W><<<k.parts * s.dtiles, s.threads, 0, st>>>(k);
  } else {
    conv_fwd<T, V, W><<<k.items * s.dtiles, s.threads, 0, st>>>(k);
  }
  HB_LAUNCH_OK();
  count_launch(1);
  if (!backward) return HASTE_B200_OK;
  SumJobs jobs;
  jobs.add(a.dweight, 0, 1, a.D * W, a.param_dtype);
  jobs.add(a.dbias, (long long)a.D * W, 1, a.D, a.param_dtype);
  return sum_parts(a.scratch, k.parts, (long long)a.D * (W + 1), jobs, st);
}

template <typename T, int V>
int by_taps(const haste_b200_causal_conv1d& a, bool backward, cudaStream_t s) {
  if (a.W == 4) return launch<T, V, 4>(a, backward, s);
  if (a.W == 3) return launch<T, V, 3>(a, backward, s);
  return launch<T, V, 2>(a, backward, s);
}

template <typename T>
int by_width(const haste_b200_causal_conv1d& a, bool backward, cudaStream_t s) {
  switch (width(a, backward)) {
    case 4: return by_taps<T, 4>(a, backward, s);
    case 2: return by_taps<T, 2>(a, backward, s);
    default: return by_taps<T, 1>(a, backward, s);
  }
}

int run(const haste_b200_causal_conv1d& a, bool backward, cudaStream_t s) {
  HB_TRY(check(a, backward));
  if (a.N == 0 || a.D == 0) return HASTE_B200_OK;
  if (a.dtype == HASTE_B200_F32) return by_width<float>(a, backward, s);
  if (a.dtype == HASTE_B200_BF16) return by_width<__nv_bfloat16>(a, backward, s);
  return by_width<__half>(a, backward, s);
}

}  // namespace

int causal_conv1d_forward(const haste_b200_causal_conv1d& a, cudaStream_t s) {
  ProfScope p(PH_OTHER, s);
  return run(a, false, s);
}
int causal_conv1d_backward(const haste_b200_causal_conv1d& a, cudaStream_t s) {
  ProfScope p(PH_OTHER, s);
  return run(a, true, s);
}
long long causal_conv1d_scratch(const haste_b200_causal_conv1d& a) {
  // (enough for every width: the pointers that decide on it may not be there yet)
  if (a.N <= 0 || a.D <= 0 || a.T < 0) return 0;
  long long rows = 0;
  for (int v = 1; v <= 4; v *= 2) rows = std::max(rows, (long long)Shape(a, v, true).parts);
  return rows * a.D * (a.W + 1);
}

}  // namespace hb
