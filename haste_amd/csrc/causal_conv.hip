// Short causal convolution over time, one filter per channel, with its input state:
//   X = [state; x],  pre[t] = bias + sum_k kernel[k] X[t+k],  y = pre sigmoid(pre)  or  pre,
//   state_out = X[length .. length+W-2]
// and its backward pass
//   dpre = dy silu'(pre),  dX[p] = sum_k kernel[k] dpre[p-k]  (+ dstate_out[p-length]),
//   dkernel[k] = sum_{t,n} dpre[t] X[t+k],  dbias = sum dpre.
//
// Bound: HBM (forward 2, backward 3 values moved for about 2W and 6W operations).  A thread owns V
// channels of a batch row and walks a run of `chunk` steps with the last W inputs in
// registers, so that every input is read once, but for the W-1 before (backward: after) a run.
#include <type_traits>

#include "sequence.h"

namespace haste_hip {
namespace {

// Channels a thread owns.  Of half tensors that is a load of 8 bytes, where 16 would take so many registers that a SIMD
// has room for two wavefronts instead of four: forward and backward, W=4 bf16, T=1024 N=8 D=1024 41 us instead of 36 (forward 11.7 and
// 10.7), T=2048 D=4096 178 and 170.
constexpr int V = 4;

// Steps whose elements a thread fetches while those before them are computed.  Two backward, where they are of two tensors:
// with four a SIMD has room for three wavefronts instead of four (T=2048 N=8 D=4096 W=4 bf16: 126 us instead of 104).
constexpr int kForwardAhead = 4, kBackwardAhead = 2;

struct ConvShape {
  int T, N, D, chunk;
  int silu;
};

// The channels of thread `vector` of a row.  The last one's are the row's last V, some of them also its neighbour's: both
// compute and write the same, and no thread has channels beyond the row.  Not where a thread might read what its neighbour has
// written: a state in place.
__device__ __forceinline__ int first_channel(unsigned vector, int D, bool overlap) {
  const int c = (int)vector * V;
  return overlap && D >= V ? min(c, D - V) : c;
}

// X[p] for p >= 0: the state's rows, then the sequence.
template <typename T>
__device__ __forceinline__ void load_padded(const Rows<const T>& x, const T* state, int W, int p, int n, int c,
                                            int N, int D, float (&f)[V]) {
  if (p >= W - 1) {
    load_channels<V>(x.at(p - (W - 1), n), c, D, f);
  } else if (state != nullptr) {
    load_channels<V>(state + ((size_t)p * N + n) * D, c, D, f);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = 0.f;
  }
}

// V channels of U steps, packed in the tensor's own type until they are worked on.
template <typename T, int U>
struct HeldSteps {
  typedef T packed_t __attribute__((ext_vector_type(V)));
  packed_t v[U];
  __device__ __forceinline__ void load(const Rows<const T>& rows, int t, int end, int n, int c, int D) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u] = t + u < end ? load_packed<V>(rows.at(t + u, n), c, D) : packed_t{};
    }
  }
  __device__ __forceinline__ void get(int u, float (&f)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = (float)v[u][i];
  }
};
template <typename T, int W>
__global__ __launch_bounds__(256)
void causal_conv_forward_kernel(ConvShape s, Rows<const T> x, const float* __restrict__ kernel,
                                const float* __restrict__ bias, const T* state, const long long* __restrict__ lengths,
                                T* __restrict__ y, T* state_out) {
  const int T_ = s.T, N = s.N, D = s.D;
  const unsigned vectors = (D + V - 1) / V;
  const unsigned item = blockIdx.x * 256 + threadIdx.x, n = item / vectors;
  if (n >= (unsigned)N) return;
  const int c = first_channel(item % vectors, D, state_out == nullptr || state_out != state);
  const int t0 = blockIdx.y * s.chunk, t1 = min(T_, t0 + s.chunk);
  const Extent e = extent_of(lengths, n, T_);
  const int end = min(t1, e.steps);
  const Rows<T> out = packed_rows(y, N, D);

  // Everything the run starts from is requested before the first use of any of it.
  float w[W][V], b[V];
#pragma unroll
  for (int k = 0; k < W; ++k) load_channels<V>(kernel + (size_t)k * D, c, D, w[k]);
#pragma unroll
  for (int v = 0; v < V; ++v) b[v] = 0.f;
  if (bias != nullptr) load_channels<V>(bias, c, D, b);
  HeldSteps<T, kForwardAhead> coming;
  coming.load(x, t0, end, n, c, D);
  float win[W][V];  // X[t .. t+W-1], the last of them filled in by every step
  if (t0 < end) {
#pragma unroll
    for (int j = 0; j + 1 < W; ++j) load_padded(x, state, W, t0 + j, n, c, N, D, win[j]);
  }
  if (blockIdx.y == 0 && state_out != nullptr) {
    // read before any of it is written: state_out may be state (no other thread reads these: a run
    // that is not the first starts W-1 steps or more behind the state)
    float last[W > 1 ? W - 1 : 1][V];
#pragma unroll
    for (int j = 0; j + 1 < W; ++j) load_padded(x, state, W, e.steps + j, n, c, N, D, last[j]);
#pragma unroll
    for (int j = 0; j + 1 < W; ++j) {
      if (e.fill != 0.f) {  // NaN
#pragma unroll
        for (int v = 0; v < V; ++v) last[j][v] = e.fill;
      }
      store_channels<V>(state_out + ((size_t)j * N + n) * D, c, D, last[j]);
    }
  }
  if (t0 < end) {
    auto step = [&](int t) {
      float o[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float pre = b[v];
#pragma unroll
        for (int k = 0; k < W; ++k) pre += w[k][v] * win[k][v];
        o[v] = s.silu ? pre * sigmoid_of(pre) : pre;
      }
      store_channels<V>(out.at(t, n), c, D, o);
#pragma unroll
      for (int k = 0; k + 1 < W; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) win[k][v] = win[k + 1][v];
    };
    constexpr int U = kForwardAhead;
    for (int t = t0; t < end; t += U) {
      const HeldSteps<T, U> now = coming;
      if (t + U < end) coming.load(x, t + U, end, n, c, D);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        now.get(u, win[W - 1]);
        if (t + u < end) step(t + u);
      }
    }
  }
  float fill[V];
#pragma unroll
  for (int v = 0; v < V; ++v) fill[v] = e.fill;
  for (int t = max(t0, end); t < t1; ++t) store_channels<V>(out.at(t, n), c, D, fill);
}

// A run computes dX for the steps t0 .. t1-1 of x (the first also for the state): dpre of step t goes
// into dX[t .. t+W-1], so it needs dpre of W-1 steps behind the run too.  Step t finishes dX[t].
template <typename T, int W>
__global__ __launch_bounds__(256)
void causal_conv_backward_kernel(ConvShape s, Rows<const T> x, const float* __restrict__ kernel,
                                 const float* __restrict__ bias, const T* __restrict__ state,
                                 const long long* __restrict__ lengths, Rows<const T> dy,
                                 const T* __restrict__ dstate_out, T* __restrict__ dx, T* __restrict__ dstate,
                                 float* __restrict__ partial) {
  const int T_ = s.T, N = s.N, D = s.D;
  const unsigned vectors = (D + V - 1) / V;
  const unsigned item = blockIdx.x * 256 + threadIdx.x, n = item / vectors;
  if (n >= (unsigned)N) return;
  const int c = first_channel(item % vectors, D, true);
  const int t0 = blockIdx.y * s.chunk, t1 = min(T_, t0 + s.chunk);
  const Extent e = extent_of(lengths, n, T_);
  const int own = min(t1, e.steps);                // dpre of steps below it counts towards dkernel here
  const int given = min(e.steps, t1 + W - 1);      // dpre of steps at and behind it is 0, or not needed
  const Rows<T> out = packed_rows(dx, N, D);

  float w[W][V], b[V], dw[W][V], db[V];
#pragma unroll
  for (int k = 0; k < W; ++k) {
    load_channels<V>(kernel + (size_t)k * D, c, D, w[k]);
#pragma unroll
    for (int v = 0; v < V; ++v) dw[k][v] = 0.f;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) b[v] = db[v] = 0.f;
  if (bias != nullptr) load_channels<V>(bias, c, D, b);

  float win[W][V], acc[W][V];  // X[t .. t+W-1]; dX[t .. t+W-1] so far
#pragma unroll
  for (int k = 0; k < W; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v) win[k][v] = acc[k][v] = 0.f;
  if (t0 < given) {
#pragma unroll
    for (int j = 0; j + 1 < W; ++j) load_padded(x, state, W, t0 + j, n, c, N, D, win[j]);
  }
  auto emit = [&](int t) {  // dX[t] is complete: row t of the state, or step t-(W-1) of x
    float o[V];
    const int beyond = t - e.steps;
    if (dstate_out != nullptr && beyond >= 0 && beyond < W - 1 && e.fill == 0.f)
      load_channels<V>(dstate_out + ((size_t)beyond * N + n) * D, c, D, o);
    else {
#pragma unroll
      for (int v = 0; v < V; ++v) o[v] = e.fill;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] += acc[0][v];
    if (t >= W - 1) {
      const int to = t - (W - 1);
      if (to >= t0) store_channels<V>(out.at(to, n), c, D, o);
    } else if (t0 == 0 && dstate != nullptr) {
      store_channels<V>(dstate + ((size_t)t * N + n) * D, c, D, o);
    }
  };
  auto shift = [&] {
#pragma unroll
    for (int k = 0; k < W; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (k + 1 < W) win[k][v] = win[k + 1][v];
        acc[k][v] = k + 1 < W ? acc[k + 1][v] : 0.f;
      }
  };
  auto step = [&](int t, const float (&in)[V], const float (&g)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      win[W - 1][v] = in[v];
      float d = g[v];
      if (s.silu) {
        float pre = b[v];
#pragma unroll
        for (int k = 0; k < W; ++k) pre += w[k][v] * win[k][v];
        d *= silu_slope(pre, sigmoid_of(pre));
      }
#pragma unroll
      for (int k = 0; k < W; ++k) acc[k][v] += w[k][v] * d;
      const float mine = t < own ? d : 0.f;
      db[v] += mine;
#pragma unroll
      for (int k = 0; k < W; ++k) dw[k][v] += mine * win[k][v];
    }
    emit(t);
    shift();
  };
  constexpr int U = kBackwardAhead;
  HeldSteps<T, U> x_coming, dy_coming;
  x_coming.load(x, t0, given, n, c, D);
  dy_coming.load(dy, t0, given, n, c, D);
  int t = t0;
  for (; t < given; t += U) {
    const HeldSteps<T, U> x_now = x_coming, dy_now = dy_coming;
    if (t + U < given) {
      x_coming.load(x, t + U, given, n, c, D);
      dy_coming.load(dy, t + U, given, n, c, D);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float in[V], g[V];
      x_now.get(u, in);
      dy_now.get(u, g);
      if (t + u < given) step(t + u, in, g);
    }
  }
  t = max(t0, given);
  for (; t < t1 + W - 1; ++t) {
    emit(t);
    shift();
  }
  // partial[run][row][kernel, bias][D]
  float* mine = partial + ((size_t)blockIdx.y * N + n) * (W + 1) * D;
#pragma unroll
  for (int k = 0; k < W; ++k) store_channels<V>(mine + (size_t)k * D, c, D, dw[k]);
  store_channels<V>(mine + (size_t)W * D, c, D, db);
}

// Threads that a run of every row takes.
size_t items_of(int N, int D) { return (size_t)N * ((D + V - 1) / V); }

// Steps in a run: 64, and down to 8 (the W-1 steps read twice must stay few) where that leaves fewer
// than two wavefronts a SIMD.
int run_length(int T, size_t items) {
  int chunk = 64;
  while (chunk > 8 && items * ((T + chunk - 1) / chunk) < (size_t)device_cu_count() * 4 * 2 * 64) chunk /= 2;
  while ((size_t)(T + chunk - 1) / chunk > kGridLimitYZ) chunk *= 2;
  return chunk;
}

// Floats of workspace a backward pass needs: the runs' partials [parts][columns], and what adding them takes.
struct ConvPartials {
  size_t parts, columns, floats, total;
};
ConvPartials partials_of(int T, int N, int D, int W) {
  ConvPartials p;
  const size_t chunk = run_length(T, items_of(N, D));
  p.parts = (T + chunk - 1) / chunk * N;
  p.columns = (size_t)(W + 1) * D;
  p.floats = p.parts * p.columns;
  p.total = p.floats + column_sums_scratch(p.parts, p.columns);
  return p;
}

template <typename T, int W>
int forward(hipStream_t stream, ConvShape s, const Rows<const T>& x, const float* kernel, const float* bias, const T* state,
            const long long* lengths, T* y, T* state_out) {
  const size_t items = items_of(s.N, s.D), blocks = (items + 255) / 256;
  s.chunk = run_length(s.T, items);
  ScopedKernelTimer timer("causal_conv_forward", stream);
  dim3 grid((unsigned)blocks, (s.T + s.chunk - 1) / s.chunk);
  causal_conv_forward_kernel<T, W><<<grid, 256, 0, stream>>>(s, x, kernel, bias, state, lengths, y, state_out);
  HASTE_HIP_TRY(hipGetLastError());
  return HASTE_HIP_OK;
}

template <typename T, int W>
int backward(hipStream_t stream, ConvShape s, const Rows<const T>& x, const float* kernel, const float* bias, const T* state,
             const long long* lengths, const Rows<const T>& dy, const T* dstate_out, T* dx, float* dkernel,
             float* dbias, T* dstate, float* workspace, size_t workspace_bytes) {
  const size_t items = items_of(s.N, s.D), blocks = (items + 255) / 256;
  s.chunk = run_length(s.T, items);
  const ConvPartials p = partials_of(s.T, s.N, s.D, W);
  if (workspace_bytes < p.total * sizeof(float)) return too_large("causal_conv_backward: the workspace is too small");
  {
    ScopedKernelTimer timer("causal_conv_backward", stream);
    dim3 grid((unsigned)blocks, (s.T + s.chunk - 1) / s.chunk);
    causal_conv_backward_kernel<T, W><<<grid, 256, 0, stream>>>(s, x, kernel, bias, state, lengths, dy, dstate_out, dx,
                                                                   dstate, workspace);
    HASTE_HIP_TRY(hipGetLastError());
  }
  const ColumnOutputs to = {{dkernel, dbias, nullptr, nullptr}, {(size_t)W * s.D, p.columns, p.columns, p.columns}};
  return column_sums(stream, p.parts, p.columns, workspace, workspace + p.floats, to);
}

constexpr int kMaxWidth = 8;

template <typename F>
int with_width(int W, F&& f) {
  switch (W) {
    case 1: return f(std::integral_constant<int, 1>());
    case 2: return f(std::integral_constant<int, 2>());
    case 3: return f(std::integral_constant<int, 3>());
    case 4: return f(std::integral_constant<int, 4>());
    case 5: return f(std::integral_constant<int, 5>());
    case 6: return f(std::integral_constant<int, 6>());
    case 7: return f(std::integral_constant<int, 7>());
    case 8: return f(std::integral_constant<int, 8>());
  }
  return too_large("causal_conv: kernels of up to 8 steps are implemented");
}

bool sizes_ok(int T, int N, int D, int W) { return T > 0 && N > 0 && D > 0 && W > 0; }
// For the calls and for the size of their workspace alike.
int check_limits(int T, int N, int D) {
  if (T > kSizeLimit || N > kSizeLimit || D > kSizeLimit / kMaxWidth) return too_large("causal_conv: sizes beyond 2^30");
  if ((items_of(N, D) + 255) / 256 > kGridLimit) return too_large("causal_conv: too many rows of channels");
  return HASTE_HIP_OK;
}

template <typename T>
int forward_entry(int steps, int batch_size, int channels, int width, const void* x, size_t x_step, size_t x_row,
                  const float* kernel, const float* bias, int silu, const void* state, const void* lengths, void* y,
                  void* state_out, void* stream) {
  HASTE_HIP_REQUIRE(sizes_ok(steps, batch_size, channels, width));
  HASTE_HIP_REQUIRE(x && kernel && y);
  HASTE_HIP_PROPAGATE(check_limits(steps, batch_size, channels));
  return with_width(width, [&](auto w) {
    return forward<T, w()>(as_stream(stream), {steps, batch_size, channels, 0, silu}, {static_cast<const T*>(x), x_step, x_row},
                           kernel, bias, static_cast<const T*>(state), static_cast<const long long*>(lengths),
                           static_cast<T*>(y), static_cast<T*>(state_out));
  });
}

template <typename T>
int backward_entry(int steps, int batch_size, int channels, int width, const void* x, size_t x_step, size_t x_row,
                   const float* kernel, const float* bias, int silu, const void* state, const void* lengths, const void* dy,
                   size_t dy_step, size_t dy_row, const void* dstate_out, void* dx, float* dkernel, float* dbias,
                   void* dstate, void* workspace, size_t workspace_bytes, void* stream) {
  HASTE_HIP_REQUIRE(sizes_ok(steps, batch_size, channels, width));
  HASTE_HIP_REQUIRE(x && kernel && dy && dx && dkernel && workspace);
  HASTE_HIP_PROPAGATE(check_limits(steps, batch_size, channels));
  return with_width(width, [&](auto w) {
    return backward<T, w()>(as_stream(stream), {steps, batch_size, channels, 0, silu},
                            {static_cast<const T*>(x), x_step, x_row}, kernel, bias, static_cast<const T*>(state),
                            static_cast<const long long*>(lengths), {static_cast<const T*>(dy), dy_step, dy_row},
                            static_cast<const T*>(dstate_out), static_cast<T*>(dx), dkernel, dbias, static_cast<T*>(dstate),
                            static_cast<float*>(workspace), workspace_bytes);
  });
}

}  // namespace
}  // namespace haste_hip

extern "C" {

using namespace haste_hip;

size_t haste_hip_causal_conv_workspace_bytes(int steps, int batch_size, int channels, int width) {
  if (!sizes_ok(steps, batch_size, channels, width) || width > kMaxWidth) return 0;
  if (check_limits(steps, batch_size, channels) != HASTE_HIP_OK) return 0;
  return partials_of(steps, batch_size, channels, width).total * sizeof(float);
}

#define HASTE_HIP_CAUSAL_CONV(SUFFIX, T)                                                                               \
  int haste_hip_causal_conv_forward_##SUFFIX(int steps, int batch_size, int channels, int width, const void* x,       \
                                             size_t x_step, size_t x_row, const float* kernel, const float* bias,     \
                                             int silu, const void* state, const void* lengths, void* y,               \
                                             void* state_out, void* stream) {                                         \
    return forward_entry<T>(steps, batch_size, channels, width, x, x_step, x_row, kernel, bias, silu, state, lengths, y, \
                            state_out, stream);                                                                       \
  }                                                                                                                   \
  int haste_hip_causal_conv_backward_##SUFFIX(int steps, int batch_size, int channels, int width, const void* x,      \
                                              size_t x_step, size_t x_row, const float* kernel, const float* bias,    \
                                              int silu, const void* state, const void* lengths, const void* dy,       \
                                              size_t dy_step, size_t dy_row, const void* dstate_out, void* dx,        \
                                              float* dkernel, float* dbias, void* dstate, void* workspace,            \
                                              size_t workspace_bytes, void* stream) {                                 \
    return backward_entry<T>(steps, batch_size, channels, width, x, x_step, x_row, kernel, bias, silu, state, lengths, dy, \
                             dy_step, dy_row, dstate_out, dx, dkernel, dbias, dstate, workspace, workspace_bytes,     \
                             stream);                                                                                 \
  }

HASTE_HIP_CAUSAL_CONV(f32, float)
HASTE_HIP_CAUSAL_CONV(f16, _Float16)
HASTE_HIP_CAUSAL_CONV(bf16, __bf16)

}  // extern "C"
