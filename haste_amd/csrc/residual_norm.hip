// The norms around a block, its gate and its residual scale in one pass:
//   n = norm(update) after_weight,  out = residual + scale n silu(gate),
//   normed = norm(out) before_weight + before_bias
// (out leaves the block, normed enters the next one), each part of which may be absent, and the backward
// pass.  norm is v / sqrt(mean v^2 + eps), or that of v - mean v (centered).  With u, o the normed values
// before their weights, gated = n silu(gate) and 1/sigma their factors:
//   e = dnormed before_weight,  d = dout + (e - o mean(e o) [- mean e]) / sigma_out,
//   dresidual = d,  dscale = sum d gated,  dgate = d scale n silu'(gate),  dbefore = sum dnormed o,
//   f = d scale silu(gate) after_weight,  dupdate = (f - u mean(f u) [- mean f]) / sigma_update,
//   dafter = sum d scale silu(gate) u,  dbias = sum dnormed.
//
// Bound: HBM.  A row lies in the registers of THREADS threads, eight elements each, from its load to its
// last use; the weights, and backward the sums over rows, stay in registers while a workgroup goes
// through its rows.  The backward pass computes `out` again from what the forward pass read rather than
// reading its rounded values: the sums over rows then carry no rounding of them, for the same bytes.
#include <type_traits>

#include "sequence.h"

namespace haste_hip {
namespace {

constexpr int EACH = 8;          // elements of a thread
constexpr int kMaxChannels = 1024 * EACH;
constexpr int kSums = 4;         // dscale, dafter, dbefore, dbias

struct NormShape {
  int T, N, D;
  int centered;
  float eps;
};

template <typename T>
struct NormInputs {
  Rows<const T> update, residual, gate;                 // the latter two may have null pointers
  const float *scale, *after, *before, *before_bias;    // each may be null
};

// A thread's elements of a row: pieces of V neighbouring ones.
template <typename T, int THREADS>
struct Share {
  static constexpr int V = 16 / sizeof(T) < EACH ? 16 / sizeof(T) : EACH;
  static constexpr int kPieces = EACH / V;
  static __device__ __forceinline__ int column(int piece, int thread) { return (piece * THREADS + thread) * V; }
};

template <typename T, int THREADS, typename U>
__device__ __forceinline__ void load_share(const U* row, int thread, int D, float (&f)[EACH]) {
  typedef Share<T, THREADS> S;
#pragma unroll
  for (int p = 0; p < S::kPieces; ++p) {
    float v[S::V];
    const int c = S::column(p, thread);
    if (c < D) {
      load_channels<S::V>(row, c, D, v);
    } else {
#pragma unroll
      for (int i = 0; i < S::V; ++i) v[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < S::V; ++i) f[p * S::V + i] = v[i];
  }
}

template <typename T, int THREADS, typename U>
__device__ __forceinline__ void store_share(U* row, int thread, int D, const float (&f)[EACH]) {
  typedef Share<T, THREADS> S;
#pragma unroll
  for (int p = 0; p < S::kPieces; ++p) {
    float v[S::V];
#pragma unroll
    for (int i = 0; i < S::V; ++i) v[i] = f[p * S::V + i];
    const int c = S::column(p, thread);
    if (c < D) store_channels<S::V>(row, c, D, v);
  }
}

template <typename T, int THREADS>
__device__ __forceinline__ void load_or(const float* weights, float otherwise, int thread, int D, float (&f)[EACH]) {
  if (weights != nullptr) {
    load_share<T, THREADS>(weights, thread, D, f);
  } else {
#pragma unroll
    for (int i = 0; i < EACH; ++i) f[i] = otherwise;
  }
}

template <int THREADS, typename T>
__device__ __forceinline__ void load_or_zero(const Rows<const T>& rows, int t, int n, int thread, int D, float (&f)[EACH]) {
  if (rows.p != nullptr) {
    load_share<T, THREADS>(rows.at(t, n), thread, D, f);
  } else {
#pragma unroll
    for (int i = 0; i < EACH; ++i) f[i] = 0.f;
  }
}

// Sums of two values over the threads of a row.  Rows of more than one wavefront meet in LDS, in one of
// two places in turn, so that a sum needs one barrier.
template <int THREADS>
struct RowSums {
  static constexpr int kWaves = THREADS / 64;
  float2* lds;  // [2][kWaves] of this row
  int turn;
  __device__ __forceinline__ void operator()(float& a, float& b) {
    a = wave_sum(a);
    b = wave_sum(b);
    if (kWaves == 1) return;
    float2* place = lds + turn * kWaves;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) place[threadIdx.x / 64 % kWaves] = make_float2(a, b);
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      a += place[w].x;
      b += place[w].y;
    }
  }
};

// (mean, 1 / sigma) of a row's elements; mean 0 unless centered.  The squares are those of the centered
// values: the difference of two large sums would lose them.
template <typename T, int THREADS>
__device__ __forceinline__ float2 statistics(RowSums<THREADS>& sums, const float (&v)[EACH], const NormShape& s, int thread) {
  typedef Share<T, THREADS> S;
  float mean = 0.f, unused = 0.f;
  auto inside = [&](int i) { return S::column(i / S::V, thread) + i % S::V < s.D; };
  if (s.centered) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) mean += inside(i) ? v[i] : 0.f;
    sums(mean, unused);
    mean /= s.D;
  }
  float square = 0.f;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const float c = inside(i) ? v[i] - mean : 0.f;
    square += c * c;
  }
  sums(square, unused);
  return make_float2(mean, 1.0f / sqrtf(square / s.D + s.eps));
}

template <int THREADS>
struct Launch {
  static constexpr int kBlock = THREADS < 256 ? 256 : THREADS;
  static constexpr int kRows = kBlock / THREADS;  // rows a workgroup works on side by side
};

template <typename T, int THREADS>
__global__ __launch_bounds__(Launch<THREADS>::kBlock)
void residual_norm_forward_kernel(NormShape s, NormInputs<T> in, T* __restrict__ out, T* __restrict__ normed,
                                  float* __restrict__ stats) {
  typedef Launch<THREADS> L;
  __shared__ float2 lds[L::kRows][2 * RowSums<THREADS>::kWaves];
  const int thread = threadIdx.x % THREADS, group = threadIdx.x / THREADS;
  RowSums<THREADS> sums = {lds[group], 0};
  const size_t rows = (size_t)s.T * s.N;
  float scale[EACH], after[EACH], before[EACH], before_bias[EACH];
  load_or<T, THREADS>(in.scale, 1.f, thread, s.D, scale);
  load_or<T, THREADS>(in.after, 1.f, thread, s.D, after);
  load_or<T, THREADS>(in.before, 1.f, thread, s.D, before);
  load_or<T, THREADS>(in.before_bias, 0.f, thread, s.D, before_bias);

  // every thread of the workgroup takes part in all turns: there are barriers in them
  for (size_t first = (size_t)blockIdx.x * L::kRows; first < rows; first += (size_t)gridDim.x * L::kRows) {
    const size_t row = first + group;
    const bool live = row < rows;
    const int t = live ? (int)(row / s.N) : 0, n = live ? (int)(row % s.N) : 0;
    float v[EACH], gate[EACH], o[EACH];
    load_share<T, THREADS>(in.update.at(t, n), thread, s.D, v);
    if (in.gate.p != nullptr) load_share<T, THREADS>(in.gate.at(t, n), thread, s.D, gate);
    if (in.residual.p != nullptr) load_share<T, THREADS>(in.residual.at(t, n), thread, s.D, o);
    float2 first_stats = make_float2(0.f, 1.f), second_stats = make_float2(0.f, 1.f);
    if (in.after != nullptr) first_stats = statistics<T, THREADS>(sums, v, s, thread);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      float p = (v[i] - first_stats.x) * first_stats.y * after[i] * scale[i];
      if (in.gate.p != nullptr) p *= gate[i] * sigmoid_of(gate[i]);
      o[i] = in.residual.p != nullptr ? o[i] + p : p;
    }
    if (live) store_share<T, THREADS>(out + row * s.D, thread, s.D, o);
    if (in.before != nullptr) {
      second_stats = statistics<T, THREADS>(sums, o, s, thread);
#pragma unroll
      for (int i = 0; i < EACH; ++i) o[i] = (o[i] - second_stats.x) * second_stats.y * before[i] + before_bias[i];
      if (live) store_share<T, THREADS>(normed + row * s.D, thread, s.D, o);
    }
    if (live && thread == 0 && stats != nullptr)
      reinterpret_cast<float4*>(stats)[row] = make_float4(first_stats.x, first_stats.y, second_stats.x, second_stats.y);
  }
}

template <typename T>
struct NormGradients {
  T *update, *residual, *gate;  // the latter two may be null
  float* partial;               // [groups of rows][kSums][D]
};

template <typename T, int THREADS>
__global__ __launch_bounds__(Launch<THREADS>::kBlock)
void residual_norm_backward_kernel(NormShape s, NormInputs<T> in, const float* __restrict__ stats, Rows<const T> dout,
                                   Rows<const T> dnormed, NormGradients<T> to) {
  typedef Launch<THREADS> L;
  typedef Share<T, THREADS> S;
  __shared__ float2 lds[L::kRows][2 * RowSums<THREADS>::kWaves];
  const int thread = threadIdx.x % THREADS, group = threadIdx.x / THREADS;
  RowSums<THREADS> sums = {lds[group], 0};
  const size_t rows = (size_t)s.T * s.N;
  float scale[EACH], after[EACH], before[EACH];
  load_or<T, THREADS>(in.scale, 1.f, thread, s.D, scale);
  load_or<T, THREADS>(in.after, 1.f, thread, s.D, after);
  load_or<T, THREADS>(in.before, 1.f, thread, s.D, before);
  float dscale[EACH], dafter[EACH], dbefore[EACH], dbias[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) dscale[i] = dafter[i] = dbefore[i] = dbias[i] = 0.f;

  for (size_t first = (size_t)blockIdx.x * L::kRows; first < rows; first += (size_t)gridDim.x * L::kRows) {
    const size_t row = first + group;
    const bool live = row < rows;
    const int t = live ? (int)(row / s.N) : 0, n = live ? (int)(row % s.N) : 0;
    float u[EACH], gate[EACH], o[EACH], d[EACH], e[EACH];
    load_share<T, THREADS>(in.update.at(t, n), thread, s.D, u);
    if (in.gate.p != nullptr) load_share<T, THREADS>(in.gate.at(t, n), thread, s.D, gate);
    load_or_zero<THREADS>(in.residual, t, n, thread, s.D, o);
    load_or_zero<THREADS>(dout, t, n, thread, s.D, d);
    load_or_zero<THREADS>(dnormed, t, n, thread, s.D, e);
    const float4 st = live ? reinterpret_cast<const float4*>(stats)[row] : make_float4(0.f, 0.f, 0.f, 0.f);
    if (!live) {
#pragma unroll
      for (int i = 0; i < EACH; ++i) u[i] = o[i] = d[i] = e[i] = 0.f;
    }
    float silu[EACH];
    float along = 0.f, mean = 0.f;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      silu[i] = in.gate.p != nullptr ? gate[i] * sigmoid_of(gate[i]) : 1.f;
      u[i] = (u[i] - st.x) * st.y;
      if (in.before != nullptr) {
        o[i] = (o[i] + scale[i] * (u[i] * after[i] * silu[i]) - st.z) * st.w;
        dbefore[i] += e[i] * o[i];
        dbias[i] += e[i];
        e[i] *= before[i];
        along += e[i] * o[i];
        mean += e[i];
      }
    }
    if (in.before != nullptr) {
      sums(along, mean);
      along /= s.D;
      mean = s.centered ? mean / s.D : 0.f;
#pragma unroll
      for (int i = 0; i < EACH; ++i) d[i] += (e[i] - o[i] * along - mean) * st.w;
    }
    if (live && to.residual != nullptr) store_share<T, THREADS>(to.residual + row * s.D, thread, s.D, d);
    along = mean = 0.f;
    float dgate[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const bool inside = S::column(i / S::V, thread) + i % S::V < s.D;
      const float n_i = u[i] * after[i];
      dscale[i] += d[i] * (n_i * silu[i]);
      const float ds = d[i] * scale[i];
      if (in.gate.p != nullptr) dgate[i] = ds * n_i * silu_slope(gate[i], sigmoid_of(gate[i]));
      const float dn = ds * silu[i];
      dafter[i] += dn * u[i];
      d[i] = inside ? dn * after[i] : 0.f;
      along += d[i] * u[i];
      mean += d[i];
    }
    if (live && to.gate != nullptr) store_share<T, THREADS>(to.gate + row * s.D, thread, s.D, dgate);
    if (in.after != nullptr) {
      sums(along, mean);
      along /= s.D;
      mean = s.centered ? mean / s.D : 0.f;
#pragma unroll
      for (int i = 0; i < EACH; ++i) d[i] = (d[i] - u[i] * along - mean) * st.y;
    }
    if (live) store_share<T, THREADS>(to.update + row * s.D, thread, s.D, d);
  }
  float* partial = to.partial + ((size_t)blockIdx.x * L::kRows + group) * kSums * s.D;
  store_share<T, THREADS>(partial, thread, s.D, dscale);
  store_share<T, THREADS>(partial + s.D, thread, s.D, dafter);
  store_share<T, THREADS>(partial + 2 * (size_t)s.D, thread, s.D, dbefore);
  store_share<T, THREADS>(partial + 3 * (size_t)s.D, thread, s.D, dbias);
}

// Threads of a row of D: the least power of two that holds it, a wavefront or more.
int threads_for(int D) {
  int threads = 64;
  while (threads * EACH < D) threads *= 2;
  return threads;
}

template <typename F>
int with_threads(int D, F&& f) {
  switch (threads_for(D)) {
    case 64: return f(std::integral_constant<int, 64>());
    case 128: return f(std::integral_constant<int, 128>());
    case 256: return f(std::integral_constant<int, 256>());
    case 512: return f(std::integral_constant<int, 512>());
    default: return f(std::integral_constant<int, 1024>());
  }
}

// Workgroups: enough to fill the chip `waves` wavefronts a SIMD deep, which then go through the rows.
int workgroups(size_t rows, int D, int waves) {
  const int threads = threads_for(D), block = threads < 256 ? 256 : threads;
  const size_t wanted = (size_t)device_cu_count() * 4 * waves * 64 / block;
  const size_t most = (rows + block / threads - 1) / (block / threads);
  return (int)(wanted > 0 && wanted < most ? wanted : most < kGridLimit ? most : kGridLimit);
}
constexpr int kForwardWaves = 8, kBackwardWaves = 4;

struct NormPartials {
  int parts;
  size_t columns, floats, total;
};
NormPartials partials_of(int T, int N, int D) {
  NormPartials p;
  const int threads = threads_for(D), block = threads < 256 ? 256 : threads;
  p.parts = workgroups((size_t)T * N, D, kBackwardWaves) * (block / threads);
  p.columns = (size_t)kSums * D;
  p.floats = p.parts * p.columns;
  p.total = p.floats + column_sums_scratch(p.parts, p.columns);
  return p;
}

int check_sizes(int T, int N, int D) {
  HASTE_HIP_REQUIRE(T > 0 && N > 0 && D > 0);
  if (D > kMaxChannels) return too_large("residual_norm: rows of up to 8192 channels are implemented");
  if (T > kSizeLimit || N > kSizeLimit || (size_t)T * N > (size_t)kSizeLimit) return too_large("residual_norm: more than 2^30 rows");
  return HASTE_HIP_OK;
}

template <typename T>
int forward_entry(int steps, int batch_size, int channels, const NormInputs<T>& in, int centered, float eps, T* out, T* normed,
                  float* stats, void* stream) {
  HASTE_HIP_PROPAGATE(check_sizes(steps, batch_size, channels));
  HASTE_HIP_REQUIRE(in.update.p && out);
  HASTE_HIP_REQUIRE((in.before != nullptr) == (normed != nullptr) && (in.before != nullptr || in.before_bias == nullptr));
  const NormShape s = {steps, batch_size, channels, centered, eps};
  ScopedKernelTimer timer("residual_norm_forward", as_stream(stream));
  return with_threads(channels, [&](auto threads) {
    residual_norm_forward_kernel<T, threads()><<<workgroups((size_t)steps * batch_size, channels, kForwardWaves),
                                                 Launch<threads()>::kBlock, 0, as_stream(stream)>>>(s, in, out, normed, stats);
    HASTE_HIP_TRY(hipGetLastError());
    return HASTE_HIP_OK;
  });
}

template <typename T>
int backward_entry(int steps, int batch_size, int channels, const NormInputs<T>& in, int centered, const float* stats,
                   const Rows<const T>& dout, const Rows<const T>& dnormed, const NormGradients<T>& grads, float* dscale,
                   float* dafter, float* dbefore, float* dbias, size_t workspace_bytes, void* stream) {
  HASTE_HIP_PROPAGATE(check_sizes(steps, batch_size, channels));
  HASTE_HIP_REQUIRE(in.update.p && stats && grads.update && grads.partial);
  HASTE_HIP_REQUIRE(in.before != nullptr || dnormed.p == nullptr);
  const NormPartials p = partials_of(steps, batch_size, channels);
  if (workspace_bytes < p.total * sizeof(float)) return too_large("residual_norm_backward: the workspace is too small");
  const NormShape s = {steps, batch_size, channels, centered, 0.f};
  {
    ScopedKernelTimer timer("residual_norm_backward", as_stream(stream));
    HASTE_HIP_PROPAGATE(with_threads(channels, [&](auto threads) {
      residual_norm_backward_kernel<T, threads()><<<workgroups((size_t)steps * batch_size, channels, kBackwardWaves),
                                                    Launch<threads()>::kBlock, 0, as_stream(stream)>>>(s, in, stats, dout, dnormed, grads);
      HASTE_HIP_TRY(hipGetLastError());
      return HASTE_HIP_OK;
    }));
  }
  const size_t D = channels;
  const ColumnOutputs sums = {{dscale, dafter, dbefore, dbias}, {D, 2 * D, 3 * D, 4 * D}};
  return column_sums(as_stream(stream), p.parts, p.columns, grads.partial, grads.partial + p.floats, sums);
}

}  // namespace
}  // namespace haste_hip

extern "C" {

using namespace haste_hip;

size_t haste_hip_residual_norm_workspace_bytes(int steps, int batch_size, int channels) {
  if (check_sizes(steps, batch_size, channels) != HASTE_HIP_OK) return 0;
  return partials_of(steps, batch_size, channels).total * sizeof(float);
}

#define HASTE_HIP_NORM_INPUTS                                                                                         \
  const void *update, size_t update_step, size_t update_row, const void *residual, size_t residual_step,              \
      size_t residual_row, const void *gate, size_t gate_step, size_t gate_row, const float *scale,                   \
      const float *after_weight, const float *before_weight
#define HASTE_HIP_NORM_IN(T, BIAS)                                                                                    \
  NormInputs<T>{{static_cast<const T*>(update), update_step, update_row},                                             \
                {static_cast<const T*>(residual), residual_step, residual_row},                                       \
                {static_cast<const T*>(gate), gate_step, gate_row}, scale, after_weight, before_weight, BIAS}

#define HASTE_HIP_RESIDUAL_NORM(SUFFIX, T)                                                                            \
  int haste_hip_residual_norm_forward_##SUFFIX(int steps, int batch_size, int channels, HASTE_HIP_NORM_INPUTS,        \
                                               const float* before_bias, int centered, float eps, void* out,          \
                                               void* normed, float* stats, void* stream) {                            \
    return forward_entry<T>(steps, batch_size, channels, HASTE_HIP_NORM_IN(T, before_bias), centered, eps,            \
                            static_cast<T*>(out), static_cast<T*>(normed), stats, stream);                            \
  }                                                                                                                   \
  int haste_hip_residual_norm_backward_##SUFFIX(                                                                      \
      int steps, int batch_size, int channels, HASTE_HIP_NORM_INPUTS, int centered, const float* stats,               \
      const void* dout, size_t dout_step, size_t dout_row, const void* dnormed, size_t dnormed_step,                  \
      size_t dnormed_row, void* dupdate, void* dresidual, void* dgate, float* dscale, float* dafter_weight,           \
      float* dbefore_weight, float* dbefore_bias, void* workspace, size_t workspace_bytes, void* stream) {            \
    return backward_entry<T>(steps, batch_size, channels, HASTE_HIP_NORM_IN(T, nullptr), centered, stats,             \
                             {static_cast<const T*>(dout), dout_step, dout_row},                                      \
                             {static_cast<const T*>(dnormed), dnormed_step, dnormed_row},                             \
                             {static_cast<T*>(dupdate), static_cast<T*>(dresidual), static_cast<T*>(dgate),           \
                              static_cast<float*>(workspace)},                                                        \
                             dscale, dafter_weight, dbefore_weight, dbefore_bias, workspace_bytes, stream);           \
  }

HASTE_HIP_RESIDUAL_NORM(f32, float)
HASTE_HIP_RESIDUAL_NORM(f16, _Float16)
HASTE_HIP_RESIDUAL_NORM(bf16, __bf16)

}  // extern "C"
