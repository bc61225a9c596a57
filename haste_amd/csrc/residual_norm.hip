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
  static __device__ __forceinline__ int column_of(int i, int thread) { return column(i / V, thread) + i % V; }
};

// They in the tensor's own type, as they are fetched a row ahead; those beyond the row 0.
template <typename T, int THREADS>
struct Held {
  typedef Share<T, THREADS> S;
  typedef T packed_t __attribute__((ext_vector_type(S::V)));
  packed_t v[S::kPieces];
  __device__ __forceinline__ void load(const T* row, int thread, int D) {
#pragma unroll
    for (int p = 0; p < S::kPieces; ++p) {
      v[p] = load_packed<S::V>(row, S::column(p, thread), D);
    }
  }
  __device__ __forceinline__ float get(int i) const { return (float)v[i / S::V][i % S::V]; }
};

template <typename T, int THREADS, typename U>
__device__ __forceinline__ void store_share(U* row, int thread, int D, const float (&f)[EACH]) {
  typedef Share<T, THREADS> S;
#pragma unroll
  for (int p = 0; p < S::kPieces; ++p) {
    float v[S::V];
#pragma unroll
    for (int i = 0; i < S::V; ++i) v[i] = f[p * S::V + i];
    store_channels<S::V>(row, S::column(p, thread), D, v);
  }
}

// A weight's elements, 0 beyond the row; a weight that is absent is `otherwise` everywhere.
template <typename T, int THREADS>
__device__ __forceinline__ void load_or(const float* weights, float otherwise, int thread, int D, float (&f)[EACH]) {
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int c = Share<T, THREADS>::column_of(i, thread);
    f[i] = weights == nullptr ? otherwise : c < D ? weights[c] : 0.f;
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
  auto inside = [&](int i) { return S::column_of(i, thread) < s.D; };
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

  struct Raw {
    Held<T, THREADS> update, gate, residual;
  } coming = {};
  const bool gated = in.gate.p != nullptr, added = in.residual.p != nullptr;
  const size_t stride = (size_t)gridDim.x * L::kRows;
  auto fetch = [&](size_t row) {
    if (row >= rows) return;
    const int t = (int)((unsigned)row / (unsigned)s.N), n = (int)((unsigned)row % (unsigned)s.N);
    coming.update.load(in.update.at(t, n), thread, s.D);
    if (gated) coming.gate.load(in.gate.at(t, n), thread, s.D);
    if (added) coming.residual.load(in.residual.at(t, n), thread, s.D);
  };
  fetch((size_t)blockIdx.x * L::kRows + group);
  // every thread of the workgroup takes part in all turns: there are barriers in them
  for (size_t first = (size_t)blockIdx.x * L::kRows; first < rows; first += stride) {
    const size_t row = first + group;
    const bool live = row < rows;
    float v[EACH], o[EACH];
    const Raw now = coming;
    fetch(row + stride);
#pragma unroll
    for (int i = 0; i < EACH; ++i) v[i] = now.update.get(i);
    float2 first_stats = make_float2(0.f, 1.f), second_stats = make_float2(0.f, 1.f);
    if (in.after != nullptr) first_stats = statistics<T, THREADS>(sums, v, s, thread);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      float p = (v[i] - first_stats.x) * first_stats.y * after[i] * scale[i];
      const float gate = now.gate.get(i), silu = gate * sigmoid_of(gate);
      p = gated ? p * silu : p;
      o[i] = added ? now.residual.get(i) + p : p;
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
  float* partial;               // [groups of rows][kSums, or kSums - 1 without dbias][D]
};

// BIAS: whether the gradient of before_bias is wanted; its sums would take registers.
template <typename T, int THREADS, bool BIAS>
__global__ __launch_bounds__(Launch<THREADS>::kBlock)
void residual_norm_backward_kernel(NormShape s, NormInputs<T> in, const float* __restrict__ stats, Rows<const T> dout,
                                   Rows<const T> dnormed, NormGradients<T> to) {
  typedef Launch<THREADS> L;
  typedef Share<T, THREADS> S;
  __shared__ float2 lds[L::kRows][2 * RowSums<THREADS>::kWaves];
  const int thread = threadIdx.x % THREADS, group = threadIdx.x / THREADS;
  RowSums<THREADS> sums = {lds[group], 0};
  const size_t rows = (size_t)s.T * s.N;
  // A workgroup of 1024 threads has 128 registers a thread: the sums over its rows lie in LDS, and rows are not fetched ahead.  It spills
  // 116 to 148 bytes a thread all the same, and takes twice its bytes' time: D=8192 T=512 N=8 bf16 219 us, D=4096 64.
  constexpr bool kAhead = THREADS < 1024;
  constexpr int kWanted = BIAS ? kSums : kSums - 1;
  __shared__ float sums_lds[kAhead ? 1 : kWanted][kAhead ? 1 : EACH][kAhead ? 1 : THREADS];
  float scale[EACH], after[EACH], before[EACH];
  load_or<T, THREADS>(in.scale, 1.f, thread, s.D, scale);
  load_or<T, THREADS>(in.after, 1.f, thread, s.D, after);
  load_or<T, THREADS>(in.before, 1.f, thread, s.D, before);
  float over_rows[kAhead ? kWanted : 1][EACH];  // dscale, dafter, dbefore, dbias
#pragma unroll
  for (int k = 0; k < kWanted; ++k)
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      if (kAhead) over_rows[kAhead ? k : 0][i] = 0.f;
      else sums_lds[kAhead ? 0 : k][kAhead ? 0 : i][kAhead ? 0 : thread] = 0.f;
    }
  auto add = [&](int k, int i, float v) {
    if (kAhead) over_rows[kAhead ? k : 0][i] += v;
    else sums_lds[kAhead ? 0 : k][kAhead ? 0 : i][kAhead ? 0 : thread] += v;
  };

  struct Raw {
    Held<T, THREADS> update, gate, residual, dout, dnormed;
    float4 stats;
  } coming = {};
  const bool gated = in.gate.p != nullptr, second = in.before != nullptr;
  const size_t stride = (size_t)gridDim.x * L::kRows;
  auto fetch = [&](size_t row) {
    if (row >= rows) {  // a turn whose row is not there adds nothing
      coming = {};
      return;
    }
    const int t = (int)((unsigned)row / (unsigned)s.N), n = (int)((unsigned)row % (unsigned)s.N);
    coming.update.load(in.update.at(t, n), thread, s.D);
    if (gated) coming.gate.load(in.gate.at(t, n), thread, s.D);
    if (in.residual.p != nullptr) coming.residual.load(in.residual.at(t, n), thread, s.D);
    if (dout.p != nullptr) coming.dout.load(dout.at(t, n), thread, s.D);
    if (dnormed.p != nullptr) coming.dnormed.load(dnormed.at(t, n), thread, s.D);
    coming.stats = reinterpret_cast<const float4*>(stats)[row];
  };
  if (kAhead) fetch((size_t)blockIdx.x * L::kRows + group);
  for (size_t first = (size_t)blockIdx.x * L::kRows; first < rows; first += stride) {
    const size_t row = first + group;
    const bool live = row < rows;
    if (!kAhead) fetch(row);
    const Raw now = coming;
    if (kAhead) fetch(row + stride);
    float u[EACH], sigmoid[EACH], o[EACH], d[EACH];
    float along = 0.f, mean = 0.f;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const float gate = now.gate.get(i);
      sigmoid[i] = sigmoid_of(gate);
      u[i] = (now.update.get(i) - now.stats.x) * now.stats.y;
      d[i] = now.dout.get(i);
      const float p = scale[i] * (u[i] * after[i]), e = now.dnormed.get(i);
      o[i] = (now.residual.get(i) + (gated ? p * (gate * sigmoid[i]) : p) - now.stats.z) * now.stats.w;
      add(2, i, e * o[i]);
      if (BIAS) add(3, i, e);
      along += e * before[i] * o[i];
      mean += e * before[i];
    }
    if (second) {
      sums(along, mean);
      along /= s.D;
      mean = s.centered ? mean / s.D : 0.f;
#pragma unroll
      for (int i = 0; i < EACH; ++i) d[i] += (now.dnormed.get(i) * before[i] - o[i] * along - mean) * now.stats.w;
    }
    if (live && to.residual != nullptr) store_share<T, THREADS>(to.residual + row * s.D, thread, s.D, d);
    along = mean = 0.f;
    float dgate[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const float gate = now.gate.get(i), silu = gated ? gate * sigmoid[i] : 1.f, n_i = u[i] * after[i];
      add(0, i, d[i] * (n_i * silu));
      const float ds = d[i] * scale[i];
      dgate[i] = ds * n_i * silu_slope(gate, sigmoid[i]);
      const float dn = ds * silu;
      add(1, i, dn * u[i]);
      d[i] = S::column_of(i, thread) < s.D ? dn * after[i] : 0.f;
      along += d[i] * u[i];
      mean += d[i];
    }
    if (live && to.gate != nullptr) store_share<T, THREADS>(to.gate + row * s.D, thread, s.D, dgate);
    if (in.after != nullptr) {
      sums(along, mean);
      along /= s.D;
      mean = s.centered ? mean / s.D : 0.f;
#pragma unroll
      for (int i = 0; i < EACH; ++i) d[i] = (d[i] - u[i] * along - mean) * now.stats.y;
    }
    if (live) store_share<T, THREADS>(to.update + row * s.D, thread, s.D, d);
  }
  float* partial = to.partial + ((size_t)blockIdx.x * L::kRows + group) * kWanted * s.D;
#pragma unroll
  for (int k = 0; k < kWanted; ++k) {
    float sum[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) sum[i] = kAhead ? over_rows[kAhead ? k : 0][i] : sums_lds[kAhead ? 0 : k][kAhead ? 0 : i][kAhead ? 0 : thread];
    store_share<T, THREADS>(partial + (size_t)k * s.D, thread, s.D, sum);
  }
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
constexpr int kForwardWaves = 4, kBackwardWaves = 2;

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
      const dim3 grid(workgroups((size_t)steps * batch_size, channels, kBackwardWaves)), block(Launch<threads()>::kBlock);
      if (dbias != nullptr)
        residual_norm_backward_kernel<T, threads(), true><<<grid, block, 0, as_stream(stream)>>>(s, in, stats, dout, dnormed, grads);
      else
        residual_norm_backward_kernel<T, threads(), false><<<grid, block, 0, as_stream(stream)>>>(s, in, stats, dout, dnormed, grads);
      HASTE_HIP_TRY(hipGetLastError());
      return HASTE_HIP_OK;
    }));
  }
  const size_t D = channels;
  const ColumnOutputs sums = {{dscale, dafter, dbefore, dbias}, {D, 2 * D, 3 * D, 4 * D}};
  return column_sums(as_stream(stream), p.parts, (dbias != nullptr ? kSums : kSums - 1) * D, grads.partial, grads.partial + p.floats, sums);
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
