// Shared by the operators of a state space block (causal_conv.hip, selective_scan.hip,
// residual_norm.hip): element types, rows of channels, lengths, sums over lanes and over partials.
//
// Tensors are time-major [T,N,D]; what the operators read may have any strides between steps and
// between batch rows (column blocks of a projection, batch-first tensors), channels are contiguous.
// Activations are float, _Float16 or __bf16 and are widened to float as they are read; every sum,
// state and statistic is float, and a result is rounded once, as it is stored.
#pragma once

#include "common.h"

namespace haste_hip {

// A tensor [T,N,D]: the strides between steps and between rows, in elements.
template <typename T>
struct Rows {
  T* p;
  size_t step, row;
  __device__ __forceinline__ T* at(int t, int n) const { return p + (size_t)t * step + (size_t)n * row; }
};

template <typename T>
__host__ __device__ inline Rows<T> packed_rows(T* p, int N, int D) { return {p, (size_t)N * D, (size_t)D}; }

// V consecutive elements, loaded and stored by one instruction.  Rows may start anywhere: the type's
// alignment is the element's (a wide access needs no more on this hardware).
template <typename T, int V>
struct Wide {
  typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};

// Channels c .. c+V-1 of a row of D, those beyond it 0.
template <int V, typename T>
__device__ __forceinline__ void load_channels(const T* row, int c, int D, float (&f)[V]) {
  if (c + V <= D) {
    const typename Wide<T, V>::type w = *reinterpret_cast<const typename Wide<T, V>::type*>(row + c);
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = (float)w[v];
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = c + v < D ? (float)row[c + v] : 0.f;
  }
}

template <int V, typename T>
__device__ __forceinline__ void store_channels(T* row, int c, int D, const float (&f)[V]) {
  if (c + V <= D) {
    typename Wide<T, V>::type w;
#pragma unroll
    for (int v = 0; v < V; ++v) w[v] = (T)f[v];
    *reinterpret_cast<typename Wide<T, V>::type*>(row + c) = w;
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (c + v < D) row[c + v] = (T)f[v];
  }
}

// Steps of batch row n: all T, or lengths[n] of them, counted from the end when negative.  A length
// that names no step gives none, and NaNs (`fill`) where an empty row has zeros.
struct Extent {
  int steps;
  float fill;
};
__device__ __forceinline__ Extent extent_of(const long long* lengths, int n, int T) {
  if (lengths == nullptr) return {T, 0.f};
  long long l = lengths[n];
  if (l < 0) l += (long long)T + 1;
  if (l < 0 || l > T) return {0, __builtin_nanf("")};
  return {(int)l, 0.f};
}

// exp and sigmoid on the hardware exp2 and reciprocal (1 ulp each).
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ float sigmoid_of(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_of(-x)); }
// d/dx (x sigmoid(x)), s = sigmoid(x).
__device__ __forceinline__ float silu_slope(float x, float s) { return s * (1.0f + x * (1.0f - s)); }

// Adding across lanes: within rows of 16 by the data path's own permutations, across them by swaps.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kHalfMirror = 0x141, kRor4 = 0x124, kRor8 = 0x128;
__device__ __forceinline__ float swap_add_halves(float a, float b) {  // lower half: a's sum, upper: b's
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float swap_add_rows(float a, float b) {  // even rows: a's sum, odd: b's
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Sum over all 64 lanes, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
  v += dpp<kXor1>(v);
  v += dpp<kXor2>(v);
  v += dpp<kHalfMirror>(v);
  v += dpp<kRor8>(v);
  v = swap_add_rows(v, v);
  return swap_add_halves(v, v);
}

// Sums over p < parts of partial[p][columns]: partials of many workgroups, added in an order that depends
// on the sizes alone.  Columns below end[0] go to out[0], further ones below end[1] to out[1] and so on; a
// null output is left out.  `scratch` holds column_sums_scratch(parts, columns) floats.
struct ColumnOutputs {
  float* out[4];
  size_t end[4];
};
size_t column_sums_scratch(int parts, size_t columns);
int column_sums(hipStream_t stream, int parts, size_t columns, const float* partial, float* scratch,
                const ColumnOutputs& to);

constexpr size_t kGridLimit = (size_t(1) << 22) - 1;  // workgroups along x: threads along an axis are counted in 32 bits
constexpr size_t kGridLimitYZ = 65535;
constexpr int kSizeLimit = 1 << 30;  // steps, rows, channels: sums of a few of them stay below 2^31

inline int too_large(const char* text) {
  set_error_text(text);
  return HASTE_HIP_ERROR_UNSUPPORTED_SIZE;
}

}  // namespace haste_hip
