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

// V elements in registers, a half type's two to a register.
template <typename T, int V>
struct Packed {
  typedef T type __attribute__((ext_vector_type(V)));
};

// Where a row ends within a thread's V channels (c < D < c + V), those of a half type are read as the V before the row's end and
// moved down, and written in pieces of 4, 2 and 1; an element at a time is a chain of conversions and waits: a norm and its gradient
// of rows of 1023 in bf16, 33 and 92 us against 42 and 124.  In float it is not: 31 and 104 an element at a time, 33 and 116 moved.
template <int V, typename T>
__device__ __forceinline__ typename Packed<T, V>::type load_tail(const T* row, int c, int D) {
  typename Packed<T, V>::type w = {};
  if constexpr (V > 1 && sizeof(T) == 2) {
    if (D >= V) {
      constexpr int WORDS = V / 2;
      unsigned u[WORDS];
      const typename Wide<T, V>::type last = *reinterpret_cast<const typename Wide<T, V>::type*>(row + D - V);
      __builtin_memcpy(u, &last, sizeof(u));
      const int down = c + V - D;
#pragma unroll
      for (int step = V / 2; step >= 2; step /= 2)
#pragma unroll
        for (int i = 0; i < WORDS; ++i) u[i] = !(down & step) ? u[i] : i + step / 2 < WORDS ? u[i + step / 2] : 0u;
#pragma unroll
      for (int i = 0; i < WORDS; ++i)
        u[i] = down & 1 ? __builtin_amdgcn_alignbit(i + 1 < WORDS ? u[i + 1] : 0u, u[i], 16) : u[i];
      __builtin_memcpy(&w, u, sizeof(u));
      return w;
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (c + v < D) w[v] = row[c + v];
  return w;
}

template <int V, typename T>
__device__ __forceinline__ void store_tail(T* row, int c, int D, const typename Packed<T, V>::type& w) {
  if constexpr (V > 1 && sizeof(T) == 2) {
    constexpr int WORDS = V / 2;
    unsigned u[WORDS];
    __builtin_memcpy(u, &w, sizeof(u));
    T* to = row + c;
    const int count = D - c;
#pragma unroll
    for (int step = V / 2; step >= 2; step /= 2) {
      if (count & step) {
        __builtin_memcpy(to, u, step * sizeof(T));
        to += step;
#pragma unroll
        for (int i = 0; i < WORDS; ++i) u[i] = i + step / 2 < WORDS ? u[i + step / 2] : 0u;
      }
    }
    if (count & 1) __builtin_memcpy(to, u, sizeof(T));
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (c + v < D) row[c + v] = w[v];
  }
}

// Channels c .. c+V-1 of a row of D, those beyond it 0.
template <int V, typename T>
__device__ __forceinline__ typename Packed<T, V>::type load_packed(const T* row, int c, int D) {
  typename Packed<T, V>::type w = {};
  if (c + V <= D) w = *reinterpret_cast<const typename Wide<T, V>::type*>(row + c);
  else if (c < D) w = load_tail<V>(row, c, D);
  return w;
}
template <int V, typename T>
__device__ __forceinline__ void load_channels(const T* row, int c, int D, float (&f)[V]) {
  const typename Packed<T, V>::type w = load_packed<V>(row, c, D);
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = (float)w[v];
}

template <int V, typename T>
__device__ __forceinline__ void store_channels(T* row, int c, int D, const float (&f)[V]) {
  typename Packed<T, V>::type w;
#pragma unroll
  for (int v = 0; v < V; ++v) w[v] = (T)f[v];
  if (c + V <= D) *reinterpret_cast<typename Wide<T, V>::type*>(row + c) = w;
  else if (c < D) store_tail<V>(row, c, D, w);
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
size_t column_sums_scratch(size_t parts, size_t columns);
int column_sums(hipStream_t stream, size_t parts, size_t columns, const float* partial, float* scratch,
                const ColumnOutputs& to);

constexpr size_t kGridLimit = (size_t(1) << 22) - 1;  // workgroups along x: threads along an axis are counted in 32 bits
constexpr size_t kGridLimitYZ = 65535;
constexpr int kSizeLimit = 1 << 30;  // steps, rows, channels: sums of a few of them stay below 2^31

inline int too_large(const char* text) {
  set_error_text(text);
  return HASTE_HIP_ERROR_UNSUPPORTED_SIZE;
}

}  // namespace haste_hip
