// The global norm of many gradients, and their clipping by it: norm = sqrt(sum of g^2 over all elements of all tensors),
//   out = g min(1, max_norm / (norm + 1e-6)).
//
// Bound: HBM, twice the gradients in (the norm comes first) and once out; where they fit the last-level cache the second reading is
// cheap.  Tensors are cut into chunks of kChunk bytes; a workgroup takes chunks in turn, so that many small tensors and
// few large ones fill the device alike.  Where tensors lie is an argument of the kernels (kTensors to a launch): nothing is copied to the
// device, and a captured launch keeps it.  Squares are added in double, a lane's, a workgroup's and all: no gradient in float or half overflows
// or vanishes by being squared, and an element costs two operations at a rate that the memory does not reach (those of doubles do from 1.4e154 on
// and below 1.5e-162: the norm is infinite, or is without them).  Sums are parked per workgroup and added in order.
//
// The gradients are scaled from the last chunk to the first, and neither they nor the results are kept in the caches any more: what the norm
// read last is then still in the last-level cache.  us, forwards / backwards / and so: 537 million gradients (1.07 GB) 611 / 608 / 560, 67
// million in bf16 (134 MB) 84 / 84 / 69.
//
// Where nothing is to be clipped the factor is 1, and what lies in place is left alone.
#include <algorithm>
#include <type_traits>
#include <vector>

#include "sequence.h"

namespace haste_hip {
namespace {

constexpr int kTensors = 112;            // of a launch: 32 bytes each, beside the rest below the 4 KiB of arguments
constexpr int kFewTensors = 12;          // of a short one, whose arguments are sooner on the device
constexpr size_t kChunk = 32768;         // bytes of a tensor that a workgroup takes at a time
constexpr int kThreads = 256;

enum { kF32, kF16, kBF16, kF64 };
constexpr int kSize[] = {4, 2, 2, 8};

template <int MOST>
struct Tensors {
  const void* in[MOST];
  void* out[MOST];
  size_t count[MOST];                    // elements
  unsigned first[MOST];                  // chunks before the tensor's
  unsigned char type[MOST];
  int tensors;
  unsigned chunks;
};

// Runs f(type's zero, elements of the chunk, where it starts) for this workgroup's chunks.
// BACK: from the last.
template <bool BACK, int MOST, class F>
__device__ __forceinline__ void for_chunks(const Tensors<MOST>& list, F f) {
  for (unsigned turn = blockIdx.x; turn < list.chunks; turn += gridDim.x) {
    const unsigned chunk = BACK ? list.chunks - 1 - turn : turn;
    int low = 0, high = list.tensors - 1;  // the last tensor whose chunks start at or before this one
    while (low < high) {
      const int middle = (low + high + 1) / 2;
      if (list.first[middle] <= chunk) low = middle;
      else high = middle - 1;
    }
    const int type = list.type[low], size = type == kF64 ? 8 : type == kF32 ? 4 : 2;
    const size_t start = (size_t)(chunk - list.first[low]) * (kChunk / size), left = list.count[low] - start;
    const int n = (int)(left < kChunk / size ? left : kChunk / size);
    if (type == kF32) f(0.f, low, start, n);
    else if (type == kBF16) f((__bf16)0.f, low, start, n);
    else if (type == kF16) f((_Float16)0.f, low, start, n);
    else f(0.0, low, start, n);
  }
}

template <typename T>
constexpr int kVector = 16 / sizeof(T);

__device__ __forceinline__ double workgroup_sum(double v) {
  __shared__ double lds[kThreads / 64];
  __syncthreads();  // a sum before this one has been read
  for (int step = 32; step > 0; step /= 2) v += __shfl_down(v, step, 64);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x / 64] = v;
  __syncthreads();
  v = 0.0;
  for (int w = 0; w < kThreads / 64; ++w) v += lds[w];
  return v;
}

template <int MOST>
__global__ __launch_bounds__(kThreads)
void gradient_squares_kernel(Tensors<MOST> list, double* __restrict__ partial) {
  double sum = 0.0;
  for_chunks<false>(list, [&](auto zero, int tensor, size_t start, int n) {
    typedef decltype(zero) T;
    constexpr int V = kVector<T>, EACH = kChunk / 16 / kThreads;
    const T* p = static_cast<const T*>(list.in[tensor]) + start;
    if (n == (int)(kChunk / sizeof(T))) {
      typename Packed<T, V>::type v[EACH];
#pragma unroll
      for (int i = 0; i < EACH; ++i) v[i] = *reinterpret_cast<const typename Wide<T, V>::type*>(p + (i * kThreads + threadIdx.x) * V);
#pragma unroll
      for (int i = 0; i < EACH; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) sum = fma((double)v[i][e], (double)v[i][e], sum);
    } else {
      int i = threadIdx.x * V;
      for (; i + V <= n; i += kThreads * V) {
        const typename Packed<T, V>::type v = *reinterpret_cast<const typename Wide<T, V>::type*>(p + i);
#pragma unroll
        for (int e = 0; e < V; ++e) sum = fma((double)v[e], (double)v[e], sum);
      }
      for (const int last = i + V < n ? i + V : n; i < last; ++i) sum = fma((double)p[i], (double)p[i], sum);
    }
  });
  sum = workgroup_sum(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// The sum of what the workgroups left.
__device__ __forceinline__ double sum_of_parts(int parts, const double* partial) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < parts; i += kThreads) sum += partial[i];
  return workgroup_sum(sum);
}

__device__ __forceinline__ void store_norm(void* norm, int in_double, double value) {
  if (in_double) *static_cast<double*>(norm) = value;
  else *static_cast<float*>(norm) = (float)value;
}

__global__ __launch_bounds__(kThreads)
void gradient_norm_kernel(int parts, const double* partial, double* total, void* __restrict__ norm, int in_double) {
  const double sum = sum_of_parts(parts, partial);
  if (threadIdx.x != 0) return;
  store_norm(norm, in_double, sqrt(sum));
  if (total != nullptr) *total = sum;
}

// parts: those of the norm, which every workgroup adds up for itself and the first hands out (a launch less: 2 us, and 4 of the host);
// 0: it is there.
template <int MOST>
__global__ __launch_bounds__(kThreads)
void gradient_scale_kernel(Tensors<MOST> list, void* __restrict__ norm, int in_double, double max_norm, int parts,
                           const double* __restrict__ partial) {
  double length;
  if (parts > 0) {
    length = sqrt(sum_of_parts(parts, partial));
    if (blockIdx.x == 0 && threadIdx.x == 0) store_norm(norm, in_double, length);
    // As it is handed out, so that the gradients are the same where it is given; beyond a float's range, where it is handed out as
    // infinite, as it is: finite gradients of such a norm are not zeros.
    const float rounded = (float)length;
    if (!in_double && rounded <= 0x1.fffffep127f) length = rounded;
  } else {
    length = in_double ? *static_cast<const double*>(norm) : (double)*static_cast<const float*>(norm);
  }
  double factor = max_norm / (length + 1e-6);
  factor = factor > 1.0 ? 1.0 : factor;  // (a NaN stays)
  // A factor below a float's normal range goes into the product in two: the first lifts it by a power of 2, which the product, below 4, has room for.
  const double lift = factor < 0x1p-126 ? 0x1p120 : 1.0;
  for_chunks<true>(list, [&](auto zero, int tensor, size_t start, int n) {
    typedef decltype(zero) T;
    typedef typename std::conditional<sizeof(T) == 8, double, float>::type scale_t;
    constexpr int V = kVector<T>, EACH = kChunk / 16 / kThreads;
    const T* p = static_cast<const T*>(list.in[tensor]) + start;
    T* to = static_cast<T*>(list.out[tensor]) + start;
    if (factor == 1.0 && p == to) return;
    const scale_t by = (scale_t)(factor * lift), down = (scale_t)(1.0 / lift);
    if (n == (int)(kChunk / sizeof(T))) {
      typename Packed<T, V>::type v[EACH];
#pragma unroll
      for (int i = 0; i < EACH; ++i)
        v[i] = __builtin_nontemporal_load(reinterpret_cast<const typename Wide<T, V>::type*>(p + (i * kThreads + threadIdx.x) * V));
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[i][e] = (T)((scale_t)v[i][e] * by * down);
        __builtin_nontemporal_store(v[i], reinterpret_cast<typename Wide<T, V>::type*>(to + (i * kThreads + threadIdx.x) * V));
      }
    } else {
      int i = threadIdx.x * V;
      for (; i + V <= n; i += kThreads * V) {
        typename Packed<T, V>::type v = *reinterpret_cast<const typename Wide<T, V>::type*>(p + i);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (T)((scale_t)v[e] * by * down);
        *reinterpret_cast<typename Wide<T, V>::type*>(to + i) = v;
      }
      for (const int last = i + V < n ? i + V : n; i < last; ++i) to[i] = (T)((scale_t)p[i] * by * down);
    }
  });
}

// ---- host --------------------------------------------------------------------------------
struct Call {
  int count;
  const void* const* in;
  void* const* out;  // null: the norm alone
  const size_t* elements;
  const int* types;
};

size_t chunks_of(size_t elements, int type) {
  const size_t each = kChunk / kSize[type];
  return (elements + each - 1) / each;
}

// Calls run(list, workgroups) for every MOST tensors; at most `most` workgroups of a list.
template <int MOST, class Run>
int for_lists_of(const Call& call, size_t most, Run run) {
  Tensors<MOST> list;
  int t = 0;
  while (t < call.count) {
    list.tensors = 0;
    size_t chunks = 0;
    for (; t < call.count && list.tensors < MOST; ++t) {
      if (call.elements[t] == 0) continue;
      const size_t here = chunks_of(call.elements[t], call.types[t]);
      const int i = list.tensors++;
      list.in[i] = call.in[t];
      list.out[i] = call.out != nullptr ? call.out[t] : nullptr;
      list.count[i] = call.elements[t];
      list.type[i] = (unsigned char)call.types[t];
      list.first[i] = (unsigned)chunks;
      chunks += here;
    }
    if (list.tensors == 0) break;
    list.chunks = (unsigned)chunks;
    HASTE_HIP_PROPAGATE(run(list, (unsigned)(chunks < most ? chunks : most)));
  }
  return HASTE_HIP_OK;
}
template <class Run>
int for_lists(const Call& call, size_t most, Run run) {
  return call.count <= kFewTensors ? for_lists_of<kFewTensors>(call, most, run) : for_lists_of<kTensors>(call, most, run);
}

size_t workgroups() { return (size_t)(device_cu_count() > 0 ? device_cu_count() : 256) * 8; }

int check(const Call& call) {
  HASTE_HIP_REQUIRE(call.count >= 0 && (call.count == 0 || (call.in != nullptr && call.elements != nullptr && call.types != nullptr)));
  size_t chunks = 0;
  for (int t = 0; t < call.count; ++t) {
    HASTE_HIP_REQUIRE(call.types[t] >= kF32 && call.types[t] <= kF64);
    HASTE_HIP_REQUIRE(call.elements[t] == 0 || (call.in[t] != nullptr && (call.out == nullptr || call.out[t] != nullptr)));
    if (call.elements[t] > (size_t(1) << 40)) return too_large("gradient_norm: a tensor of more than 2^40 elements");
    chunks += chunks_of(call.elements[t], call.types[t]);
    if (chunks >= (size_t(1) << 31)) return too_large("gradient_norm: more than 2^46 bytes of gradients");
  }
  return HASTE_HIP_OK;
}

// What is written may be what is read of the same tensor, and overlap nothing else, the norm included.
int check_apart(const Call& call, const void* norm, size_t norm_bytes, bool norm_given) {
  struct Span {
    uintptr_t begin, end;
    bool written;
  };
  try {
    std::vector<Span> spans;
    spans.reserve((size_t)call.count * 2 + 1);
    const uintptr_t at = reinterpret_cast<uintptr_t>(norm);
    spans.push_back({at, at + norm_bytes, !norm_given});
    for (int t = 0; t < call.count; ++t) {
      if (call.elements[t] == 0) continue;
      const size_t bytes = call.elements[t] * kSize[call.types[t]];
      const uintptr_t out = reinterpret_cast<uintptr_t>(call.out[t]), in = reinterpret_cast<uintptr_t>(call.in[t]);
      spans.push_back({out, out + bytes, true});
      if (in != out) spans.push_back({in, in + bytes, false});
    }
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
    uintptr_t written = 0, read = 0;  // the ends of what begins so far
    for (const Span& s : spans) {
      if (s.begin < written || (s.written && s.begin < read)) {
        set_error_text("clip_gradients: what is written overlaps another gradient");
        return HASTE_HIP_ERROR_INVALID_ARGUMENT;
      }
      uintptr_t& end = s.written ? written : read;
      end = s.end > end ? s.end : end;
    }
  } catch (...) {
    set_error_text("clip_gradients: out of host memory");
    return HASTE_HIP_ERROR_RUNTIME;
  }
  return HASTE_HIP_OK;
}

size_t lists_of(int count) { return ((size_t)count + kTensors - 1) / kTensors; }
constexpr size_t kMostLists = 1u << 16;

// Leaves the parts of the norm in the workspace.
int squares_of(const Call& call, int* parts, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (lists_of(call.count) > kMostLists) return too_large("gradient_norm: more than 7340032 gradients");
  HASTE_HIP_REQUIRE(workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 7u) == 0 &&
                    workspace_bytes >= haste_hip_gradient_norm_workspace_bytes(call.count));
  double* partial = static_cast<double*>(workspace);
  *parts = 0;
  ScopedKernelTimer timer("gradient_squares", stream);
  return for_lists(call, workgroups(), [&](const auto& list, unsigned groups) {
    gradient_squares_kernel<<<groups, kThreads, 0, stream>>>(list, partial + *parts);
    *parts += (int)groups;
    HASTE_HIP_TRY(hipGetLastError());
    return HASTE_HIP_OK;
  });
}

// total: where the sum of the squares is left too, or null.
int norm_of(int parts, double* total, void* norm, int in_double, const void* workspace, hipStream_t stream) {
  ScopedKernelTimer timer("gradient_norm", stream);
  gradient_norm_kernel<<<1, kThreads, 0, stream>>>(parts, static_cast<const double*>(workspace), total, norm, in_double);
  HASTE_HIP_TRY(hipGetLastError());
  return HASTE_HIP_OK;
}

// Parts that every workgroup may add up for itself: eight a thread.
constexpr int kOwnParts = 8 * kThreads;

}  // namespace
}  // namespace haste_hip

extern "C" {

using namespace haste_hip;

size_t haste_hip_gradient_norm_workspace_bytes(int count) {
  if (count < 0 || lists_of(count) > kMostLists) return 0;
  return (lists_of(count) + 1) * workgroups() * sizeof(double);
}

int haste_hip_gradient_norm(int count, const void* const* gradients, const size_t* elements, const int* types, void* norm,
                            int norm_in_double, void* workspace, size_t workspace_bytes, void* stream) {
  const Call call = {count, gradients, nullptr, elements, types};
  HASTE_HIP_PROPAGATE(check(call));
  HASTE_HIP_REQUIRE(norm != nullptr);
  int parts = 0;
  HASTE_HIP_PROPAGATE(squares_of(call, &parts, workspace, workspace_bytes, as_stream(stream)));
  return norm_of(parts, nullptr, norm, norm_in_double, workspace, as_stream(stream));
}

int haste_hip_clip_gradients(int count, const void* const* gradients, void* const* clipped, const size_t* elements, const int* types,
                             double max_norm, int norm_given, void* norm, int norm_in_double, void* workspace,
                             size_t workspace_bytes, void* stream) {
  const Call call = {count, gradients, clipped, elements, types};
  HASTE_HIP_REQUIRE(count == 0 || clipped != nullptr);
  HASTE_HIP_PROPAGATE(check(call));
  HASTE_HIP_REQUIRE(norm != nullptr && max_norm >= 0.0);
  HASTE_HIP_PROPAGATE(check_apart(call, norm, norm_in_double ? 8 : 4, norm_given != 0));
  int parts = 0;
  double* partial = static_cast<double*>(workspace);
  if (!norm_given) {
    HASTE_HIP_PROPAGATE(squares_of(call, &parts, workspace, workspace_bytes, as_stream(stream)));
    if (parts == 0 || parts > kOwnParts) {  // none: there is nothing to scale behind it
      HASTE_HIP_PROPAGATE(norm_of(parts, partial + parts, norm, norm_in_double, workspace, as_stream(stream)));
      partial += parts;  // their sum, for which the workspace has room behind those of all lists
      parts = 1;
    }
  }
  ScopedKernelTimer timer("gradient_scale", as_stream(stream));
  return for_lists(call, workgroups(), [&](const auto& list, unsigned groups) {
    gradient_scale_kernel<<<groups, kThreads, 0, as_stream(stream)>>>(list, norm, norm_in_double, max_norm, parts, partial);
    HASTE_HIP_TRY(hipGetLastError());
    return HASTE_HIP_OK;
  });
}

}  // extern "C"
