// Column sums of partials that many workgroups left, in a fixed order and without atomics.
//
// A workgroup adds up to kPartsPerGroup rows of 64 columns, four wavefronts a quarter of them each; more
// rows than that leave one row per such group, which is added the same way again.  Rows of 64 floats are
// read as 256-byte segments, eight in flight.
#include "sequence.h"

namespace haste_hip {
namespace {

constexpr int kPartsPerGroup = 256;

__global__ __launch_bounds__(256)
void column_sums_kernel(int parts, size_t columns, const float* __restrict__ partial,
                        float* __restrict__ stage, ColumnOutputs to) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const size_t col = (size_t)blockIdx.x * 64 + lane;
  const int first = blockIdx.y * kPartsPerGroup, last = min(parts, first + kPartsPerGroup);
  float sum = 0.f;
  if (col < columns) {
    int p = first + w;
    for (; p + 28 < last; p += 32) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = partial[(size_t)(p + 4 * i) * columns + col];
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += v[i];
    }
    for (; p < last; p += 4) sum += partial[(size_t)p * columns + col];
  }
  red[w][lane] = sum;
  __syncthreads();
  if (w != 0 || col >= columns) return;
  const float total = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
  if (stage != nullptr) {
    stage[(size_t)blockIdx.y * columns + col] = total;
  } else {
    size_t begin = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (col >= begin && col < to.end[j] && to.out[j] != nullptr) to.out[j][col - begin] = total;
      begin = to.end[j];
    }
  }
}

int groups_of(int parts) { return (parts + kPartsPerGroup - 1) / kPartsPerGroup; }

}  // namespace

size_t column_sums_scratch(int parts, size_t columns) {
  size_t floats = 0;
  for (int g = groups_of(parts); g > 1; g = groups_of(g)) floats += (size_t)g * columns;
  return floats;
}

int column_sums(hipStream_t stream, int parts, size_t columns, const float* partial, float* scratch,
                const ColumnOutputs& to) {
  const size_t blocks = (columns + 63) / 64;
  if (blocks > kGridLimit || (size_t)groups_of(parts) > kGridLimitYZ) return too_large("too many partial sums");
  ScopedKernelTimer timer("column_sums", stream);
  for (;;) {
    const int groups = groups_of(parts);
    dim3 grid((unsigned)blocks, groups);
    column_sums_kernel<<<grid, 256, 0, stream>>>(parts, columns, partial, groups > 1 ? scratch : nullptr, to);
    HASTE_HIP_TRY(hipGetLastError());
    if (groups == 1) return HASTE_HIP_OK;
    partial = scratch;
    scratch += (size_t)groups * columns;
    parts = groups;
  }
}

}  // namespace haste_hip
