// Column sums of partials that many workgroups left, in a fixed order and without atomics.
//
// A workgroup adds up to kPartsPerGroup rows of 64 columns, four wavefronts a quarter of them each; more
// rows than that leave one row per such group, which is added the same way again.  Rows of 64 floats are
// read as 256-byte segments, eight in flight.  What exceeds a grid, columns or groups, goes by turns: a
// caller's sums are never refused when its own kernel already runs.
#include "sequence.h"

namespace haste_hip {
namespace {

constexpr size_t kPartsPerGroup = 256;

__global__ __launch_bounds__(256)
void column_sums_kernel(size_t parts, size_t columns, const float* __restrict__ partial,
                        float* __restrict__ stage, ColumnOutputs to) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (size_t first = (size_t)blockIdx.y * kPartsPerGroup; first < parts; first += (size_t)gridDim.y * kPartsPerGroup) {
    const size_t last = parts - first < kPartsPerGroup ? parts : first + kPartsPerGroup;
    for (size_t block = blockIdx.x * (size_t)64; block < columns; block += (size_t)gridDim.x * 64) {
      const size_t col = block + lane;
      float sum = 0.f;
      if (col < columns) {
        size_t p = first + w;
        for (; p + 28 < last; p += 32) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = partial[(p + 4 * i) * columns + col];
#pragma unroll
          for (int i = 0; i < 8; ++i) sum += v[i];
        }
        for (; p < last; p += 4) sum += partial[p * columns + col];
      }
      red[w][lane] = sum;
      __syncthreads();
      if (w == 0 && col < columns) {
        const float total = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
        if (stage != nullptr) {
          stage[first / kPartsPerGroup * columns + col] = total;
        } else {
          size_t begin = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (col >= begin && col < to.end[j] && to.out[j] != nullptr) to.out[j][col - begin] = total;
            begin = to.end[j];
          }
        }
      }
      __syncthreads();  // red is written again
    }
  }
}

size_t groups_of(size_t parts) { return (parts + kPartsPerGroup - 1) / kPartsPerGroup; }

}  // namespace

size_t column_sums_scratch(size_t parts, size_t columns) {
  size_t floats = 0;
  for (size_t g = groups_of(parts); g > 1; g = groups_of(g)) floats += g * columns;
  return floats;
}

int column_sums(hipStream_t stream, size_t parts, size_t columns, const float* partial, float* scratch,
                const ColumnOutputs& to) {
  const size_t blocks = (columns + 63) / 64;
  ScopedKernelTimer timer("column_sums", stream);
  for (;;) {
    const size_t groups = groups_of(parts);
    dim3 grid((unsigned)(blocks < kGridLimit ? blocks : kGridLimit), (unsigned)(groups < kGridLimitYZ ? groups : kGridLimitYZ));
    column_sums_kernel<<<grid, 256, 0, stream>>>(parts, columns, partial, groups > 1 ? scratch : nullptr, to);
    HASTE_HIP_TRY(hipGetLastError());
    if (groups == 1) return HASTE_HIP_OK;
    partial = scratch;
    scratch += groups * columns;
    parts = groups;
  }
}

}  // namespace haste_hip
