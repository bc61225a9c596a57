// A gated linear recurrence, one state a channel:
//   r = sigmoid(forget + forget_bias),  i = sigmoid(admit + admit_bias),
//   with a decay:     a = exp(-decay r),  u = sqrt(1 - a^2) i x     (without an admit gate i = 1)
//   without a decay:  a = r,              u = i x                   (without an admit gate u = (1 - r) x)
//   h[t] = a h[t-1] + u,  y = h silu(z)                             (without z y = h)
// and its backward pass, with c the gradient that reaches h[t] from behind (at the end that of h_last):
//   g = dy silu(z) + c,  c' = a g (for the step before; at the first step the gradient of h0),
//   dz = dy h silu'(z),  dx = g du/dx,  dadmit = g du/di i (1 - i),  dforget = (dL or da) r (1 - r),
//   with a decay dL = g (h[t-1] a - i x a^2 / sqrt(1 - a^2)) is that of log a: dforget = -decay dL r (1 - r), ddecay = -sum dL r.
//
// Bound: HBM, 2 to 4 inputs in and one output out, backward those and dy in and as many gradients out.  Steps are
// composed: a run of steps maps h to A h + B.  A workgroup takes 128 channels of a row through time in tiles of kTile steps;
// a wavefront has kEach steps of a tile in registers, two channels a lane, composes them and leaves (A, B) in LDS; after one barrier each
// has what the wavefronts before it hand over, and goes through its steps again.  Inputs are read once, a tile ahead.
// A pass in training keeps the state before each tile (4 bytes for kTile elements); the backward pass goes through tiles from the last
// to the first, composing both ways at once (the products A are the same), so that it reads inputs once as well.
// Where rows and channels make few workgroups the time axis is cut into segments: a first pass composes each, and each joins
// those before it (backward: behind it) itself.
#include <type_traits>

#include "sequence.h"

namespace haste_hip {
namespace {

constexpr int V = 2;                     // channels of a lane
constexpr int kStrip = 64 * V;           // of a workgroup
constexpr int kEach = 4;                 // steps of a wavefront
constexpr int kWaves = 16;
constexpr int kTile = kEach * kWaves;
constexpr int kSums = 3;                 // dforget_bias, dadmit_bias, ddecay

struct Shape {
  int T, N, D, strips, segments, tiles_each;  // tiles of a segment
  __host__ __device__ int tiles() const { return (T + kTile - 1) / kTile; }
};

template <typename T>
struct Inputs {
  Rows<const T> x, forget, admit, z;               // admit, z: may be absent
  const float *decay, *forget_bias, *admit_bias;   // each may be null
  const long long* lengths;
};

template <typename T>
using Raw = typename Packed<T, V>::type;

// sigmoid(v) and 1 - sigmoid(v), each with all its bits.
struct Sigmoid {
  float s, c;
};
__device__ __forceinline__ Sigmoid sigmoid_both(float v) {
  const float e = exp_of(-fabsf(v)), large = __builtin_amdgcn_rcpf(1.0f + e), small = e * large;
  return v >= 0.f ? Sigmoid{large, small} : v < 0.f ? Sigmoid{small, large} : Sigmoid{large, large};  // (the last: 0.5, or NaN)
}

// sqrt(1 - exp(-2 w)) of w >= 0, a = exp(-w): below 2 w = 0.5 by the series of 1 - exp.
__device__ __forceinline__ float complement(float w, float a) {
  const float y = 2.0f * w;
  float p = 1.0f / 40320.0f;
  p = 1.0f / 5040.0f - y * p;
  p = 1.0f / 720.0f - y * p;
  p = 1.0f / 120.0f - y * p;
  p = 1.0f / 24.0f - y * p;
  p = 1.0f / 6.0f - y * p;
  p = 0.5f - y * p;
  p = y * (1.0f - y * p);
  return sqrtf(y < 0.5f ? p : 1.0f - a * a);
}

// One channel's constants.
struct Channel {
  float decay, forget_bias, admit_bias;
};

// A step's factors: a, and by what x enters.  The rest is for the gradients.
struct Gates {
  float a, scale, m;
  Sigmoid r, i;
};
template <bool DECAY, bool ADMIT>
__device__ __forceinline__ Gates gates_of(const Channel& c, float forget, float admit) {
  Gates g;
  g.r = sigmoid_both(forget + c.forget_bias);
  g.m = 1.0f;
  if constexpr (DECAY) {
    const float w = c.decay * g.r.s;
    g.a = exp_of(-w);
    g.m = complement(w, g.a);
  } else {
    g.a = g.r.s;
  }
  if constexpr (ADMIT) {
    g.i = sigmoid_both(admit + c.admit_bias);
    g.scale = DECAY ? g.m * g.i.s : g.i.s;
  } else {
    g.i = {1.0f, 0.0f};
    g.scale = DECAY ? g.m : g.r.c;
  }
  return g;
}

template <bool DECAY, bool ADMIT, typename T>
__device__ __forceinline__ void load_constants(const Inputs<T>& in, int c0, int D, Channel (&ch)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const bool inside = c0 + v < D;
    ch[v].decay = DECAY && inside ? in.decay[c0 + v] : 0.f;
    ch[v].forget_bias = in.forget_bias != nullptr && inside ? in.forget_bias[c0 + v] : 0.f;
    ch[v].admit_bias = ADMIT && in.admit_bias != nullptr && inside ? in.admit_bias[c0 + v] : 0.f;
  }
}

// A wavefront's steps of a tensor, as they are fetched; steps from `end` on are not read.
template <typename T>
__device__ __forceinline__ void fetch(const Rows<const T>& rows, int t, int end, int n, int c0, int D, Raw<T> (&raw)[kEach]) {
#pragma unroll
  for (int l = 0; l < kEach; ++l) {
    raw[l] = Raw<T>{};
    if (t + l < end) raw[l] = load_packed<V>(rows.at(t + l, n), c0, D);
  }
}

struct Place {
  int c0, n, segment;
};
__device__ __forceinline__ Place place_of(const Shape& s) {
  const unsigned strip = blockIdx.x % s.strips, rest = blockIdx.x / s.strips;
  return {(int)(strip * kStrip + (threadIdx.x & 63) * V), (int)(rest % s.N), (int)(rest / s.N)};
}

// What a segment does to a state, composed by its first pass: [segment][2][N][D].
__device__ __forceinline__ float* composed(float* at, const Shape& s, int segment, int which, int n) {
  return at + (((size_t)segment * 2 + which) * s.N + n) * s.D;
}

// The state (backward: the gradient) that enters a segment, from what enters the first (last) one and the segments between.
template <bool BACKWARD>
__device__ __forceinline__ void join_segments(const Shape& s, const Place& at, const float* sums, float (&h)[V]) {
  const int count = BACKWARD ? s.segments - 1 - at.segment : at.segment;
  for (int j = 0; j < count; ++j) {
    const int seg = BACKWARD ? s.segments - 1 - j : j;
    float A[V], B[V];
    load_channels<V>(composed(const_cast<float*>(sums), s, seg, 0, at.n), at.c0, s.D, A);
    load_channels<V>(composed(const_cast<float*>(sums), s, seg, 1, at.n), at.c0, s.D, B);
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = A[v] * h[v] + B[v];
  }
}

// ---- the first pass over a cut time axis --------------------------------------------------
// A wavefront takes a run of the segment's steps through by itself; the runs meet at the end.
template <typename T, bool DECAY, bool ADMIT, bool BACKWARD>
__global__ __launch_bounds__(64 * kWaves)
void gated_compose_kernel(Shape s, Inputs<T> in, Rows<const T> dy, float* __restrict__ sums) {
  __shared__ float2 lds[kWaves][kStrip];
  Place at = place_of(s);
  at.segment += BACKWARD ? 1 : 0;  // the last one's is not needed (backward: the first one's)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Extent extent = extent_of(in.lengths, at.n, s.T);
  const int begin = at.segment * s.tiles_each * kTile;
  const int each = s.tiles_each * kEach;  // steps of a wavefront
  const int first = begin + wave * each;
  const int end = extent.steps < first + each ? extent.steps : first + each;
  Channel ch[V];
  load_constants<DECAY, ADMIT>(in, at.c0, s.D, ch);
  float A[V], B[V];
#pragma unroll
  for (int v = 0; v < V; ++v) A[v] = 1.f, B[v] = 0.f;
  const int blocks = end > first ? (end - first + kEach - 1) / kEach : 0;
  for (int b = 0; b < blocks; ++b) {
    const int t = first + (BACKWARD ? blocks - 1 - b : b) * kEach;
    Raw<T> f[kEach], other[kEach], gate[kEach] = {};
    fetch(in.forget, t, end, at.n, at.c0, s.D, f);
    if constexpr (BACKWARD) {
      fetch(dy, t, end, at.n, at.c0, s.D, other);
      if (in.z.p != nullptr) fetch(in.z, t, end, at.n, at.c0, s.D, gate);
    } else {
      fetch(in.x, t, end, at.n, at.c0, s.D, other);
      if constexpr (ADMIT) fetch(in.admit, t, end, at.n, at.c0, s.D, gate);
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int l = BACKWARD ? kEach - 1 - k : k;
      if (t + l >= end) continue;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Gates g = gates_of<DECAY, ADMIT>(ch[v], (float)f[l][v], BACKWARD ? 0.f : (float)gate[l][v]);
        const float value = (float)other[l][v], z = (float)gate[l][v];
        if constexpr (BACKWARD) B[v] = g.a * (B[v] + (in.z.p != nullptr ? value * (z * sigmoid_of(z)) : value));
        else B[v] = g.a * B[v] + g.scale * value;
        A[v] *= g.a;
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) lds[wave][lane * V + v] = make_float2(A[v], B[v]);
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int v = 0; v < V; ++v) A[v] = 1.f, B[v] = 0.f;
  for (int k = 0; k < kWaves; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float2 m = lds[BACKWARD ? kWaves - 1 - k : k][lane * V + v];
      B[v] = m.x * B[v] + m.y;
      A[v] *= m.x;
    }
  store_channels<V>(composed(sums, s, at.segment, 0, at.n), at.c0, s.D, A);
  store_channels<V>(composed(sums, s, at.segment, 1, at.n), at.c0, s.D, B);
}

// ---- forward -----------------------------------------------------------------------------
template <typename T, bool DECAY, bool ADMIT>
__global__ __launch_bounds__(64 * kWaves)
void gated_forward_kernel(Shape s, Inputs<T> in, const float* __restrict__ h0, T* __restrict__ y, float* __restrict__ h_last,
                          float* __restrict__ kept, const float* __restrict__ sums) {
  __shared__ float2 lds[2][kWaves][kStrip];
  const Place at = place_of(s);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c0 = at.c0, n = at.n;
  const Extent extent = extent_of(in.lengths, n, s.T);
  const bool gated = in.z.p != nullptr;
  Channel ch[V];
  load_constants<DECAY, ADMIT>(in, c0, s.D, ch);
  float h[V] = {};  // the state before the tile
  if (h0 != nullptr) load_channels<V>(h0 + (size_t)n * s.D, c0, s.D, h);
  join_segments<false>(s, at, sums, h);

  const int first = at.segment * s.tiles_each;
  const int last = first + s.tiles_each < s.tiles() ? first + s.tiles_each : s.tiles();
  Raw<T> x[kEach], f[kEach], g[kEach] = {}, z[kEach] = {};
  auto fetch_tile = [&](int tile) {
    const int t = tile * kTile + wave * kEach;
    fetch(in.x, t, extent.steps, n, c0, s.D, x);
    fetch(in.forget, t, extent.steps, n, c0, s.D, f);
    if constexpr (ADMIT) fetch(in.admit, t, extent.steps, n, c0, s.D, g);
    if (gated) fetch(in.z, t, extent.steps, n, c0, s.D, z);
  };
  fetch_tile(first);
  for (int tile = first; tile < last; ++tile) {
    const int t = tile * kTile + wave * kEach;
    float a[kEach][V], u[kEach][V], gate[kEach][V], A[V], B[V];
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1.f, B[v] = 0.f;
#pragma unroll
    for (int l = 0; l < kEach; ++l) {
      const bool inside = t + l < extent.steps;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Gates k = gates_of<DECAY, ADMIT>(ch[v], (float)f[l][v], ADMIT ? (float)g[l][v] : 0.f);
        a[l][v] = inside ? k.a : 1.f;
        u[l][v] = inside ? k.scale * (float)x[l][v] : 0.f;
        const float zv = (float)z[l][v];
        gate[l][v] = gated ? zv * sigmoid_of(zv) : 1.f;
        B[v] = a[l][v] * B[v] + u[l][v];
        A[v] *= a[l][v];
      }
    }
    if (tile + 1 < last) fetch_tile(tile + 1);
    float2(*places)[kStrip] = lds[tile & 1];
#pragma unroll
    for (int v = 0; v < V; ++v) places[wave][lane * V + v] = make_float2(A[v], B[v]);
    __syncthreads();
    float mine[V];  // the state before this wavefront's steps
    if (kept != nullptr && wave == 0) store_channels<V>(kept + ((size_t)tile * s.N + n) * s.D, c0, s.D, h);
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float2 m = places[w][lane * V + v];
        if (w == wave) mine[v] = h[v];
        h[v] = m.x * h[v] + m.y;
      }
#pragma unroll
    for (int l = 0; l < kEach; ++l) {
      float out[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        mine[v] = a[l][v] * mine[v] + u[l][v];
        out[v] = t + l < extent.steps ? mine[v] * gate[l][v] : extent.fill;
      }
      if (t + l < s.T) store_channels<V>(y + ((size_t)(t + l) * s.N + n) * s.D, c0, s.D, out);
    }
  }
  if (last == s.tiles() && wave == 0 && h_last != nullptr) {
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] += extent.fill;
    store_channels<V>(h_last + (size_t)n * s.D, c0, s.D, h);
  }
}

// ---- backward ----------------------------------------------------------------------------
template <typename T>
struct Gradients {
  T *dx, *dforget, *dadmit, *dz;  // packed [T,N,D]; dadmit, dz null where there is no such input
  float* dh0;                     // may be null
  float* partial;                 // [N segments][kSums][D]
};

template <typename T, bool DECAY, bool ADMIT>
__global__ __launch_bounds__(64 * kWaves)
void gated_backward_kernel(Shape s, Inputs<T> in, const float* __restrict__ kept, Rows<const T> dy, const float* __restrict__ dh_last,
                           Gradients<T> out, const float* __restrict__ sums) {
  struct Run {
    float A, B, Q;
  };
  __shared__ Run lds[2][kWaves][kStrip];
  const Place at = place_of(s);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c0 = at.c0, n = at.n;
  const Extent extent = extent_of(in.lengths, n, s.T);
  const bool gated = in.z.p != nullptr;
  Channel ch[V];
  load_constants<DECAY, ADMIT>(in, c0, s.D, ch);
  float c[V] = {};  // the gradient that reaches the tile from behind
  if (dh_last != nullptr) load_channels<V>(dh_last + (size_t)n * s.D, c0, s.D, c);
  join_segments<true>(s, at, sums, c);

  const int first = at.segment * s.tiles_each;
  const int last = first + s.tiles_each < s.tiles() ? first + s.tiles_each : s.tiles();
  Raw<T> x[kEach], f[kEach], g[kEach] = {}, z[kEach] = {}, d[kEach];
  float before[V];
  auto fetch_tile = [&](int tile) {
    const int t = tile * kTile + wave * kEach;
    fetch(in.x, t, extent.steps, n, c0, s.D, x);
    fetch(in.forget, t, extent.steps, n, c0, s.D, f);
    if constexpr (ADMIT) fetch(in.admit, t, extent.steps, n, c0, s.D, g);
    if (gated) fetch(in.z, t, extent.steps, n, c0, s.D, z);
    fetch(dy, t, extent.steps, n, c0, s.D, d);
    load_channels<V>(kept + ((size_t)tile * s.N + n) * s.D, c0, s.D, before);
  };
  float sum_forget[V] = {}, sum_admit[V] = {}, sum_decay[V] = {};
  fetch_tile(last - 1);
  for (int tile = last - 1; tile >= first; --tile) {
    const int t = tile * kTile + wave * kEach;
    Gates k[kEach][V];
    float xs[kEach][V], ds[kEach][V], q[kEach][V], zs[kEach][V], h[V];
    Run run[V];
#pragma unroll
    for (int v = 0; v < V; ++v) run[v] = {1.f, 0.f, 0.f}, h[v] = before[v];
#pragma unroll
    for (int l = 0; l < kEach; ++l) {
      const bool inside = t + l < extent.steps;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        k[l][v] = gates_of<DECAY, ADMIT>(ch[v], (float)f[l][v], ADMIT ? (float)g[l][v] : 0.f);
        k[l][v].a = inside ? k[l][v].a : 1.f;
        xs[l][v] = (float)x[l][v];  // 0 behind the row's end, as are z and dy
        zs[l][v] = (float)z[l][v];
        ds[l][v] = (float)d[l][v];
        q[l][v] = gated ? ds[l][v] * (zs[l][v] * sigmoid_of(zs[l][v])) : ds[l][v];
        run[v].B = k[l][v].a * run[v].B + k[l][v].scale * xs[l][v];
        // step l's share goes back through the steps before it
        run[v].A *= k[l][v].a;
        run[v].Q += run[v].A * q[l][v];
      }
    }
    if (tile > first) fetch_tile(tile - 1);
    Run(*places)[kStrip] = lds[tile & 1];
#pragma unroll
    for (int v = 0; v < V; ++v) places[wave][lane * V + v] = run[v];
    __syncthreads();
    float mine[V];
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (w < wave) {
          const Run m = places[w][lane * V + v];
          h[v] = m.A * h[v] + m.B;
        }
#pragma unroll
    for (int w = kWaves - 1; w >= 0; --w)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Run m = places[w][lane * V + v];
        if (w == wave) mine[v] = c[v];
        c[v] = m.A * c[v] + m.Q;
      }
    float hs[kEach + 1][V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      hs[0][v] = h[v];
#pragma unroll
      for (int l = 0; l < kEach; ++l) hs[l + 1][v] = k[l][v].a * hs[l][v] + k[l][v].scale * xs[l][v];
    }
    float tile_forget[V] = {}, tile_admit[V] = {}, tile_decay[V] = {};
#pragma unroll
    for (int l = kEach - 1; l >= 0; --l) {
      const bool inside = t + l < extent.steps;
      float dx[V], df[V], da[V], dz[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Gates& e = k[l][v];
        const float grad = q[l][v] + mine[v], was = hs[l][v], xv = xs[l][v];
        dx[v] = grad * e.scale;
        if constexpr (DECAY) {
          const float fed = ADMIT ? xv * e.i.s : xv;
          const float slope = e.m > 0.f ? e.a * e.a / e.m : 0.f;  // no steps towards a decay of exactly 1
          const float dlog = grad * (was * e.a - fed * slope);
          tile_decay[v] -= inside ? dlog * e.r.s : 0.f;
          df[v] = -ch[v].decay * dlog * (e.r.s * e.r.c);
          if constexpr (ADMIT) da[v] = grad * e.m * xv * (e.i.s * e.i.c);
        } else if constexpr (ADMIT) {
          df[v] = grad * was * (e.r.s * e.r.c);
          da[v] = grad * xv * (e.i.s * e.i.c);
        } else {
          df[v] = grad * (was - xv) * (e.r.s * e.r.c);
        }
        if (!inside) dx[v] = df[v] = da[v] = extent.fill;
        tile_forget[v] += df[v];
        if constexpr (ADMIT) tile_admit[v] += da[v];
        if (gated) {
          const float sg = sigmoid_of(zs[l][v]);
          dz[v] = inside ? ds[l][v] * hs[l + 1][v] * silu_slope(zs[l][v], sg) : extent.fill;
        }
        mine[v] = e.a * grad;
      }
      if (t + l < s.T) {
        const size_t row = ((size_t)(t + l) * s.N + n) * s.D;
        store_channels<V>(out.dx + row, c0, s.D, dx);
        store_channels<V>(out.dforget + row, c0, s.D, df);
        if constexpr (ADMIT) store_channels<V>(out.dadmit + row, c0, s.D, da);
        if (gated) store_channels<V>(out.dz + row, c0, s.D, dz);
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) sum_forget[v] += tile_forget[v], sum_admit[v] += tile_admit[v], sum_decay[v] += tile_decay[v];
  }
  if (first == 0 && wave == 0 && out.dh0 != nullptr) {
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] += extent.fill;
    store_channels<V>(out.dh0 + (size_t)n * s.D, c0, s.D, c);
  }
  // the sums over a workgroup's steps, the wavefronts' in order
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) lds[0][wave][lane * V + v] = {sum_forget[v], sum_admit[v], sum_decay[v]};
  __syncthreads();
  if (wave != 0) return;
  float total[kSums][V] = {};
  for (int w = 0; w < kWaves; ++w)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const Run m = lds[0][w][lane * V + v];
      total[0][v] += m.A;
      total[1][v] += m.B;
      total[2][v] += m.Q;
    }
  float* to = out.partial + ((size_t)at.segment * s.N + n) * kSums * s.D;
#pragma unroll
  for (int j = 0; j < kSums; ++j) store_channels<V>(to + (size_t)j * s.D, c0, s.D, total[j]);
}

// ---- a single step -----------------------------------------------------------------------
template <typename T, bool DECAY, bool ADMIT>
__global__ __launch_bounds__(256)
void gated_step_kernel(int N, int D, Inputs<T> in, const float* __restrict__ h, T* __restrict__ y, float* __restrict__ h_out) {
  const unsigned groups = (D + V - 1) / V;
  for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < (size_t)N * groups; i += (size_t)gridDim.x * 256) {
    const int n = (int)(i / groups), c0 = (int)(i % groups) * V;
    Channel ch[V];
    load_constants<DECAY, ADMIT>(in, c0, D, ch);
    float x[V], f[V], g[V] = {}, z[V] = {}, state[V], out[V];
    load_channels<V>(in.x.at(0, n), c0, D, x);
    load_channels<V>(in.forget.at(0, n), c0, D, f);
    if constexpr (ADMIT) load_channels<V>(in.admit.at(0, n), c0, D, g);
    if (in.z.p != nullptr) load_channels<V>(in.z.at(0, n), c0, D, z);
    load_channels<V>(h + (size_t)n * D, c0, D, state);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const Gates k = gates_of<DECAY, ADMIT>(ch[v], f[v], g[v]);
      state[v] = k.a * state[v] + k.scale * x[v];
      out[v] = in.z.p != nullptr ? state[v] * (z[v] * sigmoid_of(z[v])) : state[v];
    }
    store_channels<V>(y + (size_t)n * D, c0, D, out);
    store_channels<V>(h_out + (size_t)n * D, c0, D, state);
  }
}

// ---- host --------------------------------------------------------------------------------
int check_sizes(int T, int N, int D) {
  HASTE_HIP_REQUIRE(T > 0 && N > 0 && D > 0);
  if (T > kSizeLimit || N > kSizeLimit || D > kSizeLimit) return too_large("gated_recurrence: a size beyond 2^30");
  const size_t strips = ((size_t)D + kStrip - 1) / kStrip;
  if (strips * N > kGridLimit / 16) return too_large("gated_recurrence: more rows of channels than a grid takes");
  return HASTE_HIP_OK;
}

Shape shape_of(int T, int N, int D) {
  Shape s = {T, N, D, (D + kStrip - 1) / kStrip, 1, 0};
  const int cus = device_cu_count() > 0 ? device_cu_count() : 256;
  const int tiles = s.tiles();
  const long long groups = (long long)s.strips * N;
  int segments = 1;
  if (groups < cus / 2) {
    segments = (int)(cus / groups);
    const int most = tiles / 2;
    segments = segments < most ? segments : most;
    segments = segments < 16 ? segments : 16;
    segments = segments > 1 ? segments : 1;
  }
  s.tiles_each = (tiles + segments - 1) / segments;
  s.segments = (tiles + s.tiles_each - 1) / s.tiles_each;
  return s;
}

size_t segment_floats(const Shape& s) { return s.segments > 1 ? (size_t)s.segments * 2 * s.N * s.D : 0; }
size_t partial_floats(const Shape& s) {
  const size_t parts = (size_t)s.segments * s.N, columns = (size_t)kSums * s.D;
  return parts * columns + column_sums_scratch(parts, columns);
}

template <typename T, class Run>
int with_gates(const Inputs<T>& in, Run run) {
  using Y = std::true_type;
  using N = std::false_type;
  if (in.decay != nullptr) return in.admit.p != nullptr ? run(Y(), Y()) : run(Y(), N());
  return in.admit.p != nullptr ? run(N(), Y()) : run(N(), N());
}

unsigned grid_of(const Shape& s, int segments) { return (unsigned)((size_t)s.strips * s.N * segments); }

bool workspace_ok(const void* workspace, size_t bytes, size_t floats) {
  return floats == 0 || (workspace != nullptr && bytes >= floats * sizeof(float) && (reinterpret_cast<uintptr_t>(workspace) & 3u) == 0);
}

template <typename T>
int forward_entry(int steps, int N, int D, const Inputs<T>& in, const float* h0, T* y, float* h_last, float* kept, void* workspace,
                  size_t workspace_bytes, void* stream) {
  HASTE_HIP_PROPAGATE(check_sizes(steps, N, D));
  HASTE_HIP_REQUIRE(in.x.p != nullptr && in.forget.p != nullptr && y != nullptr);
  const Shape s = shape_of(steps, N, D);
  HASTE_HIP_REQUIRE(workspace_ok(workspace, workspace_bytes, segment_floats(s)));
  float* sums = static_cast<float*>(workspace);
  return with_gates(in, [&](auto decay, auto admit) {
    constexpr bool DECAY = decltype(decay)::value, ADMIT = decltype(admit)::value;
    if (s.segments > 1) {
      ScopedKernelTimer timer("gated_compose", as_stream(stream));
      gated_compose_kernel<T, DECAY, ADMIT, false><<<grid_of(s, s.segments - 1), 64 * kWaves, 0, as_stream(stream)>>>(s, in, {}, sums);
      HASTE_HIP_TRY(hipGetLastError());
    }
    ScopedKernelTimer timer("gated_forward", as_stream(stream));
    gated_forward_kernel<T, DECAY, ADMIT><<<grid_of(s, s.segments), 64 * kWaves, 0, as_stream(stream)>>>(s, in, h0, y, h_last, kept, sums);
    HASTE_HIP_TRY(hipGetLastError());
    return HASTE_HIP_OK;
  });
}

template <typename T>
int backward_entry(int steps, int N, int D, const Inputs<T>& in, const float* kept, const Rows<const T>& dy, const float* dh_last,
                   Gradients<T> out, float* ddecay, float* dforget_bias, float* dadmit_bias, void* workspace, size_t workspace_bytes,
                   void* stream) {
  HASTE_HIP_PROPAGATE(check_sizes(steps, N, D));
  HASTE_HIP_REQUIRE(in.x.p != nullptr && in.forget.p != nullptr && kept != nullptr && dy.p != nullptr && out.dx != nullptr);
  HASTE_HIP_REQUIRE(out.dforget != nullptr && (in.admit.p == nullptr || out.dadmit != nullptr) && (in.z.p == nullptr || out.dz != nullptr));
  const Shape s = shape_of(steps, N, D);
  const size_t cut = segment_floats(s);
  HASTE_HIP_REQUIRE(workspace_ok(workspace, workspace_bytes, cut + partial_floats(s)));
  float* sums = static_cast<float*>(workspace);
  out.partial = sums + cut;
  HASTE_HIP_PROPAGATE(with_gates(in, [&](auto decay, auto admit) {
    constexpr bool DECAY = decltype(decay)::value, ADMIT = decltype(admit)::value;
    if (s.segments > 1) {
      ScopedKernelTimer timer("gated_compose", as_stream(stream));
      gated_compose_kernel<T, DECAY, ADMIT, true><<<grid_of(s, s.segments - 1), 64 * kWaves, 0, as_stream(stream)>>>(s, in, dy, sums);
      HASTE_HIP_TRY(hipGetLastError());
    }
    ScopedKernelTimer timer("gated_backward", as_stream(stream));
    gated_backward_kernel<T, DECAY, ADMIT><<<grid_of(s, s.segments), 64 * kWaves, 0, as_stream(stream)>>>(s, in, kept, dy, dh_last, out, sums);
    HASTE_HIP_TRY(hipGetLastError());
    return HASTE_HIP_OK;
  }));
  if (ddecay == nullptr && dforget_bias == nullptr && dadmit_bias == nullptr) return HASTE_HIP_OK;
  const size_t parts = (size_t)s.segments * N, width = D;
  return column_sums(as_stream(stream), parts, kSums * width, out.partial, out.partial + parts * kSums * width,
                     {{dforget_bias, dadmit_bias, ddecay, nullptr}, {width, 2 * width, 3 * width, 3 * width}});
}

template <typename T>
int iterate_entry(int N, int D, const Inputs<T>& in, const float* h, T* y, float* h_out, void* stream) {
  HASTE_HIP_PROPAGATE(check_sizes(1, N, D));
  HASTE_HIP_REQUIRE(in.x.p != nullptr && in.forget.p != nullptr && h != nullptr && y != nullptr && h_out != nullptr);
  const size_t blocks = ((size_t)N * ((D + V - 1) / V) + 255) / 256;
  return with_gates(in, [&](auto decay, auto admit) {
    ScopedKernelTimer timer("gated_step", as_stream(stream));
    gated_step_kernel<T, decltype(decay)::value, decltype(admit)::value>
        <<<(unsigned)(blocks < 65536 ? blocks : 65536), 256, 0, as_stream(stream)>>>(N, D, in, h, y, h_out);
    HASTE_HIP_TRY(hipGetLastError());
    return HASTE_HIP_OK;
  });
}

}  // namespace
}  // namespace haste_hip

extern "C" {

using namespace haste_hip;

size_t haste_hip_gated_recurrence_workspace_bytes(int backward, int steps, int batch_size, int channels) {
  if (check_sizes(steps, batch_size, channels) != HASTE_HIP_OK) return 0;
  const Shape s = shape_of(steps, batch_size, channels);
  return (segment_floats(s) + (backward ? partial_floats(s) : 0)) * sizeof(float);
}

size_t haste_hip_gated_recurrence_kept_bytes(int steps, int batch_size, int channels) {
  if (check_sizes(steps, batch_size, channels) != HASTE_HIP_OK) return 0;
  return (size_t)shape_of(steps, batch_size, channels).tiles() * batch_size * channels * sizeof(float);
}

#define HASTE_HIP_GATED_INPUTS                                                                                              \
  const void *x, size_t x_step, size_t x_row, const void *forget, size_t forget_step, size_t forget_row, const void *admit, \
      size_t admit_step, size_t admit_row, const void *z, size_t z_step, size_t z_row, const float *decay,                  \
      const float *forget_bias, const float *admit_bias
#define HASTE_HIP_GATED_IN(T)                                                                                               \
  Inputs<T>{{static_cast<const T*>(x), x_step, x_row}, {static_cast<const T*>(forget), forget_step, forget_row},            \
            {static_cast<const T*>(admit), admit_step, admit_row}, {static_cast<const T*>(z), z_step, z_row},               \
            decay, forget_bias, admit_bias, static_cast<const long long*>(lengths)}

#define HASTE_HIP_GATED_RECURRENCE(SUFFIX, T)                                                                               \
  int haste_hip_gated_recurrence_forward_##SUFFIX(int steps, int batch_size, int channels, HASTE_HIP_GATED_INPUTS,          \
                                                  const float* h0, const void* lengths, void* y, float* h_last,             \
                                                  float* kept, void* workspace, size_t workspace_bytes, void* stream) {     \
    return forward_entry<T>(steps, batch_size, channels, HASTE_HIP_GATED_IN(T), h0, static_cast<T*>(y), h_last, kept,       \
                            workspace, workspace_bytes, stream);                                                            \
  }                                                                                                                         \
  int haste_hip_gated_recurrence_backward_##SUFFIX(                                                                         \
      int steps, int batch_size, int channels, HASTE_HIP_GATED_INPUTS, const void* lengths, const float* kept,              \
      const void* dy, size_t dy_step, size_t dy_row, const float* dh_last, void* dx, void* dforget, void* dadmit, void* dz, \
      float* ddecay, float* dforget_bias, float* dadmit_bias, float* dh0, void* workspace, size_t workspace_bytes,          \
      void* stream) {                                                                                                       \
    return backward_entry<T>(steps, batch_size, channels, HASTE_HIP_GATED_IN(T), kept,                                      \
                             {static_cast<const T*>(dy), dy_step, dy_row}, dh_last,                                         \
                             {static_cast<T*>(dx), static_cast<T*>(dforget), static_cast<T*>(dadmit), static_cast<T*>(dz),  \
                              dh0, nullptr},                                                                                \
                             ddecay, dforget_bias, dadmit_bias, workspace, workspace_bytes, stream);                        \
  }                                                                                                                         \
  int haste_hip_gated_recurrence_iterate_##SUFFIX(                                                                          \
      int batch_size, int channels, const void* x, size_t x_row, const void* forget, size_t forget_row, const void* admit,  \
      size_t admit_row, const void* z, size_t z_row, const float* decay, const float* forget_bias, const float* admit_bias, \
      const float* h, void* y, float* h_out, void* stream) {                                                                \
    const size_t x_step = 0, forget_step = 0, admit_step = 0, z_step = 0;                                                   \
    const void* lengths = nullptr;                                                                                          \
    return iterate_entry<T>(batch_size, channels, HASTE_HIP_GATED_IN(T), h, static_cast<T*>(y), h_out, stream);             \
  }

HASTE_HIP_GATED_RECURRENCE(f32, float)
HASTE_HIP_GATED_RECURRENCE(f16, _Float16)
HASTE_HIP_GATED_RECURRENCE(bf16, __bf16)

}  // extern "C"
