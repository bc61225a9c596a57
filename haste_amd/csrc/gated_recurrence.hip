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
// composed: a run of steps maps h to A h + B.  A workgroup takes 64 lanes' channels of a row through time in tiles of kTile steps;
// a wavefront has kEach steps of a tile in registers, composes them and leaves (A, B) in LDS; after one barrier each
// has what the wavefronts before it hand over, and goes through its steps again.  Inputs are read once, a tile ahead.
// A pass in training keeps the state before each tile (4 bytes for kTile elements); the backward pass goes through tiles from the last
// to the first, composing both ways at once (the products A are the same), so that it reads inputs once as well.
// Where rows and channels make few workgroups the time axis is cut into segments: a first pass composes each, and each joins
// those before it (backward: behind it) itself.  Its arithmetic is then done twice, and that bounds it: some 50 issue slots an
// element, half of them exponentials, reciprocals and roots at a quarter of the rate.
//
// Forward and backward of T x N x D, us, at kEach 4 and kWaves 8 / kEach 8 / kEach 2 / kWaves 4:
//   2048 x 8 x 4096, bf16, all parts          366 / 885 / 430 / 428   (1.90 GB, 5.2 TB/s; eight steps do not fit the registers)
//    500 x 37 x 300, float, all parts          87 /  84 /  92 / 100   (312 MB)
//   1024 x 8 x 1024, bf16, x and forget alone  51 /  53 /  58 /  54   (136 MB; 4 segments of 256 steps)
//   4096 x 1 x 2048, bf16, all, forward alone  34 /  40 /  37 /  36   (84 MB; 16 segments of 256 steps: first pass 13.7, second 21.7)
#include <type_traits>

#include "sequence.h"

namespace haste_hip {
namespace {

constexpr int kEach = 4;                 // steps of a wavefront: its share of a tile is held in registers
constexpr int kWaves = 8;                // of a tile, each of which reads what all leave
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

template <typename T, int V>
using Raw = typename Packed<T, V>::type;

constexpr float kLog2e = 1.44269504088896341f;

// sigmoid(v) and 1 - sigmoid(v), each with all its bits, of v = -l / log2 e: 1 / (1 + e) and e / (1 + e), whose factors are kept in
// range (an infinite e times 0).  A NaN is one in the first.
struct Sigmoid {
  float s, c, e;
};
__device__ __forceinline__ Sigmoid sigmoid_both(float l) {
  const float e = __builtin_amdgcn_exp2f(l), s = __builtin_amdgcn_rcpf(1.0f + e);
  return {s, fminf(e, 0x1p126f) * fmaxf(s, 0x1p-126f), e};
}

// 1 - exp(-y) of y >= 0, a = exp(-y / 2).  Below 0.6 by the polynomial for (1 - exp(-y)) / y of degree 5 with the least
// largest relative error there, 4e-9.
__device__ __forceinline__ float complement(float y, float a) {
  float p = -1.0748759327e-03f;
  p = p * y + 8.1288257559e-03f;
  p = p * y - 4.1603583380e-02f;
  p = p * y + 1.6665774386e-01f;
  p = p * y - 4.9999953290e-01f;
  p = p * y + 1.0f;
  p *= y;
  asm volatile("" : "+v"(p));  // worked out either way: a branch costs more
  return y < 0.6f ? p : 1.0f - a * a;
}

// One channel's constants: the decay, and what is left of it in the exponents of 2; the biases times -log2 e.
struct Channel {
  float decay, exponent, forget_bias, admit_bias;
};

// A step's factors: a, and by what x enters.  The rest is for the gradients (of which those that are not used cost nothing):
// slope = a^2 / (1 - a^2), 0 where the divisor is below a float's normal range.
struct Gates {
  float a, scale, slope;
  Sigmoid r, i;
};
template <bool DECAY, bool ADMIT>
__device__ __forceinline__ Gates gates_of(const Channel& c, float forget, float admit) {
  Gates g;
  g.r = sigmoid_both(fmaf(forget, -kLog2e, c.forget_bias));
  g.i = ADMIT ? sigmoid_both(fmaf(admit, -kLog2e, c.admit_bias)) : Sigmoid{1.0f, 0.0f, 0.0f};
  g.slope = 0.0f;
  if constexpr (DECAY) {
    g.a = __builtin_amdgcn_exp2f(c.exponent * g.r.s);
    const float p = complement(2.0f * c.decay * g.r.s, g.a);
    const float m = __builtin_amdgcn_sqrtf(p);
    g.scale = ADMIT ? m * g.i.s : m;
    const float least = 0x1p-126f;
    g.slope = (p > least ? g.a * g.a : 0.0f) * __builtin_amdgcn_rcpf(__builtin_elementwise_maximum(p, least));
  } else {
    // From its complement where that is the smaller: the reciprocal's last bit is not even-handed, and a gate near 1 goes into hundreds of
    // products (470 steps of gates of 0.62 to 0.9975: the state 2.4e-7 off instead of 6.8e-7).
    g.a = g.r.s >= 0.5f ? fmaf(-g.r.e, g.r.s, 1.0f) : g.r.s;
    g.scale = ADMIT ? g.i.s : g.r.c;
  }
  return g;
}

template <bool DECAY, bool ADMIT, int V, typename T>
__device__ __forceinline__ void load_constants(const Inputs<T>& in, int c0, Channel (&ch)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    ch[v].decay = DECAY ? in.decay[c0 + v] : 0.f;
    ch[v].exponent = ch[v].decay * -kLog2e;
    ch[v].forget_bias = in.forget_bias != nullptr ? in.forget_bias[c0 + v] * -kLog2e : 0.f;
    ch[v].admit_bias = ADMIT && in.admit_bias != nullptr ? in.admit_bias[c0 + v] * -kLog2e : 0.f;
  }
}

// A lane's channels, V of them in a row from c0 on: the last vector of a row is moved back to end with it, and lanes beyond it
// take that one too; they compute and write the same.
template <int V, typename U>
__device__ __forceinline__ void load_floats(const U* row, int c0, float (&f)[V]) {
  const typename Wide<U, V>::type w = *reinterpret_cast<const typename Wide<U, V>::type*>(row + c0);
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = (float)w[v];
}
template <int V, typename U>
__device__ __forceinline__ void store_floats(U* row, int c0, const float (&f)[V]) {
  typename Wide<U, V>::type w;
#pragma unroll
  for (int v = 0; v < V; ++v) w[v] = (U)f[v];
  *reinterpret_cast<typename Wide<U, V>::type*>(row + c0) = w;
}

// Addresses: those of rows are the same for all lanes and stay in scalar registers, stepped from row to row (the compiler would make
// a pair of vector registers and a wide addition of each); a lane's channels are `offset` bytes behind.  With two wavefronts a SIMD
// every instruction counts, a scalar one too.
typedef __attribute__((address_space(1))) char* Address;
__device__ __forceinline__ Address scalar(Address p) {
  asm volatile("" : "+s"(p));
  return p;
}
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_at(Address row, unsigned offset) {
  typedef typename Wide<T, V>::type wide_t;
  return *(const __attribute__((address_space(1))) wide_t*)(row + offset);
}
template <typename T, int V>
__device__ __forceinline__ void store_at(Address row, unsigned offset, const Raw<T, V>& w) {
  typedef typename Wide<T, V>::type wide_t;
  *(__attribute__((address_space(1))) wide_t*)(row + offset) = w;
}

// A wavefront's way through a tensor: the address of its next step, and the bytes between steps.
template <typename T>
struct Walk {
  Address p;
  long long step;
  __device__ __forceinline__ Walk(const Rows<const T>& rows, int t, int n)
      : p((Address)(void*)rows.at(t, n)), step(rows.step * sizeof(T)) {}
  __device__ __forceinline__ void move(int steps) { p += steps * step; }
  // kEach steps from p on, of which the first `count` (at least 0) are there: zeros for the rest.
  template <bool FULL, int V>
  __device__ __forceinline__ void fetch(int count, unsigned offset, Raw<T, V> (&raw)[kEach]) const {
    Address row = scalar(p);
#pragma unroll
    for (int l = 0; l < kEach; ++l) {
      if (FULL) {
        raw[l] = load_at<T, V>(row, offset);
      } else {
        raw[l] = Raw<T, V>{};
        if (l < count) raw[l] = load_at<T, V>(row, offset);
      }
      if (l + 1 < kEach) row = scalar(row + step);
    }
  }
};
// The same steps of a packed output, from element `first` on.
template <bool FULL, int V, typename T>
__device__ __forceinline__ void put(T* to, long long first, long long step, int count, unsigned offset, const float (&f)[kEach][V]) {
  Address row = scalar((Address)(void*)(to + first));
#pragma unroll
  for (int l = 0; l < kEach; ++l) {
    Raw<T, V> w;
#pragma unroll
    for (int v = 0; v < V; ++v) w[v] = (T)f[l][v];
    if (FULL || l < count) store_at<T, V>(row, offset, w);
    if (l + 1 < kEach) row = scalar(row + step * (long long)sizeof(T));
  }
}

struct Place {
  int c0, n, segment;
};
template <int V>
__device__ __forceinline__ Place place_of(const Shape& s) {
  const unsigned strip = blockIdx.x % s.strips, rest = blockIdx.x / s.strips;
  const int c0 = (int)(strip * (64 * V) + (threadIdx.x & 63) * V);
  return {c0 < s.D - V ? c0 : s.D - V, (int)(rest % s.N), (int)(rest / s.N)};
}
// The wavefront's number again, in a vector register: what is compared with it stays no mask in scalar registers.
__device__ __forceinline__ int lane_wave(int wave) {
  asm volatile("" : "+v"(wave));
  return wave;
}
__device__ __forceinline__ int wave_of() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// What a segment does to a state, composed by its first pass: [segment][2][N][D].
__device__ __forceinline__ float* composed(float* at, const Shape& s, int segment, int which, int n) {
  return at + (((size_t)segment * 2 + which) * s.N + n) * s.D;
}

// The state (backward: the gradient) that enters a segment, from what enters the first (last) one and the segments between.
template <bool BACKWARD, int V>
__device__ __forceinline__ void join_segments(const Shape& s, const Place& at, const float* sums, float (&h)[V]) {
  const int count = BACKWARD ? s.segments - 1 - at.segment : at.segment;
  constexpr int AT_ONCE = 8;
  for (int j = 0; j < count; j += AT_ONCE) {
    float A[AT_ONCE][V], B[AT_ONCE][V];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int k = j + i < count ? j + i : count - 1, seg = BACKWARD ? s.segments - 1 - k : k;
      load_floats<V>(composed(const_cast<float*>(sums), s, seg, 0, at.n), at.c0, A[i]);
      load_floats<V>(composed(const_cast<float*>(sums), s, seg, 1, at.n), at.c0, B[i]);
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = j + i < count ? A[i][v] * h[v] + B[i][v] : h[v];
  }
}

// ---- the first pass over a cut time axis --------------------------------------------------
// A wavefront takes a run of the segment's steps through by itself; the runs meet at the end.
template <typename T, int V, bool DECAY, bool ADMIT, bool BACKWARD>
__global__ __launch_bounds__(64 * kWaves)
void gated_compose_kernel(Shape s, Inputs<T> in, Rows<const T> dy, float* __restrict__ sums) {
  __shared__ float2 lds[kWaves][64 * V];
  Place at = place_of<V>(s);
  at.segment += BACKWARD ? 1 : 0;  // the last one's is not needed (backward: the first one's)
  const int lane = threadIdx.x & 63, wave = wave_of();
  const Extent extent = extent_of(in.lengths, at.n, s.T);
  const int begin = at.segment * s.tiles_each * kTile;
  const int each = s.tiles_each * kEach;  // steps of a wavefront
  const int first = begin + wave * each;
  const int end = extent.steps < first + each ? extent.steps : first + each;
  Channel ch[V];
  load_constants<DECAY, ADMIT>(in, at.c0, ch);
  float A[V], B[V];
#pragma unroll
  for (int v = 0; v < V; ++v) A[v] = 1.f, B[v] = 0.f;
  // whole blocks of kEach steps, and what is left at the end: two blocks are on their way while one is composed
  const int steps = end > first ? end - first : 0, blocks = steps / kEach, left = steps % kEach;
  const unsigned offset = at.c0 * sizeof(T);
  const int start = first + (BACKWARD ? (left > 0 ? blocks : blocks - 1) * kEach : 0);
  Walk<T> forget(in.forget, start, at.n), entering(BACKWARD ? dy : in.x, start, at.n), gates(BACKWARD ? in.z : in.admit, start, at.n);
  const bool with_gate = BACKWARD ? in.z.p != nullptr : ADMIT;
  Raw<T, V> f[2][kEach], other[2][kEach], gate[2][kEach] = {};
  auto fetch = [&](auto set, auto full, int count) {
    constexpr int next = BACKWARD ? -kEach : kEach;
    forget.template fetch<full(), V>(count, offset, f[set]);
    entering.template fetch<full(), V>(count, offset, other[set]);
    if (with_gate) gates.template fetch<full(), V>(count, offset, gate[set]);
    forget.move(next);
    entering.move(next);
    if (with_gate) gates.move(next);
  };
  auto compose = [&](auto set, auto full, int count, bool ahead) {
    Raw<T, V> fs[kEach], others[kEach], gs[kEach];
#pragma unroll
    for (int l = 0; l < kEach; ++l) fs[l] = f[set][l], others[l] = other[set][l], gs[l] = gate[set][l];
    if (ahead) fetch(set, std::true_type(), kEach);
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int l = BACKWARD ? kEach - 1 - k : k;
      if (!full() && l >= count) continue;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Gates g = gates_of<DECAY, ADMIT>(ch[v], (float)fs[l][v], BACKWARD ? 0.f : (float)gs[l][v]);
        const float value = (float)others[l][v], z = (float)gs[l][v];
        if constexpr (BACKWARD) B[v] = g.a * (B[v] + (in.z.p != nullptr ? value * (z * sigmoid_of(z)) : value));
        else B[v] = g.a * B[v] + g.scale * value;
        A[v] *= g.a;
      }
    }
  };
  constexpr std::integral_constant<int, 0> even;
  constexpr std::integral_constant<int, 1> odd;
  auto rest = [&] {
    if (left == 0) return;
    fetch(even, std::false_type(), left);
    compose(even, std::false_type(), left, false);
  };
  if constexpr (BACKWARD) rest();
  if (blocks > 0) fetch(even, std::true_type(), kEach);
  if (blocks > 1) fetch(odd, std::true_type(), kEach);
  for (int b = 0; b < blocks; b += 2) {
    compose(even, std::true_type(), kEach, b + 2 < blocks);
    if (b + 1 < blocks) compose(odd, std::true_type(), kEach, b + 3 < blocks);
  }
  if constexpr (!BACKWARD) rest();
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
  store_floats<V>(composed(sums, s, at.segment, 0, at.n), at.c0, A);
  store_floats<V>(composed(sums, s, at.segment, 1, at.n), at.c0, B);
}

// ---- forward -----------------------------------------------------------------------------
template <typename T, int V, bool DECAY, bool ADMIT>
__global__ __launch_bounds__(64 * kWaves)
void gated_forward_kernel(Shape s, Inputs<T> in, const float* __restrict__ h0, T* __restrict__ y, float* __restrict__ h_last,
                          float* __restrict__ kept, const float* __restrict__ sums) {
  __shared__ float2 lds[2][kWaves][64 * V];
  const Place at = place_of<V>(s);
  const int lane = threadIdx.x & 63, wave = wave_of(), c0 = at.c0, n = at.n;
  const Extent extent = extent_of(in.lengths, n, s.T);
  const bool gated = in.z.p != nullptr;
  Channel ch[V];
  load_constants<DECAY, ADMIT>(in, c0, ch);
  float h[V] = {};  // the state before the tile
  if (h0 != nullptr) load_floats<V>(h0 + (size_t)n * s.D, c0, h);
  join_segments<false, V>(s, at, sums, h);

  const int first = at.segment * s.tiles_each;
  const int last = first + s.tiles_each < s.tiles() ? first + s.tiles_each : s.tiles();
  Raw<T, V> x2[2][kEach], f2[2][kEach], g2[2][kEach] = {}, z2[2][kEach] = {};
  const unsigned offset = c0 * sizeof(T);
  const int t0 = first * kTile + wave * kEach;
  Walk<T> wx(in.x, t0, n), wf(in.forget, t0, n), wg(in.admit, t0, n), wz(in.z, t0, n);
  const long long step = (long long)s.N * s.D;  // elements of a step
  auto fetch_tile = [&](auto set, auto full, int count) {
    wx.template fetch<full(), V>(count, offset, x2[set]);
    wx.move(kTile);
    wf.template fetch<full(), V>(count, offset, f2[set]);
    wf.move(kTile);
    if constexpr (ADMIT) {
      wg.template fetch<full(), V>(count, offset, g2[set]);
      wg.move(kTile);
    }
    if (gated) {
      wz.template fetch<full(), V>(count, offset, z2[set]);
      wz.move(kTile);
    }
  };
  // A tile: FULL, its steps are all inside the row.  `ahead`: whether the one after the next is to be fetched.
  auto run_tile = [&](auto set, auto full, int tile, bool ahead) {
    Raw<T, V>(&x)[kEach] = x2[set], (&f)[kEach] = f2[set], (&g)[kEach] = g2[set], (&z)[kEach] = z2[set];
    const int t = tile * kTile + wave * kEach;
    float a[kEach][V], u[kEach][V], gate[kEach][V], A[V], B[V];
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1.f, B[v] = 0.f;
#pragma unroll
    for (int l = 0; l < kEach; ++l) {
      const bool inside = full() || t + l < extent.steps;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Gates k = gates_of<DECAY, ADMIT>(ch[v], (float)f[l][v], ADMIT ? (float)g[l][v] : 0.f);
        a[l][v] = inside ? k.a : 1.f;
        u[l][v] = inside ? k.scale * (float)x[l][v] : 0.f;
        gate[l][v] = 1.f;
        B[v] = a[l][v] * B[v] + u[l][v];
        A[v] *= a[l][v];
      }
    }
    if (gated) {
#pragma unroll
      for (int l = 0; l < kEach; ++l)
#pragma unroll
        for (int v = 0; v < V; ++v) gate[l][v] = (float)z[l][v] * sigmoid_of((float)z[l][v]);
    }
    if (ahead) fetch_tile(set, std::true_type(), kEach);
    float2(*places)[64 * V] = lds[set];
#pragma unroll
    for (int v = 0; v < V; ++v) places[wave][lane * V + v] = make_float2(A[v], B[v]);
    __syncthreads();
    float mine[V] = {};  // the state before this wavefront's steps
    const int here = lane_wave(wave);
    if (kept != nullptr && wave == 0) store_floats<V>(kept + ((size_t)tile * s.N + n) * s.D, c0, h);
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float2 m = places[w][lane * V + v];
        mine[v] = w == here ? h[v] : mine[v];
        h[v] = m.x * h[v] + m.y;
      }
#pragma unroll
    for (int l = 0; l < kEach; ++l)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        mine[v] = a[l][v] * mine[v] + u[l][v];
        gate[l][v] = full() || t + l < extent.steps ? mine[v] * gate[l][v] : extent.fill;
      }
    put<full()>(y, t * step + (long long)n * s.D, step, s.T - t, offset, gate);
  };
  constexpr std::integral_constant<int, 0> even;
  constexpr std::integral_constant<int, 1> odd;
  const int whole = extent.steps / kTile < last ? extent.steps / kTile : last;  // tiles of the row that are full
  if (first < whole) fetch_tile(even, std::true_type(), kEach);
  if (first + 1 < whole) fetch_tile(odd, std::true_type(), kEach);
  int tile = first;
  for (; tile < whole; tile += 2) {
    run_tile(even, std::true_type(), tile, tile + 2 < whole);
    if (tile + 1 < whole) run_tile(odd, std::true_type(), tile + 1, tile + 3 < whole);
  }
  for (tile = whole > first ? whole : first; tile < last; ++tile) {
    const int left = extent.steps - tile * kTile - wave * kEach;
    fetch_tile(even, std::false_type(), left > 0 ? left : 0);
    __syncthreads();  // what the tile before left in LDS has been read
    run_tile(even, std::false_type(), tile, false);
  }
  if (last == s.tiles() && wave == 0 && h_last != nullptr) {
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] += extent.fill;
    store_floats<V>(h_last + (size_t)n * s.D, c0, h);
  }
}

// ---- backward ----------------------------------------------------------------------------
template <typename T>
struct Gradients {
  T *dx, *dforget, *dadmit, *dz;  // packed [T,N,D]; dadmit, dz null where there is no such input
  float* dh0;                     // may be null
  float* partial;                 // [N segments][kSums][D]
};

template <typename T, int V, bool DECAY, bool ADMIT>
__global__ __launch_bounds__(64 * kWaves, 2)
void gated_backward_kernel(Shape s, Inputs<T> in, const float* __restrict__ kept, Rows<const T> dy, const float* __restrict__ dh_last,
                           Gradients<T> out, const float* __restrict__ sums) {
  __shared__ float2 lds[2][kWaves][64 * V];   // A, B: what the steps do to a state
  __shared__ float lds_q[2][kWaves][64 * V];  // and A, Q to the gradient that comes back
  const Place at = place_of<V>(s);
  const int lane = threadIdx.x & 63, wave = wave_of(), c0 = at.c0, n = at.n;
  const Extent extent = extent_of(in.lengths, n, s.T);
  const bool gated = in.z.p != nullptr;
  Channel ch[V];
  load_constants<DECAY, ADMIT>(in, c0, ch);
  float c[V] = {};  // the gradient that reaches the tile from behind
  if (dh_last != nullptr) load_floats<V>(dh_last + (size_t)n * s.D, c0, c);
  join_segments<true, V>(s, at, sums, c);

  const int first = at.segment * s.tiles_each;
  const int last = first + s.tiles_each < s.tiles() ? first + s.tiles_each : s.tiles();
  Raw<T, V> x2[2][kEach], f2[2][kEach], g2[2][kEach] = {}, z2[2][kEach] = {}, d2[2][kEach];
  float before2[2][V];
  const unsigned offset = c0 * sizeof(T);
  const int t0 = (last - 1) * kTile + wave * kEach;
  Walk<T> wx(in.x, t0, n), wf(in.forget, t0, n), wg(in.admit, t0, n), wz(in.z, t0, n), wd(dy, t0, n);
  const long long step = (long long)s.N * s.D;
  const float* states = kept + ((size_t)(last - 1) * s.N + n) * s.D;
  auto fetch_tile = [&](auto set, auto full, int count) {
    wx.template fetch<full(), V>(count, offset, x2[set]);
    wx.move(-kTile);
    wf.template fetch<full(), V>(count, offset, f2[set]);
    wf.move(-kTile);
    if constexpr (ADMIT) {
      wg.template fetch<full(), V>(count, offset, g2[set]);
      wg.move(-kTile);
    }
    if (gated) {
      wz.template fetch<full(), V>(count, offset, z2[set]);
      wz.move(-kTile);
    }
    wd.template fetch<full(), V>(count, offset, d2[set]);
    wd.move(-kTile);
    load_floats<V>(states, c0, before2[set]);
    states -= (size_t)s.N * s.D;
  };
  float sum_forget[V] = {}, sum_admit[V] = {}, sum_decay[V] = {};
  auto run_tile = [&](auto set, auto full, int tile, bool ahead) {
    Raw<T, V>(&x)[kEach] = x2[set], (&f)[kEach] = f2[set], (&g)[kEach] = g2[set], (&z)[kEach] = z2[set], (&d)[kEach] = d2[set];
    float(&before)[V] = before2[set];
    const int t = tile * kTile + wave * kEach;
    // of an element: a, u = scale x, by what dx comes of g, the factors of the other gradients, and those of dy
    float a[kEach][V], u[kEach][V], scale[kEach][V], r[kEach][V], dr[kEach][V], slope[kEach][V], shut[kEach][V], q[kEach][V], e[kEach][V], h[V];
    float A[V], B[V], Q[V];
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1.f, B[v] = Q[v] = 0.f, h[v] = before[v];
#pragma unroll
    for (int l = 0; l < kEach; ++l) {
      const bool inside = full() || t + l < extent.steps;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Gates k = gates_of<DECAY, ADMIT>(ch[v], (float)f[l][v], ADMIT ? (float)g[l][v] : 0.f);
        const float xv = (float)x[l][v], dv = (float)d[l][v], zv = (float)z[l][v];  // 0 behind the row's end
        a[l][v] = inside ? k.a : 1.f;
        scale[l][v] = k.scale;
        u[l][v] = inside ? k.scale * xv : 0.f;
        dr[l][v] = DECAY ? -ch[v].decay * (k.r.s * k.r.c) : k.r.s * k.r.c;
        r[l][v] = DECAY ? k.r.s : xv;
        slope[l][v] = k.slope;
        shut[l][v] = k.i.c;
        q[l][v] = dv;
        if (gated) {
          const float sg = sigmoid_of(zv);
          q[l][v] = dv * (zv * sg);
          e[l][v] = dv * silu_slope(zv, sg);
        }
        B[v] = a[l][v] * B[v] + u[l][v];
        A[v] *= a[l][v];
        Q[v] += A[v] * q[l][v];  // step l's share goes back through the steps before it
      }
    }
    if (ahead) fetch_tile(set, std::true_type(), kEach);
    float2(*places)[64 * V] = lds[set];
    float(*back)[64 * V] = lds_q[set];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      places[wave][lane * V + v] = make_float2(A[v], B[v]);
      back[wave][lane * V + v] = Q[v];
    }
    __syncthreads();
    float mine[V] = {}, state[V];
    const int here = lane_wave(wave);
    float2 m[kWaves][V];
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
#pragma unroll
      for (int v = 0; v < V; ++v) m[w][v] = places[w][lane * V + v];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      state[v] = h[v];
#pragma unroll
      for (int w = 0; w + 1 < kWaves; ++w) {
        state[v] = m[w][v].x * state[v] + m[w][v].y;
        h[v] = w + 1 == here ? state[v] : h[v];
      }
#pragma unroll
      for (int w = kWaves - 1; w >= 0; --w) {
        mine[v] = w == here ? c[v] : mine[v];
        c[v] = m[w][v].x * c[v] + back[w][lane * V + v];
      }
    }
    float hs[kEach + 1][V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      hs[0][v] = h[v];
#pragma unroll
      for (int l = 0; l < kEach; ++l) hs[l + 1][v] = a[l][v] * hs[l][v] + u[l][v];
    }
    float tile_forget[V] = {}, tile_admit[V] = {}, tile_decay[V] = {};
#pragma unroll
    for (int l = kEach - 1; l >= 0; --l) {
      const bool inside = full() || t + l < extent.steps;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float dx, df, da, dz;
        const float grad = q[l][v] + mine[v], was = hs[l][v];
        dx = grad * scale[l][v];
        if constexpr (DECAY) {
          const float dlog = grad * (was * a[l][v] - u[l][v] * slope[l][v]);
          tile_decay[v] -= inside ? dlog * r[l][v] : extent.fill;
          df = dlog * dr[l][v];
        } else {
          df = grad * (ADMIT ? was : was - r[l][v]) * dr[l][v];
        }
        if constexpr (ADMIT) da = grad * u[l][v] * shut[l][v];
        if (gated) dz = e[l][v] * hs[l + 1][v];
        if (!inside) dx = df = da = dz = extent.fill;
        tile_forget[v] += df;
        if constexpr (ADMIT) tile_admit[v] += da;
        mine[v] = a[l][v] * grad;
        // in the places of what is not needed any more
        scale[l][v] = dx;
        dr[l][v] = df;
        shut[l][v] = da;
        e[l][v] = dz;
      }
    }
    const int count = s.T - t;
    const long long row = t * step + (long long)n * s.D;
    put<full()>(out.dx, row, step, count, offset, scale);
    put<full()>(out.dforget, row, step, count, offset, dr);
    if constexpr (ADMIT) put<full()>(out.dadmit, row, step, count, offset, shut);
    if (gated) put<full()>(out.dz, row, step, count, offset, e);
#pragma unroll
    for (int v = 0; v < V; ++v) sum_forget[v] += tile_forget[v], sum_admit[v] += tile_admit[v], sum_decay[v] += tile_decay[v];
  };
  constexpr std::integral_constant<int, 0> even;
  constexpr std::integral_constant<int, 1> odd;
  const int whole = extent.steps / kTile < last ? extent.steps / kTile : last;  // tiles of the row that are full
  int tile = last - 1;
  for (; tile >= first && tile >= whole; --tile) {
    const int left = extent.steps - tile * kTile - wave * kEach;
    fetch_tile(even, std::false_type(), left > 0 ? left : 0);
    __syncthreads();  // what the tile before left in LDS has been read
    run_tile(even, std::false_type(), tile, false);
  }
  if (tile >= first) fetch_tile(even, std::true_type(), kEach);
  if (tile - 1 >= first) fetch_tile(odd, std::true_type(), kEach);
  __syncthreads();
  for (; tile >= first; tile -= 2) {
    run_tile(even, std::true_type(), tile, tile - 2 >= first);
    if (tile - 1 >= first) run_tile(odd, std::true_type(), tile - 1, tile - 3 >= first);
  }
  if (first == 0 && wave == 0 && out.dh0 != nullptr) {
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] += extent.fill;
    store_floats<V>(out.dh0 + (size_t)n * s.D, c0, c);
  }
  // the sums over a workgroup's steps, the wavefronts' in order
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) {
    lds[0][wave][lane * V + v] = make_float2(sum_forget[v], sum_admit[v]);
    lds_q[0][wave][lane * V + v] = sum_decay[v];
  }
  __syncthreads();
  if (wave != 0) return;
  float total[kSums][V] = {};
  for (int w = 0; w < kWaves; ++w)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      total[0][v] += lds[0][w][lane * V + v].x;
      total[1][v] += lds[0][w][lane * V + v].y;
      total[2][v] += lds_q[0][w][lane * V + v];
    }
  float* to = out.partial + ((size_t)at.segment * s.N + n) * kSums * s.D;
#pragma unroll
  for (int j = 0; j < kSums; ++j) store_floats<V>(to + (size_t)j * s.D, c0, total[j]);
}

// ---- a single step -----------------------------------------------------------------------
// Two channels a thread; none is taken twice, the state may be written where it was read.
template <typename T, bool DECAY, bool ADMIT>
__global__ __launch_bounds__(256)
void gated_step_kernel(int N, int D, Inputs<T> in, const float* __restrict__ h, T* __restrict__ y, float* __restrict__ h_out) {
  constexpr int V = 2;
  const unsigned groups = (D + V - 1) / V;
  for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < (size_t)N * groups; i += (size_t)gridDim.x * 256) {
    const int n = (int)(i / groups), c0 = (int)(i % groups) * V;
    float x[V], f[V], g[V] = {}, z[V] = {}, state[V], out[V], decay[V] = {}, forget_bias[V] = {}, admit_bias[V] = {};
    load_channels<V>(in.x.at(0, n), c0, D, x);
    load_channels<V>(in.forget.at(0, n), c0, D, f);
    if constexpr (ADMIT) load_channels<V>(in.admit.at(0, n), c0, D, g);
    if (in.z.p != nullptr) load_channels<V>(in.z.at(0, n), c0, D, z);
    load_channels<V>(h + (size_t)n * D, c0, D, state);
    if constexpr (DECAY) load_channels<V>(in.decay, c0, D, decay);
    if (in.forget_bias != nullptr) load_channels<V>(in.forget_bias, c0, D, forget_bias);
    if (ADMIT && in.admit_bias != nullptr) load_channels<V>(in.admit_bias, c0, D, admit_bias);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const Channel ch = {decay[v], decay[v] * -kLog2e, forget_bias[v] * -kLog2e, admit_bias[v] * -kLog2e};
      const Gates k = gates_of<DECAY, ADMIT>(ch, f[v], g[v]);
      state[v] = k.a * state[v] + k.scale * x[v];
      out[v] = in.z.p != nullptr ? state[v] * (z[v] * sigmoid_of(z[v])) : state[v];
    }
    store_channels<V>(y + (size_t)n * D, c0, D, out);
    store_channels<V>(h_out + (size_t)n * D, c0, D, state);
  }
}

// ---- host --------------------------------------------------------------------------------
int cus() { return device_cu_count() > 0 ? device_cu_count() : 256; }

// Channels of a lane: two where that leaves three quarters of a workgroup a CU, otherwise one, for twice as many workgroups (two on a
// cut time axis, with segments half as long: 4096 x 1 x 2048 36 us instead of 34, 500 x 37 x 300 119 instead of 87).
int vector_of(int N, int D) { return D > 1 && ((long long)D + 127) / 128 * N >= cus() * 3 / 4 ? 2 : 1; }

int check_sizes(int T, int N, int D) {
  HASTE_HIP_REQUIRE(T > 0 && N > 0 && D > 0);
  if (T > kSizeLimit || N > kSizeLimit || D > kSizeLimit) return too_large("gated_recurrence: a size beyond 2^30");
  const size_t strip = 64 * vector_of(N, D);
  if ((D + strip - 1) / strip * N > kGridLimit) return too_large("gated_recurrence: more rows of channels than a grid takes");
  return HASTE_HIP_OK;
}

// The time axis is cut where there are fewer workgroups than five eighths of the CUs, for about two a CU, of two tiles at least.
Shape shape_of(int T, int N, int D) {
  const int strip = 64 * vector_of(N, D);
  Shape s = {T, N, D, (D + strip - 1) / strip, 1, 0};
  const int tiles = s.tiles();
  const long long groups = (long long)s.strips * N;
  int segments = 1;
  if (groups <= cus() * 5 / 8) {
    segments = (int)(2 * cus() / groups);
    const int most = tiles / 2 < 64 ? tiles / 2 : 64;
    segments = segments < most ? segments : most;
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

// run(channels of a lane, whether there is a decay, whether an admit gate)
template <typename T, class Run>
int with_kind(const Inputs<T>& in, int vector, Run run) {
  using Y = std::true_type;
  using N = std::false_type;
  auto gates = [&](auto v) {
    if (in.decay != nullptr) return in.admit.p != nullptr ? run(v, Y(), Y()) : run(v, Y(), N());
    return in.admit.p != nullptr ? run(v, N(), Y()) : run(v, N(), N());
  };
  return vector == 1 ? gates(std::integral_constant<int, 1>()) : gates(std::integral_constant<int, 2>());
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
  return with_kind(in, vector_of(N, D), [&](auto vector, auto decay, auto admit) {
    constexpr int V = decltype(vector)::value;
    constexpr bool DECAY = decltype(decay)::value, ADMIT = decltype(admit)::value;
    if constexpr (V == 1) if (s.segments > 1) {  // (where lanes take two channels there are too many workgroups for a cut)
      ScopedKernelTimer timer("gated_compose", as_stream(stream));
      gated_compose_kernel<T, V, DECAY, ADMIT, false><<<grid_of(s, s.segments - 1), 64 * kWaves, 0, as_stream(stream)>>>(s, in, {}, sums);
      HASTE_HIP_TRY(hipGetLastError());
    }
    ScopedKernelTimer timer("gated_forward", as_stream(stream));
    gated_forward_kernel<T, V, DECAY, ADMIT><<<grid_of(s, s.segments), 64 * kWaves, 0, as_stream(stream)>>>(s, in, h0, y, h_last, kept, sums);
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
  HASTE_HIP_PROPAGATE(with_kind(in, vector_of(N, D), [&](auto vector, auto decay, auto admit) {
    constexpr int V = decltype(vector)::value;
    constexpr bool DECAY = decltype(decay)::value, ADMIT = decltype(admit)::value;
    if constexpr (V == 1) if (s.segments > 1) {
      ScopedKernelTimer timer("gated_compose", as_stream(stream));
      gated_compose_kernel<T, V, DECAY, ADMIT, true><<<grid_of(s, s.segments - 1), 64 * kWaves, 0, as_stream(stream)>>>(s, in, dy, sums);
      HASTE_HIP_TRY(hipGetLastError());
    }
    ScopedKernelTimer timer("gated_backward", as_stream(stream));
    gated_backward_kernel<T, V, DECAY, ADMIT><<<grid_of(s, s.segments), 64 * kWaves, 0, as_stream(stream)>>>(s, in, kept, dy, dh_last, out, sums);
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
  const size_t blocks = ((size_t)N * ((D + 1) / 2) + 255) / 256;
  return with_kind(in, 2, [&](auto, auto decay, auto admit) {
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
