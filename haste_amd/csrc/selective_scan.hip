// Selective state space scan: every channel d carries S states that decay and take input at rates that
// the input sets,
//   dt = softplus(delta + delta_bias) (or their sum),  a = exp(dt A[d,s]),
//   h[t] = a h[t-1] + dt x B[t,g,s],  y = (sum_s C[t,g,s] h[t] + D x) silu(z),
// g the group of channels d belongs to, and its backward pass, walking down with
// q = dy silu(z), ypre the bracket above, G[T-1] the gradient of the last state:
//   g[t] = q C + G[t],  G[t-1] = a g[t],  w = G[t-1] h[t-1],
//   dC = sum_d q h[t],  dB = sum_d g dt x,  du = sum_s g B,  ddt = x du + sum_s A w,  dA = sum_tn dt w,
//   dx = dt du + D q,  ddelta = ddt sigmoid(delta + delta_bias),  dz = dy ypre silu'(z),  dD = sum q x.
//
// Bound: the vector ALUs.  A state's step is four operations and an exp2 forward (fourteen and the sums
// over channels backward), at 16 states a channel several times what moving the channel's few bytes
// takes.  A lane keeps four states of one channel in registers, LANES lanes make up the channel, and a
// workgroup of four wavefronts takes 256 / LANES channels of a batch row through time in tiles of 16
// steps: what there is once per channel (softplus, products, the gate) is computed by one thread for
// every element of a tile and handed over through LDS, B and C are read from there by all channels.
//
// The time axis is cut into chunks where there are too few rows and channels to fill the chip: a first
// pass finds what each chunk adds to a state of zero and sum dt, by which it decays what it is given
// (exp(A sum dt)); the second pass runs all chunks at once, each from what those before it hand over.
// The same backwards with G.
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "channel_share.h"
#include "sequence.h"

namespace haste_hip {
namespace {

constexpr int TS = 16;           // steps of a tile; a training pass keeps the states at every tile's start
constexpr int K = 4;             // states of a lane
constexpr int kMaxStates = 64;
constexpr float kLog2e = 1.44269504088896341f;
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef float float2_t __attribute__((ext_vector_type(2)));

struct ScanShape {
  int T, N, D, S, G;
  int blocks_group;    // workgroups of a group
  ChannelShare share;  // of its D / G channels among them
  int chunk, chunks;   // steps of a chunk (a multiple of TS)
  int softplus;
};

template <typename T>
struct ScanInputs {
  Rows<const T> x, delta, B, C, z;  // z.p may be null
  const float *A, *skip, *bias;     // skip (D), bias may be null
  const long long* lengths;
};

// log(1 + e) for 0 <= e <= 1, exact to a few ulp however small e is: log(w) has the error of w = 1 + e,
// and e / (w - 1) takes it back out.
__device__ __forceinline__ float log1p_of(float e) {
  const float w = 1.0f + e, d = w - 1.0f;
  const float l = __builtin_amdgcn_logf(w) * 0.693147180559945309f;
  return d == 0.f ? e : l * (e * __builtin_amdgcn_rcpf(d));
}
__device__ __forceinline__ float softplus_of(float v) { return fmaxf(v, 0.f) + log1p_of(exp_of(-fabsf(v))); }
// The same with its derivative, sigmoid(v).
__device__ __forceinline__ float softplus_of(float v, float* slope) {
  const float e = exp_of(-fabsf(v)), r = __builtin_amdgcn_rcpf(1.0f + e);
  *slope = v >= 0.f ? r : e * r;
  return fmaxf(v, 0.f) + log1p_of(e);
}
// Chosen, not branched to, like everything between the steps of a scan: a branch would part it from them.
__device__ __forceinline__ float step_size(float raw, int softplus, bool inside) {
  const float soft = softplus_of(raw), dt = softplus ? soft : raw;
  return inside ? dt : 0.f;
}
__device__ __forceinline__ float step_size(float raw, int softplus, bool inside, float* slope) {
  const float soft = softplus_of(raw, slope), dt = softplus ? soft : raw;
  *slope = softplus ? *slope : 1.0f;
  return inside ? dt : 0.f;
}

// A lane's place in a wavefront: the lanes of a channel are neighbours, sums over them stay within a row of 16 lanes.
template <int LANES>
struct Place {
  static constexpr int kChannels = 64 / LANES;  // of a wavefront
  static constexpr int kBlock = 4 * kChannels;  // of a workgroup
  static __device__ __forceinline__ int states(int lane) { return lane % LANES; }
  static __device__ __forceinline__ int channel(int lane) { return lane / LANES; }
};

// Sum over the lanes of a channel, in each of them.
template <int LANES>
__device__ __forceinline__ float sum_states(float v) {
  if (LANES >= 2) v += dpp<kXor1>(v);
  if (LANES >= 4) v += dpp<kXor2>(v);
  if (LANES >= 8) v += dpp<kHalfMirror>(v);
  if (LANES >= 16) v += dpp<kRor8>(v);
  return v;
}

// Sums of a lane's four values over the channels of the wavefront (parts 1), or of each of its rows of 16 lanes (parts 4).
template <int LANES>
struct ChannelSums {
  static constexpr int kParts = 1;
  static __device__ __forceinline__ int part(int) { return 0; }
  // the value whose sum a lane gets: rows 0, 2, 1, 3
  static __device__ __forceinline__ int value(int lane) { return (lane >> 4 & 1) << 1 | lane >> 5; }
  static __device__ __forceinline__ float sum(const float (&v)[K]) {
    float s = swap_add_rows(swap_add_halves(v[0], v[1]), swap_add_halves(v[2], v[3]));
    if (LANES <= 8) s += dpp<kRor8>(s);
    if (LANES <= 4) s += dpp<kRor4>(s);
    if (LANES <= 2) s += dpp<kXor2>(s);
    return s;
  }
};
// With four lanes a channel the channels of a row are its four banks, and additions that write some banks only leave each bank with
// one of the four values: six of them, 24 cycles, for the 44 of swapping rows and halves too, against four times the parts to add
// up from LDS.  Forward and backward, both builds in turn: T=2048 N=8 D=4096 S=16 bf16 1257 us without, 1211 so (runs differ by 1 %),
// T=1024 D=1024 239 and 232.
// (The assembler's form: of the compiler's every addition that leaves banks as they are is a move and an addition.)
template <>
struct ChannelSums<4> {
  static constexpr int kParts = 4;
  static __device__ __forceinline__ int part(int lane) { return lane >> 4; }
  static __device__ __forceinline__ int value(int lane) { return (lane >> 2 & 1 ? 0 : 2) | (lane >> 3 & 1); }
  static __device__ __forceinline__ float sum(const float (&v)[K]) {
    float low, high, s;
    // a lane read by another needs two instructions after its write; rotating right, lane i reads i - 8, i - 4, i - 12 (i + 4)
    asm("s_nop 1\n\t"
        "v_add_f32_dpp %0, %3, %3 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
        "v_add_f32_dpp %1, %5, %5 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
        "v_add_f32_dpp %0, %4, %4 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %1, %6, %6 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "s_nop 1\n\t"
        "v_add_f32_dpp %2, %0, %0 row_ror:4 row_mask:0xf bank_mask:0xa\n\t"
        "v_add_f32_dpp %2, %1, %1 row_ror:12 row_mask:0xf bank_mask:0x5"
        : "=&v"(low), "=&v"(high), "=&v"(s)
        : "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]));
    return s;
  }
};

// A channel's states [S] of float, this lane's four of them; those beyond S are 0.
__device__ __forceinline__ void load_states(const float* p, int s0, int S, float (&h)[K]) {
  load_channels<K>(p, s0, S, h);
}
__device__ __forceinline__ void store_states(float* p, int s0, int S, const float (&h)[K]) {
  store_channels<K>(p, s0, S, h);
}

// The rates of decay to base 2, all finite: a step of 0, as those behind a row's end in its last tile are, leaves as it is a state that
// forgets everything at any other.
__device__ __forceinline__ void base2_rates(const float (&A)[K], float (&A2)[K]) {
#pragma unroll
  for (int r = 0; r < K; ++r) {
    const float rate = A[r] * kLog2e;
    A2[r] = __builtin_fabsf(rate) == INFINITY ? copysignf(FLT_MAX, rate) : rate;
  }
}

// Which row and channels a workgroup works on: c0 .. c_end-1.  The workgroups of a group share its channels evenly: a share of
// 64 for all but the last one costs that one the whole time axis for the few that are left.  T=1024 N=8 S=16 bf16, forward and
// backward: D=961 242 us instead of 288, D=1025 315 instead of 385, D=1024 231 either way.
template <int LANES>
struct Block {
  int n, g, c0, c_end;
  __device__ __forceinline__ Block(const ScanShape& s, unsigned block) {
    const unsigned per_row = s.G * s.blocks_group;
    n = block / per_row;
    const unsigned rest = block % per_row;
    g = rest / s.blocks_group;
    const ChannelRange range = s.share.of((int)(rest % s.blocks_group));
    c0 = g * s.share.channels + range.first;
    c_end = g * s.share.channels + range.end;
  }
};

// A tile's elements as the threads of a workgroup share them: WIDTH channels of ITEMS rows each.
template <int LANES>
struct Tile {
  static constexpr int kBlock = Place<LANES>::kBlock;
  static constexpr int kEach = TS * kBlock / 256;
  static constexpr int WIDTH = kEach < 4 ? kEach : 4;
  static constexpr int ITEMS = kEach / WIDTH;
  static constexpr int kPerRow = kBlock / WIDTH;     // threads of a row
  static constexpr int kRowStep = 256 / kPerRow;     // rows between a thread's items
  static constexpr int kShared = (TS * LANES * K + 255) / 256;  // elements of B (of C) a thread loads
  static __device__ __forceinline__ int row(int i) { return i * kRowStep + threadIdx.x / kPerRow; }
  // This thread's columns.  Where the workgroup has fewer channels than it could take, the last threads of a row all have its last
  // ones: they compute and write the same, and no vector ends beyond the channels (`wide`).  The columns behind stay zero in LDS.
  // Only a workgroup of fewer than WIDTH channels goes by element.  With a last vector that went by element, T=1024 N=8 bf16
  // took 314 us at D=1001 and 337 at D=1023, forward and backward; so 246 at both (D=1024: 240).
  static __device__ __forceinline__ bool wide(const Block<LANES>& b) { return b.c_end - b.c0 >= WIDTH; }
  static __device__ __forceinline__ int column(const Block<LANES>& b) {
    const int c = (threadIdx.x % kPerRow) * WIDTH;
    return wide(b) ? min(c, b.c_end - b.c0 - WIDTH) : c;
  }
};

// The elements of one tensor's tile, packed in the tensor's own type until they are worked on.
template <typename T, int LANES>
struct Held {
  typedef Tile<LANES> L;
  typedef T packed_t __attribute__((ext_vector_type(L::WIDTH)));
  packed_t v[L::ITEMS];
  __device__ __forceinline__ float get(int i, int e) const { return (float)v[i][e]; }
};

// This thread's way through a tensor, tile by tile.
template <typename T, int LANES>
struct Walk {
  typedef Tile<LANES> L;
  T* p;         // of the tile's first row here
  size_t step;  // elements between steps
  __device__ __forceinline__ Walk(const Rows<T>& rows, int t0, const Block<LANES>& b)
      : p(rows.p == nullptr ? nullptr : rows.at(t0, b.n) + (size_t)L::row(0) * rows.step + b.c0 + L::column(b)), step(rows.step) {}
  __device__ __forceinline__ void forth() { p += TS * step; }
  __device__ __forceinline__ void back() { p -= TS * step; }
  // `rows` of the tile belong to the sequence; whole: all of them do, and the workgroup is wide
  template <typename U>
  __device__ __forceinline__ void load(Held<U, LANES>& to, bool whole, int rows, const Block<LANES>& b) const {
    typedef typename Wide<U, L::WIDTH>::type wide_t;
#pragma unroll
    for (int i = 0; i < L::ITEMS; ++i) {
      const T* from = p + (size_t)(i * L::kRowStep) * step;
      if (whole) {
        to.v[i] = *reinterpret_cast<const wide_t*>(from);
      } else {
        typename Held<U, LANES>::packed_t w = {};
        if (L::row(i) < rows) {
          if (L::wide(b)) {
            w = *reinterpret_cast<const wide_t*>(from);
          } else {
#pragma unroll
            for (int e = 0; e < L::WIDTH; ++e)
              if (b.c0 + L::column(b) + e < b.c_end) w[e] = from[e];
          }
        }
        to.v[i] = w;
      }
    }
  }
  __device__ __forceinline__ void store(const float (&f)[L::ITEMS][L::WIDTH], bool whole, int rows, const Block<LANES>& b) const {
    typedef typename Wide<T, L::WIDTH>::type wide_t;
#pragma unroll
    for (int i = 0; i < L::ITEMS; ++i) {
      T* to = p + (size_t)(i * L::kRowStep) * step;
      if (whole || (L::row(i) < rows && L::wide(b))) {
        wide_t w;
#pragma unroll
        for (int e = 0; e < L::WIDTH; ++e) w[e] = (T)f[i][e];
        *reinterpret_cast<wide_t*>(to) = w;
      } else if (L::row(i) < rows) {
#pragma unroll
        for (int e = 0; e < L::WIDTH; ++e)
          if (b.c0 + L::column(b) + e < b.c_end) to[e] = (T)f[i][e];
      }
    }
  }
};

// The tile of B or C: [TS][LANES * K], states beyond S and steps beyond the row's end 0.
template <typename T, int LANES>
struct HeldShared {
  typedef Tile<LANES> L;
  T v[L::kShared];
  static __device__ __forceinline__ int row(int i) { return (i * 256 + threadIdx.x) / (LANES * K); }
  static __device__ __forceinline__ int state() { return threadIdx.x % (LANES * K); }  // of every i: 256 is a multiple
  __device__ __forceinline__ void put(float4_t* lds) const {
#pragma unroll
    for (int i = 0; i < L::kShared; ++i)
      if (L::kShared * 256 == TS * LANES * K || i * 256 + (int)threadIdx.x < TS * LANES * K)
        reinterpret_cast<float*>(lds)[i * 256 + threadIdx.x] = (float)v[i];
  }
};
template <typename T, int LANES>
struct WalkShared {
  typedef HeldShared<T, LANES> H;
  const T* p;
  size_t step;
  int S;
  __device__ __forceinline__ WalkShared(const Rows<const T>& rows, int t0, const Block<LANES>& b, int S)
      : p(rows.at(t0, b.n) + (size_t)H::row(0) * rows.step + (size_t)b.g * S + H::state()), step(rows.step), S(S) {}
  __device__ __forceinline__ void forth() { p += TS * step; }
  __device__ __forceinline__ void back() { p -= TS * step; }
  __device__ __forceinline__ void load(H& to, int rows) const {
#pragma unroll
    for (int i = 0; i < H::L::kShared; ++i)
      to.v[i] = H::row(i) < (rows < TS ? rows : TS) && H::state() < S ? p[(size_t)(i * 256 / (LANES * K)) * step] : (T)0.f;
  }
};

// What the chunks before this one hand over: chunk first, first + step, ..., `count` of them, one after the other.  Chunk c
// decays what it is given (in h) over its sum of dt, sum_dt[c], and adds at[c], what it makes of a state of zero.  Every
// workgroup does this for itself: a kernel between the two passes costs more, 7 us more of 54 (T=4096 N=1 D=1024 S=16 bf16, 32 chunks)
// and 19 of 73 (T=8192 N=1 D=256, 64 and 128 chunks).
__device__ __forceinline__ void join_chunks(float (&h)[K], const float (&A2)[K], const float* at, const float* sum_dt, size_t state,
                                            size_t states, size_t channel, size_t channels, int first, int step, int count, int s0,
                                            int S) {
  constexpr int AHEAD = 4;  // chunks read at once
  for (int k = 0; k < count; k += AHEAD) {
    float added[AHEAD][K], dt[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int c = first + step * min(k + j, count - 1);
      load_states(at + c * states + state, s0, S, added[j]);
      dt[j] = sum_dt[c * channels + channel];
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (k + j >= count) break;
#pragma unroll
      for (int r = 0; r < K; ++r) {
        // In two halves: a whole chunk's decay may lie below what a float holds where the state it leaves does not, and growth
        // above.  (0 times a product of growth beyond float's range is 0, not NaN.)
        const float half = __builtin_amdgcn_exp2f(0.5f * A2[r] * dt[j]);
        h[r] = h[r] == 0.f ? added[j][r] : half * (half * h[r]) + added[j][r];
      }
    }
  }
}

// Forward pass over a chunk.  LOCAL: only what the chunk adds to a state of zero, and the sum of dt.
// added: what the chunks but the last add [chunks][N][D][S], and sum_dt [chunks][N][D] (LOCAL: out).  kept: the states at
// the tiles' starts [tiles][N][D][S], or null.
template <typename T, int LANES, bool LOCAL>
__global__ __launch_bounds__(256)
void selective_scan_forward_kernel(ScanShape s, ScanInputs<T> in, const float* __restrict__ h0, float* __restrict__ added,
                                   float* __restrict__ sum_dt, float* __restrict__ kept, T* __restrict__ y,
                                   float* __restrict__ h_last) {
  typedef Place<LANES> P;
  typedef Tile<LANES> L;
  __shared__ float2_t step_lds[2][TS][P::kBlock];  // dt, dt x
  __shared__ float4_t B_lds[2][TS * LANES], C_lds[2][LOCAL ? 1 : TS * LANES];
  __shared__ float y_lds[2][LOCAL ? 1 : TS][P::kBlock];

  const Block<LANES> b(s, blockIdx.x);
  const int column = L::column(b);
  if (b.c_end - b.c0 < P::kBlock) {  // the columns behind the last
    for (int e = threadIdx.x; e < 2 * TS * P::kBlock; e += 256) (&step_lds[0][0][0])[e] = float2_t{0.f, 0.f};
    __syncthreads();
  }
  const int t0 = blockIdx.y * s.chunk, t1 = min(s.T, t0 + s.chunk);
  const Extent extent = extent_of(in.lengths, b.n, s.T);
  const int end = min(t1, extent.steps);
  const int lane = threadIdx.x & 63, s0 = P::states(lane) * K;
  const int mine = (threadIdx.x >> 6) * P::kChannels + P::channel(lane);  // this lane's channel in the block
  const int d = b.c0 + mine;
  const bool live = d < b.c_end;
  const size_t state = ((size_t)b.n * s.D + d) * s.S, states = (size_t)s.N * s.D * s.S;

  float A2[K], h[K], dt_sum = 0.f;
#pragma unroll
  for (int r = 0; r < K; ++r) A2[r] = h[r] = 0.f;
  if (live) {
    float A[K];
    load_states(in.A + (size_t)d * s.S, s0, s.S, A);
    base2_rates(A, A2);
    if (!LOCAL) {
      if (h0 != nullptr) load_states(h0 + state, s0, s.S, h);
      if (blockIdx.y > 0)
        join_chunks(h, A2, added, sum_dt, state, states, (size_t)b.n * s.D + d, (size_t)s.N * s.D, 0, 1, blockIdx.y, s0, s.S);
    }
  }
  float bias[L::WIDTH], skip[L::WIDTH];
#pragma unroll
  for (int e = 0; e < L::WIDTH; ++e) bias[e] = skip[e] = 0.f;
  if (in.bias != nullptr) load_channels<L::WIDTH>(in.bias, b.c0 + column, b.c_end, bias);
  if (!LOCAL && in.skip != nullptr) load_channels<L::WIDTH>(in.skip, b.c0 + column, b.c_end, skip);

  // While a tile is scanned, the next one's elements are worked out between its steps, into the other half of LDS, and the one
  // after that is on its way from memory.
  struct Raw {
    Held<T, LANES> x, delta, z;
    HeldShared<T, LANES> B, C;
  } raw = {}, coming = {};
  Walk<const T, LANES> x_walk(in.x, t0, b), delta_walk(in.delta, t0, b), z_walk(in.z, t0, b);
  WalkShared<T, LANES> B_walk(in.B, t0, b, s.S), C_walk(in.C, t0, b, s.S);
  Walk<T, LANES> y_walk(packed_rows(y, s.N, s.D), t0, b);
  const bool wide = L::wide(b), gated = !LOCAL && in.z.p != nullptr;
  auto fetch = [&](Raw& to, int t) {  // the next tile of every walk, which starts at t
    const int rows = end - t;
    if (rows <= 0) return;
    const bool whole = wide && rows >= TS;
    x_walk.load(to.x, whole, rows, b);
    delta_walk.load(to.delta, whole, rows, b);
    if (gated) z_walk.load(to.z, whole, rows, b);
    B_walk.load(to.B, rows);
    if (!LOCAL) C_walk.load(to.C, rows);
    x_walk.forth();
    delta_walk.forth();
    if (gated) z_walk.forth();
    B_walk.forth();
    if (!LOCAL) C_walk.forth();
  };
  struct Rest {  // what the outputs need besides the states
    float skipped[L::ITEMS][L::WIDTH], gate[L::ITEMS][L::WIDTH];
  } before, rest, rest_next;  // of the tile before, this one and the next
  constexpr int kEach = L::ITEMS * L::WIDTH;
  auto work_out = [&](const Raw& from, int t, int half, int element, Rest& to) {
    const int i = element / L::WIDTH, e = element % L::WIDTH;
    const float xv = from.x.get(i, e);
    const float dt = step_size(from.delta.get(i, e) + bias[e], s.softplus, t + L::row(i) < end);
    step_lds[half][L::row(i)][column + e] = float2_t{dt, dt * xv};
    if (LOCAL) return;
    to.skipped[i][e] = skip[e] * xv;
    const float zv = from.z.get(i, e), silu = zv * sigmoid_of(zv);
    to.gate[i][e] = gated ? silu : 1.f;
  };
  auto put_out = [&](int half, bool whole, int rows) {
    float o[L::ITEMS][L::WIDTH];
#pragma unroll
    for (int i = 0; i < L::ITEMS; ++i)
#pragma unroll
      for (int e = 0; e < L::WIDTH; ++e)
        o[i][e] = (y_lds[half][L::row(i)][column + e] + before.skipped[i][e]) * before.gate[i][e];
    y_walk.store(o, whole, rows, b);
  };

  if (t0 < end) {
    fetch(raw, t0);
#pragma unroll
    for (int e = 0; e < kEach; ++e) work_out(raw, t0, 0, e, rest);
    raw.B.put(B_lds[0]);
    if (!LOCAL) raw.C.put(C_lds[0]);
    fetch(raw, t0 + TS);
  }
  int half = 0;
  for (int t = t0; t < end; t += TS, half ^= 1) {
    fetch(coming, t + 2 * TS);
    __syncthreads();
    if (!LOCAL && t > t0) {  // the tile before
      put_out(half ^ 1, wide, TS);
      y_walk.forth();
    }
    before = rest;
    if (!LOCAL && kept != nullptr && live) store_states(kept + (size_t)(t / TS) * states + state, s0, s.S, h);
    // a pair of steps' operands are read from LDS while the pair before is computed
    struct { float2_t dt_u[2]; float4_t B[2], C[2]; } now, next;
    auto read = [&](auto& to, int j) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        to.dt_u[i] = step_lds[half][j + i][mine];
        to.B[i] = B_lds[half][(j + i) * LANES + s0 / K];
        if (!LOCAL) to.C[i] = C_lds[half][(j + i) * LANES + s0 / K];
      }
    };
    read(now, 0);
#pragma unroll
    for (int j = 0; j < TS; j += 2) {
      if (j + 2 < TS) read(next, j + 2);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float ys = 0.f;
#pragma unroll
        for (int r = 0; r < K; ++r) {
          const float a = __builtin_amdgcn_exp2f(now.dt_u[i].x * A2[r]);
          h[r] = a * h[r] + now.dt_u[i].y * now.B[i][r];
          if (!LOCAL) ys += h[r] * now.C[i][r];
        }
        if (LOCAL) dt_sum += now.dt_u[i].x;
        else y_lds[half][j + i][mine] = sum_states<LANES>(ys);  // (the lanes of a channel write the same)
      }
#pragma unroll
      for (int e = j * kEach / TS; e < (j + 2) * kEach / TS; ++e) work_out(raw, t + TS, half ^ 1, e, rest_next);
      __builtin_amdgcn_sched_barrier(0);
      now = next;
    }
    raw.B.put(B_lds[half ^ 1]);
    if (!LOCAL) raw.C.put(C_lds[half ^ 1]);
    raw = coming;
    rest = rest_next;
  }
  if (!LOCAL && t0 < end) {
    __syncthreads();
    const int rows = (end - t0 - 1) % TS + 1;
    put_out(half ^ 1, wide && rows == TS, rows);
  }

  if (LOCAL) {
    if (live) {
      store_states(added + blockIdx.y * states + state, s0, s.S, h);
      if (s0 == 0) sum_dt[((size_t)blockIdx.y * s.N + b.n) * s.D + d] = dt_sum;
    }
    return;
  }
  float fill[L::WIDTH];
#pragma unroll
  for (int e = 0; e < L::WIDTH; ++e) fill[e] = extent.fill;
  for (int t = max(t0, end) + (int)threadIdx.x / L::kPerRow; t < t1; t += L::kRowStep)
    store_channels<L::WIDTH>(y + ((size_t)t * s.N + b.n) * s.D, b.c0 + column, b.c_end, fill);
  if (blockIdx.y + 1 == (unsigned)s.chunks && live && h_last != nullptr) {
    if (extent.fill != 0.f) {  // NaN
#pragma unroll
      for (int r = 0; r < K; ++r) h[r] = extent.fill;
    }
    store_states(h_last + state, s0, s.S, h);
  }
}

// What a backward pass writes besides dB and dC.
template <typename T>
struct ScanGradients {
  T *dx, *ddelta, *dz;  // [T,N,D]; dz null without z
  float* dh0;           // or null
  float* partial;       // [chunks * N][D * S + 2 D]: dA, dD, d delta_bias
  float *dB, *dC;       // [blocks of a group][T][N][G][S]
};

// Backward pass over a chunk.  LOCAL: only G at the chunk's start for a gradient of zero at its end, and
// the sum of dt.  added, sum_dt: as forward, of the chunks but the first.
// EVEN: the channels of a group are a multiple of WIDTH, and a thread's columns aligned to it, which lets LDS move 16 bytes at a
// time; without, T=2048 N=8 D=4096 S=16 bf16 takes 3 % more.
// Two lanes a channel (S up to 8) hold eight elements a thread of each tensor and spill: 36 to 84 bytes a thread in half types, 144 and
// 152 in float.  T=1024 N=8 D=1024 S=8 78 us in bf16 and 110 in float, where S=16 takes 111 and 113.
// A workgroup leaves S floats a step of dB and of dC, written here and read to be added up: 4 bytes an element of x at S=16, with 64
// channels a workgroup, and 64 bytes at S=64, with 16, where adding them up takes 119 us beside 860 (T=2048 N=8 D=1024 bf16).
template <typename T, int LANES, bool LOCAL, bool EVEN>
__global__ __launch_bounds__(256, 2)
void selective_scan_backward_kernel(ScanShape s, ScanInputs<T> in, const float* __restrict__ kept, Rows<const T> dy,
                                    const float* __restrict__ dh_last, float* __restrict__ added, float* __restrict__ sum_dt,
                                    ScanGradients<T> out) {
  typedef Place<LANES> P;
  typedef Tile<LANES> L;
  __shared__ float4_t step_lds[TS][P::kBlock];                // dt, dt x, q = dy silu(z), d dt / d delta
  __shared__ float2_t rest_lds[LOCAL ? 1 : TS][P::kBlock];    // x, dy silu'(z)
  __shared__ float4_t C_lds[TS * LANES], B_lds[LOCAL ? 1 : TS * LANES];
  __shared__ float ypre_lds[LOCAL ? 1 : TS][P::kBlock];
  __shared__ float2_t du_Aw_lds[LOCAL ? 1 : TS][P::kBlock];
  typedef ChannelSums<LANES> Sums;
  constexpr int kParts = 4 * Sums::kParts;  // of the workgroup; 16 floats between them keep rows that write at once in banks of their own
  __shared__ float dB_lds[LOCAL ? 1 : kParts][TS * LANES * K + 16], dC_lds[LOCAL ? 1 : kParts][TS * LANES * K + 16];

  const Block<LANES> b(s, blockIdx.x);
  const int column = EVEN ? L::column(b) / L::WIDTH * L::WIDTH : L::column(b);
  if (b.c_end - b.c0 < P::kBlock) {  // the columns behind the last
    for (int e = threadIdx.x; e < TS * P::kBlock; e += 256) (&step_lds[0][0])[e] = float4_t{0.f, 0.f, 0.f, 0.f};
    __syncthreads();
  }
  const unsigned chunk = blockIdx.y + (LOCAL ? 1 : 0);  // what goes out of the first chunk is found by the second pass
  const int t0 = chunk * s.chunk, t1 = min(s.T, t0 + s.chunk);
  const Extent extent = extent_of(in.lengths, b.n, s.T);
  const int end = min(t1, extent.steps);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, s0 = P::states(lane) * K;
  const int mine = wave * P::kChannels + P::channel(lane);
  const int part = wave * Sums::kParts + Sums::part(lane), summed = s0 + Sums::value(lane);
  const int d = b.c0 + mine;
  const bool live = d < b.c_end;
  const size_t state = ((size_t)b.n * s.D + d) * s.S, states = (size_t)s.N * s.D * s.S;
  const size_t shared_row = (size_t)s.G * s.S;  // of dB, dC

  float A[K], A2[K], G[K], dA[K], dt_sum = 0.f;
#pragma unroll
  for (int r = 0; r < K; ++r) A[r] = A2[r] = G[r] = dA[r] = 0.f;
  if (live) {
    load_states(in.A + (size_t)d * s.S, s0, s.S, A);
    base2_rates(A, A2);
    if (!LOCAL) {
      if (dh_last != nullptr) load_states(dh_last + state, s0, s.S, G);
      if (chunk + 1 < (unsigned)s.chunks)
        join_chunks(G, A2, added, sum_dt, state, states, (size_t)b.n * s.D + d, (size_t)s.N * s.D, s.chunks - 1, -1,
                    s.chunks - 1 - (int)chunk, s0, s.S);
    }
  }
  float bias[L::WIDTH], skip[L::WIDTH], dskip[L::WIDTH], dbias[L::WIDTH];
#pragma unroll
  for (int e = 0; e < L::WIDTH; ++e) bias[e] = skip[e] = dskip[e] = dbias[e] = 0.f;
  if (in.bias != nullptr) load_channels<L::WIDTH>(in.bias, b.c0 + column, b.c_end, bias);
  if (!LOCAL && in.skip != nullptr) load_channels<L::WIDTH>(in.skip, b.c0 + column, b.c_end, skip);

  if (!LOCAL) {
    float fill[L::WIDTH];
#pragma unroll
    for (int e = 0; e < L::WIDTH; ++e) fill[e] = extent.fill;
    for (int t = max(t0, end) + (int)threadIdx.x / L::kPerRow; t < t1; t += L::kRowStep) {
      const size_t at = ((size_t)t * s.N + b.n) * s.D;
      store_channels<L::WIDTH>(out.dx + at, b.c0 + column, b.c_end, fill);
      store_channels<L::WIDTH>(out.ddelta + at, b.c0 + column, b.c_end, fill);
      if (out.dz != nullptr) store_channels<L::WIDTH>(out.dz + at, b.c0 + column, b.c_end, fill);
    }
    const size_t part = (size_t)(blockIdx.x % s.blocks_group) * s.T;
    for (int e = threadIdx.x; e < (t1 - max(t0, end)) * s.S; e += 256) {
      const size_t at = ((part + max(t0, end) + e / s.S) * s.N + b.n) * shared_row + (size_t)b.g * s.S + e % s.S;
      out.dB[at] = out.dC[at] = extent.fill;
    }
  }

  const int last = t0 < end ? t0 + (end - 1 - t0) / TS * TS : t0 - TS;  // the last tile
  Held<T, LANES> x = {}, delta = {}, z = {}, up = {};
  HeldShared<T, LANES> Bt, Ct;
  const int from = max(last, t0);
  Walk<const T, LANES> x_walk(in.x, from, b), delta_walk(in.delta, from, b), z_walk(in.z, from, b), up_walk(dy, from, b);
  WalkShared<T, LANES> B_walk(in.B, from, b, s.S), C_walk(in.C, from, b, s.S);
  Walk<T, LANES> dx_walk(packed_rows(out.dx, s.N, s.D), from, b), ddelta_walk(packed_rows(out.ddelta, s.N, s.D), from, b);
  Walk<T, LANES> dz_walk(packed_rows(out.dz, s.N, s.D), from, b);
  const bool wide = L::wide(b), gated = in.z.p != nullptr;
  float start[K], start_next[K];
  auto fetch = [&](int t) {  // the tile of every walk, which starts at t
    const int rows = end - t;
    const bool whole = wide && rows >= TS;
    if (!LOCAL) {
      x_walk.load(x, whole, rows, b);
      x_walk.back();
    }
    delta_walk.load(delta, whole, rows, b);
    delta_walk.back();
    if (gated) {
      z_walk.load(z, whole, rows, b);
      z_walk.back();
    }
    up_walk.load(up, whole, rows, b);
    up_walk.back();
    C_walk.load(Ct, rows);
    C_walk.back();
    if (!LOCAL) {
      B_walk.load(Bt, rows);
      B_walk.back();
      if (live) load_states(kept + (size_t)(t / TS) * states + state, s0, s.S, start_next);
    }
  };
#pragma unroll
  for (int r = 0; r < K; ++r) start[r] = start_next[r] = 0.f;
  if (last >= t0) fetch(last);
  for (int t = last; t >= t0; t -= TS) {
#pragma unroll
    for (int i = 0; i < L::ITEMS; ++i) {
      const bool inside = t + L::row(i) < end;
#pragma unroll
      for (int e = 0; e < L::WIDTH; ++e) {
        const float xv = x.get(i, e), zv = z.get(i, e), upv = up.get(i, e), sz = sigmoid_of(zv);
        float slope;
        const float dt = step_size(delta.get(i, e) + bias[e], s.softplus, inside, &slope);
        const float q = gated ? upv * (zv * sz) : upv;
        step_lds[L::row(i)][column + e] = float4_t{dt, dt * xv, q, slope};
        if (!LOCAL) rest_lds[L::row(i)][column + e] = float2_t{xv, upv * silu_slope(zv, sz)};
      }
    }
    Ct.put(C_lds);
    if (!LOCAL) Bt.put(B_lds);
#pragma unroll
    for (int r = 0; r < K; ++r) start[r] = start_next[r];
    if (t - TS >= t0) fetch(t - TS);
    __syncthreads();

    if (LOCAL) {
#pragma unroll 4
      for (int j = TS - 1; j >= 0; --j) {
        const float dt = step_lds[j][mine].x, q = step_lds[j][mine].z;
        const float4_t Cv = C_lds[j * LANES + s0 / K];
        dt_sum += dt;
#pragma unroll
        for (int r = 0; r < K; ++r) G[r] = __builtin_amdgcn_exp2f(dt * A2[r]) * (q * Cv[r] + G[r]);
      }
      __syncthreads();
      continue;
    }

    // A step's operands are read from LDS while the step before is computed, and not earlier: the registers are
    // taken by the tile's decays and states.
    struct { float4_t dt_u_q, B, C; } now, next;
    auto read = [&](auto& to, int j) {
      to.dt_u_q = step_lds[j][mine];
      to.B = B_lds[j * LANES + s0 / K];
      to.C = C_lds[j * LANES + s0 / K];
    };
    float a[TS][K], before[TS][K];  // the decays and the states before the steps
    read(now, 0);
#pragma unroll
    for (int j = 0; j < TS; ++j) {
      read(next, j + 1 < TS ? j + 1 : j);
      float ypre = 0.f, dCv[K];
#pragma unroll
      for (int r = 0; r < K; ++r) {
        a[j][r] = __builtin_amdgcn_exp2f(now.dt_u_q.x * A2[r]);
        before[j][r] = start[r];
        start[r] = a[j][r] * start[r] + now.dt_u_q.y * now.B[r];
        ypre += start[r] * now.C[r];
        dCv[r] = now.dt_u_q.z * start[r];
      }
      ypre_lds[j][mine] = sum_states<LANES>(ypre);  // (the lanes of a channel write the same, as do those of a state below)
      dC_lds[part][j * LANES * K + summed] = Sums::sum(dCv);
      __builtin_amdgcn_sched_barrier(0);
      now = next;
    }
    // of the tile by itself: one chain over all steps would be off by sqrt(steps / 3) roundings (dA at T=2048 N=8 D=4096 S=16:
    // 9.9e-7 of it, and 5.8e-7 so; the time is the same)
    float dA_tile[K] = {};
#pragma unroll
    for (int j = TS - 1; j >= 0; --j) {
      if (j > 0) read(next, j - 1);
      float du = 0.f, Aw = 0.f, dBv[K];
#pragma unroll
      for (int r = 0; r < K; ++r) {
        const float g = now.dt_u_q.z * now.C[r] + G[r];
        dBv[r] = g * now.dt_u_q.y;
        du += g * now.B[r];
        G[r] = g * a[j][r];
        const float w = G[r] * before[j][r];
        Aw += w * A[r];
        dA_tile[r] += w * now.dt_u_q.x;
      }
      du_Aw_lds[j][mine] = float2_t{sum_states<LANES>(du), sum_states<LANES>(Aw)};
      dB_lds[part][j * LANES * K + summed] = Sums::sum(dBv);
      __builtin_amdgcn_sched_barrier(0);
      now = next;
    }
#pragma unroll
    for (int r = 0; r < K; ++r) dA[r] += dA_tile[r];
    __syncthreads();

    float dxo[L::ITEMS][L::WIDTH], ddo[L::ITEMS][L::WIDTH], dzo[L::ITEMS][L::WIDTH];
#pragma unroll
    for (int i = 0; i < L::ITEMS; ++i) {
      const int row = L::row(i);
#pragma unroll
      for (int e = 0; e < L::WIDTH; ++e) {
        const float4_t st = step_lds[row][column + e];
        const float2_t rest = rest_lds[row][column + e], du_Aw = du_Aw_lds[row][column + e];
        // (behind the row's end dt, x and q are 0: nothing is added to the sums)
        dxo[i][e] = st.x * du_Aw.x + skip[e] * st.z;
        ddo[i][e] = (rest.x * du_Aw.x + du_Aw.y) * st.w;
        dzo[i][e] = rest.y * (ypre_lds[row][column + e] + skip[e] * rest.x);
        dskip[e] += st.z * rest.x;
        dbias[e] += t + row < end ? ddo[i][e] : 0.f;
      }
    }
    const bool whole = wide && end - t >= TS;
    dx_walk.store(dxo, whole, end - t, b);
    ddelta_walk.store(ddo, whole, end - t, b);
    if (gated) dz_walk.store(dzo, whole, end - t, b);
    dx_walk.back();
    ddelta_walk.back();
    dz_walk.back();
    const size_t part = (size_t)(blockIdx.x % s.blocks_group) * s.T;
    for (int e = threadIdx.x; e < TS * LANES * K; e += 256) {
      const int j = e / (LANES * K), st = e % (LANES * K);
      if (t + j >= end || st >= s.S) continue;
      const size_t at = ((part + t + j) * s.N + b.n) * shared_row + (size_t)b.g * s.S + st;
      float dBv = 0.f, dCv = 0.f;
#pragma unroll
      for (int p = 0; p < kParts; ++p) {
        dBv += dB_lds[p][e];
        dCv += dC_lds[p][e];
      }
      out.dB[at] = dBv;
      out.dC[at] = dCv;
    }
    // No barrier: until the next one a wavefront overwrites only elements that it alone reads here, and B and C, which nobody does.
  }

  if (LOCAL) {
    if (live) {
      store_states(added + chunk * states + state, s0, s.S, G);
      if (s0 == 0) sum_dt[((size_t)chunk * s.N + b.n) * s.D + d] = dt_sum;
    }
    return;
  }
  float* partial = out.partial + ((size_t)chunk * s.N + b.n) * ((size_t)s.D * (s.S + 2));
  if (live) {
    if (chunk == 0 && out.dh0 != nullptr) {
      if (extent.fill != 0.f) {  // NaN
#pragma unroll
        for (int r = 0; r < K; ++r) G[r] = extent.fill;
      }
      store_states(out.dh0 + state, s0, s.S, G);
    }
    store_states(partial + (size_t)d * s.S, s0, s.S, dA);
  }
  // the threads of a column add theirs in order
  static_assert(256 * L::WIDTH <= TS * P::kBlock, "a row a thread of the column fits ypre_lds, and du_Aw_lds");
  float(*skip_sums)[P::kBlock] = ypre_lds;
  float(*bias_sums)[P::kBlock] = reinterpret_cast<float(*)[P::kBlock]>(&du_Aw_lds[0][0]);
  __syncthreads();
#pragma unroll
  for (int e = 0; e < L::WIDTH; ++e) {
    skip_sums[threadIdx.x / L::kPerRow][column + e] = dskip[e];
    bias_sums[threadIdx.x / L::kPerRow][column + e] = dbias[e];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < P::kBlock; e += 256) {
    if (b.c0 + e >= b.c_end) continue;
    float ds = 0.f, db = 0.f;
    for (int r = 0; r < L::kRowStep; ++r) {
      ds += skip_sums[r][e];
      db += bias_sums[r][e];
    }
    partial[(size_t)s.D * s.S + b.c0 + e] = ds;
    partial[(size_t)s.D * (s.S + 1) + b.c0 + e] = db;
  }
}

// dB, dC = the sums of the blocks' parts, rounded.  (More elements than a grid has threads go by turns.)
template <typename T>
__global__ __launch_bounds__(256)
void scan_shared_kernel(int parts, size_t count, const float* __restrict__ dB_parts, const float* __restrict__ dC_parts,
                        T* __restrict__ dB, T* __restrict__ dC) {
  const float* from = blockIdx.y == 0 ? dB_parts : dC_parts;
  T* to = blockIdx.y == 0 ? dB : dC;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (size_t)gridDim.x * 256) {
    float sum = 0.f;
#pragma unroll 8
    for (int p = 0; p < parts; ++p) sum += from[p * count + i];
    to[i] = (T)sum;
  }
}

// A single step: LANES neighbouring lanes a channel, its states in and out as whole lines.  Bound by those lines' bytes, or by
// latency.  What is the channel's (A and the like) is read once for the rows a workgroup goes through, and a row's elements
// are on their way while the row before is computed: N=128 D=4096 S=16 bf16, 72 MB, 19.1 us with a thread a row.
template <typename T, int LANES>
__global__ __launch_bounds__(256)
void selective_scan_step_kernel(ScanShape s, ScanInputs<T> in, const float* h, float* h_out, T* __restrict__ y) {
  const unsigned i = blockIdx.x * 256 + threadIdx.x, d = i / LANES, s0 = i % LANES * K;
  if (d >= (unsigned)s.D) return;  // (the lanes of a channel together)
  const size_t shared = (size_t)(d / s.share.channels) * s.S;
  float A[K], A2[K];
  load_states(in.A + (size_t)d * s.S, s0, s.S, A);
  base2_rates(A, A2);
  const float bias = in.bias != nullptr ? in.bias[d] : 0.f, skip = in.skip != nullptr ? in.skip[d] : 0.f;
  const bool gated = in.z.p != nullptr;

  struct Row {
    float h[K], B[K], C[K], x, delta, z;
  } coming;
  auto fetch = [&](int n) {
    load_states(h + ((size_t)n * s.D + d) * s.S, s0, s.S, coming.h);
    load_channels<K>(in.B.at(0, n) + shared, s0, s.S, coming.B);
    load_channels<K>(in.C.at(0, n) + shared, s0, s.S, coming.C);
    coming.x = (float)in.x.at(0, n)[d];
    coming.delta = (float)in.delta.at(0, n)[d];
    coming.z = gated ? (float)in.z.at(0, n)[d] : 0.f;
  };
  fetch(blockIdx.y);
  for (int n = blockIdx.y; n < s.N; n += gridDim.y) {
    Row now = coming;
    if (n + (int)gridDim.y < s.N) fetch(n + gridDim.y);
    const float dt = step_size(now.delta + bias, s.softplus, true), u = dt * now.x;
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < K; ++r) {
      now.h[r] = __builtin_amdgcn_exp2f(dt * A2[r]) * now.h[r] + u * now.B[r];
      sum += now.h[r] * now.C[r];
    }
    store_states(h_out + ((size_t)n * s.D + d) * s.S, s0, s.S, now.h);
    if (LANES >= 2) sum += dpp<kXor1>(sum);
    if (LANES >= 4) sum += dpp<kXor2>(sum);
    if (LANES >= 8) sum += dpp<kHalfMirror>(sum);
    if (LANES >= 16) sum += dpp<kRor8>(sum);
    sum += skip * now.x;
    sum = gated ? sum * (now.z * sigmoid_of(now.z)) : sum;
    if (s0 == 0) y[(size_t)n * s.D + d] = (T)sum;
  }
}

int lanes_for(int S) { return S <= 8 ? 2 : S <= 16 ? 4 : S <= 32 ? 8 : 16; }

template <typename F>
int with_lanes(int S, F&& f) {
  switch (lanes_for(S)) {
    case 2: return f(std::integral_constant<int, 2>());
    case 4: return f(std::integral_constant<int, 4>());
    case 8: return f(std::integral_constant<int, 8>());
    default: return f(std::integral_constant<int, 16>());
  }
}

size_t blocks_of(const ScanShape& s) { return (size_t)s.N * s.G * s.blocks_group; }

// The time axis is cut where rows and channels make too few workgroups, into chunks that make about two a CU, of no fewer than 4
// tiles, and of no more than so many that joining them (a memory round trip for every four) takes the time of the steps saved:
// 3 sqrt(tiles), T=8192 N=1 D=128 and T=32768 N=1 D=64 forward 46 and 110 us with 64 chunks, 55 and 85 with 128, 54 and 158 with 512.
// The first of the two passes costs two thirds of the second.  Forward that is not won back by two chunks: one and two with T=2048
// N=4 D=4096 S=16 bf16 (256 workgroups) 244 and 254 us, T=128 N=32 D=512 18 and 22.  Backward, where it costs two fifths,
// it is: 680 and 559, 53 and 50.
// From 257 workgroups on there is one chunk.  The backward pass has room for two workgroups a CU (LDS and registers), so that 257
// to 512 of them take about the time of 512, and a few more those of another round: T=2048 D=4096 S=16 bf16 backward 434 + 131 us at
// N=4 (two chunks), 844 to 848 at N=5, 6 and 8, 1366 at N=9.
ScanShape shape_of(int T, int N, int D, int S, int G, int softplus, bool backward) {
  const int block = 256 / lanes_for(S), workgroups = (D / G + block - 1) / block;
  ScanShape s = {T, N, D, S, G, workgroups, {D / G, workgroups}, 0, 0, softplus};
  const size_t blocks = blocks_of(s), tiles = ((size_t)T + TS - 1) / TS;
  const size_t least = backward ? 2 : 3, most = tiles / 4, join = (size_t)(3.0 * std::sqrt((double)tiles));
  size_t chunks = 2 * (size_t)device_cu_count() / blocks;
  chunks = chunks < most ? chunks : most;
  chunks = chunks < join ? chunks : join;
  if (chunks < least) chunks = 1;
  s.chunk = (int)((tiles + chunks - 1) / chunks) * TS;
  s.chunks = (int)(((size_t)T + s.chunk - 1) / s.chunk);
  return s;
}

// For the calls and for the size of their workspace alike.
int check_grid(const ScanShape& s) {
  if (blocks_of(s) > kGridLimit || (size_t)s.chunks > kGridLimitYZ) return too_large("selective_scan: too many rows of channels");
  return HASTE_HIP_OK;
}

// Floats of workspace, in the order they lie there.
struct ScanWorkspace {
  size_t added, sum_dt, partial, sums, dB, dC, total;
};
ScanWorkspace forward_workspace(const ScanShape& s) {
  ScanWorkspace w = {};
  if (s.chunks > 1) {
    w.sum_dt = (size_t)s.chunks * s.N * s.D * s.S;
    w.total = w.sum_dt + (size_t)s.chunks * s.N * s.D;
  }
  return w;
}
ScanWorkspace backward_workspace(const ScanShape& s) {
  ScanWorkspace w = forward_workspace(s);
  const size_t parts = (size_t)s.chunks * s.N, columns = (size_t)s.D * (s.S + 2);
  w.partial = w.total;
  w.sums = w.partial + parts * columns;
  w.dB = w.sums + column_sums_scratch(parts, columns);
  w.dC = w.dB + (size_t)s.blocks_group * s.T * s.N * s.G * s.S;
  w.total = w.dC + (w.dC - w.dB);
  return w;
}

template <typename T>
int forward(hipStream_t stream, const ScanShape& s, const ScanInputs<T>& in, const float* h0, T* y, float* h_last, float* kept,
            float* workspace, size_t workspace_bytes) {
  const size_t blocks = blocks_of(s);
  const ScanWorkspace w = forward_workspace(s);
  HASTE_HIP_PROPAGATE(check_grid(s));
  if (workspace_bytes < w.total * sizeof(float)) return too_large("selective_scan_forward: the workspace is too small");
  HASTE_HIP_REQUIRE(workspace != nullptr || w.total == 0);
  float *added = workspace, *sum_dt = s.chunks > 1 ? workspace + w.sum_dt : nullptr;
  return with_lanes(s.S, [&](auto lanes) {
    dim3 grid((unsigned)blocks, s.chunks);
    if (s.chunks > 1) {
      ScopedKernelTimer timer("selective_scan_chunks", stream);
      selective_scan_forward_kernel<T, lanes(), true><<<dim3(grid.x, grid.y - 1), 256, 0, stream>>>(s, in, nullptr, added, sum_dt, nullptr, nullptr, nullptr);
      HASTE_HIP_TRY(hipGetLastError());
    }
    ScopedKernelTimer timer("selective_scan_forward", stream);
    selective_scan_forward_kernel<T, lanes(), false><<<grid, 256, 0, stream>>>(s, in, h0, added, sum_dt, kept, y, h_last);
    HASTE_HIP_TRY(hipGetLastError());
    return HASTE_HIP_OK;
  });
}

template <typename T>
int backward(hipStream_t stream, const ScanShape& s, const ScanInputs<T>& in, const float* kept, const Rows<const T>& dy,
             const float* dh_last, T* dx, T* ddelta, float* dA, T* dB, T* dC, float* dskip, T* dz, float* dbias, float* dh0,
             float* workspace, size_t workspace_bytes) {
  const size_t blocks = blocks_of(s);
  const size_t shared = (size_t)s.T * s.N * s.G * s.S, columns = (size_t)s.D * (s.S + 2);
  const ScanWorkspace w = backward_workspace(s);
  HASTE_HIP_PROPAGATE(check_grid(s));
  if (workspace_bytes < w.total * sizeof(float)) return too_large("selective_scan_backward: the workspace is too small");
  float *added = workspace + w.added, *sum_dt = workspace + w.sum_dt;
  const ScanGradients<T> out = {dx, ddelta, dz, dh0, workspace + w.partial, workspace + w.dB, workspace + w.dC};
  auto launch = [&](auto lanes, auto even) {
    dim3 grid((unsigned)blocks, s.chunks);
    if (s.chunks > 1) {
      ScopedKernelTimer timer("selective_scan_chunks", stream);
      selective_scan_backward_kernel<T, lanes(), true, even()><<<dim3(grid.x, grid.y - 1), 256, 0, stream>>>(s, in, nullptr, dy, dh_last, added, sum_dt, out);
      HASTE_HIP_TRY(hipGetLastError());
    }
    ScopedKernelTimer timer("selective_scan_backward", stream);
    selective_scan_backward_kernel<T, lanes(), false, even()><<<grid, 256, 0, stream>>>(s, in, kept, dy, dh_last, added, sum_dt, out);
    HASTE_HIP_TRY(hipGetLastError());
    return HASTE_HIP_OK;
  };
  HASTE_HIP_PROPAGATE(with_lanes(s.S, [&](auto lanes) {
    if constexpr (Tile<lanes()>::WIDTH > 1) {
      if (s.share.channels % Tile<lanes()>::WIDTH != 0) return launch(lanes, std::false_type());
    }
    return launch(lanes, std::true_type());
  }));
  {
    ScopedKernelTimer timer("selective_scan_shared", stream);
    const size_t groups = (shared + 255) / 256;
    scan_shared_kernel<T><<<dim3((unsigned)(groups < kGridLimit ? groups : kGridLimit), 2), 256, 0, stream>>>(s.blocks_group, shared, out.dB, out.dC, dB, dC);
    HASTE_HIP_TRY(hipGetLastError());
  }
  const size_t first = (size_t)s.D * s.S;
  const ColumnOutputs to = {{dA, dskip, dbias, nullptr}, {first, first + s.D, columns, columns}};
  return column_sums(stream, (size_t)s.chunks * s.N, columns, out.partial, workspace + w.sums, to);
}

int check_sizes(int T, int N, int D, int S, int G) {
  HASTE_HIP_REQUIRE(T > 0 && N > 0 && D > 0 && S > 0 && G > 0 && D % G == 0);
  if (S > kMaxStates) return too_large("selective_scan: up to 64 states a channel are implemented");
  if (T > kSizeLimit || N > kSizeLimit || D > kSizeLimit / (kMaxStates + 2)) return too_large("selective_scan: sizes beyond 2^30");
  return HASTE_HIP_OK;
}

template <typename T>
ScanInputs<T> inputs_of(const void* x, size_t x_step, size_t x_row, const void* delta, size_t delta_step, size_t delta_row,
                        const float* A, const void* B, size_t B_step, size_t B_row, const void* C, size_t C_step, size_t C_row,
                        const float* D, const void* z, size_t z_step, size_t z_row, const float* delta_bias,
                        const void* lengths) {
  return {{static_cast<const T*>(x), x_step, x_row}, {static_cast<const T*>(delta), delta_step, delta_row},
          {static_cast<const T*>(B), B_step, B_row}, {static_cast<const T*>(C), C_step, C_row},
          {static_cast<const T*>(z), z_step, z_row}, A, D, delta_bias, static_cast<const long long*>(lengths)};
}

template <typename T>
int step(hipStream_t stream, int N, int D, int S, int G, int softplus, const ScanInputs<T>& in, const float* h, T* y,
         float* h_out) {
  const ScanShape s = {1, N, D, S, G, 1, {D / G, 1}, TS, 1, softplus};
  return with_lanes(S, [&](auto lanes) {
    const size_t across = ((size_t)D * lanes() + 255) / 256;  // at most 2^22: D is at most 2^30 / 66
    if (across > kGridLimit) return too_large("selective_scan: too many channels");
    const size_t wanted = (size_t)device_cu_count() * 8 / across;  // workgroups that fill the chip, per 256 lanes
    const size_t down = wanted < 1 ? 1 : wanted < (size_t)N ? wanted : (size_t)N;
    ScopedKernelTimer timer("selective_scan_iterate", stream);
    selective_scan_step_kernel<T, lanes()><<<dim3((unsigned)across, (unsigned)down), 256, 0, stream>>>(s, in, h, h_out, y);
    HASTE_HIP_TRY(hipGetLastError());
    return HASTE_HIP_OK;
  });
}

}  // namespace
}  // namespace haste_hip

extern "C" {

using namespace haste_hip;

size_t haste_hip_selective_scan_workspace_bytes(int backward, int steps, int batch_size, int channels, int states, int groups) {
  if (check_sizes(steps, batch_size, channels, states, groups) != HASTE_HIP_OK) return 0;
  const ScanShape s = shape_of(steps, batch_size, channels, states, groups, 0, backward != 0);
  if (check_grid(s) != HASTE_HIP_OK) return 0;
  return (backward ? backward_workspace(s) : forward_workspace(s)).total * sizeof(float);
}

size_t haste_hip_selective_scan_kept_bytes(int steps, int batch_size, int channels, int states) {
  if (check_sizes(steps, batch_size, channels, states, 1) != HASTE_HIP_OK) return 0;
  return (size_t)((steps + TS - 1) / TS) * batch_size * channels * states * sizeof(float);
}

#define HASTE_HIP_SCAN_INPUTS                                                                                          \
  const void *x, size_t x_step, size_t x_row, const void *delta, size_t delta_step, size_t delta_row, const float *A,  \
      const void *B, size_t B_step, size_t B_row, const void *C, size_t C_step, size_t C_row, const float *D,          \
      const void *z, size_t z_step, size_t z_row, const float *delta_bias, int delta_softplus

#define HASTE_HIP_SELECTIVE_SCAN(SUFFIX, T)                                                                            \
  int haste_hip_selective_scan_forward_##SUFFIX(int steps, int batch_size, int channels, int states, int groups,       \
                                                HASTE_HIP_SCAN_INPUTS, const float* h0, const void* lengths, void* y,  \
                                                float* h_last, float* kept, void* workspace, size_t workspace_bytes,   \
                                                void* stream) {                                                        \
    HASTE_HIP_PROPAGATE(check_sizes(steps, batch_size, channels, states, groups));                                     \
    HASTE_HIP_REQUIRE(x && delta && A && B && C && y);                                                                 \
    return forward<T>(as_stream(stream), shape_of(steps, batch_size, channels, states, groups, delta_softplus, false), \
                      inputs_of<T>(x, x_step, x_row, delta, delta_step, delta_row, A, B, B_step, B_row, C, C_step,     \
                                   C_row, D, z, z_step, z_row, delta_bias, lengths),                                   \
                      h0, static_cast<T*>(y), h_last, kept, static_cast<float*>(workspace), workspace_bytes);          \
  }                                                                                                                    \
  int haste_hip_selective_scan_backward_##SUFFIX(                                                                      \
      int steps, int batch_size, int channels, int states, int groups, HASTE_HIP_SCAN_INPUTS, const void* lengths,     \
      const float* kept, const void* dy, size_t dy_step, size_t dy_row, const float* dh_last, void* dx, void* ddelta,  \
      float* dA, void* dB, void* dC, float* dD, void* dz, float* ddelta_bias, float* dh0, void* workspace,             \
      size_t workspace_bytes, void* stream) {                                                                          \
    HASTE_HIP_PROPAGATE(check_sizes(steps, batch_size, channels, states, groups));                                     \
    HASTE_HIP_REQUIRE(x && delta && A && B && C && kept && dy && dx && ddelta && dA && dB && dC && workspace);         \
    HASTE_HIP_REQUIRE((z == nullptr) == (dz == nullptr));                                                              \
    return backward<T>(as_stream(stream), shape_of(steps, batch_size, channels, states, groups, delta_softplus, true), \
                       inputs_of<T>(x, x_step, x_row, delta, delta_step, delta_row, A, B, B_step, B_row, C, C_step,    \
                                    C_row, D, z, z_step, z_row, delta_bias, lengths),                                  \
                       kept, {static_cast<const T*>(dy), dy_step, dy_row}, dh_last, static_cast<T*>(dx),               \
                       static_cast<T*>(ddelta), dA, static_cast<T*>(dB), static_cast<T*>(dC), dD, static_cast<T*>(dz), \
                       ddelta_bias, dh0, static_cast<float*>(workspace), workspace_bytes);                             \
  }                                                                                                                    \
  int haste_hip_selective_scan_iterate_##SUFFIX(                                                                       \
      int batch_size, int channels, int states, int groups, const void* x, size_t x_row, const void* delta,            \
      size_t delta_row, const float* A, const void* B, size_t B_row, const void* C, size_t C_row, const float* D,      \
      const void* z, size_t z_row, const float* delta_bias, int delta_softplus, const float* h, void* y, float* h_out, \
      void* stream) {                                                                                                  \
    HASTE_HIP_PROPAGATE(check_sizes(1, batch_size, channels, states, groups));                                         \
    HASTE_HIP_REQUIRE(x && delta && A && B && C && h && y && h_out);                                                   \
    return step<T>(as_stream(stream), batch_size, channels, states, groups, delta_softplus,                            \
                   inputs_of<T>(x, 0, x_row, delta, 0, delta_row, A, B, 0, B_row, C, 0, C_row, D, z, 0, z_row,         \
                                delta_bias, nullptr),                                                                  \
                   h, static_cast<T*>(y), h_out);                                                                      \
  }

HASTE_HIP_SELECTIVE_SCAN(f32, float)
HASTE_HIP_SELECTIVE_SCAN(f16, _Float16)
HASTE_HIP_SELECTIVE_SCAN(bf16, __bf16)

}  // extern "C"
