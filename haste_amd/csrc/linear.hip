// A projection with what follows it: y[R,D] = act(x[R,C] W[C,D] + bias) + residual, and its gradients
//   d = dy act'(pre),  dx = d W^T,  dW = x^T d,  dbias = sum over rows of d.
// act: none, gelu (v Phi(v), Phi the normal distribution function) or silu (v sigmoid(v)).
//
// Half types (f16, bf16).  Bound: the matrix cores (2 R C D flops, dense peak 2.5 PFLOP/s); below some hundred rows the bytes
// of W.  Products of the matrix cores are exact, sums are float from the first to the last; an output is rounded once.  d is rounded to
// the activations' type, the matrix cores take no other: what it costs is a rounding of each term of sums that are rounded
// to that type themselves.  act'(pre) is what the forward pass leaves for the backward pass, beside bf16 in half: it lies between -0.2 and
// 1.2, where half is eight times as fine as bfloat16, and a float would be as many bytes again as y.  Beside f16 it is a float: rounded to
// half it would cost as much precision as d (dx and dW 2.9e-4 off by the 2-norm instead of 3.7e-4, where 2.1e-4 is the results' own rounding).
//
// One tile kernel makes all three products.  An operand is either stored with the contraction index contiguous (x and d in
// x W and d W^T, W in d W^T) or with it as the slow index (W in x W, x and d in x^T d).  Tiles go from memory straight into LDS
// (buffer loads that write LDS: no registers, no wait in between), two stages of BK of the contraction: while one is multiplied the next
// is on its way, and what has been read of the first is replaced piece by piece.  A contiguous operand lies in LDS as rows of BK elements,
// 16-byte chunk c of row r at position c ^ turn(r), so that 16 rows of one chunk cover all banks; an operand of the instruction is one
// 16-byte read.  A slow one lies as rows of k, 32-byte piece g of row k at g ^ turn_slow(k), and is read transposed (ds_read_b64_tr_b16: in
// each 16 lanes, lane i receives element i % 4 of what lanes i / 4 + 4 j address).  Loads beyond an operand's end give zeros.
// Tiles of 256 x 256 halve what the L2s have to deliver (at 128 x 128 it is their rate that bounds); bands of kTallest of them, gone through
// column by column, keep what an XCD works on in its L2.  bf16, x W / d W^T / x^T d of R x C x D, us (TFLOP/s):
//   16384 x 4096 x 4096   406 (1353) / 390 (1410) / 411 (1339)   tiles of 128 x 128   498 / 462 / 527   kTallest 1   429 / 421 / 431
//    4096 x 4096 x 4096   103 (1336) / 100 (1374) / 104 (1319)                        124 / 116 / 136                105 / 101 / 105
//    8192 x 1024 x 2048    32 (1061) /  33 (1053) /  48 (719)                          37 /  33 /  48                 32 /  33 /  47
// (kTallest 32: 431 / 417 / 404 of the first).  The matrix cores are busy for 71 to 80 % of the cycles, at the 1.75 to 1.9 GHz that are left of
// the clock under this load.
// Operands that are not laid out in 16-byte pieces are copied once, rows padded with zeros: unaligned 16-byte loads are two to four
// times as slow (8191 x 2047 x 1023 through registers 96 us, with copies 50).
//
// Float: large products by gemm.hip (the bf16 matrix cores on floats split in three: 190 TFLOP/s), with a pass for what follows them;
// small ones by the tile kernel, with the float instruction.
#include <cmath>
#include <type_traits>

#include "sequence.h"

namespace haste_hip {
namespace {

typedef float float4_t __attribute__((ext_vector_type(4)));
typedef unsigned int uint4_t __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));

enum Activation { kNone, kGelu, kSilu };

// Phi(v) and e = exp(-v^2 / 2) for halves: Phi(-x) = t P(t) e with t = 1 / (1 + 0.3 x / sqrt 2) for x >= 0, P the polynomial of
// degree 8 with the least largest relative error, 4e-8 (fitted to exp(x^2) erfc(x) over 0 <= x <= 14).  For floats the library's
// function, whose last bits are right too.
template <typename T>
__device__ __forceinline__ float normal_below(float v, float& e) {
  e = __builtin_amdgcn_exp2f(v * v * -0.72134752044f);
  if constexpr (sizeof(T) == 4) return 0.5f * erfcf(v * -0.70710678119f);
  const float t = __builtin_amdgcn_rcpf(1.0f + 0.21213203436f * fabsf(v));
  float p = -6.330811700e-02f;
  p = p * t + 2.359122957e-01f;
  p = p * t - 2.423442380e-01f;
  p = p * t + 2.585225439e-01f;
  p = p * t - 3.702330108e-02f;
  p = p * t + 1.031920523e-01f;
  p = p * t + 7.523456362e-02f;
  p = p * t + 8.521184213e-02f;
  p = p * t + 8.460237762e-02f;
  const float below = p * t * e;
  return v < 0.f ? below : 1.0f - below;
}

// act(v), and its slope.
template <typename T>
__device__ __forceinline__ float activated(int act, float v, float& slope) {
  if (act == kGelu) {
    float e;
    const float below = normal_below<T>(v, e);
    slope = below + v * e * 0.39894228040f;
    return v * below;
  }
  if (act == kSilu) {
    const float s = sigmoid_of(v);
    slope = silu_slope(v, s);
    return v * s;
  }
  slope = 1.0f;
  return v;
}

// What becomes of a product's elements.
template <typename T>
struct Finish {
  typedef typename std::conditional<std::is_same<T, __bf16>::value, _Float16, float>::type slope_t;
  T* out;
  size_t ld;
  int act;
  const T* bias;                                                              // may be null, like the rest
  const T* residual;
  size_t residual_ld;
  slope_t* slope;                                                             // [rows][columns]
};

// Eight neighbouring elements of a row, with the bias of their columns.
template <typename T>
__device__ __forceinline__ void finish(const Finish<T>& to, float (&v)[8], const float (&bias)[8], size_t row, int col, int columns) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] += bias[i];
  if (to.act != kNone) {
    float slope[8];
    if (to.act == kGelu) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = activated<T>(kGelu, v[i], slope[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = activated<T>(kSilu, v[i], slope[i]);
    }
    if (to.slope != nullptr) store_channels<8>(to.slope + row * columns, col, columns, slope);
  }
  if (to.residual != nullptr) {
    float r[8];
    load_channels<8>(to.residual + row * to.residual_ld, col, columns, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += r[i];
  }
  store_channels<8>(to.out + row * to.ld, col, columns, v);
}

template <typename T>
__device__ __forceinline__ void load_bias(const Finish<T>& to, int col, int columns, float (&bias)[8]) {
  if (to.bias != nullptr) {
    load_channels<8>(to.bias, col, columns, bias);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) bias[i] = 0.f;
  }
}

// ---- the tile kernel ---------------------------------------------------------------------
__device__ __forceinline__ float4_t mfma(_Float16, uint4_t a, uint4_t b, float4_t c) {
  typedef _Float16 v __attribute__((ext_vector_type(8)));
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v, a), __builtin_bit_cast(v, b), c, 0, 0, 0);
}
__device__ __forceinline__ float4_t mfma(__bf16, uint4_t a, uint4_t b, float4_t c) {
  typedef __bf16 v __attribute__((ext_vector_type(8)));
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v, a), __builtin_bit_cast(v, b), c, 0, 0, 0);
}

constexpr int kStageBytes = 128;                // of the contraction in a stage: whole cache lines
constexpr int BK = 64;                          // of halves; pieces of a product are cut at multiples of it
constexpr unsigned int kNowhere = 0x7ffffff0u;  // an offset beyond any resource: the load gives zeros

__device__ __forceinline__ uint4_t resource(const void* base, long long bytes) {
  const unsigned long long a = reinterpret_cast<unsigned long long>(base);
  const long long most = 0x7fffffe0ll;
  return uint4_t{(unsigned)a, (unsigned)(a >> 32) & 0xffffu, (unsigned)(bytes < 0 ? 0 : bytes < most ? bytes : most), 0x00020000u};
}

// 16 bytes a lane from the resource into LDS at `lds` and the 1008 bytes behind it, lane by lane.  The load has no register
// to write; it is waited for by count, in tile_ready().  m0 is named, so that the compiler does not take what it put there for what is there still
// (its warning is that it does not save what the register holds, which is right).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(unsigned lds, unsigned offset, uint4_t from, unsigned shift) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(offset), "s"(from),
               "s"(shift)
               : "memory", "m0");
}
#pragma clang diagnostic pop

// Waits until at most LEFT of this wavefront's loads are on their way and all its reads of LDS have returned, then for the others.
template <int LEFT>
__device__ __forceinline__ void tile_ready() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

// Waits for this wavefront's reads of LDS, then for the others'.
__device__ __forceinline__ void all_have_read() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// What is written before stays before.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

// One operand's part of a stage: WIDTH rows (columns) of the product, kStageBytes of the contraction in elements of E bytes, loaded by
// WAVES wavefronts.
template <int E, bool SLOW, int WIDTH, int WAVES>
struct Panel {
  static constexpr int kBytes = WIDTH * kStageBytes, kChunk = 16 / E;  // elements of 16 bytes
  static constexpr int kLoads = kBytes / 1024 / WAVES;  // of a wavefront
  static_assert(kLoads * 1024 * WAVES == kBytes && WAVES % 2 == 0, "a stage is loaded in whole kilobytes");
  static __device__ __forceinline__ int turn(int row) { return (row >> 1) & 7; }
  static constexpr int kPiece = E == 2 ? 32 : 64;  // bytes of 16 neighbours, which are read together
  static __device__ __forceinline__ int turn_slow(int k) {
    if (E == 4) return (k >> 2) & 3;                                               // four rows of k at once, four apart
    return WIDTH == 64 ? (k & 2) + ((k >> 3) & 1) : 2 * (k & 3) + ((k >> 3) & 1);  // (rows of 128 bytes: two lie side by side)
  }

  const char* base;
  long long ld_bytes;
  unsigned offset[kLoads];
  int columns;     // SLOW: those from the tile's first on, in whole chunks (a load that ends beyond a resource loses its last elements)
  unsigned chunk;  // contiguous: the lane's first k of a stage
  uint4_t from;    // what the stage in hand is loaded from
  unsigned shift;
  bool gone;

  // first: of the tile's rows (columns), of `count` in all.
  __device__ __forceinline__ void start(const void* p, long long ld, int first, int count, int k_end, int wave, int lane) {
    ld_bytes = ld * E;
    shift = 0;
    gone = false;
    const int left = count - first;
    if constexpr (SLOW) {
      base = static_cast<const char*>(p) + (size_t)first * E;
      columns = (left + kChunk - 1) & ~(kChunk - 1);
      constexpr int LANES = WIDTH / kChunk, ROWS = 64 / LANES, CHUNKS = kPiece / 16;  // lanes of a row of k, rows of a load, loads of a piece
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int k = (i * WAVES + wave) * ROWS + lane / LANES, unit = lane % LANES;
        const int column = ((unit / CHUNKS) ^ turn_slow(k)) * 16 + unit % CHUNKS * kChunk;
        offset[i] = column < left ? (unsigned)(k * ld_bytes + column * E) : kNowhere;
      }
    } else {
      base = static_cast<const char*>(p) + (size_t)first * ld_bytes;
      const int rows = left < WIDTH ? left : WIDTH;
      from = resource(base, (rows - 1) * ld_bytes + (long long)((k_end + kChunk - 1) & ~(kChunk - 1)) * E);
      const int in_load = lane / 8;  // a load's eight rows start at a multiple of 8 that has the wavefront's parity
      chunk = ((lane % 8) ^ turn(in_load + 8 * (wave & 1))) * kChunk;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row = (i * WAVES + wave) * 8 + in_load;
        offset[i] = row < rows ? (unsigned)(row * ld_bytes + chunk * E) : kNowhere;
      }
    }
  }
  // The stage that starts at k0, and load i of it into LDS at `lds`.
  __device__ __forceinline__ void stage(int k0, int k_end) {
    if constexpr (SLOW) {
      from = resource(base + k0 * ld_bytes, (long long)(k_end - k0 - 1) * ld_bytes + (long long)columns * E);
    } else {
      shift = (unsigned)k0 * E;
      gone = k0 + (int)chunk >= k_end;
    }
  }
  __device__ __forceinline__ void load(int i, unsigned lds, int wave) const {
    load_to_lds(lds + (i * WAVES + wave) * 1024, !SLOW && gone ? kNowhere : offset[i], from, shift);
  }
  // 16 bytes of k of row (column) `first` + lane % 16: those from kChunk (4 half + lane / 16) on.
  static __device__ __forceinline__ uint4_t operand(const char* stage, int first, int half, int lane) {
    if constexpr (SLOW && E == 4) {
      uint4_t v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = 16 * half + 4 * (lane >> 4) + e;
        v[e] = *reinterpret_cast<const unsigned*>(stage + k * (WIDTH * 4) + ((first >> 4) ^ turn_slow(k)) * kPiece + (lane & 15) * 4);
      }
      return v;
    } else if constexpr (SLOW) {
      uint4_t v;
      const int q = lane >> 4, i = lane & 15;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = 32 * half + 8 * q + 4 * h + (i >> 2);
        const int piece = (first >> 4) ^ turn_slow(k);
        typedef __attribute__((address_space(3))) short4_t* lds_t;
        const short4_t part = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(stage + k * (WIDTH * 2) + piece * 32 + (i & 3) * 8));
        __builtin_memcpy(reinterpret_cast<char*>(&v) + 8 * h, &part, 8);
      }
      return v;
    } else {
      const int row = first + (lane & 15), c = 4 * half + (lane >> 4);
      return *reinterpret_cast<const uint4_t*>(stage + row * kStageBytes + (c ^ turn(row)) * 16);
    }
  }
};

template <int E, bool A_SLOW_, bool B_SLOW_, int BM_, int BN_, int WAVES_M_, int WAVES_N_, int STAGES_ = 2>
struct Tile {
  static constexpr int STAGES = STAGES_, ON_A_SIMD = STAGES == 2 ? 2 : 3;  // wavefronts that registers and LDS leave room for
  static constexpr bool A_SLOW = A_SLOW_, B_SLOW = B_SLOW_;
  static constexpr int BM = BM_, BN = BN_, WAVES_M = WAVES_M_, WAVES_N = WAVES_N_, WAVES = WAVES_M * WAVES_N;
  static constexpr int MI = BM / WAVES_M / 16, NJ = BN / WAVES_N / 16;  // of 16 x 16 elements
  typedef Panel<E, A_SLOW, BM, WAVES> PA;
  typedef Panel<E, B_SLOW, BN, WAVES> PB;
  static constexpr int kStage = PA::kBytes + PB::kBytes;
  static constexpr int kSlabLd = NJ * 16 + 4;           // floats of a row of a wavefront's results in LDS
  static constexpr int kSlabs = WAVES * 32 * kSlabLd * 4;
  static constexpr int kLds = STAGES * kStage > kSlabs ? STAGES * kStage : kSlabs;
};

struct Product {
  int M, N, K;
  const void *A, *B;
  long long lda, ldb;
  int tiles_m, tiles_n, k_per_piece;  // tiles whole, or cut along K
  float* partial;                     // [piece][M][N to whole eights], null: whole
};
__host__ __device__ constexpr long long eights(long long n) { return (n + 7) / 8 * 8; }

// Workgroups go to the XCDs in turn; each XCD is given a range of a product's work.
__device__ __forceinline__ unsigned work_of_xcd(unsigned block, unsigned blocks) {
  const unsigned each = blocks >> 3, rest = blocks & 7, xcd = block & 7;
  return xcd * each + (xcd < rest ? xcd : rest) + (block >> 3);
}

constexpr int kTallest = 8;  // rows of tiles that are gone through side by side

template <typename T, class G>
__device__ __forceinline__ void store_tile(char* lds, const Product& p, const Finish<T>& to, const float4_t (&acc)[G::MI][G::NJ], int piece, int m0,
                                           int n0) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / G::WAVES_N * (G::MI * 16), wn = wave % G::WAVES_N * (G::NJ * 16);
  // 32 rows of a wavefront's results at a time go through LDS, so that a lane has eight neighbouring elements of a row.
  float* slab = reinterpret_cast<float*>(lds) + wave * 32 * G::kSlabLd;
  constexpr int LANES = G::NJ * 2, ROWS = 64 / LANES;  // lanes of a row, rows at a time
  const int col = n0 + wn + lane % LANES * 8;
  float bias[8];
  if (p.partial == nullptr) load_bias(to, col, p.N, bias);
#pragma unroll
  for (int i = 0; i < G::MI / 2; ++i) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < G::NJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          slab[(16 * h + 4 * (lane >> 4) + e) * G::kSlabLd + 16 * j + (lane & 15)] = acc[2 * i + h][j][e];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll 2
    for (int r = 0; r < 32; r += ROWS) {
      const int in_slab = r + lane / LANES, row = m0 + wm + 32 * i + in_slab;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = slab[in_slab * G::kSlabLd + lane % LANES * 8 + e];
      if (row < p.M) {
        if (p.partial != nullptr) store_channels<8>(p.partial + ((size_t)piece * p.M + row) * eights(p.N), col, (int)eights(p.N), v);
        else finish(to, v, bias, row, col, p.N);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// What a workgroup has to do.
struct Work {
  int piece, m0, n0, k_begin, k_end;
};
template <class G>
__device__ __forceinline__ Work work_of(const Product& p, unsigned turn) {
  const unsigned tiles = (unsigned)p.tiles_m * p.tiles_n;  // it goes through blocks of them that share rows of A and columns of B
  const int piece = turn / tiles, tile = turn % tiles;
  const int band = tile / (kTallest * p.tiles_n), in_band = tile % (kTallest * p.tiles_n);
  const int tall = p.tiles_m - band * kTallest < kTallest ? p.tiles_m - band * kTallest : kTallest;
  const int k_begin = piece * p.k_per_piece;
  return {piece, (band * kTallest + in_band % tall) * G::BM, in_band / tall * G::BN, k_begin,
          k_begin + p.k_per_piece < p.K ? k_begin + p.k_per_piece : p.K};
}

template <typename T, class G>
__device__ __forceinline__ void multiply_tile(char* lds, const Product& p, const Finish<T>& to, unsigned turn) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Work work = work_of<G>(p, turn);
  const int k_begin = work.k_begin, k_end = work.k_end;
  const int wm = wave / G::WAVES_N * (G::MI * 16), wn = wave % G::WAVES_N * (G::NJ * 16);

  typename G::PA pa;
  typename G::PB pb;
  pa.start(p.A, p.lda, work.m0, p.M, k_end, wave, lane);
  pb.start(p.B, p.ldb, work.n0, p.N, k_end, wave, lane);
  const unsigned lds_at = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)lds;

  float4_t acc[G::MI][G::NJ];
#pragma unroll
  for (int i = 0; i < G::MI; ++i)
#pragma unroll
    for (int j = 0; j < G::NJ; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;

  const int steps = (k_end - k_begin + BK - 1) / BK;
  // A stage is multiplied in four quarters: each half of its k with each half of the wavefront's rows.
  constexpr int kLoads = G::PA::kLoads + G::PB::kLoads, RI = G::MI / 2, kProducts = RI * G::NJ;
  uint4_t a[2][RI], b[2][G::NJ];  // the operands of a quarter and of the next, of a half and of the next
  auto stage = [&](int step) {
    pa.stage(k_begin + step * BK, k_end);
    pb.stage(k_begin + step * BK, k_end);
  };
  // A wavefront's loads of a stage, in the order in which what they replace has been read: those of A that quarters 0 and 1 (SLOW), or
  // 0 and 2, read, those of B, the rest of A.
  constexpr int kEarly = G::PA::kLoads / 2 + G::PB::kLoads;
  auto load = [&](int i, int step) {
    const unsigned at = lds_at + (step & 1) * G::kStage;
    const int late = i >= kEarly, of_a = late ? i - kEarly : i;
    if (!late && i >= G::PA::kLoads / 2) pb.load(i - G::PA::kLoads / 2, at + G::PA::kBytes, wave);
    else pa.load(G::A_SLOW ? of_a + late * (G::PA::kLoads / 2) : 2 * of_a + late, at, wave);
  };
  auto read_a = [&](int i, int step, int quarter) {
    const char* from = lds + (step & 1) * G::kStage;
    a[quarter & 1][i] = G::PA::operand(from, wm + 16 * ((quarter & 1) * RI + i), quarter >> 1, lane);
  };
  auto read_b = [&](int j, int step, int half) {
    b[half][j] = G::PB::operand(lds + (step & 1) * G::kStage + G::PA::kBytes, wn + 16 * j, half, lane);
  };
  // The products of a quarter; beside each of them goes what `beside` has for its place, in that order: reads of LDS in a row
  // would fill its queue, and the products wait for their turn behind them.
  auto multiply = [&](int quarter, auto beside) {
#pragma unroll
    for (int i = 0; i < RI; ++i)
#pragma unroll
      for (int j = 0; j < G::NJ; ++j) {
        float4_t& to = acc[(quarter & 1) * RI + i][j];
        to = mfma(T(), a[quarter & 1][i], b[quarter >> 1][j], to);
        in_order();
        beside(i * G::NJ + j);
        in_order();
      }
  };
  // things [0, count) spread over the places of a quarter
  auto spread = [&](int place, int count, auto thing) {
#pragma unroll
    for (int r = place * count / kProducts; r < (place + 1) * count / kProducts; ++r) thing(r);
  };
  // A step: its operands are read a quarter ahead.  Behind the barrier in its middle all have read B and half of A, behind the one
  // before the last quarter the rest: into their places the step after the next is loaded (LOAD), which has a step and a quarter to arrive.
  // Behind the second the next step's has (NEXT).  No branch within: where two ways meet, the compiler waits for the reads of both.
  auto step = [&](auto load_c, auto next_c, int s) {
    constexpr bool LOAD = decltype(load_c)::value, NEXT = decltype(next_c)::value;
    multiply(0, [&](int place) {
      spread(place, RI + G::NJ / 2, [&](int r) { r < RI ? read_a(r, s, 1) : read_b(r - RI, s, 1); });
    });
    multiply(1, [&](int place) {
      spread(place, RI + G::NJ / 2, [&](int r) { r < RI ? read_a(r, s, 2) : read_b(r - RI + G::NJ / 2, s, 1); });
    });
    if constexpr (LOAD) {
      all_have_read();
      stage(s + 2);
      in_order();
    }
    multiply(2, [&](int place) {
      spread(place, RI, [&](int r) { read_a(r, s, 3); });
      if constexpr (LOAD) spread(place, kEarly, [&](int r) { load(r, s + 2); });
    });
    if constexpr (NEXT) tile_ready<LOAD ? kEarly : 0>();
    in_order();
    multiply(3, [&](int place) {
      if constexpr (NEXT) spread(place, RI + G::NJ, [&](int r) { r < G::NJ ? read_b(r, s + 1, 0) : read_a(r - G::NJ, s + 1, 0); });
      if constexpr (LOAD) spread(place, kLoads - kEarly, [&](int r) { load(kEarly + r, s + 2); });
    });
  };
  for (int s = 0; s < 2 && s < steps; ++s) {
    stage(s);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load(i, s);
  }
  if (steps > 1) tile_ready<kLoads>();
  else tile_ready<0>();
#pragma unroll
  for (int i = 0; i < RI; ++i) read_a(i, 0, 0);
#pragma unroll
  for (int j = 0; j < G::NJ; ++j) read_b(j, 0, 0);
  int s = 0;
  for (; s + 2 < steps; ++s) step(std::true_type(), std::true_type(), s);
  if (s + 1 < steps) step(std::false_type(), std::true_type(), s++);
  step(std::false_type(), std::false_type(), s);
  tile_ready<0>();

  store_tile<T, G>(lds, p, to, acc, work.piece, work.m0, work.n0);
}

// Few tiles, of which each has its steps' latency to bear: STAGES of them in a ring, all but one on their way, and three workgroups a CU. A
// k of one takes 4.2 ns, of two on a CU 6.3, of three 8.4 (128 x 128: 9.0, of two 13.9).  Eight stages, which leave one a CU, 512 x 2048 x 2048 16.1
// us instead of 13.1; operands read half a stage ahead 13.4.
// Floats go through the float instruction, four k at a time, of which lane group q has 4 q + e at turn e; a stage's sum is added to what there
// is as a whole, so that a sum of K is rounded K / 32 + 32 times.
template <typename T, class G>
__device__ __forceinline__ void multiply_narrow_tile(char* lds, const Product& p, const Finish<T>& to, unsigned turn) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Work work = work_of<G>(p, turn);
  const int wm = wave / G::WAVES_N * (G::MI * 16), wn = wave % G::WAVES_N * (G::NJ * 16);
  typename G::PA pa;
  typename G::PB pb;
  pa.start(p.A, p.lda, work.m0, p.M, work.k_end, wave, lane);
  pb.start(p.B, p.ldb, work.n0, p.N, work.k_end, wave, lane);
  const unsigned lds_at = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)lds;
  constexpr int kLoads = G::PA::kLoads + G::PB::kLoads, kStep = kStageBytes / (int)sizeof(T);
  auto load = [&](int step, int place) {  // beyond the last step: zeros, so that as many are on their way
    const int k0 = work.k_begin + step * kStep;
    pa.stage(k0, work.k_end);
    pb.stage(k0, work.k_end);
    const unsigned at = lds_at + place * G::kStage;
#pragma unroll
    for (int i = 0; i < G::PA::kLoads; ++i) pa.load(i, at, wave);
#pragma unroll
    for (int i = 0; i < G::PB::kLoads; ++i) pb.load(i, at + G::PA::kBytes, wave);
  };
  float4_t acc[G::MI][G::NJ];
#pragma unroll
  for (int i = 0; i < G::MI; ++i)
#pragma unroll
    for (int j = 0; j < G::NJ; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;
  const int steps = (work.k_end - work.k_begin + kStep - 1) / kStep;
#pragma unroll
  for (int s = 0; s < G::STAGES - 1; ++s) load(s, s);
  int place = 0, free = G::STAGES - 1;
  for (int s = 0; s < steps; ++s) {
    tile_ready<kLoads * (G::STAGES - 2)>();  // and all have read what the next goes into
    load(s + G::STAGES - 1, free);
    free = place;
    const char* stage = lds + place * G::kStage;
    place = place + 1 < G::STAGES ? place + 1 : 0;
    float4_t sum[sizeof(T) == 4 ? G::MI : 1][G::NJ] = {};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint4_t a[G::MI], b[G::NJ];
#pragma unroll
      for (int i = 0; i < G::MI; ++i) a[i] = G::PA::operand(stage, wm + 16 * i, half, lane);
#pragma unroll
      for (int j = 0; j < G::NJ; ++j) b[j] = G::PB::operand(stage + G::PA::kBytes, wn + 16 * j, half, lane);
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int i = 0; i < G::MI; ++i)
#pragma unroll
            for (int j = 0; j < G::NJ; ++j)
              sum[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i][e]), __uint_as_float(b[j][e]), sum[i][j], 0, 0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < G::MI; ++i)
#pragma unroll
          for (int j = 0; j < G::NJ; ++j) acc[i][j] = mfma(T(), a[i], b[j], acc[i][j]);
      }
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < G::MI; ++i)
#pragma unroll
        for (int j = 0; j < G::NJ; ++j) acc[i][j] += sum[i][j];
    }
  }
  tile_ready<0>();
  store_tile<T, G>(lds, p, to, acc, work.piece, work.m0, work.n0);
}

template <typename T, class G>
__device__ __forceinline__ void multiply(char* lds, const Product& p, const Finish<T>& to, unsigned block, unsigned blocks) {
  if constexpr (G::STAGES == 2) multiply_tile<T, G>(lds, p, to, work_of_xcd(block, blocks));
  else multiply_narrow_tile<T, G>(lds, p, to, work_of_xcd(block, blocks));
}

template <typename T, class G>
__global__ __launch_bounds__(64 * G::WAVES, G::ON_A_SIMD)
void linear_tile_kernel(Product p, Finish<T> to) {
  __shared__ __attribute__((aligned(1024))) char lds[G::kLds];
  multiply<T, G>(lds, p, to, blockIdx.x, gridDim.x);
}

// ---- few rows ----------------------------------------------------------------------------
// Up to 16 MT rows, the whole product in one launch.  Bound: how fast a CU takes in pieces of rows of W and x, some 2 ns each whether they
// have 32 or 64 bytes; the fewer columns a workgroup has, the more CUs take part.  Each of its wavefronts takes the 32 k of every eighth unit,
// two units on their way while two are multiplied: W goes through registers (rows may start anywhere, what is beyond them is 0) into the
// wavefront's own part of LDS and comes back transposed, x comes as the instruction wants it.  The wavefronts' sums meet in LDS.
// C x D = 1024 x 4096 and 4096 x 4096, 1 / 16 / 32 rows: 4.2 / 4.7 / 5.5 and 10.5 / 12.4 / 15.9 us (tiles, and the sums of their
// pieces, 7.8 / 7.3 / 7.8 and 13.1 / 13.7 / 14.5); with four units 4.8 / 5.1 / 5.8 and 11.4 / 13.1 / 16.6.
constexpr int kRowWaves = 8, kUnits = 2;
template <typename T, int MT, int COLUMNS>
__global__ __launch_bounds__(64 * kRowWaves, 2)
void linear_rows_kernel(int R, int D, int K, const T* __restrict__ x, size_t x_ld, const T* __restrict__ W, Finish<T> to) {
  typedef typename Packed<T, 8>::type vec_t;
  constexpr int kUnitBytes = 32 * COLUMNS * 2, kPitch = COLUMNS + 4, NJ = COLUMNS / 16;
  constexpr int LANES = COLUMNS / 8, ROWS = 64 / LANES, kLoads = 32 / ROWS;  // lanes of a row of W, rows of a load, loads of a unit
  constexpr int kTurned = kRowWaves * kUnits * kUnitBytes, kSums = kRowWaves * MT * 16 * kPitch * 4;
  __shared__ __attribute__((aligned(16))) char lds[kTurned > kSums ? kTurned : kSums];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = work_of_xcd(blockIdx.x, gridDim.x) * COLUMNS;  // (a cache line has the columns of several workgroups)
  char* own = lds + wave * kUnits * kUnitBytes;
  const int units = (K + 31) / 32;
  const int col = n0 + lane % LANES * 8;
  // Where 32 bytes of row k of a unit lie: what half a wavefront reads at once, rows 0 .. 3 and 8 .. 11, on different banks.
  auto place = [](int k, int piece) {
    const int turn = k >> 3 & 1;
    return COLUMNS == 16 ? (k ^ 4 * turn) * 32 : k * 64 + (piece ^ turn) * 32;
  };

  vec_t w[2][kUnits][kLoads], a[2][kUnits][MT];
  const T* rows[MT];  // those beyond the last are not wanted: it once more
#pragma unroll
  for (int m = 0; m < MT; ++m) rows[m] = x + (size_t)(16 * m + (lane & 15) < R ? 16 * m + (lane & 15) : R - 1) * x_ld;
  auto fetch = [&](auto set, int first) {  // the units first + wave, first + wave + kRowWaves ..
    if ((first + kUnits * kRowWaves) * 32 <= K && n0 + COLUMNS <= D) {  // nothing to leave out
#pragma unroll
      for (int g = 0; g < kUnits; ++g) {
        const int k0 = (first + g * kRowWaves + wave) * 32;
#pragma unroll
        for (int h = 0; h < kLoads; ++h)
          w[set][g][h] = *reinterpret_cast<const typename Wide<T, 8>::type*>(W + (size_t)(k0 + ROWS * h + lane / LANES) * D + col);
#pragma unroll
        for (int m = 0; m < MT; ++m) a[set][g][m] = *reinterpret_cast<const typename Wide<T, 8>::type*>(rows[m] + k0 + lane / 16 * 8);
      }
      return;
    }
#pragma unroll
    for (int g = 0; g < kUnits; ++g) {
      const int k0 = (first + g * kRowWaves + wave) * 32;
#pragma unroll
      for (int h = 0; h < kLoads; ++h) {
        const int k = k0 + ROWS * h + lane / LANES;
        w[set][g][h] = vec_t{};
        if (k < K) w[set][g][h] = load_packed<8>(W + (size_t)k * D, col, D);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) a[set][g][m] = load_packed<8>(rows[m], k0 + lane / 16 * 8, K);
    }
  };
  float4_t acc[MT][NJ];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[m][j] = float4_t{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](auto set) {
#pragma unroll
    for (int g = 0; g < kUnits; ++g)
#pragma unroll
      for (int h = 0; h < kLoads; ++h)
        *reinterpret_cast<vec_t*>(own + g * kUnitBytes + place(ROWS * h + lane / LANES, lane % LANES >> 1) + (lane & 1) * 16) = w[set][g][h];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int g = 0; g < kUnits; ++g)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        uint4_t b;
        const int q = lane >> 4, i = lane & 15;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          typedef __attribute__((address_space(3))) short4_t* lds_t;
          const short4_t part =
              __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(own + g * kUnitBytes + place(8 * q + 4 * h + (i >> 2), j) + (i & 3) * 8));
          __builtin_memcpy(reinterpret_cast<char*>(&b) + 8 * h, &part, 8);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m][j] = mfma(T(), __builtin_bit_cast(uint4_t, a[set][g][m]), b, acc[m][j]);
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  constexpr std::integral_constant<int, 0> even;
  constexpr std::integral_constant<int, 1> odd;
  constexpr int kGroup = kUnits * kRowWaves;
  fetch(even, 0);
  for (int u = 0; u < units; u += 2 * kGroup) {
    if (u + kGroup < units) fetch(odd, u + kGroup);
    multiply(even);
    if (u + kGroup < units) {
      if (u + 2 * kGroup < units) fetch(even, u + 2 * kGroup);
      multiply(odd);
    }
  }
  __syncthreads();
  float(*sums)[MT * 16][kPitch] = reinterpret_cast<float(*)[MT * 16][kPitch]>(lds);
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[wave][16 * m + 4 * (lane >> 4) + e][16 * j + (lane & 15)] = acc[m][j][e];
  __syncthreads();
  const int row = threadIdx.x / LANES, c = threadIdx.x % LANES * 8;
  if (row >= MT * 16 || row >= R) return;
  float v[8], bias[8];
  load_bias(to, n0 + c, D, bias);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = sums[0][row][c + e];
#pragma unroll
  for (int z = 1; z < kRowWaves; ++z)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += sums[z][row][c + e];
  finish(to, v, bias, row, n0 + c, D);
}

// ---- what is done before and behind the products: each in one launch, whose workgroups are dealt out to its parts -----------
// rows x columns of an operand in 16-byte pieces: rows padded with zeros to a multiple of eight elements.
template <typename T>
struct Copy {
  int rows, columns;
  const T* in;
  size_t ld;
  T* out;
  unsigned blocks;  // 0: none
};
template <typename T>
__device__ __forceinline__ void make_copy(const Copy<T>& c, unsigned block) {
  const unsigned groups = (c.columns + 7) / 8;
  for (size_t i = block * (size_t)256 + threadIdx.x; i < (size_t)c.rows * groups; i += (size_t)c.blocks * 256) {
    const size_t row = i / groups;
    const int col = (int)(i % groups) * 8;
    *reinterpret_cast<typename Packed<T, 8>::type*>(c.out + i * 8) = load_packed<8>(c.in + row * c.ld, col, c.columns);
  }
}

// d = dy slope, rows padded as above, and its sums over the rows of a workgroup.  Bound: HBM.  A workgroup takes 512 columns,
// eight a lane; its four wavefronts take the rows of its share in turn.  16384 x 4096 in bf16 (403 MB in and out) 75 us, 5.3 TB/s.
constexpr int kSumColumns = 512;
template <typename T>
struct Slopes {
  int M, N, rows_each;
  const T* dy;
  size_t dy_ld;
  const typename Finish<T>::slope_t* slope;  // null: 1
  T* d;                                      // null: not wanted
  size_t d_ld;
  float* partial;                            // null: not wanted
  unsigned across, blocks;                   // 0: none
};
template <typename T>
__device__ __forceinline__ void apply_slopes(const Slopes<T>& s, unsigned block) {
  __shared__ float red[4][kSumColumns];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned part = block / s.across, first_col = block % s.across * kSumColumns;
  const int col = first_col + lane * 8;
  const int first = part * s.rows_each, last = s.M - first < s.rows_each ? s.M : first + s.rows_each;
  float sum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[i] = 0.f;
#pragma unroll 4
  for (int row = first + wave; row < last; row += 4) {
    float v[8];
    load_channels<8>(s.dy + row * s.dy_ld, col, s.N, v);
    if (s.slope != nullptr) {
      float by[8];
      load_channels<8>(s.slope + (size_t)row * s.N, col, s.N, by);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= by[i];
    }
    if (s.d != nullptr && col < (int)s.d_ld) store_channels<8>(s.d + row * s.d_ld, col, (int)s.d_ld, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += v[i];
  }
  if (s.partial == nullptr) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) red[wave][lane * 8 + i] = sum[i];
  __syncthreads();
  for (int c = threadIdx.x; c < kSumColumns; c += 256)
    if (first_col + c < (unsigned)s.N) s.partial[(size_t)part * s.N + first_col + c] = (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
}

template <typename T>
__global__ __launch_bounds__(256)
void linear_prepare_kernel(Slopes<T> slopes, Copy<T> first, Copy<T> second) {
  unsigned block = blockIdx.x;
  if (block < slopes.blocks) return apply_slopes(slopes, block);
  block -= slopes.blocks;
  if (block < first.blocks) return make_copy(first, block);
  make_copy(second, block - first.blocks);
}

// The pieces of a product, added in order, and what follows.  Bound: HBM; 2 pieces of 128 x 4096 4.2 us.  No pieces: the elements lie in `to.out` already (float).
template <typename T>
struct Join {
  int M, N, pieces;
  const float* partial;
  Finish<T> to;
  unsigned blocks;  // 0: none
};
__device__ __forceinline__ void load_floats(const float* from, float (&v)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) *reinterpret_cast<float4_t*>(v + 4 * h) = *reinterpret_cast<const float4_t*>(from + 4 * h);
}
template <typename T>
__device__ __forceinline__ void join_pieces(const Join<T>& j, unsigned block) {
  const unsigned groups = (j.N + 7) / 8;
  for (size_t i = block * (size_t)256 + threadIdx.x; i < (size_t)j.M * groups; i += (size_t)j.blocks * 256) {
    const size_t row = i / groups;
    const int col = (int)(i % groups) * 8;
    float v[8], bias[8];
    load_bias(j.to, col, j.N, bias);
    if (j.partial == nullptr) {
      load_channels<8>(j.to.out + row * j.to.ld, col, j.N, v);
    } else {
      const size_t piece = (size_t)j.M * groups * 8;
      const float* from = j.partial + i * 8;
      load_floats(from, v);
      constexpr int AT_ONCE = 8;
      for (int z = 1; z < j.pieces; z += AT_ONCE) {
        float w[AT_ONCE][8];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k)  // beyond the last piece it once more, not added
          load_floats(from + (z + k < j.pieces ? z + k : j.pieces - 1) * piece, w[k]);
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += z + k < j.pieces ? w[k][e] : 0.f;
      }
    }
    finish(j.to, v, bias, row, col, j.N);
  }
}

// The gradient of the bias from what the workgroups of d left: 16 columns a workgroup, whose 16 groups of lanes take the parts in turn, 16 of
// them on their way.
constexpr int kBiasColumns = 16;
template <typename T>
struct Bias {
  int parts, N;
  const float* partial;
  T* out;
  unsigned blocks;  // 0: none
};
template <typename T>
__device__ __forceinline__ void add_bias(const Bias<T>& b, unsigned block) {
  constexpr int GROUPS = 256 / kBiasColumns, AT_ONCE = 16;
  __shared__ float red[GROUPS][kBiasColumns];
  const int lane = threadIdx.x % kBiasColumns, group = threadIdx.x / kBiasColumns, col = block * kBiasColumns + lane;
  float sum = 0.f;
  if (col < b.N) {
    for (int p = group; p < b.parts; p += AT_ONCE * GROUPS) {
      float v[AT_ONCE];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) v[i] = b.partial[(size_t)(p + GROUPS * i < b.parts ? p + GROUPS * i : p) * b.N + col];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) sum += p + GROUPS * i < b.parts ? v[i] : 0.f;
    }
  }
  red[group][lane] = sum;
  __syncthreads();
  if (group != 0 || col >= b.N) return;
  for (int g = 1; g < GROUPS; ++g) sum += red[g][lane];
  b.out[col] = (T)sum;
}

template <typename T>
__global__ __launch_bounds__(256)
void linear_finish_kernel(Bias<T> bias, Join<T> first, Join<T> second) {
  unsigned block = blockIdx.x;
  if (block < bias.blocks) return add_bias(bias, block);
  block -= bias.blocks;
  if (block < first.blocks) return join_pieces(first, block);
  join_pieces(second, block - first.blocks);
}

// Two products that do not wait for one another, and (of 256 threads) the gradient of the bias ahead of them.  The workgroups [first, first + blocks)
// behind those are the first product's.
template <typename T, class G, class H>
__global__ __launch_bounds__(64 * G::WAVES, G::ON_A_SIMD < H::ON_A_SIMD ? G::ON_A_SIMD : H::ON_A_SIMD)
void linear_gradients_kernel(Bias<T> bias, Product p, Finish<T> to, unsigned first, unsigned blocks, Product q, Finish<T> q_to) {
  static_assert(G::WAVES == H::WAVES, "one shape of workgroups");
  __shared__ __attribute__((aligned(1024))) char lds[G::kLds > H::kLds ? G::kLds : H::kLds];
  if constexpr (64 * G::WAVES == 256)
    if (blockIdx.x < bias.blocks) return add_bias(bias, blockIdx.x);
  const unsigned block = blockIdx.x - bias.blocks, others = gridDim.x - bias.blocks - blocks;
  if (block - first < blocks) multiply<T, G>(lds, p, to, block - first, blocks);
  else multiply<T, H>(lds, q, q_to, block < first ? block : block - blocks, others);
}

// ---- plans -------------------------------------------------------------------------------
int cus() { return device_cu_count() > 0 ? device_cu_count() : 256; }

enum { kLarge, kSmall, kNarrow, kTiles };
struct Plan {
  int kind;  // tiles of 256 x 256, 128 x 128 or 64 x 64
  int tiles_m, tiles_n, pieces, k_per_piece;
  size_t floats;
  double cost;  // ns
};

// What a k of a tile was measured to cost, in ns, by how many of its kind a CU has: one to three.
constexpr int kSide[kTiles] = {256, 128, 64}, kPerCu[kTiles] = {1, 2, 3};
constexpr double kStep[kTiles][3] = {{21.0}, {9.0, 13.9}, {4.2, 6.3, 8.4}}, kRound[kTiles] = {5000, 3500, 3500};
constexpr double kFloatStep[3] = {23.0, 38.0, 56.0};  // floats, 64 x 64
double step_cost(int element, int kind, int on_a_cu) { return element == 4 ? kFloatStep[on_a_cu - 1] : kStep[kind][on_a_cu - 1]; }

// Adding pieces up, 2500 ns and 1000 for a launch more, which the host bears; and writing and reading their elements at 4 TB/s. (The 1000 is
// in the estimates below and not in what the device was measured to take.)
double join_cost(int pieces, int M, int N) { return pieces > 1 ? 3500 + (double)pieces * M * N * 8 / 4000 : 0.0; }

// The cheapest of the tiles from `first` to `last` and of 1 to 32 pieces by cost(kind, workgroups, k of a workgroup), and its joins.
template <class Cost>
Plan cheapest(int cus, int first, int last, int M, int N, int K, Cost cost) {
  Plan best = {};
  best.cost = 1e300;
  for (int kind = first; kind <= last; ++kind) {
    const int side = kSide[kind];
    const long long tm = ((long long)M + side - 1) / side, tn = ((long long)N + side - 1) / side, tiles = tm * tn;
    if (kind == kNarrow && tiles > (long long)kGridLimit) break;
    for (int s = 1; s <= 32; ++s) {
      int per = (K + s - 1) / s;
      per = (per + BK - 1) / BK * BK;
      if (s > 1 && (per < 2 * BK || tiles * s > 2ll * kPerCu[kind] * cus)) break;
      if ((K + per - 1) / per != s) continue;
      const double here = cost(kind, tiles * s, per) + join_cost(s, M, N);
      if (here < best.cost) best = {kind, (int)tm, (int)tn, s, per, s > 1 ? (size_t)s * M * eights(N) : 0, here};
    }
  }
  return best;
}

// A product by itself: its steps in rounds of workgroups.  us, estimate / measured: 128 x 4096 x 4096 (M, K, N) in 4 / 8
// pieces of 128 x 128 20.4 / 18.3, 20.0 / 18.8, in 8 of 256 x 256 28 / 24, in 2 / 4 of 64 x 64 17.7 / 16.8, 17.6 / 17.0; 1024 x 8192 x 2048 in 4 of
// 128 x 128 52 / 48, in 8 of 256 x 256 64 / 51; 512 x 16384 x 512 in 16 of 128 x 128 25 / 26; 8192 x 2048 x 1024 whole, 128 x 128 / 256 x 256 32, 48 /
// 34, 48; 512 x 2048 x 2048 whole of 64 x 64 12 / 13 (before there were those: 20.7), 1024 x 1024 x 1024 7.8 / 8.6 (14.0), 512 x 512 x 512 5.7 / 5.7
// (9.1), 2048 x 2048 x 2048 whole of 128 x 128 22 / 24, of 64 x 64 33 / 29.
Plan plan_product(int cus, int element, int first, int last, int M, int N, int K) {
  return cheapest(cus, first, last, M, N, K, [=](int kind, long long workgroups, int per) {
    const unsigned slots = (unsigned)(kPerCu[kind] * cus), all = (unsigned)workgroups, rounds = all / slots, rest = all % slots;
    return (double)rounds * (step_cost(element, kind, kPerCu[kind]) * per + kRound[kind]) +
           (rest > 0 ? step_cost(element, kind, (int)((rest - 1) / (unsigned)cus) + 1) * per + kRound[kind] : 0.0);
  });
}

// One that is launched with `other`: all workgroups' shares of a full CU, which has as many as fit of the larger tiles, or the
// longest's time where that is more.  us, estimate / measured: both gradients of
// 8192 x 1024 x 2048 with that of the kernel in 2 / 3 / 4 pieces 74 / 76, 79 / 80, 84 / 81 (by itself 4 would be best), of 4096 x 2048 x 1024 in 2 / 4
// 46 / 45, 56 / 49.
Plan plan_product_beside(int cus, int element, const Plan& other, int M, int N, int K) {
  const double others = (double)other.tiles_m * other.tiles_n * other.pieces;
  return cheapest(cus, element == 4 ? kNarrow : kSmall, kNarrow, M, N, K, [&](int kind, long long workgroups, int per) {
    const int fit = kPerCu[kind] < kPerCu[other.kind] ? kPerCu[kind] : kPerCu[other.kind];
    const double on_a_cu = (workgroups + others) / cus;
    const int here = on_a_cu < fit ? (int)std::ceil(on_a_cu) : fit;
    const double longest = step_cost(element, kind, here) * per + kRound[kind];
    const double shares = (workgroups * (step_cost(element, kind, fit) * per + kRound[kind]) +
                           others * (step_cost(element, other.kind, fit) * other.k_per_piece + kRound[other.kind])) / ((double)fit * cus);
    return shares > longest ? shares : longest;
  });
}

// The same with one of 256 x 256, of which a CU has one at a time: those that take longer come first, the others where there is room. us, both
// gradients apart or of smaller tiles / so: 8192 x 2048 x 2048 149 / 128, 8192 x 1024 x 2048 78 / 72, 65536 x 512 x 512 105 / 95, 16384 x 4096 x 4096 817 / 802.
Plan plan_large_beside(int cus, const Plan& other, int M, int N, int K) {
  const long long others = (long long)other.tiles_m * other.tiles_n * other.pieces;
  return cheapest(cus, kLarge, kLarge, M, N, K, [&](int, long long workgroups, int per) {
    const bool longer = per > other.k_per_piece;
    const double slow = kStep[kLarge][0] * (longer ? per : other.k_per_piece) + kRound[kLarge];
    const double quick = kStep[kLarge][0] * (longer ? other.k_per_piece : per) + kRound[kLarge];
    const long long first = longer ? workgroups : others, second = longer ? others : workgroups;
    const long long rounds = first / cus, late = first % cus;  // CUs that have one more of the first
    const auto room = [&](double until) {
      const double early = std::floor((until - rounds * slow) / quick + 1e-6), there = std::floor((until - (rounds + 1) * slow) / quick + 1e-6);
      return (early > 0 ? early : 0) * (double)(cus - late) + (there > 0 ? there : 0) * (double)late;
    };
    double low = (rounds + (late > 0)) * slow, high = low + ((double)second / cus + 1) * quick;
    if (room(low) >= (double)second) return low;
    for (int i = 0; i < 24; ++i) (room(0.5 * (low + high)) >= (double)second ? high : low) = 0.5 * (low + high);
    return high;
  });
}

// Whether linear_rows_kernel has the forward product: with more than 16 rows of a long contraction tiles are faster.
bool few_rows(int element, int R, int K) { return element == 2 && R <= (K <= 2048 ? 32 : 16); }

template <typename T>
int product_of_few_rows(hipStream_t stream, int R, int D, int K, const T* x, size_t x_ld, const T* W, const Finish<T>& to) {
  ScopedKernelTimer timer("linear_rows", stream);
  const bool narrow = D <= 32 * cus();
  const dim3 grid((unsigned)((D + (narrow ? 15 : 31)) / (narrow ? 16 : 32)));
#define HASTE_LAUNCH_ROWS(MT_, COLUMNS_) \
  linear_rows_kernel<T, MT_, COLUMNS_><<<grid, 64 * kRowWaves, 0, stream>>>(R, D, K, x, x_ld, W, to)
  if (R <= 16 && narrow) HASTE_LAUNCH_ROWS(1, 16);
  else if (R <= 16) HASTE_LAUNCH_ROWS(1, 32);
  else if (narrow) HASTE_LAUNCH_ROWS(2, 16);
  else HASTE_LAUNCH_ROWS(2, 32);
#undef HASTE_LAUNCH_ROWS
  HASTE_HIP_TRY(hipGetLastError());
  return HASTE_HIP_OK;
}

int blocks_for(size_t threads) {
  const size_t b = (threads + 255) / 256, most = (size_t)cus() * 32;
  return (int)(b < most ? b : most);
}

// A product as plan_product() says, and as much scratch for its pieces.
Product product_of(const Plan& plan, int M, int N, int K, const void* A, size_t lda, const void* B, size_t ldb, char* scratch) {
  return {M, N, K, A, B, (long long)lda, (long long)ldb, plan.tiles_m, plan.tiles_n, plan.k_per_piece,
          plan.pieces > 1 ? reinterpret_cast<float*>(scratch) : nullptr};
}
unsigned workgroups(const Plan& plan) { return (unsigned)(plan.tiles_m * plan.tiles_n * plan.pieces); }

// What is left to be done behind it.
template <typename T>
Join<T> joined(const Plan& plan, const Product& p, const Finish<T>& to) {
  if (plan.pieces <= 1) return {};
  return {p.M, p.N, plan.pieces, p.partial, to, (unsigned)blocks_for((size_t)p.M * ((p.N + 7) / 8))};
}

template <int E, bool A_SLOW, bool B_SLOW>
struct Tiles {
  typedef Tile<E, A_SLOW, B_SLOW, 256, 256, 2, 4> large;
  typedef Tile<E, A_SLOW, B_SLOW, 128, 128, 2, 2> small;
  typedef Tile<E, A_SLOW, B_SLOW, 64, 64, 2, 2, 3> narrow;
};

template <typename T, class TILES>
int multiply(hipStream_t stream, const Plan& plan, const Product& p, const Finish<T>& to) {
  ScopedKernelTimer timer("linear_product", stream);
  const unsigned blocks = workgroups(plan);
  if constexpr (sizeof(T) == 2) {
    if (plan.kind == kLarge) linear_tile_kernel<T, typename TILES::large><<<blocks, 64 * TILES::large::WAVES, 0, stream>>>(p, to);
    else if (plan.kind == kSmall) linear_tile_kernel<T, typename TILES::small><<<blocks, 256, 0, stream>>>(p, to);
  }
  if (plan.kind == kNarrow) linear_tile_kernel<T, typename TILES::narrow><<<blocks, 256, 0, stream>>>(p, to);
  HASTE_HIP_TRY(hipGetLastError());
  return HASTE_HIP_OK;
}

template <typename T, class G, class H>
int both_gradients(hipStream_t stream, const Bias<T>& bias, const Plan& plan, const Product& p, const Finish<T>& to, const Plan& q_plan,
                   const Product& q, const Finish<T>& q_to) {
  ScopedKernelTimer timer("linear_product", stream);
  const unsigned blocks = workgroups(plan), others = workgroups(q_plan);
  const unsigned first = q_plan.k_per_piece > plan.k_per_piece ? others : 0;  // those that take longer start first
  linear_gradients_kernel<T, G, H><<<bias.blocks + blocks + others, 64 * G::WAVES, 0, stream>>>(bias, p, to, first, blocks, q, q_to);
  HASTE_HIP_TRY(hipGetLastError());
  return HASTE_HIP_OK;
}

template <typename T>
int prepare(hipStream_t stream, const Slopes<T>& slopes, const Copy<T>& first, const Copy<T>& second) {
  const unsigned blocks = slopes.blocks + first.blocks + second.blocks;
  if (blocks == 0) return HASTE_HIP_OK;
  ScopedKernelTimer timer("linear_prepare", stream);
  linear_prepare_kernel<T><<<blocks, 256, 0, stream>>>(slopes, first, second);
  HASTE_HIP_TRY(hipGetLastError());
  return HASTE_HIP_OK;
}

template <typename T>
int finish_all(hipStream_t stream, const Bias<T>& bias, const Join<T>& first, const Join<T>& second) {
  const unsigned blocks = bias.blocks + first.blocks + second.blocks;
  if (blocks == 0) return HASTE_HIP_OK;
  ScopedKernelTimer timer("linear_finish", stream);
  linear_finish_kernel<T><<<blocks, 256, 0, stream>>>(bias, first, second);
  HASTE_HIP_TRY(hipGetLastError());
  return HASTE_HIP_OK;
}

size_t whole(size_t bytes) { return (bytes + 255) / 256 * 256; }
struct SumPlan {
  int blocks, rows_each;
  size_t floats;
};
SumPlan plan_sums(int rows, int columns) {
  const int across = (columns + kSumColumns - 1) / kSumColumns;
  long long blocks = (4ll * cus() + across - 1) / across;
  const long long most = (rows + 15) / 16;
  blocks = blocks < most ? blocks : most;
  SumPlan s;
  s.rows_each = (int)((rows + blocks - 1) / blocks);
  s.blocks = (rows + s.rows_each - 1) / s.rows_each;
  s.floats = (size_t)s.blocks * columns;
  return s;
}

// Where what a call keeps in its workspace lies; sizes in bytes.
struct Layout {
  size_t x, kernel, d, sums, product, product_kernel, total;
  bool tiles;              // otherwise the products are those of gemm.hip
  bool together;           // both gradients in one launch
  Plan plan, plan_kernel;  // of the product forward, or of dx and dkernel
};

// What gemm.hip's product of M rows takes, ns: 190 TFLOP/s, and beside them less for few rows.  Products of floats go by tiles of the float
// instruction where those cost less, which have no pass behind them.  us, tiles / gemm.hip: 512 x 512 x 512 (R, C, D) 10.9 / 15.7, both
// gradients 16.2 / 33.8; 1024 x 1024 x 1024 27.7 / 31.7, 43 / 65; 1296 x 224 x 630 12.4 / 18.9; 3071 x 300 x 1001 28.5 / 28.8, 59 / 68;
// 64 x 1024 x 4096 14.4 / 17.6, but 64 x 4096 x 4096 31.1 / 27.6; 2048 x 1024 x 1024 41.6 / 38.5, 99 / 77; 2048 x 2048 x 2048 150 / 99.
double product_of_floats(int M, int R, int C, int D) { return (M < 80 ? 9500 + 80.0 * M : 16000) + 2.0 * R * C * D / 190e3; }

Layout layout_of(bool backward, int element, int R, int C, int D, bool aligned) {
  Layout l = {};
  if (!backward && few_rows(element, R, C)) return l;
  const int cus = haste_hip::cus(), first = element == 4 ? kNarrow : kLarge;
  double cost;
  if (!backward) {
    l.plan = plan_product(cus, element, first, kNarrow, R, D, C);
    cost = l.plan.cost;
  } else {
    l.plan = plan_product(cus, element, first, kNarrow, R, C, D);
    l.plan_kernel = plan_product(cus, element, first, kNarrow, C, D, R);
    cost = l.plan.cost + l.plan_kernel.cost;
    const auto consider = [&](const Plan& plan, const Plan& plan_kernel) {  // in one launch
      const double here = plan_kernel.cost + join_cost(plan.pieces, R, C);
      if (here < cost) l.plan = plan, l.plan_kernel = plan_kernel, cost = here, l.together = true;
    };
    // (floats have the narrow tiles alone; where those are too many for a grid there is no plan)
    const Plan small = l.plan.kind >= kSmall || element == 4 ? l.plan : plan_product(cus, element, kSmall, kNarrow, R, C, D);
    if (small.cost < 1e300) consider(small, plan_product_beside(cus, element, small, C, D, R));
    if (element == 2) {
      Plan whole = plan_product(cus, element, kLarge, kLarge, R, C, D);
      whole.pieces = 1, whole.k_per_piece = (D + BK - 1) / BK * BK, whole.floats = 0;
      consider(whole, plan_large_beside(cus, whole, C, D, R));
    }
  }
  l.tiles = element == 2 || cost < product_of_floats(R, R, C, D) + (backward ? product_of_floats(C, R, C, D) : 0.0);
  const int piece = 16 / element;
  size_t at = 0;
  auto place = [&](size_t bytes) {
    const size_t here = at;
    at += whole(bytes);
    return here;
  };
  l.x = place(l.tiles && (!aligned || C % piece != 0) ? (size_t)R * eights(C) * element : 0);
  l.kernel = place(!l.tiles ? (backward ? (size_t)C * D * 4 : 0) : !aligned || D % piece != 0 ? (size_t)C * eights(D) * element : 0);
  if (backward) {
    l.d = place((size_t)R * (l.tiles ? eights(D) : D) * element);
    const SumPlan s = plan_sums(R, D);
    l.sums = place(s.floats * sizeof(float));
  }
  l.product = at;
  size_t need;
  if (l.tiles) {
    l.product_kernel = l.product + whole(l.plan.floats * sizeof(float));
    need = l.product_kernel - l.product + l.plan_kernel.floats * sizeof(float);
  } else {
    // (how far apart rows are, by which a contraction may be cut into runs, is not known here)
    const size_t a = backward ? gemm_f32_scratch_bound(R, C, D) : gemm_f32_scratch_bound(R, D, C);
    const size_t b = backward ? gemm_f32_scratch_bound(C, D, R) : 0;
    need = a > b ? a : b;
  }
  l.total = at + whole(need);
  return l;
}

int check_sizes(int R, int C, int D, int element) {
  HASTE_HIP_REQUIRE(R > 0 && C > 0 && D > 0);
  if (R > kSizeLimit || C > (1 << 20) || D > (1 << 20)) return too_large("linear: more than 2^30 rows or 2^20 columns");
  const auto tiles = [](long long m, long long n) { return ((m + 127) / 128) * ((n + 127) / 128); };
  const long long most = element == 2 ? (1ll << 22) : (1ll << 24);
  if (tiles(R, D) >= most || tiles(R, C) >= most || tiles(C, D) >= most) return too_large("linear: more tiles than a grid takes");
  return HASTE_HIP_OK;
}

bool in_pieces(const void* p, size_t ld, int element) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld * element % 16 == 0; }

// An operand in 16-byte pieces: itself, or a copy that is to be made.  The rows of a contiguous operand have to end with zeros.
template <typename T>
Copy<T> placed(int rows, int columns, const T*& p, size_t& ld, T* copy) {
  if (columns * sizeof(T) % 16 == 0 && in_pieces(p, ld, sizeof(T))) return {};
  const Copy<T> c = {rows, columns, p, ld, copy, (unsigned)blocks_for((size_t)rows * ((columns + 7) / 8))};
  p = copy;
  ld = (size_t)eights(columns);
  return c;
}

bool workspace_ok(const void* workspace, size_t bytes, size_t need) {
  return need == 0 || (workspace != nullptr && bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0);
}

template <typename T>
int forward_entry(int R, int C, int D, const T* x, size_t x_row, const T* kernel, const T* bias, int act, const T* residual,
                  size_t residual_row, T* y, void* cache, void* workspace, size_t workspace_bytes, void* stream_) {
  HASTE_HIP_PROPAGATE(check_sizes(R, C, D, sizeof(T)));
  HASTE_HIP_REQUIRE(x != nullptr && kernel != nullptr && y != nullptr && act >= kNone && act <= kSilu);
  HASTE_HIP_REQUIRE(R == 1 || x_row >= (size_t)C);
  const bool aligned = in_pieces(x, R == 1 ? 8 : x_row, sizeof(T)) && in_pieces(kernel, 8, sizeof(T));
  if (R == 1) x_row = C;
  if (x_row > (size_t)(1 << 22)) return too_large("linear: rows of x more than 2^22 elements apart");
  hipStream_t stream = as_stream(stream_);
  const Layout l = layout_of(false, sizeof(T), R, C, D, aligned);
  HASTE_HIP_REQUIRE(workspace_ok(workspace, workspace_bytes, l.total));
  char* ws = static_cast<char*>(workspace);
  typedef typename Finish<T>::slope_t slope_t;
  const Finish<T> to = {y, (size_t)D, act, bias, residual, residual_row, act == kNone ? nullptr : static_cast<slope_t*>(cache)};
  if constexpr (sizeof(T) == 4) {
    if (!l.tiles) {
      {
        CallerScratch scratch(ws + l.product, l.total - l.product);
        HASTE_HIP_PROPAGATE(gemm_f32(stream, false, R, D, C, x, (int)x_row, kernel, D, y, D, false));
      }
      if (act == kNone && bias == nullptr && residual == nullptr) return HASTE_HIP_OK;
      return finish_all<T>(stream, {}, {R, D, 0, nullptr, to, (unsigned)blocks_for((size_t)R * ((D + 7) / 8))}, {});
    }
  } else if (few_rows(sizeof(T), R, C)) {
    return product_of_few_rows(stream, R, D, C, x, x_row, kernel, to);
  }
  size_t kernel_row = D;
  const Copy<T> of_x = placed(R, C, x, x_row, reinterpret_cast<T*>(ws + l.x));
  const Copy<T> of_kernel = placed(C, D, kernel, kernel_row, reinterpret_cast<T*>(ws + l.kernel));
  HASTE_HIP_PROPAGATE(prepare<T>(stream, {}, of_x, of_kernel));
  const Product p = product_of(l.plan, R, D, C, x, x_row, kernel, kernel_row, ws + l.product);
  HASTE_HIP_PROPAGATE((multiply<T, Tiles<sizeof(T), false, true>>(stream, l.plan, p, to)));
  return finish_all<T>(stream, {}, joined(l.plan, p, to), {});
}

template <typename T>
int backward_entry(int R, int C, int D, const T* x, size_t x_row, const T* kernel, int act, const void* cache, const T* dy, size_t dy_row,
                   T* dx, T* dkernel, T* dbias, void* workspace, size_t workspace_bytes, void* stream_) {
  HASTE_HIP_PROPAGATE(check_sizes(R, C, D, sizeof(T)));
  HASTE_HIP_REQUIRE(x != nullptr && kernel != nullptr && dy != nullptr && act >= kNone && act <= kSilu);
  HASTE_HIP_REQUIRE(act == kNone || cache != nullptr);
  HASTE_HIP_REQUIRE(R == 1 || (x_row >= (size_t)C && dy_row >= (size_t)D));
  const bool aligned = in_pieces(x, R == 1 ? 8 : x_row, sizeof(T)) && in_pieces(kernel, 8, sizeof(T));
  if (R == 1) x_row = C, dy_row = D;
  if (x_row > (size_t)(1 << 22) || dy_row > (size_t)(1 << 22)) return too_large("linear: rows more than 2^22 elements apart");
  hipStream_t stream = as_stream(stream_);
  const Layout l = layout_of(true, sizeof(T), R, C, D, aligned);
  HASTE_HIP_REQUIRE(workspace_ok(workspace, workspace_bytes, l.total));
  char* ws = static_cast<char*>(workspace);
  // d and its sums
  const T* d = dy;
  size_t d_row = dy_row;
  const bool own = act != kNone || (l.tiles && (D * sizeof(T) % 16 != 0 || !in_pieces(dy, dy_row, sizeof(T))));
  if (own) {
    d = reinterpret_cast<T*>(ws + l.d);
    d_row = l.tiles ? (size_t)eights(D) : (size_t)D;
  }
  Slopes<T> slopes = {};
  Bias<T> of_bias = {};
  if (own || dbias != nullptr) {
    const SumPlan s = plan_sums(R, D);
    const unsigned across = (unsigned)((D + kSumColumns - 1) / kSumColumns);
    float* sums = dbias != nullptr ? reinterpret_cast<float*>(ws + l.sums) : nullptr;
    slopes = {R, D, s.rows_each, dy, dy_row, act == kNone ? nullptr : static_cast<const typename Finish<T>::slope_t*>(cache),
              own ? reinterpret_cast<T*>(ws + l.d) : nullptr, d_row, sums, across, across * s.blocks};
    if (dbias != nullptr) of_bias = {s.blocks, D, sums, dbias, (unsigned)((D + kBiasColumns - 1) / kBiasColumns)};
  }
  if constexpr (sizeof(T) == 4) {
    if (!l.tiles) {
      HASTE_HIP_PROPAGATE(prepare<T>(stream, slopes, {}, {}));
      HASTE_HIP_PROPAGATE(finish_all<T>(stream, of_bias, {}, {}));
      CallerScratch scratch(ws + l.product, l.total - l.product);
      if (dx != nullptr) {
        float* turned = reinterpret_cast<float*>(ws + l.kernel);
        HASTE_HIP_PROPAGATE(haste_hip_transpose_f32(C, D, kernel, turned, stream_));
        HASTE_HIP_PROPAGATE(gemm_f32(stream, false, R, C, D, d, (int)d_row, turned, C, dx, C, false));
      }
      if (dkernel != nullptr) HASTE_HIP_PROPAGATE(gemm_f32(stream, true, C, D, R, x, (int)x_row, d, (int)d_row, dkernel, D, false));
      return HASTE_HIP_OK;
    }
  }
  size_t kernel_row = D;
  Copy<T> of_kernel = {}, of_x = {};
  if (dx != nullptr) of_kernel = placed(C, D, kernel, kernel_row, reinterpret_cast<T*>(ws + l.kernel));
  if (dkernel != nullptr) of_x = placed(R, C, x, x_row, reinterpret_cast<T*>(ws + l.x));
  HASTE_HIP_PROPAGATE(prepare<T>(stream, slopes, of_kernel, of_x));
  const Finish<T> to_dx = {dx, (size_t)C, kNone, nullptr, nullptr, 0, nullptr};
  const Finish<T> to_dkernel = {dkernel, (size_t)D, kNone, nullptr, nullptr, 0, nullptr};
  const Product of_dx = product_of(l.plan, R, C, D, d, d_row, kernel, kernel_row, ws + l.product);
  const Product of_dkernel = product_of(l.plan_kernel, C, D, R, x, x_row, d, d_row, ws + l.product_kernel);
  typedef Tiles<sizeof(T), false, false> tiles_dx;
  typedef Tiles<sizeof(T), true, true> tiles_dkernel;
  if (dx != nullptr && dkernel != nullptr && l.together) {
    const auto run = [&](auto of_first, auto of_second) {
      typedef decltype(of_first) first_t;
      const bool with_bias = 64 * first_t::WAVES == 256;
      HASTE_HIP_PROPAGATE((both_gradients<T, first_t, decltype(of_second)>(stream, with_bias ? of_bias : Bias<T>(), l.plan, of_dx, to_dx, l.plan_kernel,
                                                                          of_dkernel, to_dkernel)));
      if (with_bias) of_bias.blocks = 0;
      return HASTE_HIP_OK;
    };
    const typename tiles_dx::narrow narrow_dx;
    const typename tiles_dkernel::narrow narrow_dkernel;
    if constexpr (sizeof(T) == 2) {
      const typename tiles_dx::small small_dx;
      const typename tiles_dkernel::small small_dkernel;
      if (l.plan.kind == kLarge) HASTE_HIP_PROPAGATE(run(typename tiles_dx::large(), typename tiles_dkernel::large()));
      else if (l.plan.kind == kSmall) HASTE_HIP_PROPAGATE(l.plan_kernel.kind == kSmall ? run(small_dx, small_dkernel) : run(small_dx, narrow_dkernel));
      else HASTE_HIP_PROPAGATE(l.plan_kernel.kind == kSmall ? run(narrow_dx, small_dkernel) : run(narrow_dx, narrow_dkernel));
    } else {
      HASTE_HIP_PROPAGATE(run(narrow_dx, narrow_dkernel));
    }
  } else {
    if (dx != nullptr) HASTE_HIP_PROPAGATE((multiply<T, tiles_dx>(stream, l.plan, of_dx, to_dx)));
    if (dkernel != nullptr) HASTE_HIP_PROPAGATE((multiply<T, tiles_dkernel>(stream, l.plan_kernel, of_dkernel, to_dkernel)));
  }
  return finish_all(stream, of_bias, dx != nullptr ? joined(l.plan, of_dx, to_dx) : Join<T>(),
                    dkernel != nullptr ? joined(l.plan_kernel, of_dkernel, to_dkernel) : Join<T>());
}

}  // namespace
}  // namespace haste_hip

extern "C" {

using namespace haste_hip;

size_t haste_hip_linear_workspace_bytes(int backward, int element_bytes, int rows, int inputs, int outputs, int aligned) {
  if ((element_bytes != 2 && element_bytes != 4) || check_sizes(rows, inputs, outputs, element_bytes) != HASTE_HIP_OK) return 0;
  return layout_of(backward != 0, element_bytes, rows, inputs, outputs, aligned != 0).total;
}

#define HASTE_HIP_LINEAR(SUFFIX, T)                                                                                        \
  int haste_hip_linear_forward_##SUFFIX(int rows, int inputs, int outputs, const void* x, size_t x_row, const void* kernel, \
                                        const void* bias, int activation, const void* residual, size_t residual_row,       \
                                        void* y, void* cache, void* workspace, size_t workspace_bytes, void* stream) {     \
    return forward_entry<T>(rows, inputs, outputs, static_cast<const T*>(x), x_row, static_cast<const T*>(kernel),         \
                            static_cast<const T*>(bias), activation, static_cast<const T*>(residual), residual_row,        \
                            static_cast<T*>(y), cache, workspace, workspace_bytes, stream);                                \
  }                                                                                                                        \
  int haste_hip_linear_backward_##SUFFIX(int rows, int inputs, int outputs, const void* x, size_t x_row,                   \
                                         const void* kernel, int activation, const void* cache, const void* dy,            \
                                         size_t dy_row, void* dx, void* dkernel, void* dbias, void* workspace,             \
                                         size_t workspace_bytes, void* stream) {                                           \
    return backward_entry<T>(rows, inputs, outputs, static_cast<const T*>(x), x_row, static_cast<const T*>(kernel),        \
                             activation, cache, static_cast<const T*>(dy), dy_row, static_cast<T*>(dx),                    \
                             static_cast<T*>(dkernel), static_cast<T*>(dbias), workspace, workspace_bytes, stream);        \
  }

HASTE_HIP_LINEAR(f32, float)
HASTE_HIP_LINEAR(f16, _Float16)
HASTE_HIP_LINEAR(bf16, __bf16)

}  // extern "C"
