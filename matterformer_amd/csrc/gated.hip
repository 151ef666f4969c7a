// Gated linear layer (mf_gated_linear, mf_gated_linear_bwd) on gfx950:
//   a = x Wg^T + bg,  b = x Wu^T + bu,  h = act(a) * b,
// with Wg the first F and Wu the last F rows of one weight [2F, C].
// Backward, go = dL/dh:
//   dA = go b act'(a),  dB = go act(a),
//   dx = [dA dB] W,  dW = [dA dB]^T x,  dbias = column sums of [dA dB].
//
// The forward is one kernel: a tile of a and the matching tile of b are held by
// the same lanes, so activation and product happen on the fp32 accumulators and
// only h is written.  The backward forms a and b again (4 T C F flops) in the
// same kernel with another epilogue rather than keeping them: keeping them is
// 4 T F values more to write and read, about what the products cost at widths of
// a few hundred to a thousand (512 columns, 16384 rows, 2048 hidden: 69 GFLOP,
// 53 us at 1294 TFLOP/s, against 268 MB, 52 us at 5.14 TB/s), and would round
// them to the 16-bit type before the derivative.  [dA dB] is rounded to the operands' type for the two
// products that follow, as any 16-bit matrix product's input is.
//
// fp16 has no room for [dA dB] of large or small gradients (go of 3e4 times b of 4 overflows although dx may be small), so
// there row n is kept times 2^e_n, e_n from |dA|, |dB| <= 1.25 max|go_n| max(|x_n| max|W| + max|bias|, 1), the norms Euclidean
// (Cauchy-Schwarz; 1.25 covers the activations' derivatives, at most 1.13), so that the bound lies in [2^13, 2^14).  By row,
// because rows of dx have nothing to do with each other; dW, a sum over them, multiplies its operand by 2^(E - e_n), E the
// smallest of all.  Two launches before the products (7 and 47 us of 32768 x 768 x 2048, 7 and 9 of 2738 x 512 x 2048) and
// what it adds to them: the backward takes 888 and 120 us there, without the scales 766 and 102.
//
// All three products run on one tile kernel.  Its matrix-core "row" operand is
// the output's contiguous axis (h's columns, dx's and dW's channels), the
// "column" operand the output's rows, so that a lane ends with 16 consecutive
// output columns (see frag_row): stores of 32 bytes a lane, 128 a row and wave.
// Tiles are 128 bytes of K deep, copied from global memory straight to LDS
// (16 bytes a lane) while the previous tile is multiplied; two buffers, one
// barrier a step.  Rows past the ends are fetched from an out-of-range buffer
// offset, which reads zero, on both sides (a zero times what lies behind a
// matrix could be NaN).  Operands whose contiguous axis is K are stored as
// rows of 128 bytes and read as 16-byte pieces; operands whose K axis is the
// outer one (W in dx, both in dW) are stored as they lie and read transposed.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "mf_common.h"

namespace mf {
namespace gated {

enum Mode { kFwd, kBwd, kDx, kDw };

// -- activations: value and derivative in fp32 ---------------------------------------------------------------
// exp of -|..| only where the result must not overflow to inf / inf: 1 / (1 + exp(-a)) is 0 for a -> -inf.
template <bool FAST>
__device__ __forceinline__ float exp_(float x) {
  return FAST ? fast_exp2(x * kLog2e) : expf(x);
}
template <bool FAST>
__device__ __forceinline__ float rcp_(float x) {
  return FAST ? __builtin_amdgcn_rcpf(x) : 1.0f / x;
}
template <bool FAST>
__device__ __forceinline__ float sigmoid_(float x) {
  return rcp_<FAST>(1.0f + exp_<FAST>(-x));
}

// The normal distribution's cumulative function and density (times sqrt(2 pi)) at a.  With z = |a| / sqrt 2 and
// t = 1 / (1 + 0.4 z) (Hastings' form, Approximations for Digital Computers, 1955), erfc(z) exp(z^2) / (2 t) is within 2.1e-8
// (relative) of this polynomial on 0 < t <= 1, a Chebyshev fit of ours; evaluated in fp32 the whole comes within 4e-7, and
// the lower tail keeps that relative accuracy, as 0.5 (1 + erf) does not, because the exponential gets back what squaring a
// rounds off (without it 4e-6 at -12; left out for 16-bit outputs).  A third of erfcf's time.
template <bool FAST>
__device__ __forceinline__ void normal_cdf(float a, float& cdf, float& density) {
  const float square = a * a;
  density = exp_<FAST>(-0.5f * square);
  if constexpr (!FAST) {
    const float lost = fmaf(a, a, -square);
    density = density > 0.0f ? fmaf(density, -0.5f * lost, density) : density;  // (the square of a large a is infinite)
  }
  const float t = rcp_<FAST>(1.0f + 0.28284271247f * fabsf(a));
  constexpr float kFit[] = {0.0709634051f, -0.11936821f, 0.0707178637f, -0.0248721652f, 0.0426141247f, 0.0593170486f, 0.0859011784f, 0.10380403f, 0.112838037f, 0.112837918f};
  float q = -0.0147532262f;
#pragma unroll
  for (float c : kFit) q = fmaf(q, t, c);
  const float tail = density * t * q;
  cdf = a < 0.0f ? tail : 1.0f - tail;
}

// FAST (16-bit outputs): hardware exp2 and reciprocal, one unit in the last place of fp32 each.
template <int ACT, bool FAST>
__device__ __forceinline__ float act_value(float a) {
  if constexpr (ACT == MF_ACT_GELU) {
    float cdf, density;
    normal_cdf<FAST>(a, cdf, density);
    return a * cdf;
  } else if constexpr (ACT == MF_ACT_GELU_TANH) {
    // 0.5 (1 + tanh u) = sigmoid(2 u): no cancellation for negative u
    return a * sigmoid_<FAST>(1.5957691216057308f * (a + 0.044715f * a * a * a));
  } else if constexpr (ACT == MF_ACT_RELU) {
    return a > 0.0f ? a : (a == a ? 0.0f : a);
  } else if constexpr (ACT == MF_ACT_SIGMOID) {
    return sigmoid_<FAST>(a);
  } else {
    return a * sigmoid_<FAST>(a);
  }
}
template <int ACT, bool FAST>
__device__ __forceinline__ void act_both(float a, float& y, float& dy) {
  if constexpr (ACT == MF_ACT_GELU) {
    float cdf, density;
    normal_cdf<FAST>(a, cdf, density);
    y = a * cdf;
    dy = cdf + a * 0.3989422804014327f * density;
  } else if constexpr (ACT == MF_ACT_GELU_TANH) {
    const float a2 = a * a;
    const float u2 = 1.5957691216057308f * (a + 0.044715f * a * a2);
    const float s = sigmoid_<FAST>(u2), ns = sigmoid_<FAST>(-u2);
    y = a * s;
    dy = s + a * s * ns * 1.5957691216057308f * (1.0f + 0.134145f * a2);
  } else if constexpr (ACT == MF_ACT_RELU) {
    y = a > 0.0f ? a : (a == a ? 0.0f : a);
    dy = a > 0.0f ? 1.0f : 0.0f;
  } else if constexpr (ACT == MF_ACT_SIGMOID) {
    y = sigmoid_<FAST>(a);
    dy = y * sigmoid_<FAST>(-a);
  } else {
    const float s = sigmoid_<FAST>(a);
    y = a * s;
    dy = s * (1.0f + a * sigmoid_<FAST>(-a));
  }
}
// f(integral constant of the activation): one branch around an epilogue instead of one per element
template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
  switch (act) {
    case MF_ACT_GELU: f(std::integral_constant<int, MF_ACT_GELU>()); break;
    case MF_ACT_GELU_TANH: f(std::integral_constant<int, MF_ACT_GELU_TANH>()); break;
    case MF_ACT_RELU: f(std::integral_constant<int, MF_ACT_RELU>()); break;
    case MF_ACT_SIGMOID: f(std::integral_constant<int, MF_ACT_SIGMOID>()); break;
    default: f(std::integral_constant<int, MF_ACT_SILU>()); break;
  }
}

// -- 16 bytes of K as one matrix-core operand: one product for 16-bit types, four (parts) for fp32 ---------------
template <typename T>
struct Mma {
  using Frag = typename Elem<T>::Operand;
  static constexpr int kParts = 1;
  __device__ static __forceinline__ void run(Frag a, Frag b, mf_f32x4& c, int) { c = Elem<T>::mma(a, b, c); }
};
template <>
struct Mma<float> {
  using Frag = mf_f32x4;
  static constexpr int kParts = 4;
  __device__ static __forceinline__ void run(Frag a, Frag b, mf_f32x4& c, int e) {
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  }
};

constexpr int kRowBytes = 128;                        // K bytes of a tile
template <typename T> constexpr int kBK = kRowBytes / int(sizeof(T));
template <typename T> constexpr int kEpc = 16 / int(sizeof(T));  // elements per 16-byte chunk

// Row operand ("A", M axis): lane r of fragment j in a group of 64 holds group row 16 (r >> 2) + 4 j + (r & 3),
// so accumulator register q of fragment j in lane group g is row 16 g + 4 j + q: over j and q, 16 rows in order.
__device__ __forceinline__ int frag_row(int r, int j) { return ((r >> 2) << 4) + 4 * j + (r & 3); }

// Chunk swizzles (16-byte chunks of a stored row) that spread a wave's reads over the LDS banks.
// K-contiguous rows: the eight rows that eight consecutive lanes read get eight different chunk positions.
template <bool ROW_OPERAND>
__device__ __forceinline__ int swz_row(int row) {
  return ROW_OPERAND ? (row & 3) | ((row >> 2) & 4) : row & 7;
}
// K-outer rows (one k each): see read_frag.
template <typename T, bool ROW_OPERAND>
__device__ __forceinline__ int swz_k(int k) {
  if constexpr (sizeof(T) == 2) return ROW_OPERAND ? (k & 1) | ((k & 2) << 2) : 2 * (k & 3) | ((k >> 3) & 1) << 3;
  else return ROW_OPERAND ? (k >> 2) & 3 : ((k >> 2) & 3) << 2;
}

// One operand's tile: EXT rows (or columns) of the M or N axis by 128 bytes of K, loaded by NW waves.
// KOUT: K is the outer axis in memory.
template <typename T, bool KOUT, bool ROW_OPERAND, int EXT, int NW>
struct Tile {
  static constexpr int kBytes = EXT * kRowBytes;
  static constexpr int kLoads = kBytes / (64 * 16 * NW);  // 16-byte loads per lane
  static_assert(kLoads * 64 * 16 * NW == kBytes, "tile shape");
  static constexpr int kPitch = KOUT ? EXT * int(sizeof(T)) : kRowBytes;
  static_assert(!KOUT || EXT >= 128, "the swizzle of K-outer rows needs 16 chunks");
  unsigned off[kLoads];  // buffer offset of the lane's chunk, or kLdsCopyOutside for a row or column past the end
  int k[kLoads];         // its first k within the tile

  // `valid`: rows (columns) of the tile that exist; K-contiguous rows r >= split continue at +jump bytes
  __device__ __forceinline__ void init(int wave, int lane, int64_t ld_bytes, int valid, int split, int valid2,
                                       int64_t jump) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int q = (wave * kLoads + i) * 64 + lane;
      if constexpr (KOUT) {
        const int row = q / (kPitch / 16), pos = q % (kPitch / 16);
        const int c = pos ^ swz_k<T, ROW_OPERAND>(row);
        k[i] = row;
        off[i] = c * kEpc<T> < valid ? unsigned(row * ld_bytes + c * 16) : kLdsCopyOutside;
      } else {
        const int row = q >> 3, pos = q & 7;
        const int c = pos ^ swz_row<ROW_OPERAND>(row);
        k[i] = c * kEpc<T>;
        const bool second = row >= split;
        const int r = second ? row - split : row;
        off[i] = r < (second ? valid2 : valid) ? unsigned(r * ld_bytes + (second ? jump : 0) + c * 16) : kLdsCopyOutside;
      }
    }
  }
  // base: the tile's first byte at this K step; left: K entries that remain
  __device__ __forceinline__ void load(const char* base, int left, char* lds, int wave) const {
    const mf_i32x4 source = lds_copy_source(base);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      lds_copy16(source, k[i] < left ? off[i] : kLdsCopyOutside, lds + (wave * kLoads + i) * 1024);
  }
};

// The 16-byte K piece kk (of 2) of a fragment.  row operand: group base + frag_row(r16, j); column operand: base + 16 j
// + r16.  16-bit types: k = 32 kk + 8 g + i; fp32: k = 16 kk + 4 g + i.
template <typename T, bool KOUT, bool ROW_OPERAND, int EXT>
__device__ __forceinline__ typename Mma<T>::Frag read_frag(const char* lds, int base, int j, int kk, int lane) {
  using Frag = typename Mma<T>::Frag;
  const int g = lane >> 4, r = lane & 15;
  if constexpr (!KOUT) {
    const int row = base + (ROW_OPERAND ? frag_row(r, j) : 16 * j + r);
    return *reinterpret_cast<const Frag*>(lds + row * kRowBytes + (((kk * 4 + g) ^ (r & 7)) << 4));
  } else if constexpr (sizeof(T) == 2) {
    // lane 4 e + a of a 16-lane group addresses 4 elements of row k = .. + e; the transposing read gives lane
    // 4 a + c element c of the pieces of rows e = 0..3
    const int e = r >> 2, a = r & 3;
    const int col = base + (ROW_OPERAND ? 16 * a + 4 * j : 16 * j + 4 * a);
    typedef __attribute__((__vector_size__(4 * sizeof(T)))) T Op4;
    Op4 h[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int k = 32 * kk + 8 * g + 4 * s + e;
      h[s] = read_tr16(reinterpret_cast<const T*>(lds + k * (EXT * 2) + (((col >> 3) ^ swz_k<T, ROW_OPERAND>(k)) << 4) +
                                                  (col & 4) * 2));
    }
    return __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
    const int col = base + (ROW_OPERAND ? frag_row(r, j) : 16 * j + r);
    Frag f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = 16 * kk + 4 * g + e;
      f[e] = *reinterpret_cast<const float*>(lds + k * (EXT * 4) + (((col >> 2) ^ swz_k<T, ROW_OPERAND>(k)) << 4) +
                                             (col & 3) * 4);
    }
    return f;
  }
}

struct Params {
  const char* a;      // row operand: W (kFwd, kBwd, kDx), x (kDw)
  const char* b;      // column operand: x (kFwd, kBwd), [dA dB] (kDx, kDw)
  int64_t lda, ldb;   // bytes between their rows
  int M, N, K;        // output columns (kFwd, kBwd: F), output rows (kDw: 2 Fp), K extent
  int F, Fp;          // hidden width, and its multiple of 64 that [dA dB] is laid out by
  int act;
  int mt, nt;         // tiles along M and N
  int full, tail;     // tiles computed whole, and tiles after them whose K is split
  int splits, steps;  // K splits of a tail tile, K steps of one
  void* out;          // h, [dA dB], dx or dW
  int64_t ldo;        // elements between its rows
  float* part;        // kDx, kDw: sums of the tail tiles' splits, fp32 [tail][splits][BN][BM]; kBwd: bias sums
                      // [column tiles' waves][2 Fp]
  const void* bias;   // [2F] or null
  const void* go;     // kBwd: [N, F]
  // fp16's [dA dB]: row n is kept times 2^exps[n] (kBwd, kDx); *lowest is the smallest of them (kBwd, kDw) and factors[n]
  // 2^(*lowest - exps[n]), zero up to a multiple of 64 (written by kBwd, read by kDw)
  int* exps;
  int* lowest;
  _Float16* factors;
};

// 16 consecutive elements, of which the first n exist; rows of odd lengths start off 16 bytes, which wide accesses may
template <typename T>
__device__ __forceinline__ void store16(T* p, const float (&v)[16], int n) {
  typedef T V __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
  constexpr int E = kEpc<T>;
  if (n >= 16) {
#pragma unroll
    for (int i = 0; i < 16 / E; ++i) {
      V o;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = Elem<T>::from_f32(v[i * E + e]);
      reinterpret_cast<V*>(p)[i] = o;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < n) p[i] = Elem<T>::from_f32(v[i]);
  }
}
template <typename T>
__device__ __forceinline__ void load16(const T* p, float (&v)[16], int n) {
  typedef T V __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
  constexpr int E = kEpc<T>;
  if (n >= 16) {
#pragma unroll
    for (int i = 0; i < 16 / E; ++i) {
      const V o = reinterpret_cast<const V*>(p)[i];
#pragma unroll
      for (int e = 0; e < E; ++e) v[i * E + e] = Elem<T>::to_f32(o[e]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = i < n ? Elem<T>::to_f32(p[i]) : 0.0f;
  }
}

// Row n of the product as a row of the output: kDw's run over [dA dB]'s columns, each half padded to Fp.
template <int MODE>
__device__ __forceinline__ bool out_row(const Params& p, int& n) {
  if (n >= p.N) return false;
  if constexpr (MODE == kDw) {
    const int f = n >= p.Fp ? n - p.Fp : n;
    n = n >= p.Fp ? p.F + f : f;
    return f < p.F;
  }
  return true;
}

// Tile t of the walk: groups of 8 column tiles, so that the tiles resident together share rows of both operands.
__device__ __forceinline__ void tile_of(const Params& p, int t, int& tm, int& tn) {
  const int group = t / (8 * p.mt);
  t -= group * 8 * p.mt;
  const int gn = min(8, p.nt - group * 8);
  tm = t / gn;
  tn = group * 8 + (t - tm * gn);
}

// WM waves of 128 rows (two groups of 64: gate and up of the same 64 hidden columns in kFwd and kBwd) by WN waves of
// 16 NT columns.
template <typename T, int MODE, int WM, int WN, int NT>
__global__ void __launch_bounds__(64 * WM * WN, 2) gemm_kernel(Params p) {
  constexpr int NW = WM * WN;
  constexpr int BM = WM * 128, BN = WN * NT * 16, BK = kBK<T>;
  constexpr bool kGated = MODE == kFwd || MODE == kBwd;
  constexpr bool kAOut = MODE == kDx || MODE == kDw;  // K is the outer axis of the row operand
  constexpr bool kBOut = MODE == kDw;
  constexpr int TM = kGated ? BM / 2 : BM;            // output columns per tile
  constexpr bool kScaled = std::is_same<T, _Float16>::value && MODE != kFwd;
  constexpr bool kFactors = kScaled && MODE == kDw;
  using TileA = Tile<T, kAOut, true, BM, NW>;
  using TileB = Tile<T, kBOut, false, BN, NW>;
  using Frag = typename Mma<T>::Frag;
  // two objects per operand, so that a load into one is known not to touch the reads of the other
  __shared__ __attribute__((aligned(1024))) char a0[TileA::kBytes];
  __shared__ __attribute__((aligned(1024))) char b0[TileB::kBytes];
  __shared__ __attribute__((aligned(1024))) char a1[TileA::kBytes];
  __shared__ __attribute__((aligned(1024))) char b1[TileB::kBytes];
  // kFactors: a K step's 64 factors (128 bytes; a copy by a wave writes 256)
  __shared__ __attribute__((aligned(1024))) char fac0[kFactors ? 256 : 16];
  __shared__ __attribute__((aligned(1024))) char fac1[kFactors ? 256 : 16];

  // XCD-aware order: blockIdx.x % 8 is the XCD; each gets a contiguous range of the whole tiles, then of the tail's
  // splits
  const int xcd = blockIdx.x & 7, turn = blockIdx.x >> 3;
  const int full_per = (p.full + 7) >> 3, tail_per = (p.tail * p.splits + 7) >> 3;
  int t, split = 0;
  const bool whole = turn < full_per;
  if (whole) {
    t = xcd * full_per + turn;
    if (t >= p.full) return;
  } else {
    const int k = xcd * tail_per + turn - full_per;
    if (turn - full_per >= tail_per || k >= p.tail * p.splits) return;
    t = p.full + k / p.splits;
    split = k % p.splits;
  }
  int tm, tn;
  tile_of(p, t, tm, tn);
  const int m0 = tm * TM, n0 = tn * BN;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  TileA ta;
  TileB tb;
  const char* pa = p.a;
  const char* pb = p.b;
  if constexpr (kGated) {
    ta.init(wave, lane, p.lda, p.F - m0, BM / 2, p.F - m0, int64_t(p.F) * p.lda);
    pa += int64_t(m0) * p.lda;
  } else {
    ta.init(wave, lane, p.lda, p.M - m0, BM, 0, 0);
    pa += int64_t(m0) * sizeof(T);
  }
  tb.init(wave, lane, p.ldb, p.N - n0, BN, 0, 0);
  pb += kBOut ? int64_t(n0) * sizeof(T) : int64_t(n0) * p.ldb;

  const int steps_all = (p.K + BK - 1) / BK;
  const int s0 = split * p.steps, s1 = whole ? steps_all : min(steps_all, s0 + p.steps);
  auto load = [&](int s, char* la, char* lb, char* lf) {
    const int k0 = s * BK;
    const int left = p.K - k0;
    const char* xa;
    int left_a = left;
    if constexpr (MODE == kDx) {
      // k runs over [dA dB]'s columns; each half of Fp has F rows of W
      const int half = k0 >= p.Fp ? p.Fp : 0;
      xa = pa + int64_t(k0 - half + (half ? p.F : 0)) * p.lda;
      left_a = p.F - (k0 - half);
    } else {
      xa = kAOut ? pa + int64_t(k0) * p.lda : pa + int64_t(k0) * int(sizeof(T));
    }
    const char* xb = kBOut ? pb + int64_t(k0) * p.ldb : pb + int64_t(k0) * int(sizeof(T));
    ta.load(xa, left_a, la, wave);
    tb.load(xb, left, lb, wave);
    if (kFactors && wave == 0)
      lds_copy4(lds_copy_source(p.factors + k0), lane < 32 ? lane * 4u : kLdsCopyOutside, lf);
  };

  if constexpr (kScaled && MODE == kBwd) {
    static_assert(BN <= 64 * NW, "a thread per column");
    if (m0 == 0) {
      const int n = n0 + int(threadIdx.x);
      if (n < min(n0 + BN, (p.N + 63) / 64 * 64))
        p.factors[n] = _Float16(n < p.N ? ldexpf(1.0f, *p.lowest - p.exps[n]) : 0.0f);
    }
  }
  if (s0 < s1) load(s0, a0, b0, fac0);
  if (s0 + 1 < s1) load(s0 + 1, a1, b1, fac1);

  // lane (g, r16) holds, for column n0 + .. + 16 i + r16 of the tile, group rows 16 g .. 16 g + 15; the bias is the
  // sums' start
  const int g = lane >> 4, r16 = lane & 15;
  mf_f32x4 acc[2][4][NT];
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      mf_f32x4 start = {0.f, 0.f, 0.f, 0.f};
      if constexpr (kGated) {
        if (p.bias) {
          const int f = m0 + wm * 64 + 16 * g + 4 * j;
          const T* bias = static_cast<const T*>(p.bias) + q * p.F + f;
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (f + r < p.F) start[r] = Elem<T>::to_f32(bias[r]);
        }
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) acc[q][j][i] = start;
    }

  // A K step is two 16-byte pieces of every fragment.  While one piece is multiplied the next is read from LDS into the
  // other registers; the barrier sits between the two, where the second piece of a tile is in registers, so its buffer
  // is free for the copy of the tile after next and the next tile has had a whole step to land.
  struct Frags {
    Frag a[2][4], b[NT];
    Frag factor;  // kFactors: of the piece's eight K rows
  };
  auto read = [&](Frags& f, const char* la, const char* lb, const char* lf, int kk) {
    if constexpr (kFactors) f.factor = *reinterpret_cast<const Frag*>(lf + kk * 64 + g * 16);
#pragma unroll
    for (int i = 0; i < NT; ++i) f.b[i] = read_frag<T, kBOut, false, BN>(lb, wn * NT * 16, i, kk, lane);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int base = kGated ? q * (BM / 2) + wm * 64 : wm * 128 + q * 64;
#pragma unroll
      for (int j = 0; j < 4; ++j) f.a[q][j] = read_frag<T, kAOut, true, BM>(la, base, j, kk, lane);
    }
  };
  auto multiply = [&](const Frags& f) {
    Frag b[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      if constexpr (kFactors) b[i] = f.b[i] * f.factor;
      else b[i] = f.b[i];
    }
    // fp32: one of the four K entries at a time, so that no product waits for the one before it
#pragma unroll
    for (int e = 0; e < Mma<T>::kParts; ++e)
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < NT; ++i) Mma<T>::run(f.a[q][j], b[i], acc[q][j][i], e);
  };
  // the order of the instructions of half a step: reads spread over the products
  auto interleave = [] {
    constexpr int kReads = (kAOut ? (sizeof(T) == 2 ? 16 : 32) : 8) + (kBOut ? (sizeof(T) == 2 ? 2 : 4) * NT : NT) +
                           (kFactors ? 1 : 0);
    constexpr int kMul = 8 * NT * (sizeof(T) == 2 ? 1 : 4);
    constexpr int kEach = kMul / kReads > 0 ? kMul / kReads : 1;
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);      // one LDS read
      __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);  // products
    }
  };
  auto half = [&](Frags& f0, Frags& f1, char* ca, char* cb, char* cf, int s, const char* na, const char* nb,
                  const char* nf) {
    read(f1, ca, cb, cf, 1);
    multiply(f0);
    interleave();
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) and lgkmcnt(0): the next tile has landed, this one is read
    __syncthreads();
    if (s + 2 < s1) load(s + 2, ca, cb, cf);
    read(f0, na, nb, nf, 0);  // after the last step: stale, not used
    multiply(f1);
    interleave();
  };
  if (s0 < s1) {
    Frags f0, f1;
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    __syncthreads();
    read(f0, a0, b0, fac0, 0);
    for (int s = s0; s < s1; s += 2) {
      half(f0, f1, a0, b0, fac0, s, a1, b1, fac1);
      if (s + 1 < s1) half(f0, f1, a1, b1, fac1, s + 1, a0, b0, fac0);
    }
  }

  constexpr bool kFast = sizeof(T) == 2;
  if constexpr (kGated) {
    const int f0 = m0 + wm * 64 + 16 * g;
    const int left = p.F - f0;
    if constexpr (MODE == kFwd) {
      with_activation(p.act, [&](auto act) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const int n = n0 + (wn * NT + i) * 16 + r16;
          float h[16];
#pragma unroll
          for (int e = 0; e < 16; ++e)
            h[e] = act_value<decltype(act)::value, kFast>(acc[0][e >> 2][i][e & 3]) * acc[1][e >> 2][i][e & 3];
          if (n < p.N) store16(static_cast<T*>(p.out) + int64_t(n) * p.ldo + f0, h, left);
        }
      });
    } else {
      // dA and dB take the place of a and b
      with_activation(p.act, [&](auto act) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const int n = n0 + (wn * NT + i) * 16 + r16;
          float go[16], da[16], db[16];
          if (n < p.N) load16(static_cast<const T*>(p.go) + int64_t(n) * p.F + f0, go, left);
          const int kept = kScaled && n < p.N ? p.exps[n] : 0;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float y, dy;
            act_both<decltype(act)::value, kFast>(acc[0][e >> 2][i][e & 3], y, dy);
            if constexpr (kScaled) go[e] = ldexpf(go[e], kept);
            const bool in = n < p.N && e < left;  // columns past F are zero, whatever x holds
            da[e] = in ? go[e] * acc[1][e >> 2][i][e & 3] * dy : 0.0f;
            db[e] = in ? go[e] * y : 0.0f;
            acc[0][e >> 2][i][e & 3] = kScaled ? ldexpf(da[e], -kept) : da[e];
            acc[1][e >> 2][i][e & 3] = kScaled ? ldexpf(db[e], -kept) : db[e];
          }
          if (n < p.N && f0 < p.Fp) {
            T* o = static_cast<T*>(p.out) + int64_t(n) * p.ldo + f0;
            store16(o, da, 16);
            store16(o + p.Fp, db, 16);
          }
        }
      });
      if (p.part) {
        float* row = p.part + int64_t(tn * WN + wn) * 2 * p.Fp + f0;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          float sum[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float v = 0.0f;
#pragma unroll
            for (int i = 0; i < NT; ++i) v += acc[q][e >> 2][i][e & 3];
            sum[e] = group16_sum(v);
          }
          if (r16 == 0 && f0 < p.Fp) store16(row + q * p.Fp, sum, 16);
        }
      }
    }
  } else {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int ml = wm * 128 + q * 64 + 16 * g;
      const int m = m0 + ml;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int nl = (wn * NT + i) * 16 + r16;
        int n = n0 + nl;
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = acc[q][e >> 2][i][e & 3];
        if constexpr (kScaled) {
          const int e_n = MODE == kDw ? *p.lowest : n < p.N ? p.exps[n] : 0;
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = ldexpf(v[e], -e_n);
        }
        if (!whole) {
          store16(p.part + ((int64_t(t - p.full) * p.splits + split) * BN + nl) * BM + ml, v, 16);
        } else if (out_row<MODE>(p, n) && m < p.ldo) {
          store16(static_cast<T*>(p.out) + int64_t(n) * p.ldo + m, v, int(p.ldo) - m);
        }
      }
    }
  }
}

// The forward of few tokens (N <= 16 NT <= 64): the weights are read once, straight into the matrix operands, and the
// tile kernel's copies and barriers would only add to the latency.  A workgroup owns 16 hidden columns (their gate and
// up rows); its four waves take a quarter of K each and meet in LDS.
template <typename T, int NT>
__global__ void __launch_bounds__(256) few_kernel(Params p) {
  using Frag = typename Mma<T>::Frag;
  constexpr int E = kEpc<T>, KS = 4 * E;  // K entries of a fragment's four lane groups
  constexpr int kAhead = NT == 4 ? 2 : 4;  // steps in flight
  __shared__ mf_f32x4 part[4][2][NT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, r16 = lane & 15;
  const int f0 = blockIdx.x * 16;
  const int fr = min(f0 + r16, p.F - 1);  // rows past the end repeat the last: their results are not stored
  const T* wg = reinterpret_cast<const T*>(p.a + int64_t(fr) * p.lda) + g * E;
  const T* wu = reinterpret_cast<const T*>(p.a + (int64_t(p.F) + fr) * p.lda) + g * E;
  const T* x[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
    x[i] = reinterpret_cast<const T*>(p.b + int64_t(min(16 * i + r16, p.N - 1)) * p.ldb) + g * E;
  mf_f32x4 acc[2][NT];
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[q][i] = mf_f32x4{0.f, 0.f, 0.f, 0.f};
  const int steps = (p.K + KS - 1) / KS;
  const int quarter = (steps + 3) / 4;
  const int s1 = min(steps, (wave + 1) * quarter);
  for (int s = wave * quarter; s < s1; s += kAhead) {
    Frag a[kAhead], u[kAhead], b[kAhead][NT];
#pragma unroll
    for (int d = 0; d < kAhead; ++d) {
      const int k = (s + d) * KS;
      const bool in = s + d < s1 && k + g * E < p.K;  // K is a multiple of E
      // (one zero on each side: what lies behind a row could be NaN)
      Frag zero = {};
      a[d] = in ? *reinterpret_cast<const Frag*>(wg + k) : zero;
      u[d] = in ? *reinterpret_cast<const Frag*>(wu + k) : zero;
#pragma unroll
      for (int i = 0; i < NT; ++i) b[d][i] = in ? *reinterpret_cast<const Frag*>(x[i] + k) : zero;
    }
#pragma unroll
    for (int d = 0; d < kAhead; ++d)
#pragma unroll
      for (int e = 0; e < Mma<T>::kParts; ++e)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          Mma<T>::run(a[d], b[d][i], acc[0][i], e);
          Mma<T>::run(u[d], b[d][i], acc[1][i], e);
        }
  }
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int i = 0; i < NT; ++i) part[wave][q][i][lane] = acc[q][i];
  __syncthreads();
  // wave i finishes tokens 16 i ..: lane (g, r16) holds columns 4 g .. + 3 of token 16 i + r16
  const int i = wave, n = 16 * i + r16;
  if (i >= NT || n >= p.N) return;
  const T* bias = static_cast<const T*>(p.bias);
  with_activation(p.act, [&](auto act) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int f = f0 + 4 * g + r;
      if (f >= p.F) break;
      float a = bias ? Elem<T>::to_f32(bias[f]) : 0.0f, b = bias ? Elem<T>::to_f32(bias[p.F + f]) : 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        a += part[w][0][i][lane][r];
        b += part[w][1][i][lane][r];
      }
      static_cast<T*>(p.out)[int64_t(n) * p.ldo + f] =
          Elem<T>::from_f32(act_value<decltype(act)::value, sizeof(T) == 2>(a) * b);
    }
  });
}

// The tail tiles' outputs: each the sum of its splits, in order.  Four columns a thread.
template <typename T, int MODE>
__global__ void __launch_bounds__(256) tail_kernel(Params p, int bm, int bn) {
  const int cols = bm / 4;
  const int rows_block = 256 / cols;
  const int blocks_tile = bn / rows_block;
  const int tile = blockIdx.x / blocks_tile;
  const int nl = (blockIdx.x - tile * blocks_tile) * rows_block + threadIdx.x / cols;
  const int ml = (threadIdx.x % cols) * 4;
  int tm, tn;
  tile_of(p, p.full + tile, tm, tn);
  int n = tn * bn + nl;
  const int m = tm * bm + ml;
  if (!out_row<MODE>(p, n) || m >= p.ldo) return;
  const float* src = p.part + (int64_t(tile) * p.splits * bn + nl) * bm + ml;
  mf_f32x4 v = *reinterpret_cast<const mf_f32x4*>(src);
  for (int s = 1; s < p.splits; ++s) v += *reinterpret_cast<const mf_f32x4*>(src + int64_t(s) * bn * bm);
  T* out = static_cast<T*>(p.out) + int64_t(n) * p.ldo + m;
  if (m + 4 <= p.ldo) {
    typedef T V __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    V o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = Elem<T>::from_f32(v[e]);
    *reinterpret_cast<V*>(out) = o;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (m + e < p.ldo) out[e] = Elem<T>::from_f32(v[e]);
  }
}

// fp16's [dA dB]: how large it can get (see the top).  Two launches: of every workgroup's rows of W the largest norms and
// biases, (gate, up) each; then of every token its exponent, and the smallest of all, a minimum of integers (its order does
// not matter).  What is not finite decides nothing: a row of x or W with such an entry has no finite value in [dA dB]'s
// row or column anyway.
constexpr int kTopExp = 40;       // of a token without a gradient: 2^-24 <= B_n, so that e_n <= 37 elsewhere
constexpr int kNormBlocks = 256;  // workgroups of the first launch at most

__device__ __forceinline__ float finite_or_zero(float v) { return fabsf(v) <= 3.0e38f ? fabsf(v) : 0.0f; }

__global__ void __launch_bounds__(256) weight_reach_kernel(const char* w, int64_t ldw, const _Float16* bias, int F, int K,
                                                           float4* reach, int* lowest) {
  __shared__ float4 waves[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float4 top = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int f = blockIdx.x * 4 + wave; f < 2 * F; f += gridDim.x * 4) {
    const _Float16* row = reinterpret_cast<const _Float16*>(w + int64_t(f) * ldw);
    float sum = 0.0f;
    for (int c = lane * 8; c < K; c += 512) {  // K is a multiple of 8, the rows are aligned
      const mf_f16x8 v = *reinterpret_cast<const mf_f16x8*>(row + c);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += float(v[e]) * float(v[e]);
    }
    const float norm = sqrtf(finite_or_zero(wave_sum(sum)));
    const float b = bias ? finite_or_zero(float(bias[f])) : 0.0f;
    if (f < F) {
      top.x = fmaxf(top.x, norm);
      top.z = fmaxf(top.z, b);
    } else {
      top.y = fmaxf(top.y, norm);
      top.w = fmaxf(top.w, b);
    }
  }
  if (lane == 0) waves[wave] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 4; ++i)
      top = make_float4(fmaxf(top.x, waves[i].x), fmaxf(top.y, waves[i].y), fmaxf(top.z, waves[i].z), fmaxf(top.w, waves[i].w));
    reach[blockIdx.x] = top;
    if (blockIdx.x == 0) *lowest = kTopExp;
  }
}

// A wave per token; sixteen waves a workgroup and one workgroup a CU, because the minimum's atomics take their time (32768 x
// 768 x 2048, 184 MB: 47 us, with 4096 workgroups of four waves 65).
constexpr int kExpWaves = 16;
__global__ void __launch_bounds__(64 * kExpWaves) token_exp_kernel(const char* x, int64_t ldx, const _Float16* go, int T, int F, int K,
                                                        const float4* reach, int blocks, int* exps, int* lowest) {
  typedef _Float16 U __attribute__((ext_vector_type(8), aligned(2)));
  __shared__ int low[kExpWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float4 top = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = lane; i < blocks; i += 64) {
    const float4 r = reach[i];
    top = make_float4(fmaxf(top.x, r.x), fmaxf(top.y, r.y), fmaxf(top.z, r.z), fmaxf(top.w, r.w));
  }
  top = make_float4(wave_max(top.x), wave_max(top.y), wave_max(top.z), wave_max(top.w));
  int least = kTopExp;
  for (int64_t n = int64_t(blockIdx.x) * kExpWaves + wave; n < T; n += int64_t(gridDim.x) * kExpWaves) {
    const _Float16* row = reinterpret_cast<const _Float16*>(x + n * ldx);
    float sum = 0.0f, peak = 0.0f;
    for (int c = lane * 8; c < K; c += 512) {
      const mf_f16x8 v = *reinterpret_cast<const mf_f16x8*>(row + c);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += float(v[e]) * float(v[e]);
    }
    const _Float16* grad = go + n * F;
    for (int f = lane * 8; f < F; f += 512) {
      if (f + 8 <= F) {
        const U v = *reinterpret_cast<const U*>(grad + f);
#pragma unroll
        for (int e = 0; e < 8; ++e) peak = fmaxf(peak, finite_or_zero(float(v[e])));
      } else {
        for (int e = f; e < F; ++e) peak = fmaxf(peak, finite_or_zero(float(grad[e])));
      }
    }
    const float norm = sqrtf(finite_or_zero(wave_sum(sum)));
    peak = wave_max(peak);
    const float bound = 1.25f * peak * fmaxf(fmaxf(norm * top.x + top.z, norm * top.y + top.w), 1.0f);
    const int e = peak > 0.0f ? 13 - ilogbf(bound) : kTopExp;
    least = min(least, e);
    if (lane == 0) exps[n] = e;
  }
  if (lane == 0) low[wave] = least;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kExpWaves; ++i) least = min(least, low[i]);
    atomicMin(lowest, least);
  }
}

// dbias: column sums of `rows` partial rows of [2 Fp], 16 columns a workgroup, 16 strands of rows each.
template <typename T>
__global__ void __launch_bounds__(256) bias_kernel(const float* part, T* out, int rows, int F, int Fp) {
  __shared__ float sums[16][17];
  const int c = threadIdx.x & 15, strand = threadIdx.x >> 4;
  const int col = blockIdx.x * 16 + c;  // of the 2 Fp
  float v = 0.0f;
#pragma unroll 8
  for (int r = strand; r < rows; r += 16) v += part[int64_t(r) * 2 * Fp + col];
  sums[strand][c] = v;
  __syncthreads();
  if (strand == 0) {
    float s = 0.0f;
    for (int k = 0; k < 16; ++k) s += sums[k][c];
    const int f = col >= Fp ? col - Fp : col;
    if (f < F) out[(col >= Fp ? F : 0) + f] = Elem<T>::from_f32(s);
  }
}

// Rows of `cols` elements, `ld` apart, into rows of `pitch`, zero behind: the aligned copies of the operands whose rows
// are no multiple of 16 bytes.  16 bytes a thread and one launch for both: 9.7 us of the 27 of 1400 x 765 x 2048 bf16
// (8 MB in, 8 MB out), where an element a thread and two launches made it 33.
struct Pad {
  const void* src;
  void* dst;
  int64_t ld, chunks;
};
template <typename T>
__global__ void __launch_bounds__(256) pad_kernel(Pad x, Pad w, int cols, int pitch) {
  typedef T V __attribute__((ext_vector_type(16 / sizeof(T))));
  typedef T U __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
  constexpr int E = kEpc<T>;
  const unsigned row_chunks = pitch / E;
  // a grid of 2^32 threads and more is no launch: every thread goes on by the grid's size
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < x.chunks + w.chunks; i += int64_t(gridDim.x) * 256) {
    const bool is_x = i < x.chunks;
    const int64_t j = is_x ? i : i - x.chunks;
    const int64_t r = j >> 32 ? j / row_chunks : unsigned(j) / row_chunks;
    const int c = int(j - r * row_chunks) * E;
    const T* src = static_cast<const T*>(is_x ? x.src : w.src) + r * (is_x ? x.ld : w.ld) + c;
    V v;
    if (c + E <= cols) {
      v = *reinterpret_cast<const U*>(src);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = c + e < cols ? src[e] : T(0.0f);
    }
    reinterpret_cast<V*>(is_x ? x.dst : w.dst)[j] = v;
  }
}

// -- host ----------------------------------------------------------------------------------------------------
size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// How a product is cut.  Tiles of 256 x 256 (16-bit types) run one workgroup per CU, tiles of 128 x 128 two (fp32: one
// fills the matrix cores); `slots` is what is to be resident at once.  Tiles that fill every slot are computed whole;
// the rest, which would leave slots idle for a whole tile's time, are cut along K so that their pieces fill the slots,
// where K is long enough to pay for writing and adding the pieces' fp32 sums.
struct Cut {
  bool large;
  int bn;  // columns of a tile: 256 (large), 128 or 64
  int full, tail, splits, steps;
  size_t bytes;
};
Cut cut_tiles(int64_t m, int64_t n, int64_t k, int esize, bool large, bool split, int num_cus) {
  Cut c;
  c.large = large;
  const int b = large ? 256 : 128;
  c.bn = b;
  const int64_t tiles = ((m + b - 1) / b) * ((n + b - 1) / b);
  const int64_t slots = large || esize == 4 ? num_cus : 2 * num_cus;
  const int64_t steps = (k * esize + kRowBytes - 1) / kRowBytes;
  const int64_t tail = tiles % slots;
  int64_t s = tail > 0 ? std::min(slots / tail, steps / 4) : 1;
  if (!split || s < 2 || steps - steps / s < 16) s = 1;
  c.tail = s > 1 ? int(tail) : 0;
  c.full = int(tiles - c.tail);
  c.steps = int((steps + s - 1) / s);
  c.splits = s > 1 ? int((steps + c.steps - 1) / c.steps) : 1;
  c.bytes = round256(size_t(c.tail) * c.splits * b * b * 4);
  return c;
}
constexpr int kFewTokens = 64;  // the forward of few_kernel
// kFwd and kBwd: large tiles once the small ones need more than one round of two a CU, that is when more than half the
// CUs get a large one.  bf16, C 512, F 2048, large against small: 1400 tokens (96 large tiles) 17.6 and 13.6 us, 2000
// (128) 17.9 and 14.2, 2304 (144) 18.9 and 22.6, 3500 (224) 20.5 and 26.0 (at this width only: the rule leaves out K, and
// at 176 large tiles, 2738 tokens, 31 % of the CUs idle).  fp32, whose matrix rate is a sixteenth, takes small ones.
Cut cut_gated(int64_t f, int64_t t, int64_t k, int esize, int num_cus) {
  const bool large = esize == 2 && 2 * ((2 * f + 255) / 256) * ((t + 255) / 256) > num_cus;
  // a large tile is 128 of f and their gate and up rows, a small one 64
  Cut c = cut_tiles(2 * f, t, k, esize, large, false, num_cus);
  const int64_t fb = large ? 128 : 64;
  auto tiles = [&](int64_t bn) { return (f + fb - 1) / fb * ((t + bn - 1) / bn); };
  // fp32 products fill the matrix cores from one workgroup, so what counts is the tiles of the busiest CU: half as wide
  // ones where those add up to less (2432 rows, 1024 hidden: 3 of 64 columns instead of 2 of 128, 58 -> 47 us)
  auto busiest = [&](int64_t bn) { return (tiles(bn) + num_cus - 1) / num_cus * bn; };
  if (esize == 4 && busiest(64) < busiest(128)) c.bn = 64;
  c.full = int(tiles(c.bn));
  return c;
}
// kDx and kDw: large tiles when their K pieces can fill the CUs with at least 16 steps each.
Cut cut_product(int64_t m, int64_t n, int64_t k, int esize, int num_cus) {
  const int64_t tiles = ((m + 255) / 256) * ((n + 255) / 256);
  const int64_t steps = (k * esize + kRowBytes - 1) / kRowBytes;
  const bool large = esize == 2 && tiles * std::max<int64_t>(1, steps / 16) >= num_cus;
  return cut_tiles(m, n, k, esize, large, true, num_cus);
}

struct Plan {
  int64_t T, C, F, Fp, Cp;  // Cp: channels of the padded copies (C when none is needed)
  int esize;
  bool pad_x, pad_w;
  size_t x_bytes, w_bytes, dab_bytes, bias_bytes;
  size_t reach_bytes, exps_bytes, factors_bytes;  // fp16's backward
  Cut gated, dx, dw;
  size_t bwd_bytes() const {
    return x_bytes + w_bytes + dab_bytes + bias_bytes + reach_bytes + exps_bytes + factors_bytes + dx.bytes + dw.bytes;
  }
};

void make_plan(Plan* q, int64_t T, int64_t C, int64_t F, int64_t x_stride, const void* x, const void* w, int dtype,
               bool need_dx, bool need_dw, bool need_db, int num_cus) {
  q->T = T;
  q->C = C;
  q->F = F;
  q->esize = dtype == MF_DTYPE_F32 ? 4 : 2;
  q->Fp = (F + 63) / 64 * 64;
  const bool odd = C * q->esize % 16 != 0;
  q->pad_x = odd || x_stride * q->esize % 16 != 0 || reinterpret_cast<uintptr_t>(x) % 16 != 0;
  q->pad_w = odd || reinterpret_cast<uintptr_t>(w) % 16 != 0;
  q->Cp = (C * q->esize + 15) / 16 * 16 / q->esize;
  q->x_bytes = q->pad_x ? round256(size_t(T) * q->Cp * q->esize) : 0;
  q->w_bytes = q->pad_w ? round256(size_t(2) * F * q->Cp * q->esize) : 0;
  q->dab_bytes = need_dx || need_dw ? round256(size_t(T) * 2 * q->Fp * q->esize) : 0;
  const bool scaled = dtype == MF_DTYPE_F16 && (need_dx || need_dw || need_db);
  q->reach_bytes = scaled ? 256 + kNormBlocks * sizeof(float4) : 0;  // the smallest exponent, the weights' reach
  q->exps_bytes = scaled ? round256(size_t(T) * 4) : 0;
  q->factors_bytes = scaled ? round256(size_t((T + 63) / 64 * 64) * 2) : 0;
  q->gated = cut_gated(F, T, q->Cp, q->esize, num_cus);
  // bias sums of every column wave, four a tile
  q->bias_bytes = need_db ? round256(size_t((T + q->gated.bn - 1) / q->gated.bn) * 4 * 2 * q->Fp * 4) : 0;
  q->dx = cut_product(q->Cp, T, 2 * q->Fp, q->esize, num_cus);
  q->dw = cut_product(q->Cp, 2 * q->Fp, T, q->esize, num_cus);
  if (!need_dx) q->dx.bytes = 0;
  if (!need_dw) q->dw.bytes = 0;
}

template <typename T, int MODE>
void launch_gemm(Params p, const Cut& c, hipStream_t s) {
  const bool gated = MODE == kFwd || MODE == kBwd;
  const int b = c.large ? 256 : 128;
  const int tm = gated ? b / 2 : b;
  p.mt = (p.M + tm - 1) / tm;
  p.nt = (p.N + c.bn - 1) / c.bn;
  p.full = c.full;
  p.tail = c.tail;
  p.splits = c.splits;
  p.steps = c.steps;
  const int64_t per = (c.full + 7) / 8 + (int64_t(c.tail) * c.splits + 7) / 8;
  const dim3 grid(unsigned(per * 8));
  if constexpr (sizeof(T) == 2) {
    if (c.large) hipLaunchKernelGGL((gemm_kernel<T, MODE, 2, 4, 4>), grid, dim3(512), 0, s, p);
  }
  if constexpr (sizeof(T) == 4 && (MODE == kFwd || MODE == kBwd)) {
    if (c.bn == 64) hipLaunchKernelGGL((gemm_kernel<T, MODE, 1, 4, 1>), grid, dim3(256), 0, s, p);
  }
  if (c.bn == 128) hipLaunchKernelGGL((gemm_kernel<T, MODE, 1, 4, 2>), grid, dim3(256), 0, s, p);
  if constexpr (MODE == kDx || MODE == kDw) {
    if (c.tail > 0)
      hipLaunchKernelGGL((tail_kernel<T, MODE>), dim3(unsigned(c.tail * (b * b / 1024))), dim3(256), 0, s, p, b, b);
  }
}

// x and W, as the tile kernel reads them: in place, or their aligned copies at ws
template <typename T>
char* operands(const Plan& q, const void* x, int64_t x_stride, const void* w, char* ws, Params* p, hipStream_t s) {
  const int64_t row_chunks = q.Cp / kEpc<T>;
  Pad px = {x, ws, x_stride, q.pad_x ? q.T * row_chunks : 0};
  Pad pw = {w, ws + q.x_bytes, q.C, q.pad_w ? 2 * q.F * row_chunks : 0};
  p->a = static_cast<const char*>(q.pad_w ? pw.dst : w);
  p->lda = (q.pad_w ? q.Cp : q.C) * sizeof(T);
  p->b = static_cast<const char*>(q.pad_x ? px.dst : x);
  p->ldb = (q.pad_x ? q.Cp : x_stride) * sizeof(T);
  p->F = int(q.F);
  p->Fp = int(q.Fp);
  const int64_t blocks = (px.chunks + pw.chunks + 255) / 256;
  if (blocks > 0)
    hipLaunchKernelGGL(pad_kernel<T>, dim3(unsigned(std::min<int64_t>(blocks, 1 << 20))), dim3(256), 0, s, px, pw,
                       int(q.C), int(q.Cp));
  return ws + q.x_bytes + q.w_bytes;
}

bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

template <typename T>
int forward(const mf_gated_linear_args* a, const Plan& q, hipStream_t s) {
  Params p = {};
  operands<T>(q, a->x, a->x_stride, a->weight, static_cast<char*>(a->workspace), &p, s);
  p.M = int(q.F);
  p.N = int(q.T);
  p.K = int(q.Cp);
  p.act = a->activation;
  p.out = a->out;
  p.ldo = q.F;
  p.bias = a->bias;
  const dim3 few(unsigned((q.F + 15) / 16));
  if (q.T <= 16) hipLaunchKernelGGL((few_kernel<T, 1>), few, dim3(256), 0, s, p);
  else if (q.T <= 32) hipLaunchKernelGGL((few_kernel<T, 2>), few, dim3(256), 0, s, p);
  else if (q.T <= kFewTokens) hipLaunchKernelGGL((few_kernel<T, 4>), few, dim3(256), 0, s, p);
  else launch_gemm<T, kFwd>(p, q.gated, s);
  MF_HIP_CHECK(hipGetLastError());
  return MF_OK;
}

template <typename T>
int backward(const mf_gated_linear_bwd_args* a, const Plan& q, int num_cus, hipStream_t s) {
  const mf_gated_linear_args& f = a->fwd;
  Params p = {};
  char* ws = operands<T>(q, f.x, f.x_stride, f.weight, static_cast<char*>(a->workspace), &p, s);
  const char *w = p.a, *x = p.b;
  const int64_t ldw = p.lda, ldx = p.ldb;
  T* dab = reinterpret_cast<T*>(ws);
  ws += round256(size_t(q.T) * 2 * q.Fp * sizeof(T));
  float* sums = a->dbias ? reinterpret_cast<float*>(ws) : nullptr;
  ws += q.bias_bytes;
  p.M = int(q.F);
  p.N = int(q.T);
  p.K = int(q.Cp);
  p.act = f.activation;
  p.out = dab;
  p.ldo = 2 * q.Fp;
  p.bias = f.bias;
  p.go = a->grad_out;
  p.part = sums;
  if constexpr (std::is_same<T, _Float16>::value) {
    p.lowest = reinterpret_cast<int*>(ws);
    float4* reach = reinterpret_cast<float4*>(ws + 256);
    ws += q.reach_bytes;
    p.exps = reinterpret_cast<int*>(ws);
    ws += q.exps_bytes;
    p.factors = reinterpret_cast<_Float16*>(ws);
    ws += q.factors_bytes;
    const int blocks = int(std::min<int64_t>((2 * q.F + 3) / 4, kNormBlocks));
    hipLaunchKernelGGL(weight_reach_kernel, dim3(unsigned(blocks)), dim3(256), 0, s, w, ldw,
                       static_cast<const _Float16*>(f.bias), p.F, p.K, reach, p.lowest);
    if (q.T > 0) {
      const int64_t groups = std::min<int64_t>((q.T + kExpWaves - 1) / kExpWaves, num_cus);
      hipLaunchKernelGGL(token_exp_kernel, dim3(unsigned(groups)), dim3(64 * kExpWaves), 0, s, x, ldx,
                         static_cast<const _Float16*>(a->grad_out), p.N, p.F, p.K, reach, blocks, p.exps, p.lowest);
    }
  }
  if (q.T > 0) launch_gemm<T, kBwd>(p, q.gated, s);
  MF_HIP_CHECK(hipGetLastError());
  if (a->dbias) {
    const int rows = int((q.T + q.gated.bn - 1) / q.gated.bn) * 4;
    hipLaunchKernelGGL(bias_kernel<T>, dim3(unsigned(2 * q.Fp / 16)), dim3(256), 0, s, sums, static_cast<T*>(a->dbias),
                       rows, int(q.F), int(q.Fp));
    MF_HIP_CHECK(hipGetLastError());
  }
  if (a->dx && q.T > 0) {
    Params d = p;
    d.a = w;
    d.lda = ldw;
    d.b = reinterpret_cast<const char*>(dab);
    d.ldb = 2 * q.Fp * sizeof(T);
    d.M = int(q.Cp);
    d.N = int(q.T);
    d.K = int(2 * q.Fp);
    d.out = a->dx;
    d.ldo = q.C;
    d.part = reinterpret_cast<float*>(ws);
    launch_gemm<T, kDx>(d, q.dx, s);
    MF_HIP_CHECK(hipGetLastError());
    ws += q.dx.bytes;
  }
  if (a->dweight) {
    Params d = p;
    d.a = x;
    d.lda = ldx;
    d.b = reinterpret_cast<const char*>(dab);
    d.ldb = 2 * q.Fp * sizeof(T);
    d.M = int(q.Cp);
    d.N = int(2 * q.Fp);
    d.K = int(q.T);
    d.out = a->dweight;
    d.ldo = q.C;
    d.part = reinterpret_cast<float*>(ws);
    launch_gemm<T, kDw>(d, q.dw, s);
    MF_HIP_CHECK(hipGetLastError());
  }
  return MF_OK;
}

int check(const char* name, const mf_gated_linear_args* a) {
  const std::string n(name);
  if (!a->x || !a->weight) return fail(MF_ERR_INVALID_ARGUMENT, n + ": x and weight must be non-NULL");
  if (a->tokens < 0 || a->channels <= 0 || a->hidden <= 0 || a->x_stride < a->channels)
    return fail(MF_ERR_INVALID_ARGUMENT, n + ": tokens must be non-negative, channels and hidden positive, x_stride >= channels");
  if (a->dtype != MF_DTYPE_F32 && a->dtype != MF_DTYPE_F16 && a->dtype != MF_DTYPE_BF16)
    return fail(MF_ERR_INVALID_ARGUMENT, n + ": bad dtype");
  if (a->activation < MF_ACT_SILU || a->activation > MF_ACT_SIGMOID)
    return fail(MF_ERR_INVALID_ARGUMENT, n + ": bad activation");
  // tile-relative byte offsets are 32 bits: the weight below 2^31 bytes, 256 rows of x and of [dA dB] too
  const int64_t esize = a->dtype == MF_DTYPE_F32 ? 4 : 2;
  const int64_t reach = (int64_t(1) << 31) / (256 * esize);  // elements between rows: 2^22, of fp32 2^21
  if (a->tokens > (1 << 30)) return fail(MF_ERR_UNSUPPORTED, n + ": at most 2^30 tokens");
  if (a->x_stride >= reach)
    return fail(MF_ERR_UNSUPPORTED, n + ": rows of x " + std::to_string(reach) + " elements apart and more are not supported");
  if ((a->channels + 8) * int64_t(a->hidden) * 2 * esize >= (int64_t(1) << 31))
    return fail(MF_ERR_UNSUPPORTED, n + ": a weight of 2^31 bytes and more is not supported");
  if (2 * (int64_t(a->hidden) + 64) >= reach)
    return fail(MF_ERR_UNSUPPORTED, n + ": hidden above " + std::to_string(reach / 2 - 65) + " is not supported");
  return MF_OK;
}

}  // namespace gated
}  // namespace mf

extern "C" uint64_t mf_gated_linear_workspace_size(const mf_gated_linear_args* a) {
  using namespace mf;
  using namespace mf::gated;
  if (a == nullptr || check("mf_gated_linear_workspace_size", a) != MF_OK) return 0;
  Plan q;
  make_plan(&q, a->tokens, a->channels, a->hidden, a->x_stride, a->x, a->weight, a->dtype, false, false, false, 256);
  return q.x_bytes + q.w_bytes;
}

extern "C" int mf_gated_linear(const mf_gated_linear_args* a, void* stream) {
  using namespace mf;
  using namespace mf::gated;
  if (a == nullptr) return fail(MF_ERR_INVALID_ARGUMENT, "mf_gated_linear: args is NULL");
  int st = check("mf_gated_linear", a);
  if (st != MF_OK) return st;
  if (!a->out) return fail(MF_ERR_INVALID_ARGUMENT, "mf_gated_linear: out must be non-NULL");
  if (a->tokens == 0) return MF_OK;
  DeviceInfo info;
  st = device_info(&info);
  if (st != MF_OK) return st;
  Plan q;
  make_plan(&q, a->tokens, a->channels, a->hidden, a->x_stride, a->x, a->weight, a->dtype, false, false, false,
            info.num_cus);
  if (q.x_bytes + q.w_bytes > 0 &&
      (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < q.x_bytes + q.w_bytes))
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_gated_linear: the workspace must be 16-byte aligned and hold "
                                         "mf_gated_linear_workspace_size bytes");
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (a->dtype) {
    case MF_DTYPE_BF16: return forward<__bf16>(a, q, s);
    case MF_DTYPE_F16: return forward<_Float16>(a, q, s);
    default: return forward<float>(a, q, s);
  }
}

static int bwd_plan(const mf_gated_linear_bwd_args* a, mf::gated::Plan* q, int num_cus) {
  using namespace mf;
  using namespace mf::gated;
  const int st = check("mf_gated_linear_bwd", &a->fwd);
  if (st != MF_OK) return st;
  const mf_gated_linear_args& f = a->fwd;
  make_plan(q, f.tokens, f.channels, f.hidden, f.x_stride, f.x, f.weight, f.dtype, a->dx != nullptr,
            a->dweight != nullptr, a->dbias != nullptr, num_cus);
  q->dab_bytes = round256(size_t(q->T) * 2 * q->Fp * q->esize);
  return MF_OK;
}

extern "C" uint64_t mf_gated_linear_bwd_workspace_size(const mf_gated_linear_bwd_args* a) {
  using namespace mf;
  using namespace mf::gated;
  DeviceInfo info;
  Plan q;
  if (a == nullptr || check("mf_gated_linear_bwd_workspace_size", &a->fwd) != MF_OK) return 0;
  if (device_info(&info) != MF_OK || bwd_plan(a, &q, info.num_cus) != MF_OK) return 0;
  return q.bwd_bytes();
}

extern "C" int mf_gated_linear_bwd(const mf_gated_linear_bwd_args* a, void* stream) {
  using namespace mf;
  using namespace mf::gated;
  if (a == nullptr) return fail(MF_ERR_INVALID_ARGUMENT, "mf_gated_linear_bwd: args is NULL");
  int st = check("mf_gated_linear_bwd", &a->fwd);
  if (st != MF_OK) return st;
  if (!a->grad_out) return fail(MF_ERR_INVALID_ARGUMENT, "mf_gated_linear_bwd: grad_out must be non-NULL");
  if (!a->dx && !a->dweight && !a->dbias)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_gated_linear_bwd: nothing to compute");
  DeviceInfo info;
  st = device_info(&info);
  if (st != MF_OK) return st;
  Plan q;
  st = bwd_plan(a, &q, info.num_cus);
  if (st != MF_OK) return st;
  const size_t need = q.bwd_bytes();
  if (need > 0 && (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < need))
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_gated_linear_bwd: the workspace must be 16-byte aligned and hold "
                                         "mf_gated_linear_bwd_workspace_size bytes");
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (a->fwd.dtype) {
    case MF_DTYPE_BF16: return backward<__bf16>(a, q, info.num_cus, s);
    case MF_DTYPE_F16: return backward<_Float16>(a, q, info.num_cus, s);
    default: return backward<float>(a, q, info.num_cus, s);
  }
}
