// Gradients of attention with a bias by buckets (mf_bucket_attn_bwd) on gfx950.
// With m_i, a number near the row's maximum of x = log2(e) S (x - m_i < 1), and
// 1 / l_i, 1 over the row's sum of 2^(x - m_i), as the forward leaves them,
//   e_ij = 2^(log2(e) (scale q_i . k_j + bias_ij) - m_i),  P_ij = e_ij / l_i,
//   dv_j = sum_i P_ij go_i,           dP_ij = go_i . v_j,
//   dS_ij = P_ij (dP_ij - delta_i),   delta_i = go_i . out_i - dlse_i,
//   dq_i = scale sum_j dS_ij k_j,     dk_j = scale sum_i dS_ij q_i,
//   dtable[c, h] = sum of dS_ij over the pairs of bucket c
// (10 D flops a pair).  m and 1 / l are kept apart, and x - m is formed as the
// forward forms it: a row all of whose biases are huge and negative (a finite
// mask value) has P of one all the same, where exp(x - lse) would lose it in
// lse's rounding.
//
// Three kernels; the last two have workgroups of 128 columns, a wave 32, and
// stream 64-row tiles X and Y of the other side through LDS:
//   rows:    delta from the forward's out (and what its rounding left)
//   queries: columns are queries (Q, go in registers), rows keys (X = K, Y = V):
//            dq^T += K^T dS.  A column is one query, so dS is kept without 1 / l,
//            which the sum gets at the end.  The sum of a query's dS, which is
//            dlse_i but for delta's error (out is a product of rounded P), corrects
//            delta for the next kernel.  dq itself keeps that error, at most a
//            rounding of P in size: scale (delta's error) sum_j P_ij k_j.
//   keys:    columns are keys (K, V in registers), rows the queries of every head
//            of the key head (X = Q, Y = go): dk^T += Q^T dS, dv^T += go^T P, and
//            the table's gradient, in which delta's error would not cancel (with it
//            dtable is off by 2e-3 of the largest entry, without by 1e-6)
// On 32 x 8 heads of 512 atoms (head_dim 64, bf16) the queries' kernel takes 50 us
// (510 TFLOP/s), the keys' 85 (400; without the table's gradient 61): LDS, vector
// and matrix instructions hardly overlap at the two waves a SIMD that the registers
// allow (head_dim 128, keys: one).  Four waves of 32 columns a workgroup: with 32
// buckets two workgroups' tiles and sums (67 KB each) are in a CU's LDS.
//
// P and dS go from the accumulators of the first pair of products into the
// operands of the second without leaving the lane (bucket_tiles.h).
//
// The table's gradient needs no atomics (an fp32 one of LDS takes 193 clocks a wave,
// a read and a write 9): every lane adds dS to a sum per bucket of its own in LDS
// ([bucket][thread], one bank a lane), in the order of its pairs; the threads' sums
// are joined at the end in a fixed order and the workgroups' by table_sum_kernel.
// Two calls give identical bits.
//
// Sums are fp32; P and dS are rounded to the operands' type for the second
// products, as any 16-bit matrix product's input is.  fp16 has no room for dS of
// small or large gradients: there it is kept times 2^e, e per (batch entry, key
// head) from |dP - delta| <= 2 max|go| max|v| + max|dlse| over the rows that have
// a partner, so that it stays below 2^14 (the queries' 2^(x - m) is at most 2), and
// P times 2^12; bf16 has fp32's range and needs neither.
#include <algorithm>
#include <cmath>

#include "bucket_tiles.h"

namespace mf {
namespace bucket {

int check_attn(const mf_bucket_attn_args* a, const char* what);
int launch_table_sum(const float* parts, void* dtable, int heads, int buckets, int pieces, int dtype, hipStream_t s);

constexpr int kRowThreads = 256;
constexpr float kProb = 4096.0f;  // fp16: P is kept times this

struct BwdParams {
  const void* q;
  const void* k;
  const void* v;
  const void* table;
  const void* out;
  const void* out_lo;
  const void* go;
  const uint8_t* index;
  const uint8_t* index_t;
  const uint64_t* key_any;
  const uint64_t* query_any;
  const float* stats;  // [2, B H Nq]
  const float* dlse;
  void* dq;
  void* dk;
  void* dv;
  float* rows;    // [B H, TQ, 3, 64] m, 1 / l (fp16: times kProb), -delta
  float4* peak;   // fp16: [B H, TQ] max |go|^2 and |dlse|, then [B KV, TK] max |v|^2
  float* parts;   // [H, K, B CK pieces] sums of dS by bucket, or null
  float* split;   // pieces > 1: [units, pieces, columns, 2 or 1, DP] gradients, then the queries' sums [units, pieces, columns]
  int64_t qs[3], ks[3], vs[3], os[3], gs[3], dqs[3], dks[3], dvs[3];
  int64_t index_step, index_t_step, any_step;
  float scale;
  int B, H, KV, G, Nq, Nk, D, S, St, TQ, TK, K, table_dtype;
  int CT;  // column tiles of a head, of the kernel at hand
  int pieces, per_piece;  // the streamed row tiles in pieces, one a workgroup
  int64_t units;
};

// -- delta, and the peaks ----------------------------------------------------------------------------------------
// A workgroup takes 64 rows of one head: the first B H TQ of them queries, the others (fp16) rows of v.
template <typename T, int DP>
__global__ void __launch_bounds__(kRowThreads) bucket_rows_kernel(BwdParams p) {
  typedef T T8 __attribute__((ext_vector_type(8)));
  constexpr int L = DP / 8, RPW = 64 / L;  // lanes a row, rows a wave and pass
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t queries = int64_t(p.B) * p.H * p.TQ;
  const int64_t id = blockIdx.x;
  const bool is_query = id < queries;
  const int64_t unit = is_query ? id : id - queries;
  const int tiles = is_query ? p.TQ : p.TK, heads = is_query ? p.H : p.KV, N = is_query ? p.Nq : p.Nk;
  const int64_t bh = unit / tiles;
  const int tile = int(unit - bh * tiles);
  const int64_t b = bh / heads;
  const int h = int(bh - b * heads);
  uint64_t used = 0;  // rows with a partner: only they decide the scale
  if (p.peak)
    used = is_query ? union_of(p.query_any + b * p.any_step, p.TQ, tile, 0, p.TK)
                    : union_of(p.key_any + b * p.any_step, p.TK, tile, 0, p.TQ);
  float top = 0.0f, ltop = 0.0f;
  const int d = (lane % L) * 8;
#pragma unroll
  for (int pass = 0; pass < kTile / (4 * RPW); ++pass) {
    const int r = (pass * 4 + wave) * RPW + lane / L;
    const int row = tile * kTile + r;
    const bool in = row < N;
    float dot = 0.0f, norm = 0.0f;
    if (in && d < p.D) {
      if (is_query) {
        const T8 g = *reinterpret_cast<const T8*>(static_cast<const T*>(p.go) + b * p.gs[0] + h * p.gs[1] + row * p.gs[2] + d);
        const T8 o = *reinterpret_cast<const T8*>(static_cast<const T*>(p.out) + b * p.os[0] + h * p.os[1] + row * p.os[2] + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          dot += float(g[e]) * float(o[e]);
          norm += float(g[e]) * float(g[e]);
        }
        if (p.out_lo) {
          const T8 lo = *reinterpret_cast<const T8*>(static_cast<const T*>(p.out_lo) + (bh * p.Nq + row) * p.D + d);
#pragma unroll
          for (int e = 0; e < 8; ++e) dot += float(g[e]) * float(lo[e]);
        }
      } else {
        const T8 v = *reinterpret_cast<const T8*>(static_cast<const T*>(p.v) + b * p.vs[0] + h * p.vs[1] + row * p.vs[2] + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) norm += float(v[e]) * float(v[e]);
      }
    }
#pragma unroll
    for (int off = L / 2; off >= 1; off >>= 1) {
      dot += __shfl_xor(dot, off, 64);
      norm += __shfl_xor(norm, off, 64);
    }
    const bool counts = (used >> r) & 1;
    top = fmaxf(top, counts && norm <= 3.0e38f ? norm : 0.0f);  // (nor do rows that are not finite)
    if (is_query && lane % L == 0) {
      const float dl = in && p.dlse ? p.dlse[bh * p.Nq + row] : 0.0f;
      ltop = fmaxf(ltop, counts && fabsf(dl) <= 3.0e38f ? fabsf(dl) : 0.0f);
      float* dst = p.rows + (bh * p.TQ + tile) * 3 * kTile + r;
      const int64_t at = bh * p.Nq + row;
      const float inv = in ? p.stats[int64_t(p.B) * p.H * p.Nq + at] : 0.0f;
      dst[0] = in ? p.stats[at] : 0.0f;
      dst[kTile] = __is_same(T, _Float16) ? inv * kProb : inv;
      dst[2 * kTile] = in ? dl - dot : 0.0f;
    }
  }
  if (p.peak) {
    __shared__ float2 s[4];
    top = wave_peak(top);
    ltop = wave_peak(ltop);
    if (lane == 0) s[wave] = make_float2(top, ltop);
    __syncthreads();
    if (threadIdx.x == 0) {
      const float a = fmaxf(fmaxf(s[0].x, s[1].x), fmaxf(s[2].x, s[3].x));
      const float c = fmaxf(fmaxf(s[0].y, s[1].y), fmaxf(s[2].y, s[3].y));
      p.peak[id] = make_float4(a, c, 0.0f, 0.0f);
    }
  }
}

// fp16: the exponent of dS for the heads of a key head, which share dk.
__device__ __forceinline__ int scale_bits(const BwdParams& p, int64_t b, int kv) {
  const int lane = threadIdx.x & 63;
  float gm = 0.0f, vm = 0.0f, lm = 0.0f;
  const float4* g = p.peak + (b * p.H + int64_t(kv) * p.G) * p.TQ;
  for (int i = lane; i < p.G * p.TQ; i += 64) {
    gm = fmaxf(gm, g[i].x);
    lm = fmaxf(lm, g[i].y);
  }
  const float4* v = p.peak + int64_t(p.B) * p.H * p.TQ + (b * p.KV + kv) * p.TK;
  for (int i = lane; i < p.TK; i += 64) vm = fmaxf(vm, v[i].x);
  const float bound = 2.0f * sqrtf(wave_peak(gm)) * sqrtf(wave_peak(vm)) + wave_peak(lm);
  return bound > 0.0f && bound < 3.0e38f ? min(60, max(-60, 12 - ilogbf(bound))) : 0;
}

// -- the sums by bucket ------------------------------------------------------------------------------------------
// A lane's 16 values of a block are added to its sums in LDS while the next block is computed: a pair of values a step,
// fetched before two or more matrix instructions and put after them, so that nothing waits for LDS.  Where both values
// of a pair go to one bucket the first takes their sum and the second adds to the masked pairs' row.
template <bool ON>
struct BlockSums {
  __device__ __forceinline__ BlockSums(float*, int, int) {}
  __device__ __forceinline__ void fetch(int, int) {}
  __device__ __forceinline__ void put(int, int) {}
  __device__ __forceinline__ void take(const mf_f32x16&, const uint32_t (&)[4]) {}
};
template <>
struct BlockSums<true> {
  float* bins;
  int pitch, K;
  mf_f32x16 d;
  uint32_t word[4];
  float *b0[2], *b1[2];
  float v0[2], v1[2], s0[2], s1[2];
  __device__ __forceinline__ BlockSums(float* bins_, int pitch_, int K_) : bins(bins_), pitch(pitch_), K(K_), d(zeros16()) {
#pragma unroll
    for (int n = 0; n < 4; ++n) word[n] = 0x40404040u;
  }
  __device__ __forceinline__ void fetch(int from, int to) {  // at most two steps
#pragma unroll
    for (int step = from; step < to; ++step) {
      const int c0 = min(int(byte_of(word, 2 * step)), K), c1 = min(int(byte_of(word, 2 * step + 1)), K);
      const bool same = c0 == c1;
      const int i = step - from;
      b0[i] = bins + c0 * pitch;
      b1[i] = bins + (same ? K : c1) * pitch;
      v0[i] = same ? d[2 * step] + d[2 * step + 1] : d[2 * step];
      v1[i] = d[2 * step + 1];
      if (i == 0) {
        s0[i] = *b0[i];
        s1[i] = *b1[i];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  __device__ __forceinline__ void put(int from, int to) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int step = from; step < to; ++step) {
      const int i = step - from;
      if (i > 0) {  // the first one's may be the same places
        s0[i] = *b0[i];
        s1[i] = *b1[i];
      }
      *b0[i] = s0[i] + v0[i];
      *b1[i] = s1[i] + v1[i];
    }
  }
  __device__ __forceinline__ void take(const mf_f32x16& d_, const uint32_t (&w)[4]) {
    d = d_;
#pragma unroll
    for (int n = 0; n < 4; ++n) word[n] = w[n];
  }
};

template <typename T>
__device__ __forceinline__ void store8(T* to, const float (&x)[8]) {
  typedef __attribute__((__vector_size__(8 * sizeof(T)))) T T8;
  T8 y;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = static_cast<T>(x[e]);
  *reinterpret_cast<T8*>(to) = y;
}

// delta of query `at`, corrected by the sum of its dS: that is dlse but for delta's error.
__device__ __forceinline__ void correct_delta(const BwdParams& p, int64_t b, int h, int at, float total) {
  const int64_t bh = b * p.H + h;
  float* delta = p.rows + (bh * p.TQ + (at >> 6)) * 3 * kTile + 2 * kTile + (at & 63);  // (negative)
  *delta -= total - (p.dlse ? p.dlse[bh * p.Nq + at] : 0.0f);
}

// -- the products ------------------------------------------------------------------------------------------------
template <typename T, int DP, int W, bool KEYS, bool SUMS>
__global__ void __launch_bounds__(64 * W, (DP == 128 && (KEYS || W == 2)) || (W == 1 && DP > 32) ? 1 : 2)
    bucket_bwd_kernel(BwdParams p) {
  using Op = typename Elem<T>::Operand;
  constexpr int NK = DP / 16, ND = DP / 32;
  constexpr int kBytes = kTile * DP * 2;
  constexpr int kRowFloats = 3 * kTile;
  constexpr bool kHalf = __is_same(T, _Float16);
  // Reads of LDS are asked for a group at a time, ahead of the products or of the exp2s, where the registers allow it: left
  // to itself the compiler waits for each beside its use (head_dim 128, keys, four cells of 1997 atoms: 9 % longer).  The
  // queries' kernel of head_dim 128 fits two waves a SIMD without (130 us; with it and one wave a sixth longer).
  constexpr bool kAhead = KEYS || DP < 128;
  __shared__ __attribute__((aligned(1024))) char s_tiles[4 * kBytes];                  // X and Y of two tiles
  __shared__ __attribute__((aligned(1024))) float s_rows[KEYS ? 2 * kRowFloats : 1];  // KEYS: m, 1 / l and -delta of them
  __shared__ float s_table[kPitch];
  extern __shared__ float s_bins[];  // SUMS: [K + 1][64 W], the last one of masked pairs
  static_assert(KEYS || !SUMS, "the table's gradient is the keys' kernel's");
  const uint32_t in_order = xcd_order(blockIdx.x, gridDim.x);
  if (in_order >= p.units * p.pieces) return;
  const uint32_t id = in_order / uint32_t(p.pieces);
  const int piece = int(in_order - id * p.pieces);
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Unit of = unit_of(id, p.B, KEYS ? p.KV : p.H, KEYS ? 1 : p.G, p.CT, KEYS);
  const int uh = of.head, ct = of.tile;
  const int64_t b = of.b;
  const int kv = KEYS ? uh : uh / p.G;
  const int N = KEYS ? p.Nk : p.Nq, rows = KEYS ? p.TQ : p.TK;
  const int col = ct * 32 * W + wave * 32 + (lane & 31);
  const bool in = col < N;
  const int at = in ? col : 0;

  const LaneReads<T, DP> reads(lane);

  // which columns have a partner, and the tables of the row tiles that have
  const uint64_t* by_col = (KEYS ? p.key_any : p.query_any) + b * p.any_step;  // rows of it: row tiles
  const uint64_t* by_row = (KEYS ? p.query_any : p.key_any) + b * p.any_step;  // rows of it: column tiles
  const int c0 = ct * 32 * W / kTile, col_tiles = KEYS ? p.TK : p.TQ;
  const bool two = W == 4 && c0 + 1 < col_tiles;
  // columns: (K, V) or (Q, go), zeros where there is no partner
  Op bx[NK], by[NK];
  const T* gx = KEYS ? static_cast<const T*>(p.k) + b * p.ks[0] + kv * p.ks[1] + at * p.ks[2]
                     : static_cast<const T*>(p.q) + b * p.qs[0] + uh * p.qs[1] + at * p.qs[2];
  const T* gy = KEYS ? static_cast<const T*>(p.v) + b * p.vs[0] + kv * p.vs[1] + at * p.vs[2]
                     : static_cast<const T*>(p.go) + b * p.gs[0] + uh * p.gs[1] + at * p.gs[2];
#pragma unroll
  for (int kk = 0; kk < NK; ++kk) {
    const int d = 16 * kk + 8 * half;
    bx[kk] = *reinterpret_cast<const Op*>(gx + (d < p.D ? d : 0));
    by[kk] = *reinterpret_cast<const Op*>(gy + (d < p.D ? d : 0));
  }
  uint64_t used = union_of(by_col, col_tiles, c0, 0, rows);
  if (two) {
    const uint64_t second = union_of(by_col, col_tiles, c0 + 1, 0, rows);
    if (wave >= 2) used = second;
  }
  const bool mine = in && ((used >> (at & 63)) & 1);
#pragma unroll
  for (int kk = 0; kk < NK; ++kk) {
    if (!mine || 16 * kk + 8 * half >= p.D) {
#pragma unroll
      for (int e = 0; e < 8; ++e) bx[kk][e] = by[kk][e] = T(0.0f);
    }
  }
  float cm = 0.0f, cinv = 0.0f, cdelta = 0.0f;  // the column's row statistics
  if (!KEYS && mine) {
    const float* r = p.rows + ((b * p.H + uh) * p.TQ + (at >> 6)) * 3 * kTile + (at & 63);
    cm = r[0];
    cinv = r[kTile];
    cdelta = r[2 * kTile];
  }
  float up = 1.0f, down = p.scale;
  if constexpr (kHalf) {
    const int e = scale_bits(p, b, kv);
    up = ldexpf(1.0f, e);
    down = p.scale * ldexpf(1.0f, -e);
    if (KEYS) up *= 1.0f / kProb;  // P comes times kProb
  }
  const float slog = p.scale * kLog2e;
  // the columns' buckets: rows of the workgroup's first column on, the lane's row below 2^31 bytes further
  const int first = ct * 32 * W;
  const uint8_t* codes = KEYS ? p.index_t + b * p.index_t_step + int64_t(first) * p.St
                              : p.index + b * p.index_step + int64_t(first) * p.S;
  const uint32_t code_row = uint32_t(min(col, N - 1) - first) * uint32_t(KEYS ? p.St : p.S) + 16 * half;

  mf_f32x16 ax[ND], ay[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n) ax[n] = ay[n] = zeros16();
  float total = 0.0f;  // queries: of dS

  const char *tx = nullptr, *ty = nullptr, *tr = nullptr;
  const unsigned xstride = unsigned(KEYS ? p.qs[2] : p.ks[2]) * 2, ystride = unsigned(KEYS ? p.gs[2] : p.vs[2]) * 2;
  auto side = [&](int h) {  // the streamed side of query head h
    if (KEYS) {
      tx = reinterpret_cast<const char*>(static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[1]);
      ty = reinterpret_cast<const char*>(static_cast<const T*>(p.go) + b * p.gs[0] + h * p.gs[1]);
      tr = reinterpret_cast<const char*>(p.rows + (b * p.H + h) * p.TQ * 3 * kTile);
    } else {
      tx = reinterpret_cast<const char*>(static_cast<const T*>(p.k) + b * p.ks[0] + kv * p.ks[1]);
      ty = reinterpret_cast<const char*>(static_cast<const T*>(p.v) + b * p.vs[0] + kv * p.vs[1]);
    }
  };
  // The copies' offsets are formed for every tile where registers are short: spilled, they came back in between the copies,
  // each of which then waited for the one before.
  constexpr bool kShort = KEYS && SUMS && DP == 64;
  auto copies = [&] {
    int l = lane;
    if constexpr (kShort) asm volatile("" : "+v"(l));  // (not the ones of the last tile)
    struct Both {
      TileCopy<DP, W> x, y;
    };
    return Both{TileCopy<DP, W>(xstride, p.D, wave, l), TileCopy<DP, W>(ystride, p.D, wave, l)};
  };
  const auto kept = copies();
  auto load = [&](int tile, uint64_t set, int buffer, uint4 (&w)[2]) {
    const auto now = kShort ? copies() : kept;
    const TileCopy<DP, W>&xcopy = now.x, &ycopy = now.y;
    xcopy.copy(tx + int64_t(tile) * kTile * xstride, set, s_tiles + buffer, wave, lane);
    ycopy.copy(ty + int64_t(tile) * kTile * ystride, set, s_tiles + buffer + kBytes, wave, lane);
    if (KEYS && wave == 0) {
      const mf_i32x4 src = lds_copy_source(tr + int64_t(tile) * (kRowFloats * 4));
      const bool on = (set >> lane) & 1;  // zeros for rows without a partner here too
      float* lr = s_rows + (buffer ? kRowFloats : 0);
#pragma unroll
      for (int n = 0; n < 3; ++n) lds_copy4(src, on ? lane * 4u + n * kTile * 4u : kLdsCopyOutside, lr + n * kTile);
    }
    w[0] = *reinterpret_cast<const uint4*>(codes + int64_t(tile) * kTile + code_row);
    w[1] = *reinterpret_cast<const uint4*>(codes + int64_t(tile) * kTile + code_row + 32);
  };

  for (int g = 0; g < (KEYS ? p.G : 1); ++g) {
    const int t0 = max(0, piece * p.per_piece - g * rows), t1 = min(rows, (piece + 1) * p.per_piece - g * rows);
    const int64_t slots = int64_t(p.B) * p.CT * p.pieces;
    float* slot = SUMS ? p.parts + int64_t(kv * p.G + g) * p.K * slots + (b * p.CT + ct) * p.pieces + piece : nullptr;
    side(KEYS ? kv * p.G + g : uh);
    Tiles tiles(by_row + int64_t(c0) * rows, two ? by_row + int64_t(c0 + 1) * rows : nullptr, t0, t1);
    int tile = 0, buffer = 0;
    uint64_t set = 0;
    uint4 next[2];
    BlockSums<SUMS> sums(s_bins + threadIdx.x, 64 * W, p.K);
    bool more = tiles.next(tile, set);
    if (!more) {  // no pair
      if (SUMS && int(threadIdx.x) < p.K) slot[threadIdx.x * slots] = 0.0f;
      continue;
    }
    load(tile, set, 0, next);
    load_tables(s_table, p.table, p.table_dtype, p.K, p.H, KEYS ? kv * p.G + g : uh, 1, 64 * W);
    if constexpr (SUMS)
      for (int c = 0; c <= p.K; ++c) s_bins[c * 64 * W + threadIdx.x] = 0.0f;
    __syncthreads();  // the table and the sums
    while (more) {
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's copies into LDS have landed
      __syncthreads();
      const uint4 w[2] = {next[0], next[1]};
      const uint64_t now = set;
      const LaneReads<T, DP> at = reads.shifted(buffer);
      const float* lr = s_rows + (buffer ? kRowFloats : 0) + 16 * half;
      buffer ^= 2 * kBytes;
      more = tiles.next(tile, set);
      if (more) load(tile, set, buffer, next);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        if (uint32_t(now >> (32 * kb)) == 0) continue;  // no pair in these 32 rows
        uint32_t word[4] = {w[kb].x, w[kb].y, w[kb].z, w[kb].w};
        if (KEYS && !in) word[0] = word[1] = word[2] = word[3] = 0x40404040u;  // kMasked (not in load, which would wait for them)
        Op xa[NK], ya[NK], xt[2][ND], yt[2][ND];
        float bias[16];
        mf_f32x16 s = zeros16(), d;  // d: dP - delta, -delta as the sum's start
#pragma unroll
        for (int kk = 0; kk < (kAhead ? NK : 0); ++kk) {
          xa[kk] = at.rows(s_tiles, kb, kk);
          ya[kk] = at.rows(s_tiles + kBytes, kb, kk);
        }
#pragma unroll
        for (int t = 0; t < 16; ++t) d[t] = KEYS ? lr[2 * kTile + 32 * kb + t] : cdelta;
#pragma unroll
        for (int t = 0; t < (kAhead ? 16 : 0); ++t) bias[t] = s_table[byte_of(word, t)];
        if constexpr (kAhead) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
          sums.fetch(4 * kk / NK, 4 * (kk + 1) / NK);
          s = Mma32<T>::mma(kAhead ? xa[kk] : at.rows(s_tiles, kb, kk), bx[kk], s);
          d = Mma32<T>::mma(kAhead ? ya[kk] : at.rows(s_tiles + kBytes, kb, kk), by[kk], d);
          sums.put(4 * kk / NK, 4 * (kk + 1) / NK);
        }
        float m[16], inv[16];
        if (KEYS) {
#pragma unroll
          for (int t = 0; t < 16; ++t) {
            m[t] = lr[32 * kb + t];
            inv[t] = lr[kTile + 32 * kb + t];
          }
        }
#pragma unroll
        for (int n = 0; n < (kAhead ? ND : 0); ++n) {
          xt[0][n] = at.columns(s_tiles, kb, 0, n);
          if (KEYS) yt[0][n] = at.columns(s_tiles + kBytes, kb, 0, n);
        }
        if constexpr (kAhead) __builtin_amdgcn_sched_barrier(0);
        Op pb[2], sb[2];
#pragma unroll
        for (int t = 0; t < 16; ++t) {
          float e = fast_exp2(fmaf(s[t], slog, kAhead ? bias[t] : s_table[byte_of(word, t)]) - (KEYS ? m[t] : cm));
          if (KEYS) {
            e *= inv[t];
            pb[t >> 3][t & 7] = static_cast<T>(e);
          }
          d[t] *= e;
          sb[t >> 3][t & 7] = static_cast<T>(kHalf ? d[t] * up : d[t]);
          if (!KEYS) total += d[t];
        }
        if constexpr (kAhead) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < (kAhead ? ND : 0); ++n) {
          xt[1][n] = at.columns(s_tiles, kb, 1, n);
          if (KEYS) yt[1][n] = at.columns(s_tiles + kBytes, kb, 1, n);
        }
        if constexpr (kAhead) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int n = 0; n < ND; ++n) {
            // two steps a half: one each before and after the middle, or both at once
            const int step = 4 + 2 * u + (2 * n >= ND && n > 0);
            if (n == 0 || 2 * n == ND) sums.fetch(step, ND > 1 ? step + 1 : step + 2);
            ax[n] = Mma32<T>::mma(kAhead ? xt[u][n] : at.columns(s_tiles, kb, u, n), sb[u], ax[n]);
            if (KEYS) ay[n] = Mma32<T>::mma(kAhead ? yt[u][n] : at.columns(s_tiles + kBytes, kb, u, n), pb[u], ay[n]);
            if (2 * (n + 1) == ND || n + 1 == ND) sums.put(step, ND > 1 ? step + 1 : step + 2);
          }
        }
        sums.take(d, word);
      }
    }
    if constexpr (SUMS) {
#pragma unroll
      for (int step = 0; step < 8; ++step) {
        sums.fetch(step, step + 1);
        sums.put(step, step + 1);
      }
    }
    __syncthreads();
    if constexpr (SUMS) {
      for (int c = wave; c < p.K; c += W) {
        float v = 0.0f;
#pragma unroll
        for (int u = 0; u < W; ++u) v += s_bins[c * 64 * W + u * 64 + lane];
        v = wave_total(v) * (kHalf ? 1.0f / kProb : 1.0f);
        if (lane == 0) slot[c * slots] = v;
      }
      __syncthreads();  // the next head clears them
    }
  }

  const float fx = KEYS ? down : down * (kHalf ? cinv * (1.0f / kProb) : cinv), fy = kHalf ? 1.0f / kProb : 1.0f;
  if (!KEYS) total = pair_sum(total) * (kHalf ? cinv * (1.0f / kProb) : cinv);
  if (!in) return;
  const int64_t place = int64_t(in_order) * (32 * W) + wave * 32 + (lane & 31);  // pieces > 1
  T* ox = KEYS ? static_cast<T*>(p.dk) + b * p.dks[0] + kv * p.dks[1] + at * p.dks[2]
               : static_cast<T*>(p.dq) + b * p.dqs[0] + uh * p.dqs[1] + at * p.dqs[2];
  T* oy = static_cast<T*>(p.dv) + b * p.dvs[0] + kv * p.dvs[1] + at * p.dvs[2];
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int d0 = 32 * n + 16 * half + 8 * u;
      float x[8], y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // a column without a partner: zeros, whatever the tile's other rows hold
        x[e] = mine ? ax[n][8 * u + e] * fx : 0.0f;
        y[e] = mine ? ay[n][8 * u + e] * fy : 0.0f;
      }
      if (p.pieces > 1) {
        float* to = p.split + place * (KEYS ? 2 * DP : DP) + d0;
        store8(to, x);
        if (KEYS) store8(to + DP, y);
      } else if (d0 < p.D) {
        store8(ox + d0, x);
        if (KEYS) store8(oy + d0, y);
      }
    }
  if (!KEYS && half == 0) {
    if (p.pieces > 1) p.split[p.units * p.pieces * (32 * W) * DP + place] = total;
    else if (mine) correct_delta(p, b, uh, at, total);
  }
}

// Joins the pieces in their order: eight entries of a column a thread.
template <typename T, int DP, bool KEYS>
__global__ void __launch_bounds__(256) bucket_bwd_join_kernel(BwdParams p, int columns) {
  constexpr int L = (KEYS ? 2 : 1) * DP / 8;
  const int64_t id = int64_t(blockIdx.x) * 256 + threadIdx.x;
  const int part = int(id % L), c = int(id / L % columns);
  const int64_t unit = id / L / columns;
  if (unit >= p.units) return;
  const Unit of = unit_of(unit, p.B, KEYS ? p.KV : p.H, KEYS ? 1 : p.G, p.CT, KEYS);
  const int uh = of.head, ct = of.tile;
  const int64_t b = of.b;
  const int at = ct * columns + c, d0 = part * 8 % DP;
  if (at >= (KEYS ? p.Nk : p.Nq) || d0 >= p.D) return;
  const int64_t first = unit * p.pieces * columns + c;
  float x[8] = {};
  for (int n = 0; n < p.pieces; ++n) {
    const float4* in = reinterpret_cast<const float4*>(p.split + ((first + int64_t(n) * columns) * L + part) * 8);
    const float4 lo = in[0], hi = in[1];
    x[0] += lo.x;
    x[1] += lo.y;
    x[2] += lo.z;
    x[3] += lo.w;
    x[4] += hi.x;
    x[5] += hi.y;
    x[6] += hi.z;
    x[7] += hi.w;
  }
  if (!KEYS) {
    store8(static_cast<T*>(p.dq) + b * p.dqs[0] + uh * p.dqs[1] + at * p.dqs[2] + d0, x);
    if (part == 0) {
      float total = 0.0f;
      for (int n = 0; n < p.pieces; ++n)
        total += p.split[p.units * p.pieces * columns * DP + first + int64_t(n) * columns];
      correct_delta(p, b, uh, at, total);
    }
  } else if (part * 8 < DP) {
    store8(static_cast<T*>(p.dk) + b * p.dks[0] + uh * p.dks[1] + at * p.dks[2] + d0, x);
  } else {
    store8(static_cast<T*>(p.dv) + b * p.dvs[0] + uh * p.dvs[1] + at * p.dvs[2] + d0, x);
  }
}

namespace {

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

struct Side {  // the queries' or the keys' kernel
  int W, CT, pieces, per_piece;
  int64_t units;
  size_t split_bytes;
};
struct BwdPlan {
  int DP, TQ, TK;
  Side queries, keys;
  size_t rows, peak, parts, split;
  size_t total() const { return rows + peak + parts + split; }
};

// Few workgroups over many row tiles: the tiles in pieces, until the waves that fit (one a SIMD with head_dim 128's keys,
// two otherwise) are there, so many that none is left over.
Side side_of(int64_t batch_heads, int columns, int64_t tiles, int DP, bool keys) {
  Side z = {};
  z.W = columns <= 32 ? 1 : columns <= 64 ? 2 : 4;
  z.CT = (columns + 32 * z.W - 1) / (32 * z.W);
  z.units = batch_heads * z.CT;
  const int64_t room = 1024 * (keys && DP == 128 ? 1 : 2);
  const int64_t pieces = std::max<int64_t>(1, std::min<int64_t>(tiles, room / std::max<int64_t>(1, z.units * z.W)));
  z.per_piece = int((tiles + pieces - 1) / pieces);
  z.pieces = int((tiles + z.per_piece - 1) / z.per_piece);
  if (z.pieces > 1)
    z.split_bytes = size_t(z.units) * z.pieces * 32 * z.W * (keys ? 2 * DP : DP + 1) * sizeof(float);
  return z;
}

BwdPlan bwd_plan(const mf_bucket_attn_bwd_args* a) {
  const mf_bucket_attn_args* f = &a->fwd;
  BwdPlan z = {};
  z.DP = f->head_dim <= 32 ? 32 : f->head_dim <= 64 ? 64 : 128;
  z.TQ = (f->queries + kTile - 1) / kTile;
  z.TK = (f->keys + kTile - 1) / kTile;
  const int64_t B = f->batch;
  z.queries = side_of(B * f->heads, f->queries, z.TK, z.DP, false);
  z.keys = side_of(B * f->kv_heads, f->keys, int64_t(f->heads / f->kv_heads) * z.TQ, z.DP, true);
  const size_t qt = size_t(B) * f->heads * z.TQ, kt = size_t(B) * f->kv_heads * z.TK;
  z.rows = round256(qt * 3 * kTile * sizeof(float));
  z.peak = f->dtype == MF_DTYPE_F16 ? round256((qt + kt) * sizeof(float4)) : 0;
  z.parts = a->dtable ? round256(size_t(f->heads) * f->buckets * B * z.keys.CT * z.keys.pieces * sizeof(float)) : 0;
  z.split = round256(std::max(z.queries.split_bytes, z.keys.split_bytes));  // one kernel's at a time
  return z;
}

template <typename T, int DP, int W, bool KEYS, bool SUMS>
int launch_bwd(const BwdParams& p, hipStream_t s) {
  const int lds = SUMS ? (p.K + 1) * 64 * W * 4 : 0;
  constexpr int kMost = SUMS ? (MF_MAX_BUCKETS + 1) * 64 * W * 4 : 0;
  static_assert(kMost + 4 * kTile * DP * 2 + 4096 <= 160 * 1024, "LDS of a workgroup");
  if (const int status = ensure_dynamic_lds(reinterpret_cast<const void*>(bucket_bwd_kernel<T, DP, W, KEYS, SUMS>), kMost))
    return status;
  hipLaunchKernelGGL((bucket_bwd_kernel<T, DP, W, KEYS, SUMS>), dim3(unsigned((p.units * p.pieces + 7) / 8 * 8)), dim3(64 * W),
                     lds, s, p);
  MF_HIP_CHECK(hipGetLastError());
  if (p.pieces > 1) {
    const int64_t threads = p.units * 32 * W * (KEYS ? 2 : 1) * (DP / 8);
    hipLaunchKernelGGL((bucket_bwd_join_kernel<T, DP, KEYS>), dim3(unsigned((threads + 255) / 256)), dim3(256), 0, s, p,
                       32 * W);
    MF_HIP_CHECK(hipGetLastError());
  }
  return MF_OK;
}

template <typename T, int DP, bool KEYS, bool SUMS>
int launch_bwd(const BwdParams& p, int W, hipStream_t s) {
  if (W == 1) return launch_bwd<T, DP, 1, KEYS, SUMS>(p, s);
  if (W == 2) return launch_bwd<T, DP, 2, KEYS, SUMS>(p, s);
  return launch_bwd<T, DP, 4, KEYS, SUMS>(p, s);
}

template <typename T, int DP>
int launch_all(BwdParams p, const BwdPlan& z, hipStream_t s) {
  const int64_t blocks = int64_t(p.B) * p.H * z.TQ + (p.peak ? int64_t(p.B) * p.KV * z.TK : 0);
  hipLaunchKernelGGL((bucket_rows_kernel<T, DP>), dim3(unsigned(blocks)), dim3(kRowThreads), 0, s, p);
  MF_HIP_CHECK(hipGetLastError());
  auto take = [&p](const Side& z) {
    p.CT = z.CT;
    p.pieces = z.pieces;
    p.per_piece = z.per_piece;
    p.units = z.units;
  };
  take(z.queries);
  if (const int status = launch_bwd<T, DP, false, false>(p, z.queries.W, s)) return status;
  take(z.keys);
  return p.parts ? launch_bwd<T, DP, true, true>(p, z.keys.W, s) : launch_bwd<T, DP, true, false>(p, z.keys.W, s);
}

template <typename T>
int launch_all(const BwdParams& p, const BwdPlan& z, hipStream_t s) {
  if (z.DP == 32) return launch_all<T, 32>(p, z, s);
  if (z.DP == 64) return launch_all<T, 64>(p, z, s);
  return launch_all<T, 128>(p, z, s);
}

}  // namespace
}  // namespace bucket
}  // namespace mf

extern "C" uint64_t mf_bucket_attn_bwd_workspace_size(const mf_bucket_attn_bwd_args* a) {
  if (a == nullptr) return 0;
  const mf_bucket_attn_args* f = &a->fwd;
  if (f->batch <= 0 || f->heads <= 0 || f->kv_heads <= 0 || f->queries <= 0 || f->keys <= 0 || f->buckets <= 0) return 0;
  return mf::bucket::bwd_plan(a).total();
}

extern "C" int mf_bucket_attn_bwd(const mf_bucket_attn_bwd_args* a, void* stream) {
  using namespace mf;
  using namespace mf::bucket;
  if (a == nullptr) return fail(MF_ERR_INVALID_ARGUMENT, "mf_bucket_attn_bwd: args is NULL");
  const mf_bucket_attn_args* f = &a->fwd;
  if (const int status = check_attn(f, "mf_bucket_attn_bwd")) return status;
  if (!f->stats || !a->index_t || !a->grad_out || !a->dq || !a->dk || !a->dv)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_bucket_attn_bwd: stats, index_t, grad_out, dq, dk and dv must be non-NULL");
  for (const void* ptr : {static_cast<const void*>(a->index_t), a->grad_out, static_cast<const void*>(a->dq),
                          static_cast<const void*>(a->dk), static_cast<const void*>(a->dv)})
    if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0)
      return fail(MF_ERR_INVALID_ARGUMENT, "mf_bucket_attn_bwd: operands and gradients must be 16-byte aligned");
  for (const int64_t* s : {a->grad_out_stride, a->dq_stride, a->dk_stride, a->dv_stride})
    for (int n = 0; n < 3; ++n)
      if (s[n] % 8 != 0 || s[n] < 0)
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_bucket_attn_bwd: strides must be non-negative multiples of 8");
  if (a->grad_out_stride[2] >= (1 << 23))
    return fail(MF_ERR_UNSUPPORTED, "mf_bucket_attn_bwd: token strides must be below 2^23 elements");
  if (f->batch == 0 || f->heads == 0) return MF_OK;
  if (f->queries == 0 || f->keys == 0)
    return fail(MF_ERR_UNSUPPORTED, "mf_bucket_attn_bwd: queries and keys must be positive");
  const BwdPlan z = bwd_plan(a);
  const int64_t B = f->batch;
  // (where there are pieces, there are few units)
  const int64_t most = std::max({B * f->heads * z.TQ + B * f->kv_heads * z.TK, z.keys.units * z.keys.pieces + 8,
                                 z.queries.units * z.queries.pieces + 8});
  if (most * 256 > 0xffffffffLL)  // threads of a launch
    return fail(MF_ERR_UNSUPPORTED, "mf_bucket_attn_bwd: batch * heads * tiles too large");
  if (!a->workspace || a->workspace_bytes < z.total() || reinterpret_cast<uintptr_t>(a->workspace) % 16 != 0)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_bucket_attn_bwd: the workspace must be 16-byte aligned and hold "
                                         "mf_bucket_attn_bwd_workspace_size bytes");
  BwdParams p = {};
  p.q = f->q;
  p.k = f->k;
  p.v = f->v;
  p.table = f->table;
  p.out = f->out;
  p.out_lo = f->out_lo;
  p.go = a->grad_out;
  p.index = f->index;
  p.index_t = a->index_t;
  p.key_any = f->key_any;
  p.query_any = f->query_any;
  p.stats = f->stats;
  p.dlse = a->grad_lse;
  p.dq = a->dq;
  p.dk = a->dk;
  p.dv = a->dv;
  char* ws = static_cast<char*>(a->workspace);
  p.rows = reinterpret_cast<float*>(ws);
  p.peak = z.peak ? reinterpret_cast<float4*>(ws + z.rows) : nullptr;
  p.parts = a->dtable ? reinterpret_cast<float*>(ws + z.rows + z.peak) : nullptr;
  p.split = reinterpret_cast<float*>(ws + z.rows + z.peak + z.parts);
  for (int n = 0; n < 3; ++n) {
    p.qs[n] = f->q_stride[n];
    p.ks[n] = f->k_stride[n];
    p.vs[n] = f->v_stride[n];
    p.os[n] = f->out_stride[n];
    p.gs[n] = a->grad_out_stride[n];
    p.dqs[n] = a->dq_stride[n];
    p.dks[n] = a->dk_stride[n];
    p.dvs[n] = a->dv_stride[n];
  }
  p.scale = f->scale;
  p.B = f->batch;
  p.H = f->heads;
  p.KV = f->kv_heads;
  p.G = f->heads / f->kv_heads;
  p.Nq = f->queries;
  p.Nk = f->keys;
  p.D = f->head_dim;
  p.S = (f->keys + 63) / 64 * 64;
  p.St = (f->queries + 63) / 64 * 64;
  p.TQ = z.TQ;
  p.TK = z.TK;
  p.K = f->buckets;
  p.table_dtype = f->table_dtype;
  p.index_step = f->index_batch == 1 ? 0 : int64_t(p.Nq) * p.S;
  p.index_t_step = f->index_batch == 1 ? 0 : int64_t(p.Nk) * p.St;
  p.any_step = f->index_batch == 1 ? 0 : int64_t(p.TQ) * p.TK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int status = f->dtype == MF_DTYPE_BF16 ? launch_all<__bf16>(p, z, s) : launch_all<_Float16>(p, z, s);
  if (status != MF_OK || !a->dtable) return status;
  return launch_table_sum(p.parts, a->dtable, p.H, p.K, p.B * z.keys.CT * z.keys.pieces, p.table_dtype, s);
}
