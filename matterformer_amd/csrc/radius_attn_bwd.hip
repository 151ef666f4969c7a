// Gradients of local (radius) attention over a neighbour bit mask
// (mf_radius_attn_bwd) on gfx950.  With P = exp(scale q_i . k_j - lse_i) on the
// allowed pairs,
//   dv_j = sum_i P_ij go_i,             dP_ij = go_i . v_j,
//   dS_ij = P_ij (dP_ij - delta_i),     delta_i = go_i . out_i - dlse_i,
//   dq_i = scale sum_j dS_ij k_j,       dk_j = scale sum_i dS_ij q_i
// (10 D flops a pair).  No atomics: every gradient row has one owner, which
// sums in a fixed order, so two calls give identical bits.
//
// Three kernels.
//  - radius_tables_kernel (mf_radius_tables, once per mask): the mask transposed
//    (words per key instead of per query), and for every 64 x 64 tile which of
//    its queries have a key in it and which of its keys a query, 64 bits each:
//    also the list of tiles with an entry at all.  The forward takes the keys'.
//  - radius_rows_kernel: per row lse in log2 units and -delta.
//  - radius_bwd_kernel: a workgroup owns 64 queries (dq) or keys (dk, dv) as the
//    columns of its products, a wave 16 of them, and streams 64-row tiles of the
//    other side, X and Y = (K, V) or (Q, go), from global memory straight
//    to LDS, the next tile while the current one is multiplied.  Per 32 rows:
//      S = X cX^T, dP = Y cY^T   (rows from LDS, columns cX, cY = (Q, go) or
//                                 (K, V) in registers)
//      dX^T += X^T dS, and for keys dY^T += Y^T P
//    P and dS go from the accumulators of the first pair of products into the
//    operands of the second without leaving the lane; X^T and Y^T are read from
//    the same rows by transposing LDS reads, in the row order the operands have.
//
// delta enters every pair of a row alike, so a rounded `out` would show in dq and
// dk most of all their inputs; with out_lo, what that rounding left, it does not
// (17 neighbours, head_dim 32: error 2.6e-3 -> 2.4e-3 of the norm, where rounding
// dS and the result alone leave 2.35e-3).
//
// Sums are fp32.  P and dS are rounded to the operands' type for the second
// products, as any 16-bit matrix product's input is: bf16 gradients are off by
// 2.4e-3 of the norm, where rounding them alone leaves 1.7e-3.  (Tried: the low
// parts of P and dS as further products, 1.75e-3, for 113 us instead of 92 on 32
// cells of 512 atoms, 167 instead of 144 on four of 1997 at head_dim 128.)  fp16 has no room for dS of
// small or large gradients, so there dS is kept times 2^e, e per (molecule,
// head) from |dP - delta| <= 2 max|go| max|v| + max|dlse| (Cauchy-Schwarz, over the
// rows that have a partner) so that it stays below 2^14, and P times 2^12 (a key of
// weight 3e-9 still counts), which the stored lse carries; bf16 has fp32's range and
// needs neither.
//
// Rows that no column of the tile is paired with (padding, atoms without a
// neighbour) are staged as zeros, so that whatever they hold, NaN too, reaches
// no column; a column without a pair is stored as zeros.
#include <algorithm>
#include <cmath>

#include "mf_common.h"

namespace mf {
namespace rattn_bwd {

constexpr int kTile = 64;
constexpr int kThreads = 256;
constexpr float kProbBits = 12.0f;  // fp16: P is kept times 2^12; it is at most 1 but for the roundings of lse

struct Params {
  const void* q;
  const void* k;
  const void* v;
  const void* out;
  const void* out_lo;
  const void* go;
  const uint32_t* bits;
  const float* lse;
  const float* dlse;
  void* dq;
  void* dk;
  void* dv;
  const uint32_t* bits_t;   // [B, N, W] the transposed mask
  const uint64_t* key_any;  // [B, NB query tiles, NB key tiles] keys of the tile with a query
  const uint64_t* qry_any;  // [B, NB key tiles, NB query tiles] queries of the tile with a key
  float* rows;        // [B H, NB, 2, 64]: lse log2(e) (fp16: less kProbBits), then -delta, of every query tile
  float4* peak;       // fp16: [B H, NB] max |go|^2, |v|^2 and |dlse| of a tile
  float scale;
  int B, H, N, W, NB;
  int units;          // workgroups of one role
};

// -- the mask's tables: one wave per 64 x 64 tile, lane i its query row -------------------------------------------
struct TableParams {
  const uint32_t* bits;
  const uint8_t* block_mask;
  uint32_t* bits_t;
  uint64_t* key_any;
  uint64_t* qry_any;
  int B, N, W, NB;
};

__global__ void __launch_bounds__(kThreads) radius_tables_kernel(TableParams p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t id = int64_t(blockIdx.x) * 4 + wave;
  if (id >= int64_t(p.B) * p.NB * p.NB) return;
  const int jt = int(id % p.NB), it = int(id / p.NB % p.NB);
  const int64_t b = id / (int64_t(p.NB) * p.NB);
  const int row = it * kTile + lane;
  uint32_t lo = 0, hi = 0;
  const bool on = !p.block_mask || p.block_mask[id] != 0;
  if (on && row < p.N) {
    const uint32_t* w = p.bits + (b * p.N + row) * p.W + 2 * jt;
    lo = w[0];
    if (2 * jt + 1 < p.W) hi = w[1];
  }
  // bits of columns past N are zero by the mask's format; cleared here all the same
  const int cols = p.N - jt * kTile;
  if (cols < 64) {
    const uint64_t keep = (uint64_t(1) << cols) - 1;
    lo &= uint32_t(keep);
    hi &= uint32_t(keep >> 32);
  }
  const uint64_t qany = __ballot((lo | hi) != 0);
  uint64_t mine = 0;
  if (qany != 0) {
#pragma unroll
    for (int c = 0; c < 64; ++c) {
      const uint64_t column = __ballot(((c < 32 ? lo >> c : hi >> (c - 32)) & 1u) != 0);
      if (lane == c) mine = column;
    }
  }
  const uint64_t kany = __ballot(mine != 0);
  const int key = jt * kTile + lane;
  if (key < p.N) {
    uint32_t* w = p.bits_t + (b * p.N + key) * p.W + 2 * it;
    w[0] = uint32_t(mine);
    if (2 * it + 1 < p.W) w[1] = uint32_t(mine >> 32);
  }
  if (lane == 0) {
    p.key_any[id] = kany;
    p.qry_any[(b * p.NB + jt) * p.NB + it] = qany;
  }
}

// -- lse, delta and the peaks ------------------------------------------------------------------------------------
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) radius_rows_kernel(Params p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int unit = blockIdx.x;
  // 64 rows of one (molecule, head): D / 8 lanes a row
  constexpr int L = D / 8;
  constexpr int RPW = 64 / L;  // rows per wave and pass
  const int64_t bh = unit / p.NB;
  const int tile = unit % p.NB;
  typedef T T8 __attribute__((ext_vector_type(8)));
  float gmax = 0.0f, vmax = 0.0f, lmax = 0.0f;
  float* dst = p.rows + (bh * p.NB + tile) * 2 * kTile;
  // rows of the tile that a pair reads, as queries (go, dlse) and as keys (v): only they decide the scale
  unsigned long long queries = 0, keys = 0;
  if (p.peak) {
    const int64_t first = bh / p.H * p.NB * p.NB + tile;
    for (int t = lane; t < p.NB; t += 64) {
      queries |= p.qry_any[first + int64_t(t) * p.NB];
      keys |= p.key_any[first + int64_t(t) * p.NB];
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
      queries |= __shfl_xor(queries, off, 64);
      keys |= __shfl_xor(keys, off, 64);
    }
  }
#pragma unroll
  for (int pass = 0; pass < kTile / (4 * RPW); ++pass) {
    const int r = (pass * 4 + wave) * RPW + lane / L;
    const int row = tile * kTile + r;
    float dot = 0.0f, gg = 0.0f, vv = 0.0f;
    if (row < p.N) {
      const int64_t at = (bh * p.N + row) * D + (lane % L) * 8;
      const T8 g = *reinterpret_cast<const T8*>(static_cast<const T*>(p.go) + at);
      const T8 o = *reinterpret_cast<const T8*>(static_cast<const T*>(p.out) + at);
#pragma unroll
      for (int e = 0; e < 8; ++e) dot += Elem<T>::to_f32(g[e]) * Elem<T>::to_f32(o[e]);
      if (p.out_lo) {
        const T8 lo = *reinterpret_cast<const T8*>(static_cast<const T*>(p.out_lo) + at);
#pragma unroll
        for (int e = 0; e < 8; ++e) dot += Elem<T>::to_f32(g[e]) * Elem<T>::to_f32(lo[e]);
      }
      if constexpr (sizeof(T) == 2 && !__is_same(T, __bf16)) {
        const T8 v = *reinterpret_cast<const T8*>(static_cast<const T*>(p.v) + at);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          gg += Elem<T>::to_f32(g[e]) * Elem<T>::to_f32(g[e]);
          vv += Elem<T>::to_f32(v[e]) * Elem<T>::to_f32(v[e]);
        }
      }
    }
#pragma unroll
    for (int off = L / 2; off >= 1; off >>= 1) {
      dot += __shfl_xor(dot, off, 64);
      gg += __shfl_xor(gg, off, 64);
      vv += __shfl_xor(vv, off, 64);
    }
    // nor do rows that are not finite
    const bool query = (queries >> r) & 1, key = (keys >> r) & 1;
    gmax = fmaxf(gmax, query && gg <= 3.0e38f ? gg : 0.0f);
    vmax = fmaxf(vmax, key && vv <= 3.0e38f ? vv : 0.0f);
    if (lane % L == 0) {
      const bool in = row < p.N;
      const float dl = in && p.dlse ? p.dlse[bh * p.N + row] : 0.0f;
      lmax = fmaxf(lmax, query && fabsf(dl) <= 3.0e38f ? fabsf(dl) : 0.0f);
      constexpr float kLess = __is_same(T, _Float16) ? kProbBits : 0.0f;
      dst[r] = in ? fmaf(p.lse[bh * p.N + row], kLog2e, -kLess) : 0.0f;
      dst[kTile + r] = in ? dl - dot : 0.0f;
    }
  }
  if (p.peak) {
    __shared__ float4 s[4];
    gmax = wave_max(gmax);
    vmax = wave_max(vmax);
    lmax = wave_max(lmax);
    if (lane == 0) s[wave] = make_float4(gmax, vmax, lmax, 0.0f);
    __syncthreads();
    if (threadIdx.x == 0) {
      float4 m = s[0];
      for (int w = 1; w < 4; ++w) m = make_float4(fmaxf(m.x, s[w].x), fmaxf(m.y, s[w].y), fmaxf(m.z, s[w].z), 0.0f);
      p.peak[bh * p.NB + tile] = m;
    }
  }
}

// -- the products ------------------------------------------------------------------------------------------------
// Chunk swizzle of a staged row (16-byte chunks): eight consecutive rows read at one chunk, and eight rows read at one
// pair of chunks by the transposing reads, fall on different LDS banks.
template <int D>
__device__ __forceinline__ int swz(int row) {
  if constexpr (D == 128) return 2 * (row & 7);
  else if constexpr (D == 64) return row & 7;
  else return ((row >> 2) & 1) << 1 | ((row >> 3) & 1);
}

template <typename T, int D, bool KEYS>
__device__ __forceinline__ void bwd_unit(const Params& p, int unit, char* x0, char* y0, float* r0, char* x1, char* y1,
                                         float* r1) {
  using Op = typename Elem<T>::Operand;
  typedef __attribute__((__vector_size__(4 * sizeof(T)))) T Op4;
  constexpr int DK = D / 32, ND = D / 16, CPR = D / 8;
  constexpr int kLoads = kTile * CPR / kThreads;  // 16-byte chunks per thread and tile
  constexpr bool kHalf = __is_same(T, _Float16);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, r16 = lane & 15;
  const int ct = unit % p.NB;  // column tile
  const int64_t bh = unit / p.NB;
  const int64_t b = bh / p.H;
  const int N = p.N;
  const int64_t base = bh * N * D;
  const T* cx = static_cast<const T*>(KEYS ? p.k : p.q) + base;
  const T* cy = static_cast<const T*>(KEYS ? p.v : p.go) + base;
  const char* gx = reinterpret_cast<const char*>(static_cast<const T*>(KEYS ? p.q : p.k) + base);
  const char* gy = reinterpret_cast<const char*>(static_cast<const T*>(KEYS ? p.go : p.v) + base);
  const char* grow = reinterpret_cast<const char*>(p.rows + bh * p.NB * 2 * kTile);
  // which rows of a streamed tile have a partner among these columns
  const uint64_t* any = (KEYS ? p.qry_any : p.key_any) + (b * p.NB + ct) * p.NB;

  // columns: lane holds column r16 of the wave's 16, d = 32 kk + 8 g .. + 7
  const int col = ct * kTile + wave * 16 + r16;
  const bool col_in = col < N;
  const uint32_t* cbits = (KEYS ? p.bits_t : p.bits) + (b * N + (col_in ? col : 0)) * p.W;
  const uint32_t col_mask = col_in ? ~0u : 0u;
  Op bx[DK], by[DK];
#pragma unroll
  for (int kk = 0; kk < DK; ++kk) {
    const int64_t at = int64_t(col_in ? col : 0) * D + 8 * g + 32 * kk;
    bx[kk] = *reinterpret_cast<const Op*>(cx + at);
    by[kk] = *reinterpret_cast<const Op*>(cy + at);
  }
  float clse = 0.0f, cdelta = 0.0f;
  if (!KEYS && col_in) {
    const float* r = p.rows + (bh * p.NB + ct) * 2 * kTile + (col & 63);
    clse = r[0];
    cdelta = r[kTile];
  }
  float up = 1.0f, down = p.scale;  // dS is kept times `up` (fp16: P comes times 2^kProbBits)
  if constexpr (kHalf) {
    float gm = 0.0f, vm = 0.0f, lm = 0.0f;
    for (int i = lane; i < p.NB; i += 64) {
      const float4 m = p.peak[bh * p.NB + i];
      gm = fmaxf(gm, m.x);
      vm = fmaxf(vm, m.y);
      lm = fmaxf(lm, m.z);
    }
    gm = wave_max(gm);
    vm = wave_max(vm);
    lm = wave_max(lm);
    const float bound = 2.0f * sqrtf(gm) * sqrtf(vm) + lm;
    if (bound > 0.0f && bound < 3.0e38f) {
      const int e = min(60, max(-60, 13 - ilogbf(bound)));
      up = ldexpf(1.0f, e);
      down = p.scale * ldexpf(1.0f, -e);
    }
    up *= exp2f(-kProbBits);
  }
  const float slog = p.scale * kLog2e;

  unsigned off[kLoads];
  int srow[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int q = (wave * kLoads + i) * 64 + lane;
    srow[i] = q / CPR;
    off[i] = srow[i] * (D * 2) + (((q % CPR) ^ swz<D>(srow[i])) << 4);
  }

  // tiles with an entry, in order: 64 tiles' row sets a time in the lanes
  const uint64_t last = ~uint64_t(0) >> (p.NB * kTile - N);  // the last tile's rows
  int tbase = -64;
  uint64_t active = 0, sets = 0;
  auto next = [&](int& tile, uint64_t& set) -> bool {
    while (active == 0) {
      tbase += 64;
      if (tbase >= p.NB) return false;
      const int t = tbase + lane;
      sets = t < p.NB ? any[t] : 0;
      if (t == p.NB - 1) sets &= last;  // rows past N are read by no table
      active = __ballot(sets != 0);
    }
    const int l = __builtin_ctzll(active);
    active &= active - 1;
    tile = tbase + l;
    set = uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(sets)), l))) |
          uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(sets >> 32)), l))) << 32;
    return true;
  };
  auto load = [&](int tile, uint64_t set, char* lx, char* ly, float* lr, uint32_t (&w)[2]) {
    const int64_t first = int64_t(tile) * kTile * D * 2;
    const mf_i32x4 rx = lds_copy_source(gx + first), ry = lds_copy_source(gy + first);
    const bool all = set == ~uint64_t(0);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      unsigned o = off[i];
      if (!all) o = (set >> srow[i]) & 1 ? o : kLdsCopyOutside;
      lds_copy16(rx, o, lx + (wave * kLoads + i) * 1024);
      lds_copy16(ry, o, ly + (wave * kLoads + i) * 1024);
    }
    if (KEYS && wave == 0) {
      const mf_i32x4 rr = lds_copy_source(grow + int64_t(tile) * 512);
      const bool on = (set >> lane) & 1;  // zeros for rows without a partner here too
      lds_copy4(rr, on ? lane * 4u : kLdsCopyOutside, lr);
      lds_copy4(rr, on ? lane * 4u + kTile * 4u : kLdsCopyOutside, lr + kTile);
    }
    // (columns past the end read the first one's words, cleared where they are used)
    w[0] = cbits[2 * tile];
    w[1] = 2 * tile + 1 < p.W ? cbits[2 * tile + 1] : 0u;
  };

  uint32_t seen = 0u;  // the column has a pair
  mf_f32x4 ax[ND], ay[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n) ax[n] = ay[n] = mf_f32x4{0.f, 0.f, 0.f, 0.f};

  auto compute = [&](const char* lx, const char* ly, const float* lr, uint64_t set, const uint32_t (&words)[2]) {
#pragma unroll
    for (int pr = 0; pr < 2; ++pr) {
      if (uint32_t(set >> (32 * pr)) == 0) continue;  // no pair in these 32 rows
      const uint32_t word = words[pr] & col_mask;
      seen |= word;
      Op pb, sb;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = 32 * pr + 16 * h + r16;
        mf_f32x4 rl, d;  // d: dP - delta, -delta as the sum's start
        if constexpr (KEYS) {
          rl = *reinterpret_cast<const mf_f32x4*>(lr + 32 * pr + 16 * h + 4 * g);
          d = *reinterpret_cast<const mf_f32x4*>(lr + kTile + 32 * pr + 16 * h + 4 * g);
        } else {
          d = mf_f32x4{cdelta, cdelta, cdelta, cdelta};
        }
        mf_f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < DK; ++kk) {
          const int at = row * (D * 2) + (((4 * kk + g) ^ swz<D>(row)) << 4);
          s = Elem<T>::mma(*reinterpret_cast<const Op*>(lx + at), bx[kk], s);
          d = Elem<T>::mma(*reinterpret_cast<const Op*>(ly + at), by[kk], d);
        }
        const uint32_t bits = word >> (16 * h + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          // pairs outside the mask: P's bits are cleared (its exponent may be anything), and dS = 0 with it
          int on;
          asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(on) : "v"(bits), "n"(r));
          const float e = fast_exp2(fmaf(s[r], slog, KEYS ? -rl[r] : -clse));
          const float pv = __int_as_float(__float_as_int(e) & on);
          const float ds = kHalf ? pv * d[r] * up : pv * d[r];
          pb[4 * h + r] = Elem<T>::from_f32(pv);
          sb[4 * h + r] = Elem<T>::from_f32(ds);
        }
      }
      // operand entry 4 h + r of lane group g is row 32 pr + 16 h + 4 g + r
      const int e = r16 >> 2, a = r16 & 3;
      const int row = 32 * pr + 4 * g + e;
#pragma unroll
      for (int n = 0; n < ND; ++n) {
        const int chunk = 2 * n + (a >> 1), sub = (a & 1) * 8;
        const int lo = row * (D * 2) + ((chunk ^ swz<D>(row)) << 4) + sub;
        const int hi = (row + 16) * (D * 2) + ((chunk ^ swz<D>(row + 16)) << 4) + sub;
        const Op xt = __builtin_shufflevector(read_tr16(reinterpret_cast<const T*>(lx + lo)),
                                              read_tr16(reinterpret_cast<const T*>(lx + hi)), 0, 1, 2, 3, 4, 5, 6, 7);
        ax[n] = Elem<T>::mma(xt, sb, ax[n]);
        if constexpr (KEYS) {
          const Op yt = __builtin_shufflevector(read_tr16(reinterpret_cast<const T*>(ly + lo)),
                                                read_tr16(reinterpret_cast<const T*>(ly + hi)), 0, 1, 2, 3, 4, 5, 6, 7);
          ay[n] = Elem<T>::mma(yt, pb, ay[n]);
        }
      }
    }
  };

  auto ready = [] {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's copies into LDS have landed
    __syncthreads();
  };
  int tile = 0;
  uint64_t sa = 0, sb = 0;
  uint32_t wa[2], wb[2];
  bool more = next(tile, sa);
  if (more) load(tile, sa, x0, y0, r0, wa);
  while (more) {
    ready();
    more = next(tile, sb);
    if (more) load(tile, sb, x1, y1, r1, wb);
    compute(x0, y0, r0, sa, wa);
    if (!more) break;
    ready();
    more = next(tile, sa);
    if (more) load(tile, sa, x0, y0, r0, wa);
    compute(x1, y1, r1, sb, wb);
  }

  if (!col_in) return;
  T* ox = static_cast<T*>(KEYS ? p.dk : p.dq) + base;
  T* oy = static_cast<T*>(p.dv) + base;
#pragma unroll
  for (int n = 0; n < ND; ++n) {
    Op4 vx, vy;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      // a column without a pair: zeros, whatever it holds and whatever the tile's other rows hold
      vx[r] = Elem<T>::from_f32(seen ? ax[n][r] * down : 0.0f);
      if constexpr (KEYS) vy[r] = Elem<T>::from_f32(seen ? ay[n][r] * (kHalf ? exp2f(-kProbBits) : 1.0f) : 0.0f);
    }
    const int64_t at = int64_t(col) * D + 16 * n + 4 * g;
    *reinterpret_cast<Op4*>(ox + at) = vx;
    if constexpr (KEYS) *reinterpret_cast<Op4*>(oy + at) = vy;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, D == 128 ? 2 : 4) radius_bwd_kernel(Params p) {
  constexpr int kBytes = kTile * D * 2;
  __shared__ __attribute__((aligned(1024))) char x0[kBytes];
  __shared__ __attribute__((aligned(1024))) char y0[kBytes];
  __shared__ __attribute__((aligned(1024))) char x1[kBytes];
  __shared__ __attribute__((aligned(1024))) char y1[kBytes];
  __shared__ __attribute__((aligned(1024))) float r0[2 * kTile];
  __shared__ __attribute__((aligned(1024))) float r1[2 * kTile];
  // XCD-aware order: the column tiles of one (molecule, head), keys and queries, on one XCD and its L2
  const int per = gridDim.x >> 3;
  const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (id >= 2 * p.units) return;
  const int bh = id / (2 * p.NB), r = id - bh * 2 * p.NB;
  if (r < p.NB) bwd_unit<T, D, true>(p, bh * p.NB + r, x0, y0, r0, x1, y1, r1);
  else bwd_unit<T, D, false>(p, bh * p.NB + r - p.NB, x0, y0, r0, x1, y1, r1);
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

struct Sizes {
  int NB, W;
  size_t rows, peak;
  size_t total() const { return rows + peak; }
};
Sizes sizes(int B, int H, int N, int dtype) {
  Sizes s;
  s.NB = (N + kTile - 1) / kTile;
  s.W = (N + 31) / 32;
  s.rows = round256(size_t(B) * H * s.NB * 2 * kTile * 4);
  s.peak = dtype == MF_DTYPE_F16 ? round256(size_t(B) * H * s.NB * 16) : 0;
  return s;
}

template <typename T, int D>
int launch(Params p, hipStream_t s) {
  hipLaunchKernelGGL((radius_rows_kernel<T, D>), dim3(unsigned(p.B * p.H * p.NB)), dim3(kThreads), 0, s, p);
  MF_HIP_CHECK(hipGetLastError());
  p.units = p.B * p.H * p.NB;
  const dim3 grid(unsigned((2 * p.units + 7) / 8 * 8));
  hipLaunchKernelGGL((radius_bwd_kernel<T, D>), grid, dim3(kThreads), 0, s, p);
  MF_HIP_CHECK(hipGetLastError());
  return MF_OK;
}

template <typename T>
int dispatch(const Params& p, int D, hipStream_t s) {
  if (D == 32) return launch<T, 32>(p, s);
  if (D == 64) return launch<T, 64>(p, s);
  return launch<T, 128>(p, s);
}

}  // namespace rattn_bwd
}  // namespace mf

extern "C" int mf_radius_tables(const mf_radius_tables_args* a, void* stream) {
  using namespace mf;
  using namespace mf::rattn_bwd;
  if (a == nullptr) return fail(MF_ERR_INVALID_ARGUMENT, "mf_radius_tables: args is NULL");
  if (!a->mask_bits || !a->mask_bits_t || !a->key_any || !a->query_any)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_radius_tables: mask_bits, mask_bits_t, key_any and query_any must be non-NULL");
  if (a->batch < 0 || a->atoms < 0)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_radius_tables: batch and atoms must be non-negative");
  if (a->atoms > 65536) return fail(MF_ERR_UNSUPPORTED, "mf_radius_tables: atoms must be <= 65536");
  if (a->batch == 0 || a->atoms == 0) return MF_OK;
  TableParams p = {a->mask_bits, a->block_mask, a->mask_bits_t, a->key_any, a->query_any, a->batch, a->atoms,
                   (a->atoms + 31) / 32, (a->atoms + kTile - 1) / kTile};
  const int64_t blocks = (int64_t(p.B) * p.NB * p.NB + 3) / 4;
  if (blocks * kThreads > 0xffffffffLL)  // threads of a launch
    return fail(MF_ERR_UNSUPPORTED, "mf_radius_tables: batch * tiles too large");
  hipLaunchKernelGGL(radius_tables_kernel, dim3(unsigned(blocks)), dim3(kThreads), 0, static_cast<hipStream_t>(stream), p);
  MF_HIP_CHECK(hipGetLastError());
  return MF_OK;
}

extern "C" uint64_t mf_radius_attn_bwd_workspace_size(int32_t batch, int32_t heads, int32_t atoms, int32_t dtype) {
  if (batch <= 0 || heads <= 0 || atoms <= 0) return 0;
  return mf::rattn_bwd::sizes(batch, heads, atoms, dtype).total();
}

extern "C" int mf_radius_attn_bwd(const mf_radius_attn_bwd_args* a, void* stream) {
  using namespace mf;
  using namespace mf::rattn_bwd;
  if (a == nullptr) return fail(MF_ERR_INVALID_ARGUMENT, "mf_radius_attn_bwd: args is NULL");
  if (!a->q || !a->k || !a->v || !a->out || !a->lse || !a->grad_out || !a->dq || !a->dk || !a->dv)
    return fail(MF_ERR_INVALID_ARGUMENT,
                "mf_radius_attn_bwd: q, k, v, out, lse, grad_out, dq, dk and dv must be non-NULL");
  if (!a->mask_bits || !a->mask_bits_t || !a->key_any || !a->query_any)
    return fail(MF_ERR_INVALID_ARGUMENT,
                "mf_radius_attn_bwd: mask_bits and its tables (mf_radius_tables) must be non-NULL");
  if (a->batch < 0 || a->heads < 0 || a->atoms < 0)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_radius_attn_bwd: batch, heads and atoms must be non-negative");
  if (a->dtype != MF_DTYPE_BF16 && a->dtype != MF_DTYPE_F16)
    return fail(MF_ERR_UNSUPPORTED, "mf_radius_attn_bwd: only supports float16/bfloat16 operands");
  if (a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128)
    return fail(MF_ERR_UNSUPPORTED, "mf_radius_attn_bwd: head_dim must be 32, 64 or 128");
  if (!std::isfinite(a->scale)) return fail(MF_ERR_INVALID_ARGUMENT, "mf_radius_attn_bwd: scale must be finite");
  for (const void* ptr : {a->q, a->k, a->v, a->out, a->out_lo, a->grad_out, static_cast<const void*>(a->dq),
                          static_cast<const void*>(a->dk), static_cast<const void*>(a->dv)})
    if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0)
      return fail(MF_ERR_INVALID_ARGUMENT, "mf_radius_attn_bwd: operands and gradients must be 16-byte aligned");
  if (a->batch == 0 || a->heads == 0 || a->atoms == 0) return MF_OK;
  if (a->atoms > 65536) return fail(MF_ERR_UNSUPPORTED, "mf_radius_attn_bwd: atoms must be <= 65536");
  const Sizes z = sizes(a->batch, a->heads, a->atoms, a->dtype);
  const int64_t units = int64_t(a->batch) * a->heads * z.NB;
  if ((2 * units + 7) / 8 * 8 * kThreads > 0xffffffffLL)  // threads of a launch
    return fail(MF_ERR_UNSUPPORTED, "mf_radius_attn_bwd: batch * heads * tiles too large");
  if (!a->workspace || a->workspace_bytes < z.total() || reinterpret_cast<uintptr_t>(a->workspace) % 16 != 0)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_radius_attn_bwd: the workspace must be 16-byte aligned and hold "
                                         "mf_radius_attn_bwd_workspace_size bytes");
  Params p = {};
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.out = a->out;
  p.out_lo = a->out_lo;
  p.go = a->grad_out;
  p.bits = a->mask_bits;
  p.lse = a->lse;
  p.dlse = a->grad_lse;
  p.dq = a->dq;
  p.dk = a->dk;
  p.dv = a->dv;
  char* ws = static_cast<char*>(a->workspace);
  p.bits_t = a->mask_bits_t;
  p.key_any = a->key_any;
  p.qry_any = a->query_any;
  p.rows = reinterpret_cast<float*>(ws);
  p.peak = z.peak ? reinterpret_cast<float4*>(ws + z.rows) : nullptr;
  p.scale = a->scale;
  p.B = a->batch;
  p.H = a->heads;
  p.N = a->atoms;
  p.W = z.W;
  p.NB = z.NB;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == MF_DTYPE_BF16) return dispatch<__bf16>(p, a->head_dim, s);
  return dispatch<_Float16>(p, a->head_dim, s);
}
