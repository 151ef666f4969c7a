// Attention over all pairs with a learned bias by buckets (mf_bucket_attn) on
// gfx950: out_i = sum_j softmax_j(scale q_i . k_j + table[bucket_ij, h]) v_j over
// the pairs that are not masked.  Rows without a pair give out 0, lse 0.
//
// A wave owns 32 queries of one head as the columns of its products and streams
// 64-key tiles of K and V through LDS (copied straight from global memory, the
// next tile while the current one is multiplied; tiles in which no query of the
// workgroup has a key are left out):
//   S^T = K Q^T, x = log2(e) (scale S + bias), running maximum m and sum l of
//   2^(x - m) per column, O^T += V^T P^T
// with P^T taken from the first product's accumulators as the operand of the
// second.  A lane's 16 logits of a 32-key block belong to 16 consecutive bytes
// of its query's row of buckets, loaded from global memory in one access and
// looked up in the head's table in LDS, one bank a bucket.  fp16 keeps 2^(x - m)
// times 2^7: many keys of small weight beside a large one still count (131072
// of 2^-25 would be 0 each, 0.4 % of the row together).
//
// 32 x 8 heads of 512 atoms (head_dim 64, bf16) take 41 us (420 TFLOP/s), 2 x 12 heads
// of 8192 places, earlier keys only (head_dim 128), 494 us (834, a large product of
// the library 1232): bound by the exp2s and lookups that do not hide behind the
// products.  64 keys a tile: four buffers of it leave LDS for two workgroups and
// more a CU.
//
// Where the query heads of a key head have few queries in all (a new token), the
// heads' queries are packed into the columns of one workgroup, so that K and V
// are read once, and the keys are split over workgroups whose maxima, sums and
// outputs bucket_join_kernel joins (120001 keys of 4 key heads of 128, 12 query heads:
// 48 us, 5.1 TB/s).
#include <algorithm>
#include <cmath>

#include "bucket_tiles.h"

namespace mf {
namespace bucket {

struct FwdParams {
  const void* q;
  const void* k;
  const void* v;
  const void* table;
  const uint8_t* index;
  const uint64_t* key_any;
  const uint64_t* query_any;
  void* out;
  void* out_lo;
  float* lse;
  float* stats;
  float* part_out;  // [units, splits, columns, DP]
  float* part_ml;   // [units, splits, columns, 2]
  int64_t qs[3], ks[3], vs[3], os[3];
  int64_t index_step, any_step;  // from one batch entry to the next (0: shared)
  float slog;                    // scale * log2(e)
  int B, H, KV, G, Nq, Nk, D, S, TQ, TK, K, table_dtype;
  int packed;    // the columns are the queries of all heads of a key head
  int UH;        // heads of the units: H, or KV when packed
  int CT;        // workgroups per (batch, unit head) and split
  int splits, tiles_per_split;
  int64_t units;
};

// What column c of a unit's head stands for.
struct Column {
  int64_t b;
  int h, i;
  bool in;
};
__device__ __forceinline__ Unit unit_of(const FwdParams& p, uint32_t unit) {
  return unit_of(unit, p.B, p.UH, p.packed ? 1 : p.G, p.CT, false);
}
__device__ __forceinline__ Column column_of(const FwdParams& p, const Unit& u, int c) {
  Column r;
  r.b = u.b;
  if (p.packed) {
    const int g = c / p.Nq;
    r.in = g < p.G;
    r.h = u.head * p.G + (r.in ? g : 0);
    r.i = r.in ? c - g * p.Nq : 0;
  } else {
    r.h = u.head;
    r.in = c < p.Nq;
    r.i = r.in ? c : 0;
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void store_row(const FwdParams& p, const Column& c, int d0, const float (&x)[8]) {
  typedef __attribute__((__vector_size__(8 * sizeof(T)))) T T8;
  T8 y;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = static_cast<T>(x[e]);
  *reinterpret_cast<T8*>(static_cast<T*>(p.out) + c.b * p.os[0] + c.h * p.os[1] + c.i * p.os[2] + d0) = y;
  if (p.out_lo) {
    T8 lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) lo[e] = static_cast<T>(x[e] - float(y[e]));
    *reinterpret_cast<T8*>(static_cast<T*>(p.out_lo) + ((c.b * p.H + c.h) * p.Nq + c.i) * p.D + d0) = lo;
  }
}

constexpr float kSlack = 8.0f;         // how far x may pass m, which is not always the maximum
constexpr float kExact = 1048576.0f;   // |m| below which it may: up to there m + 8 and the like lose little

// What 2^(x - m) is kept times, as a power of two.
template <typename T>
constexpr float shift_bits() {
  return __is_same(T, _Float16) ? 15.0f - kSlack : 0.0f;
}

template <typename T>
__device__ __forceinline__ void store_stats(const FwdParams& p, const Column& c, float m, float l) {
  l *= __is_same(T, _Float16) ? 1.0f / 128.0f : 1.0f;  // 2^-shift_bits
  const int64_t at = (c.b * p.H + c.h) * p.Nq + c.i;
  if (p.stats) {
    // m, which may lag behind the maximum, is raised by the whole part of log2 l, so that 2^(x - m) < 2 for every x of the
    // row; l is what the sum from there is
    float to = m, inv = l;  // (a NaN stays one)
    if (l > 0.0f) {
      if (fabsf(m) < kExact) to = m + float(ilogbf(l));
      inv = fast_exp2(to - m) / l;
    }
    p.stats[at] = l > 0.0f ? to : 0.0f;
    p.stats[int64_t(p.B) * p.H * p.Nq + at] = inv;
  }
  if (p.lse) p.lse[at] = l > 0.0f ? (m + __log2f(l)) * kLn2 : l;
}

// Waves a SIMD that the registers are to allow: three (head_dim 128: two), or what LDS has room for.
constexpr int fwd_waves(int DP, int W, bool packed) {
  const int lds = 4 * kTile * DP * 2 + (packed ? 32 : 1) * kPitch * 4;
  const int fit = 160 * 1024 / lds * W / 4, most = DP == 128 ? 2 : 3;
  return fit < 1 ? 1 : fit < most ? fit : most;
}

template <typename T, int DP, int W, bool PACKED>
__global__ void __launch_bounds__(64 * W, fwd_waves(DP, W, PACKED)) bucket_attn_kernel(FwdParams p) {
  using Op = typename Elem<T>::Operand;
  constexpr int NK = DP / 16, ND = DP / 32;
  constexpr int kBytes = kTile * DP * 2;
  __shared__ __attribute__((aligned(1024))) char s_tiles[4 * kBytes];  // K and V of two tiles
  __shared__ float s_table[(PACKED ? 32 : 1) * kPitch];
  const uint32_t id = xcd_order(blockIdx.x, gridDim.x);
  if (id >= p.units * p.splits) return;
  const uint32_t unit = id / uint32_t(p.splits);
  const int split = int(id - unit * p.splits);
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Unit of = unit_of(p, unit);
  const int uh = of.head, ct = of.tile;
  const int64_t b = of.b;
  const Column me = column_of(p, of, ct * 32 * W + wave * 32 + (lane & 31));
  const int kv = PACKED ? uh : uh / p.G;

  const float* table = PACKED ? s_table + (me.h - uh * p.G) * kPitch : s_table;
  const LaneReads<T, DP> reads(lane);
  // the query tiles of the unit's columns
  const int qt0 = PACKED ? 0 : (ct * 32 * W) / kTile;
  const bool two = !PACKED && W == 4 && qt0 + 1 < p.TQ;
  const int t0 = split * p.tiles_per_split, t1 = min(p.TK, t0 + p.tiles_per_split);
  const uint64_t* any = p.key_any + b * p.any_step + int64_t(qt0) * p.TK;
  const uint8_t* codes = p.index + me.b * p.index_step + int64_t(me.i) * p.S + 16 * half;
  const char* gk = reinterpret_cast<const char*>(static_cast<const T*>(p.k) + b * p.ks[0] + kv * p.ks[1]);
  const char* gv = reinterpret_cast<const char*>(static_cast<const T*>(p.v) + b * p.vs[0] + kv * p.vs[1]);
  const unsigned kstride = unsigned(p.ks[2]) * 2, vstride = unsigned(p.vs[2]) * 2;

  const TileCopy<DP, W> kcopy(kstride, p.D, wave, lane), vcopy(vstride, p.D, wave, lane);
  auto load = [&](int tile, uint64_t set, char* to, uint4 (&w)[2]) {
    kcopy.copy(gk + int64_t(tile) * kTile * kstride, set, to, wave, lane);
    vcopy.copy(gv + int64_t(tile) * kTile * vstride, set, to + kBytes, wave, lane);
    w[0] = *reinterpret_cast<const uint4*>(codes + int64_t(tile) * kTile);
    w[1] = *reinterpret_cast<const uint4*>(codes + int64_t(tile) * kTile + 32);
  };

  Tiles tiles(any, two ? any + p.TK : nullptr, t0, t1);
  int tile = 0, buffer = 0;
  uint64_t set = 0;
  uint4 next[2];
  bool more = tiles.next(tile, set);
  if (more) load(tile, set, s_tiles, next);

  // while the first tile is on its way: the tables, the lane's query, and which queries have a key among this split's
  const T* gq = static_cast<const T*>(p.q) + me.b * p.qs[0] + me.h * p.qs[1] + me.i * p.qs[2];
  Op qb[NK];
#pragma unroll
  for (int kk = 0; kk < NK; ++kk) {
    const int d = 16 * kk + 8 * half;
    qb[kk] = *reinterpret_cast<const Op*>(gq + (d < p.D ? d : 0));
  }
  uint64_t used = union_of(p.query_any + b * p.any_step, p.TQ, qt0, t0, t1);
  if (two) {
    const uint64_t second = union_of(p.query_any + b * p.any_step, p.TQ, qt0 + 1, t0, t1);
    if (wave >= 2) used = second;
  }
  load_tables(s_table, p.table, p.table_dtype, p.K, p.H, PACKED ? uh * p.G : uh, PACKED ? p.G : 1, 64 * W);
  const bool mine = me.in && ((used >> (me.i & 63)) & 1);
#pragma unroll
  for (int kk = 0; kk < NK; ++kk) {
    if (!mine || 16 * kk + 8 * half >= p.D) {
#pragma unroll
      for (int e = 0; e < 8; ++e) qb[kk][e] = T(0.0f);
    }
  }
  mf_f32x16 acc[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n) acc[n] = zeros16();
  float m = -INFINITY, l = 0.0f, limit = -INFINITY;

  while (more) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's copies into LDS have landed
    __syncthreads();
    const uint4 w[2] = {next[0], next[1]};
    const LaneReads<T, DP> at = reads.shifted(buffer);
    buffer ^= 2 * kBytes;
    more = tiles.next(tile, set);
    if (more) load(tile, set, s_tiles + buffer, next);

    mf_f32x16 x[2];
    float top = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const uint32_t word[4] = {w[kb].x, w[kb].y, w[kb].z, w[kb].w};
      Op ka[NK];
      float bias[16];
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) ka[kk] = at.rows(s_tiles, kb, kk);
#pragma unroll
      for (int t = 0; t < 16; ++t) bias[t] = table[byte_of(word, t)];
      __builtin_amdgcn_sched_barrier(0);
      mf_f32x16 s = zeros16();
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) s = Mma32<T>::mma(ka[kk], qb[kk], s);
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        x[kb][t] = fmaf(s[t], p.slog, bias[t]);
        top = fmaxf(top, x[kb][t]);
      }
    }
    // m follows the maximum only where that has grown by more than kSlack, so that most tiles leave the sums alone
    top = pair_max(top);
    if (__any(top > limit)) {
      const float to = top > limit ? top : m;
      const float keep = to == -INFINITY ? 1.0f : fast_exp2(m - to);
      l *= keep;
#pragma unroll
      for (int n = 0; n < ND; ++n) acc[n] *= keep;
      m = to;
      limit = fabsf(m) < kExact ? m + kSlack : m;
    }
    const float from = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      Op pb[2], va[2][ND];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int n = 0; n < ND; ++n) va[s][n] = at.columns(s_tiles + kBytes, kb, s, n);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        // (the shift after the difference: beside a huge m it would be lost)
        const float e = fast_exp2(__is_same(T, _Float16) ? (x[kb][t] - from) + shift_bits<T>() : x[kb][t] - from);
        l += e;
        pb[t >> 3][t & 7] = static_cast<T>(e);
      }
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int n = 0; n < ND; ++n) acc[n] = Mma32<T>::mma(va[s][n], pb[s], acc[n]);
    }
  }

  l = pair_sum(l);
  if (!me.in) return;
  if (p.splits > 1) {
    const int64_t at = int64_t(id) * (32 * W) + wave * 32 + (lane & 31);
    float* o = p.part_out + at * DP;
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int t = 0; t < 16; t += 4)
        *reinterpret_cast<float4*>(o + 32 * n + 16 * half + t) =
            make_float4(acc[n][t], acc[n][t + 1], acc[n][t + 2], acc[n][t + 3]);
    if (half == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m, l);
    return;
  }
  // (a query without a pair: the sums are zero, or whatever -inf biases left of them)
  const float inv = l > 0.0f ? 1.0f / l : l;
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int d0 = 32 * n + 16 * half + 8 * u;
      if (d0 >= p.D) continue;
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = acc[n][8 * u + e] * inv;
      store_row<T>(p, me, d0, y);
    }
  if (half == 0) store_stats<T>(p, me, m, l);
}

// Joins the splits: a workgroup per column, a quarter of the splits a wave (or as many waves as there are splits for),
// DP / 8 lanes to a split's entries, the others taking the next splits.
template <typename T, int DP>
__global__ void __launch_bounds__(256) bucket_join_kernel(FwdParams p, int columns, int in_use) {
  constexpr int L = DP / 8, SG = 64 / L;
  __shared__ float s_m[4], s_l[4], s_y[4][DP];
  const uint32_t unit = blockIdx.x / uint32_t(in_use);
  const int c = int(blockIdx.x - unit * in_use);
  const Unit of = unit_of(p, unit);
  const Column me = column_of(p, of, of.tile * columns + c);
  if (!me.in) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* ml = p.part_ml + (int64_t(unit) * p.splits * columns + c) * 2;
  const float* po = p.part_out + (int64_t(unit) * p.splits * columns + c) * DP;
  const int64_t step = columns;
  float m = -INFINITY, l = 0.0f;
  for (int s = tid; s < p.splits; s += 256) m = fmaxf(m, ml[s * step * 2]);
  m = wave_max(m);
  if (lane == 0) s_m[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  const float from = m == -INFINITY ? 0.0f : m;
  const int d0 = (lane % L) * 8, g = lane / L;
  float y[8] = {};
#pragma unroll 4
  for (int s = wave * SG + g; s < p.splits; s += 4 * SG) {
    const float2 one = *reinterpret_cast<const float2*>(ml + s * step * 2);
    const float4 lo = *reinterpret_cast<const float4*>(po + s * step * DP + d0);
    const float4 hi = *reinterpret_cast<const float4*>(po + s * step * DP + d0 + 4);
    const float w = fast_exp2(one.x - from);
    l += w * one.y;
    y[0] += w * lo.x;
    y[1] += w * lo.y;
    y[2] += w * lo.z;
    y[3] += w * lo.w;
    y[4] += w * hi.x;
    y[5] += w * hi.y;
    y[6] += w * hi.z;
    y[7] += w * hi.w;
  }
#pragma unroll
  for (int off = L; off < 64; off <<= 1) {
    l += __shfl_xor(l, off, 64);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] += __shfl_xor(y[e], off, 64);
  }
  if (g == 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s_y[wave][d0 + e] = y[e];
    if (lane == 0) s_l[wave] = l;
  }
  __syncthreads();
  if (tid >= L) return;
  l = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
  const float inv = l > 0.0f ? 1.0f / l : l;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    y[e] = ((s_y[0][d0 + e] + s_y[1][d0 + e]) + (s_y[2][d0 + e] + s_y[3][d0 + e])) * inv;
  if (d0 < p.D) store_row<T>(p, me, d0, y);
  if (tid == 0) store_stats<T>(p, me, m, l);
}

namespace {

struct Plan {
  int DP, W, packed, UH, CT, splits, tiles_per_split;
  int64_t units;
  size_t out_bytes, ml_bytes;
};

Plan plan_of(const mf_bucket_attn_args* a) {
  Plan z = {};
  const int G = a->heads / a->kv_heads;
  z.DP = a->head_dim <= 32 ? 32 : a->head_dim <= 64 ? 64 : 128;
  z.packed = G > 1 && a->queries <= kTile && int64_t(G) * a->queries <= 128;
  z.UH = z.packed ? a->kv_heads : a->heads;
  const int columns = z.packed ? G * a->queries : a->queries;
  z.W = columns <= 32 ? 1 : columns <= 64 ? 2 : 4;
  z.CT = (columns + 32 * z.W - 1) / (32 * z.W);
  z.units = int64_t(a->batch) * z.UH * z.CT;
  const int TK = std::max(1, (a->keys + kTile - 1) / kTile);
  // Few workgroups over many keys: split until about 1024 waves run, a piece at least two tiles.
  const int64_t waves = z.units * z.W;
  int splits = 1;
  if (waves < 512) splits = int(std::min<int64_t>((TK + 1) / 2, (1024 + waves - 1) / waves));
  splits = std::max(splits, 1);
  z.tiles_per_split = (TK + splits - 1) / splits;
  z.splits = (TK + z.tiles_per_split - 1) / z.tiles_per_split;
  if (z.splits > 1) {
    const size_t rows = size_t(z.units) * z.splits * 32 * z.W;
    z.out_bytes = rows * z.DP * sizeof(float);
    z.ml_bytes = rows * 2 * sizeof(float);
  }
  return z;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

// 0, or the refusal of what the forward and the gradients share.
int check_attn(const mf_bucket_attn_args* a, const char* what) {
  const std::string name(what);
  if (a == nullptr) return fail(MF_ERR_INVALID_ARGUMENT, name + ": args is NULL");
  if (!a->q || !a->k || !a->v || !a->table || !a->index || !a->key_any || !a->query_any || !a->out)
    return fail(MF_ERR_INVALID_ARGUMENT,
                name + ": q, k, v, table, index, key_any, query_any and out must be non-NULL");
  if (a->batch < 0 || a->heads < 0 || a->kv_heads < 0 || a->queries < 0 || a->keys < 0)
    return fail(MF_ERR_INVALID_ARGUMENT, name + ": batch, heads, queries and keys must be non-negative");
  if (a->dtype != MF_DTYPE_BF16 && a->dtype != MF_DTYPE_F16)
    return fail(MF_ERR_UNSUPPORTED, name + ": only supports float16/bfloat16 operands");
  if (a->table_dtype != MF_DTYPE_F32 && a->table_dtype != MF_DTYPE_BF16 && a->table_dtype != MF_DTYPE_F16)
    return fail(MF_ERR_UNSUPPORTED, name + ": the table must be float32/float16/bfloat16");
  if (a->head_dim < 8 || a->head_dim > 128 || a->head_dim % 8 != 0)
    return fail(MF_ERR_UNSUPPORTED, name + ": head_dim must be a multiple of 8 up to 128");
  if (a->buckets < 1 || a->buckets > MF_MAX_BUCKETS)
    return fail(MF_ERR_UNSUPPORTED, name + ": buckets must be in [1, 64]");
  if (!std::isfinite(a->scale)) return fail(MF_ERR_INVALID_ARGUMENT, name + ": scale must be finite");
  if (a->index_batch != 1 && a->index_batch != a->batch)
    return fail(MF_ERR_INVALID_ARGUMENT, name + ": index_batch must be 1 or batch");
  if (a->queries > (1 << 24) || a->keys > (1 << 24))
    return fail(MF_ERR_UNSUPPORTED, name + ": queries and keys must be <= 2^24");
  if (a->heads > 0 && (a->kv_heads < 1 || a->heads % a->kv_heads != 0 || a->heads / a->kv_heads > 32))
    return fail(MF_ERR_UNSUPPORTED, name + ": kv_heads must divide heads, at most 32 heads to a key head");
  for (const void* ptr : {a->q, a->k, a->v, static_cast<const void*>(a->index), static_cast<const void*>(a->out),
                          static_cast<const void*>(a->out_lo)})
    if (!aligned16(ptr)) return fail(MF_ERR_INVALID_ARGUMENT, name + ": operands and outputs must be 16-byte aligned");
  for (const int64_t* s : {a->q_stride, a->k_stride, a->v_stride, a->out_stride})
    for (int n = 0; n < 3; ++n)
      if (s[n] % 8 != 0 || s[n] < 0)
        return fail(MF_ERR_INVALID_ARGUMENT, name + ": strides must be non-negative multiples of 8");
  for (const int64_t* s : {a->q_stride, a->k_stride, a->v_stride})
    if (s[2] >= (1 << 23))  // a tile's 64 rows within 2^30 bytes
      return fail(MF_ERR_UNSUPPORTED, name + ": token strides must be below 2^23 elements");
  return MF_OK;
}

template <typename T, int DP, int W, bool PACKED>
int launch_fwd(const FwdParams& p, hipStream_t s) {
  const int64_t blocks = (p.units * p.splits + 7) / 8 * 8;
  hipLaunchKernelGGL((bucket_attn_kernel<T, DP, W, PACKED>), dim3(unsigned(blocks)), dim3(64 * W), 0, s, p);
  MF_HIP_CHECK(hipGetLastError());
  if (p.splits > 1) {
    // (columns past the last are left out)
    const int columns = p.CT == 1 ? std::min(32 * W, p.packed ? p.G * p.Nq : p.Nq) : 32 * W;
    hipLaunchKernelGGL((bucket_join_kernel<T, DP>), dim3(unsigned(p.units * columns)), dim3(256), 0, s, p, 32 * W, columns);
    MF_HIP_CHECK(hipGetLastError());
  }
  return MF_OK;
}

template <typename T, int DP>
int launch_fwd(const FwdParams& p, int W, hipStream_t s) {
  if (W == 1) return p.packed ? launch_fwd<T, DP, 1, true>(p, s) : launch_fwd<T, DP, 1, false>(p, s);
  if (W == 2) return p.packed ? launch_fwd<T, DP, 2, true>(p, s) : launch_fwd<T, DP, 2, false>(p, s);
  return p.packed ? launch_fwd<T, DP, 4, true>(p, s) : launch_fwd<T, DP, 4, false>(p, s);
}

template <typename T>
int launch_fwd(const FwdParams& p, int DP, int W, hipStream_t s) {
  if (DP == 32) return launch_fwd<T, 32>(p, W, s);
  if (DP == 64) return launch_fwd<T, 64>(p, W, s);
  return launch_fwd<T, 128>(p, W, s);
}

}  // namespace bucket
}  // namespace mf

extern "C" uint64_t mf_bucket_attn_workspace_size(const mf_bucket_attn_args* a) {
  if (a == nullptr || a->batch <= 0 || a->heads <= 0 || a->kv_heads <= 0 || a->queries <= 0 || a->keys <= 0) return 0;
  const mf::bucket::Plan z = mf::bucket::plan_of(a);
  return z.out_bytes + z.ml_bytes;
}

extern "C" int mf_bucket_attn(const mf_bucket_attn_args* a, void* stream) {
  using namespace mf;
  using namespace mf::bucket;
  if (const int status = check_attn(a, "mf_bucket_attn")) return status;
  if (a->batch == 0 || a->heads == 0 || a->queries == 0) return MF_OK;
  FwdParams p = {};
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.table = a->table;
  p.index = a->index;
  p.key_any = a->key_any;
  p.query_any = a->query_any;
  p.out = a->out;
  p.out_lo = a->out_lo;
  p.lse = a->lse;
  p.stats = a->stats;
  for (int n = 0; n < 3; ++n) {
    p.qs[n] = a->q_stride[n];
    p.ks[n] = a->k_stride[n];
    p.vs[n] = a->v_stride[n];
    p.os[n] = a->out_stride[n];
  }
  p.slog = a->scale * kLog2e;
  p.B = a->batch;
  p.H = a->heads;
  p.KV = a->kv_heads;
  p.G = a->heads / a->kv_heads;
  p.Nq = a->queries;
  p.Nk = a->keys;
  p.D = a->head_dim;
  p.S = (a->keys + 63) / 64 * 64;
  p.TQ = (a->queries + kTile - 1) / kTile;
  p.TK = (a->keys + kTile - 1) / kTile;
  p.K = a->buckets;
  p.table_dtype = a->table_dtype;
  p.index_step = a->index_batch == 1 ? 0 : int64_t(p.Nq) * p.S;
  p.any_step = a->index_batch == 1 ? 0 : int64_t(p.TQ) * p.TK;
  const Plan z = plan_of(a);
  p.packed = z.packed;
  p.UH = z.UH;
  p.CT = z.CT;
  p.units = z.units;
  p.splits = z.splits;
  p.tiles_per_split = z.tiles_per_split;
  if ((p.units * p.splits + 7) / 8 * 8 * 64 * z.W > 0xffffffffLL)  // threads of a launch (few units where there are splits)
    return fail(MF_ERR_UNSUPPORTED, "mf_bucket_attn: batch * heads * queries too large");
  if (z.splits > 1) {
    if (!a->workspace || a->workspace_bytes < z.out_bytes + z.ml_bytes || !aligned16(a->workspace))
      return fail(MF_ERR_INVALID_ARGUMENT, "mf_bucket_attn: the workspace must be 16-byte aligned and hold "
                                           "mf_bucket_attn_workspace_size bytes");
    p.part_out = static_cast<float*>(a->workspace);
    p.part_ml = p.part_out + z.out_bytes / sizeof(float);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == MF_DTYPE_BF16) return launch_fwd<__bf16>(p, z.DP, z.W, s);
  return launch_fwd<_Float16>(p, z.DP, z.W, s);
}
