// Rotary positions (mf_rotary) on gfx950: every pair (x0, x1) of a head's first
// rotary_dim entries is turned by theta = pos[axis(p)] * f_p,
//   y0 = gain (x0 cos - x1 sin),   y1 = gain (x0 sin + x1 cos),
// the remaining entries and the unturned parts are copied.  The inverse (the
// gradient's direction) turns by -theta.
//
// One launch takes up to three parts (q, k, v of one projection) between any
// two strided layouts, also through the slot map of packed rows, so splitting
// the heads, turning and padding are one pass: each element is read and written
// once and the bytes are what bounds it.
//
// Angles: pos * f is formed in fp64 and reduced to a fraction of a turn there
// (a position of 10^6 in fp32 would be off by 0.06 rad); sine and cosine of what
// is left are fp32.
//
// A thread owns eight pairs of one token: it computes their sines and cosines
// once, into registers, and walks the heads of every part, four at a time (eight
// 16-byte loads in flight).  Its pairs are two pieces of eight consecutive
// entries, 16 bytes each at any alignment (the second half of the half layout
// starts at rotary_dim / 2, which need be no multiple of 8); the last unit of
// pairs starts at P - 8 and computes some pairs a second time, with equal
// results, rather than masking.  More threads of a token copy what is not turned;
// of a turned head's tail that is no multiple of 16 entries, a head at a time, each
// waiting for the one before (64 x 181 tokens, 24 heads of 64: rotary_dim 64 takes
// 16.4 us, 60 and 24 take 22.8).
#include <algorithm>
#include <cmath>

#include "mf_common.h"

namespace mf {
namespace rot {

constexpr int kThreads = 256;
constexpr int kHeads = 4;         // heads in flight per thread
constexpr int kMaxDim = 256;
constexpr int kScalarTokens = 16; // tokens per workgroup of the scalar kernel

struct Part {
  const void* src;
  void* dst;
  int64_t ss[3], ds[3];  // {batch, head, token} strides in elements
  int heads;
  int turn;
};

struct Params {
  Part part[3];
  const void* pos;
  int64_t ps[3];         // {batch, token, axis} strides of the positions
  const double* freq;
  const int32_t* slot;
  float gain;
  int pos_type, slot_side, axes, inverse;
  int nparts, B, N, D, R, interleaved;
  int TT, HS, heads;     // tokens and heads per workgroup, heads of all parts
  int units, turned;     // threads of a token, and those of them that turn pairs
};

// 8 consecutive elements in registers: one 16-byte access for 16-bit types, two for fp32.
template <typename T>
struct Chunk {
  static constexpr int kLoads = sizeof(T) / 2;
  uint4 u[kLoads];
  // any alignment: global memory takes 16-byte accesses at every byte
  __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(u, p, sizeof(u)); }
  __device__ __forceinline__ void store(T* p) const { __builtin_memcpy(p, u, sizeof(u)); }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) u[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void unpack(float (&x)[8]) const {
    typedef T V __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const V e = __builtin_bit_cast(V, u[i / int(16 / sizeof(T))]);
      x[i] = Elem<T>::to_f32(e[i % int(16 / sizeof(T))]);
    }
  }
  __device__ __forceinline__ void pack(const float (&x)[8]) {
    typedef T V __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      V e;
#pragma unroll
      for (int i = 0; i < int(16 / sizeof(T)); ++i) e[i] = Elem<T>::from_f32(x[l * int(16 / sizeof(T)) + i]);
      u[l] = __builtin_bit_cast(uint4, e);
    }
  }
};

__device__ __forceinline__ double position(const Params& p, int64_t at) {
  switch (p.pos_type) {
    case MF_POS_F64: return static_cast<const double*>(p.pos)[at];
    case MF_POS_I32: return double(static_cast<const int32_t*>(p.pos)[at]);
    case MF_POS_I64: return double(static_cast<const int64_t*>(p.pos)[at]);
    default: return double(static_cast<const float*>(p.pos)[at]);
  }
}

// cos and sin of pair pr at a position, times gain.  In fp64 the angle becomes quarter turns q and a rest x of at most
// pi / 4; their Taylor sums to x^9 and x^10 leave less than 2^-25.
__device__ __forceinline__ float2 turn_of(const Params& p, int64_t at, int pr) {
  const double turns = position(p, at) * p.freq[pr] * 0.15915494309189533577;
  const double quarters = 4.0 * (turns - rint(turns));  // in [-2, 2]
  const double whole = rint(quarters);
  const float x = float((quarters - whole) * 1.57079632679489661923);
  const int q = int(whole) & 3;
  const float z = x * x;
  const float s = x + x * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
  const float c = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 + z * (-1.0f / 3628800)))));
  const float cc = q & 1 ? s : c, sc = q & 1 ? c : s;
  const float cos = q == 1 || q == 2 ? -cc : cc, sin = q >= 2 ? -sc : sc;
  return make_float2(p.gain * cos, p.gain * (p.inverse ? -sin : sin));
}

// n < 16 elements at any alignment, in pieces of 8, 4, 2 and 1
template <typename TS, typename TD>
__device__ __forceinline__ void copy_some(const TS* src, TD* dst, int n, bool zero) {
  int at = 0;
#pragma unroll
  for (int size = 8; size >= 1; size >>= 1) {
    if (!(n & size)) continue;
    TS v[8];
    if (zero) {
#pragma unroll
      for (int e = 0; e < size; ++e) v[e] = TS(0.0f);
    } else {
      __builtin_memcpy(v, src + at, size * sizeof(TS));
    }
    TD o[8];
#pragma unroll
    for (int e = 0; e < size; ++e) o[e] = Elem<TD>::from_f32(Elem<TS>::to_f32(v[e]));
    __builtin_memcpy(dst + at, o, size * sizeof(TD));
    at += size;
  }
}

template <typename TS, typename TD, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rotary_kernel(Params p) {
  const unsigned t = threadIdx.x / unsigned(p.units);
  const int u = int(threadIdx.x - t * unsigned(p.units));
  const unsigned g = blockIdx.x * unsigned(p.TT) + t;  // below 2^31
  if (int(t) >= p.TT || g >= unsigned(p.B) * unsigned(p.N)) return;
  const unsigned b = g / unsigned(p.N), n = g - b * unsigned(p.N);
  const int P = p.R >> 1;
  const bool turner = u < p.turned;
  const int p0 = min(8 * u, P - 8);  // first pair (turners)
  int64_t row = 0;
  if (p.slot_side != MF_SLOT_NONE) row = p.slot[g];
  const bool zero = p.slot_side == MF_SLOT_SRC && row < 0;
  if (p.slot_side == MF_SLOT_DST && row < 0) return;
  float2 cs[8];
  if (turner && !zero) {
    const int per = P / p.axes;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      cs[j] = turn_of(p, b * p.ps[0] + n * p.ps[1] + ((p0 + j) / per) * p.ps[2], p0 + j);
  }
  const int h0 = blockIdx.y * p.HS, h1 = min(p.heads, h0 + p.HS);
  int base = 0;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    if (k >= p.nparts) break;
    const Part& part = p.part[k];
    const int lo = max(h0 - base, 0), hi = min(h1 - base, part.heads);
    base += part.heads;
    if (lo >= hi) continue;
    const bool turning = part.turn != 0 && turner;
    // the thread's entries: two pieces of 8, or fewer than 16 entries from e0 on
    int e0, e1, some = 16;
    if (turning) {
      e0 = INTERLEAVED ? 2 * p0 : p0;
      e1 = INTERLEAVED ? e0 + 8 : P + p0;
    } else if (part.turn) {
      e0 = p.R + 16 * (u - p.turned);
      e1 = e0 + 8;
      some = p.D - e0;
    } else {
      e0 = min(16 * u, p.D - 16);
      e1 = e0 + 8;
      if (16 * u >= p.D) continue;
    }
    const int64_t so = p.slot_side == MF_SLOT_SRC ? row * part.ss[2] : b * part.ss[0] + n * part.ss[2];
    const int64_t dst = p.slot_side == MF_SLOT_DST ? row * part.ds[2] : b * part.ds[0] + n * part.ds[2];
    const TS* s = static_cast<const TS*>(part.src) + so + lo * part.ss[1];
    TD* d = static_cast<TD*>(part.dst) + dst + lo * part.ds[1];
    if (some < 16) {
      for (int h = lo; h < hi; ++h, s += part.ss[1], d += part.ds[1]) copy_some(s + e0, d + e0, some, zero);
      continue;
    }
    for (int h = lo; h < hi; h += kHeads, s += kHeads * part.ss[1], d += kHeads * part.ds[1]) {
      Chunk<TS> a[kHeads], c[kHeads];
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        if (zero || h + i >= hi) {
          a[i].clear();
          c[i].clear();
        } else {
          a[i].load(s + i * part.ss[1] + e0);
          c[i].load(s + i * part.ss[1] + e1);
        }
      }
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        if (h + i >= hi) break;
        float x[8], y[8];
        a[i].unpack(x);
        c[i].unpack(y);
        if (turning && !zero) {
          if constexpr (INTERLEAVED) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float x0 = x[2 * j], x1 = x[2 * j + 1], y0 = y[2 * j], y1 = y[2 * j + 1];
              x[2 * j] = x0 * cs[j].x - x1 * cs[j].y;
              x[2 * j + 1] = x0 * cs[j].y + x1 * cs[j].x;
              y[2 * j] = y0 * cs[j + 4].x - y1 * cs[j + 4].y;
              y[2 * j + 1] = y0 * cs[j + 4].y + y1 * cs[j + 4].x;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float x0 = x[j], x1 = y[j];
              x[j] = x0 * cs[j].x - x1 * cs[j].y;
              y[j] = x0 * cs[j].y + x1 * cs[j].x;
            }
          }
        }
        Chunk<TD> o;
        o.pack(x);
        o.store(d + i * part.ds[1] + e0);
        o.pack(y);
        o.store(d + i * part.ds[1] + e1);
      }
    }
  }
}

// Heads too short for a thread's pieces (fewer than 8 pairs or 16 entries): one element at a time.
template <typename TS, typename TD>
__global__ void __launch_bounds__(kThreads) rotary_scalar_kernel(Params p) {
  __shared__ float2 table[kScalarTokens * 8];
  const unsigned g0 = blockIdx.x * unsigned(p.TT);  // below 2^31 tokens
  const unsigned nt = min(unsigned(p.TT), unsigned(p.B) * unsigned(p.N) - g0);
  const unsigned P = unsigned(p.R) >> 1, per = P / unsigned(p.axes);
  for (unsigned i = threadIdx.x; i < nt * P; i += kThreads) {
    const unsigned t = i / P, pr = i - t * P;
    const unsigned b = (g0 + t) / unsigned(p.N), n = g0 + t - b * unsigned(p.N);
    table[i] = turn_of(p, b * p.ps[0] + n * p.ps[1] + (pr / per) * p.ps[2], int(pr));
  }
  __syncthreads();
  const int h0 = blockIdx.y * p.HS, h1 = min(p.heads, h0 + p.HS);
  int base = 0;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    if (k >= p.nparts) break;
    const Part& part = p.part[k];
    const int lo = max(h0 - base, 0), hi = min(h1 - base, part.heads);
    base += part.heads;
    if (lo >= hi) continue;
    const unsigned D = unsigned(p.D), total = nt * unsigned(hi - lo) * D;
    for (unsigned i = threadIdx.x; i < total; i += kThreads) {
      const unsigned r = i / D, h = r / nt, t = r - h * nt;
      const int j = int(i - r * D);
      const unsigned g = g0 + t, b = g / unsigned(p.N), n = g - b * unsigned(p.N);
      const int64_t row = p.slot_side != MF_SLOT_NONE ? p.slot[g] : 0;
      const bool zero = p.slot_side == MF_SLOT_SRC && row < 0;
      if (p.slot_side == MF_SLOT_DST && row < 0) continue;
      const TS* s = static_cast<const TS*>(part.src) + (lo + h) * part.ss[1] +
                    (p.slot_side == MF_SLOT_SRC ? row * part.ss[2] : b * part.ss[0] + n * part.ss[2]);
      TD* d = static_cast<TD*>(part.dst) + (lo + h) * part.ds[1] +
              (p.slot_side == MF_SLOT_DST ? row * part.ds[2] : b * part.ds[0] + n * part.ds[2]);
      float y = zero ? 0.0f : Elem<TS>::to_f32(s[j]);
      if (part.turn && j < p.R && !zero) {
        const int Pi = int(P);
        const bool first = p.interleaved ? (j & 1) == 0 : j < Pi;
        const int other = p.interleaved ? (j ^ 1) : first ? j + Pi : j - Pi;
        const float2 c = table[t * P + (p.interleaved ? j >> 1 : first ? j : j - Pi)];
        const float o = Elem<TS>::to_f32(s[other]);
        y = y * c.x + o * (first ? -c.y : c.y);
      }
      d[j] = Elem<TD>::from_f32(y);
    }
  }
}

template <typename TS, typename TD>
void launch(bool pieces, dim3 grid, hipStream_t s, const Params& p) {
  if (!pieces) hipLaunchKernelGGL((rotary_scalar_kernel<TS, TD>), grid, dim3(kThreads), 0, s, p);
  else if (p.interleaved) hipLaunchKernelGGL((rotary_kernel<TS, TD, true>), grid, dim3(kThreads), 0, s, p);
  else hipLaunchKernelGGL((rotary_kernel<TS, TD, false>), grid, dim3(kThreads), 0, s, p);
}

template <typename TS>
void launch_to(int dst, bool pieces, dim3 grid, hipStream_t s, const Params& p) {
  switch (dst) {
    case MF_DTYPE_BF16: launch<TS, __bf16>(pieces, grid, s, p); break;
    case MF_DTYPE_F16: launch<TS, _Float16>(pieces, grid, s, p); break;
    default: launch<TS, float>(pieces, grid, s, p); break;
  }
}

bool valid_dtype(int d) { return d == MF_DTYPE_F32 || d == MF_DTYPE_F16 || d == MF_DTYPE_BF16; }

}  // namespace rot
}  // namespace mf

extern "C" int mf_rotary(const mf_rotary_args* a, void* stream) {
  using namespace mf;
  using namespace mf::rot;
  if (a == nullptr) return fail(MF_ERR_INVALID_ARGUMENT, "mf_rotary: args is NULL");
  if (a->parts < 1 || a->parts > 3) return fail(MF_ERR_INVALID_ARGUMENT, "mf_rotary: parts must be 1, 2 or 3");
  if (!a->positions || !a->frequencies)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_rotary: positions and frequencies must be non-NULL");
  if (a->batch < 0 || a->tokens < 0 || a->head_dim <= 0)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_rotary: sizes must be non-negative (head_dim positive)");
  if (a->head_dim > kMaxDim) return fail(MF_ERR_UNSUPPORTED, "mf_rotary: head_dim must be at most 256");
  if (a->axes < 1 || a->axes > 3) return fail(MF_ERR_INVALID_ARGUMENT, "mf_rotary: axes must be 1, 2 or 3");
  if (a->rotary_dim <= 0 || a->rotary_dim > a->head_dim || a->rotary_dim % (2 * a->axes) != 0)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_rotary: rotary_dim must be a positive multiple of 2 * axes, at most head_dim");
  if (!valid_dtype(a->src_dtype) || !valid_dtype(a->dst_dtype))
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_rotary: bad dtype");
  if (a->position_type < MF_POS_F32 || a->position_type > MF_POS_I64)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_rotary: bad position_type");
  if (a->slot_side < MF_SLOT_NONE || a->slot_side > MF_SLOT_DST)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_rotary: bad slot_side");
  if (a->slot_side != MF_SLOT_NONE && !a->slot)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_rotary: a slot_side needs a slot map");
  if (!std::isfinite(a->gain)) return fail(MF_ERR_INVALID_ARGUMENT, "mf_rotary: gain must be finite");
  Params p = {};
  int64_t heads = 0;
  for (int k = 0; k < a->parts; ++k) {
    if (!a->src[k] || !a->dst[k]) return fail(MF_ERR_INVALID_ARGUMENT, "mf_rotary: every part needs src and dst");
    if (a->heads[k] < 0) return fail(MF_ERR_INVALID_ARGUMENT, "mf_rotary: heads must be non-negative");
    Part& t = p.part[k];
    t.src = a->src[k];
    t.dst = a->dst[k];
    t.heads = a->heads[k];
    t.turn = a->turn[k];
    heads += t.heads;
    for (int i = 0; i < 3; ++i) {
      t.ss[i] = a->src_stride[k][i];
      t.ds[i] = a->dst_stride[k][i];
      if (t.ss[i] < 0 || t.ds[i] < 0) return fail(MF_ERR_INVALID_ARGUMENT, "mf_rotary: strides must be non-negative");
    }
  }
  const int64_t tokens = int64_t(a->batch) * a->tokens;
  if (heads * a->head_dim >= (1 << 24) || tokens >= (int64_t(1) << 31))
    return fail(MF_ERR_UNSUPPORTED, "mf_rotary: at most 2^24 elements a token and 2^31 tokens");
  if (tokens == 0 || heads == 0) return MF_OK;
  for (int i = 0; i < 3; ++i) p.ps[i] = a->position_stride[i];
  p.pos = a->positions;
  p.freq = a->frequencies;
  p.slot = a->slot;
  p.gain = a->gain;
  p.pos_type = a->position_type;
  p.slot_side = a->slot_side;
  p.axes = a->axes;
  p.inverse = a->inverse;
  p.nparts = a->parts;
  p.B = a->batch;
  p.N = a->tokens;
  p.D = a->head_dim;
  p.R = a->rotary_dim;
  p.interleaved = a->interleaved;
  p.heads = int(heads);
  const bool pieces = a->rotary_dim >= 16;
  p.turned = (a->rotary_dim / 2 + 7) / 8;
  p.units = p.turned + (a->head_dim - a->rotary_dim + 15) / 16;
  p.TT = pieces ? kThreads / p.units : kScalarTokens;
  // All heads in one workgroup, so that a token's angles are computed once; fewer while the grid would leave CUs
  // without work (a molecule of 19 atoms and 16 heads is one workgroup else), but not below the heads in flight.
  const int64_t blocks = (tokens + p.TT - 1) / p.TT;
  int64_t slices = std::max<int64_t>(1, std::min<int64_t>((heads + kHeads - 1) / kHeads, 1024 / blocks));
  p.HS = int((heads + slices - 1) / slices);
  slices = (heads + p.HS - 1) / p.HS;
  if (blocks * kThreads > 0xffffffffLL)  // threads of a launch
    return fail(MF_ERR_UNSUPPORTED, "mf_rotary: too many tokens for one launch");
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(slices));
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (a->src_dtype) {
    case MF_DTYPE_BF16: launch_to<__bf16>(a->dst_dtype, pieces, grid, s, p); break;
    case MF_DTYPE_F16: launch_to<_Float16>(a->dst_dtype, pieces, grid, s, p); break;
    default: launch_to<float>(a->dst_dtype, pieces, grid, s, p); break;
  }
  MF_HIP_CHECK(hipGetLastError());
  return MF_OK;
}
