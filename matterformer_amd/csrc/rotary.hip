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
// (a position of 10^6 in fp32 would be off by 0.06 rad), then sincospi in fp32
// with the fraction's own rounding carried as a first-order correction.  They
// are computed once per token and pair into LDS and serve every head of every
// part.
//
// A workgroup takes TT tokens of a range of heads: at most 1024 chunks of 8
// consecutive elements, four a thread, all loaded before the first is used.
// With the half layout the partner of an element lies rotary_dim / 2 away, at
// any alignment, so the raw chunks go through LDS and partners are read there
// one by one; reading them from global memory costs eight 2-byte loads a chunk.
#include <algorithm>
#include <cmath>

#include "mf_common.h"

namespace mf {
namespace rot {

constexpr int kThreads = 256;
constexpr int kChunks = 4;                       // chunks of 8 elements per thread
constexpr int kBlockChunks = kThreads * kChunks;
constexpr int kMaxTokens = 16;                   // tokens per workgroup
constexpr int kMaxPairs = 128;                   // head_dim <= 256

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
};

// 8 consecutive elements in registers: one 16-byte load for 16-bit types, two for fp32.
template <typename T>
struct Chunk {
  static constexpr int kLoads = sizeof(T) / 2;
  uint4 u[kLoads];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) reinterpret_cast<uint4*>(p)[i] = u[i];
  }
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

// The workgroup's first token, and its others: a token is few steps behind it, so the molecule is found by counting on
// (a 64-bit division per chunk costs more than the rest of its arithmetic).
struct First {
  int b, n;
};
__device__ __forceinline__ First first_token(const Params& p, unsigned g0) {
  const unsigned b = g0 / unsigned(p.N);
  return {int(b), int(g0 - b * unsigned(p.N))};
}
__device__ __forceinline__ void token_at(const Params& p, First f, int t, int& b, int& n) {
  b = f.b;
  n = f.n + t;
  while (n >= p.N) {
    n -= p.N;
    ++b;
  }
}

// cos and sin (times gain) of every (token, pair) of the workgroup
__device__ __forceinline__ void fill_table(const Params& p, First f, int nt, float2* table) {
  const unsigned P = unsigned(p.R) >> 1, per = P / unsigned(p.axes);
  for (unsigned i = threadIdx.x; i < nt * P; i += kThreads) {
    const unsigned t = i / P, pr = i - t * P;
    int b, n;
    token_at(p, f, int(t), b, n);
    const double turns = position(p, b * p.ps[0] + n * p.ps[1] + (pr / per) * p.ps[2]) * p.freq[pr] *
                         0.15915494309189533577;
    const double half = 2.0 * (turns - rint(turns));  // the angle in units of pi, in [-1, 1]
    const float a = float(half);
    const float d = float(half - double(a)) * 3.14159265f;
    float s, c;
    sincospif(a, &s, &c);
    const float cc = c - d * s, sc = s + d * c;
    table[i] = make_float2(p.gain * cc, p.gain * (p.inverse ? -sc : sc));
  }
}

struct Where {
  const char* src;  // the head row, or null where the source has none
  char* dst;        // the head row, or null where the destination has none
  int t;            // token within the workgroup
  int turn;
};

__device__ __forceinline__ Where locate(const Params& p, First f, int t, int hh, int ssize, int dsize) {
  Where w;
  w.t = t;
  // the part by comparison: an index into the arguments would put them in scratch memory
  const bool one = hh >= p.part[0].heads;
  const bool two = p.nparts > 2 && hh >= p.part[0].heads + p.part[1].heads;
  const int h = hh - (one ? p.part[0].heads : 0) - (two ? p.part[1].heads : 0);
#define MF_PICK(field) (two ? p.part[2].field : one ? p.part[1].field : p.part[0].field)
  int b, n;
  token_at(p, f, t, b, n);
  int64_t so = b * MF_PICK(ss[0]) + n * MF_PICK(ss[2]);
  int64_t dst = b * MF_PICK(ds[0]) + n * MF_PICK(ds[2]);
  bool src_ok = true, dst_ok = true;
  if (p.slot_side != MF_SLOT_NONE) {
    const int64_t row = p.slot[int64_t(b) * p.N + n];
    if (p.slot_side == MF_SLOT_SRC) {
      src_ok = row >= 0;
      so = row * MF_PICK(ss[2]);
    } else {
      dst_ok = row >= 0;
      dst = row * MF_PICK(ds[2]);
    }
  }
  so += h * MF_PICK(ss[1]);
  dst += h * MF_PICK(ds[1]);
  w.src = src_ok ? static_cast<const char*>(MF_PICK(src)) + so * ssize : nullptr;
  w.dst = dst_ok ? static_cast<char*>(MF_PICK(dst)) + dst * dsize : nullptr;
  w.turn = MF_PICK(turn);
#undef MF_PICK
  return w;
}

// Rows of 16-byte aligned chunks of 8 elements.
template <typename TS, typename TD>
__global__ void __launch_bounds__(kThreads) rotary_kernel(Params p) {
  __shared__ float2 table[kMaxTokens * kMaxPairs];
  __shared__ __attribute__((aligned(16))) TS raw[kBlockChunks * 8];
  const unsigned g0 = blockIdx.x * unsigned(p.TT);  // below 2^31 tokens
  const int nt = min(p.TT, int(unsigned(p.B) * unsigned(p.N) - g0));
  const First first = first_token(p, g0);
  const int h0 = blockIdx.y * p.HS;
  const int nh = min(p.HS, p.heads - h0);
  const int DC = p.D >> 3;
  const int total = nt * nh * DC;
  const int rdc = (65536 + DC - 1) / DC, rnt = (65536 + nt - 1) / nt;
  Chunk<TS> v[kChunks];
  Where w[kChunks];
  int col[kChunks];
#pragma unroll
  for (int k = 0; k < kChunks; ++k) {
    const int i = threadIdx.x + k * kThreads;
    if (i >= total) continue;
    // i < 1024, DC <= 32, nt <= 16: the products with the reciprocals' ceilings below are exact quotients
    const int r = (i * rdc) >> 16;
    const int hh = (r * rnt) >> 16;
    col[k] = (i - r * DC) * 8;
    w[k] = locate(p, first, r - hh * nt, h0 + hh, sizeof(TS), sizeof(TD));
    if (w[k].src) v[k].load(reinterpret_cast<const TS*>(w[k].src) + col[k]);
    else v[k].clear();
  }
  fill_table(p, first, nt, table);
  if (!p.interleaved) {
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int i = threadIdx.x + k * kThreads;
      if (i < total) v[k].store(raw + i * 8);
    }
  }
  __syncthreads();
  const int P = p.R >> 1;
#pragma unroll
  for (int k = 0; k < kChunks; ++k) {
    const int i = threadIdx.x + k * kThreads;
    if (i >= total || !w[k].dst) continue;
    float x[8];
    v[k].unpack(x);
    if (w[k].turn && w[k].src) {
      const float2* cs = table + w[k].t * P;
      if (p.interleaved) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          if (col[k] + e < p.R) {
            const float2 c = cs[(col[k] + e) >> 1];
            const float a = x[e], b = x[e + 1];
            x[e] = a * c.x - b * c.y;
            x[e + 1] = a * c.y + b * c.x;
          }
        }
      } else {
        const TS* row = raw + (i * 8 - col[k]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = col[k] + e;
          if (j < p.R) {
            const bool first = j < P;
            const float2 c = cs[first ? j : j - P];
            const float o = Elem<TS>::to_f32(row[first ? j + P : j - P]);
            x[e] = x[e] * c.x + o * (first ? -c.y : c.y);
          }
        }
      }
    }
    Chunk<TD> o;
    o.pack(x);
    o.store(reinterpret_cast<TD*>(w[k].dst) + col[k]);
  }
}

// Any head_dim, strides and alignment: one element at a time.
template <typename TS, typename TD>
__global__ void __launch_bounds__(kThreads) rotary_scalar_kernel(Params p) {
  __shared__ float2 table[kMaxTokens * kMaxPairs];
  const unsigned g0 = blockIdx.x * unsigned(p.TT);  // below 2^31 tokens
  const int nt = min(p.TT, int(unsigned(p.B) * unsigned(p.N) - g0));
  const First first = first_token(p, g0);
  const int h0 = blockIdx.y * p.HS;
  const int nh = min(p.HS, p.heads - h0);
  const int total = nt * nh * p.D;
  fill_table(p, first, nt, table);
  __syncthreads();
  const int P = p.R >> 1;
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int r = i / p.D;
    const int hh = r / nt;
    const int j = i - r * p.D;
    const Where w = locate(p, first, r - hh * nt, h0 + hh, sizeof(TS), sizeof(TD));
    if (!w.dst) continue;
    const TS* src = reinterpret_cast<const TS*>(w.src);
    float y = src ? Elem<TS>::to_f32(src[j]) : 0.0f;
    if (w.turn && j < p.R && src) {
      const bool first = p.interleaved ? (j & 1) == 0 : j < P;
      const int other = p.interleaved ? (j ^ 1) : first ? j + P : j - P;
      const float2 c = table[w.t * P + (p.interleaved ? j >> 1 : first ? j : j - P)];
      const float o = Elem<TS>::to_f32(src[other]);
      y = y * c.x + o * (first ? -c.y : c.y);
    }
    reinterpret_cast<TD*>(w.dst)[j] = Elem<TD>::from_f32(y);
  }
}

template <typename TS, typename TD>
void launch(bool vec, dim3 grid, hipStream_t s, const Params& p) {
  if (vec) hipLaunchKernelGGL((rotary_kernel<TS, TD>), grid, dim3(kThreads), 0, s, p);
  else hipLaunchKernelGGL((rotary_scalar_kernel<TS, TD>), grid, dim3(kThreads), 0, s, p);
}

template <typename TS>
void launch_to(int dst, bool vec, dim3 grid, hipStream_t s, const Params& p) {
  switch (dst) {
    case MF_DTYPE_BF16: launch<TS, __bf16>(vec, grid, s, p); break;
    case MF_DTYPE_F16: launch<TS, _Float16>(vec, grid, s, p); break;
    default: launch<TS, float>(vec, grid, s, p); break;
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
  if (a->head_dim > 2 * kMaxPairs) return fail(MF_ERR_UNSUPPORTED, "mf_rotary: head_dim must be at most 256");
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
  const int ssize = a->src_dtype == MF_DTYPE_F32 ? 4 : 2, dsize = a->dst_dtype == MF_DTYPE_F32 ? 4 : 2;
  bool vec = a->head_dim % 8 == 0;
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
    vec = vec && reinterpret_cast<uintptr_t>(t.src) % 16 == 0 && reinterpret_cast<uintptr_t>(t.dst) % 16 == 0;
    for (int i = 0; i < 3; ++i) {
      t.ss[i] = a->src_stride[k][i];
      t.ds[i] = a->dst_stride[k][i];
      if (t.ss[i] < 0 || t.ds[i] < 0) return fail(MF_ERR_INVALID_ARGUMENT, "mf_rotary: strides must be non-negative");
      vec = vec && t.ss[i] * ssize % 16 == 0 && t.ds[i] * dsize % 16 == 0;
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
  // Heads per workgroup: all that fit with one token; tokens: what fills the
  // workgroup's chunks, fewer while the grid would leave CUs without work.
  const int dc = (a->head_dim + 7) / 8;
  p.HS = std::min(p.heads, kBlockChunks / dc);
  const int slices = (p.heads + p.HS - 1) / p.HS;
  p.HS = (p.heads + slices - 1) / slices;
  int tt = std::min(kMaxTokens, kBlockChunks / (dc * p.HS));
  while (tt > 1 && (tokens + tt - 1) / tt * slices < 512) tt = (tt + 1) / 2;
  p.TT = tt;
  const dim3 grid(unsigned((tokens + tt - 1) / tt), unsigned(slices));
  if (grid.y > 65535) return fail(MF_ERR_UNSUPPORTED, "mf_rotary: too many heads");
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (a->src_dtype) {
    case MF_DTYPE_BF16: launch_to<__bf16>(a->dst_dtype, vec, grid, s, p); break;
    case MF_DTYPE_F16: launch_to<_Float16>(a->dst_dtype, vec, grid, s, p); break;
    default: launch_to<float>(a->dst_dtype, vec, grid, s, p); break;
  }
  MF_HIP_CHECK(hipGetLastError());
  return MF_OK;
}
