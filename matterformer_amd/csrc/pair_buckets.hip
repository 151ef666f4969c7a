// Buckets of the pairs of a batch and the learned bias they give, on gfx950
// (mf_pair_buckets, mf_bucket_bias, mf_bucket_bias_bwd).
//
// pair_buckets_kernel: bucket(i, j) = how many of the rising edges are at or
// below the pair's value (a distance, an offset, a given number).  A workgroup
// writes a tile of 64 queries by 64 keys, a thread 16 keys of one query, and
// through LDS the same tile transposed, with the words that say which of its
// keys and queries have a pair at all.  Distances are compared as squares, in
// fp64 without contraction, so that the bucket is that of the exact distance of
// the fp32 coordinates but for the roundings of fp64.
//
// bucket_bias_kernel: a thread reads 16 buckets once and writes their biases for
// every head; the tables lie in LDS, one bank a bucket.  Bound by its writes.
//
// bucket_bias_bwd_kernel: sums by bucket without atomics between lanes.  Every
// lane keeps a sum per bucket of its own in LDS ([bucket][thread]: one bank a
// lane whatever the buckets), to which it adds in the order of its pairs; then
// the threads' sums are joined in a fixed order, and table_sum_kernel joins the
// workgroups' in fp64.  Two calls give identical bits.  Bound by reading dbias.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "bucket_tiles.h"

namespace mf {
namespace bucket {

constexpr int kThreads = 256;

// Bucket of a value: a table by the leading bits of its fp32 rounding (an order-preserving integer) gives how many edges
// lie in lower cells; those in the value's own cell, mostly none or one, are compared with it.  1024 cells over the
// edges' range: 157 an octave for distances of 0.1 to 9, where a count of 32 compares takes four times as long.
constexpr int kCells = 1024;

struct BucketParams {
  const void* query_pos;
  const void* key_pos;
  const void* values;
  const uint8_t* query_pad;
  const uint8_t* key_pad;
  uint8_t* index;
  uint8_t* index_t;
  uint64_t* key_any;
  uint64_t* query_any;
  int64_t query_step, key_step;
  double cutoff;
  int64_t first, tiles;  // workgroups before this launch's, and in all
  int symmetric;         // index_t is index: tiles on and above the diagonal, each written twice
  int buckets, causal, Nq, Nk, TQ, TK;
  int base, shift;
  double edges[MF_MAX_BUCKETS];  // the last one (behind num_edges) NaN
  uint8_t cells[kCells];
};

__host__ __device__ __forceinline__ int ordered_bits(float x) {
#ifdef __HIP_DEVICE_COMPILE__
  const int b = __float_as_int(x);
#else
  int b;
  __builtin_memcpy(&b, &x, 4);
#endif
  return b ^ ((b >> 31) & 0x7fffffff);
}
__host__ __device__ __forceinline__ int cell_of(float x, int base, int shift) {
  const int c = (ordered_bits(x) >> shift) - base;
  return c < 0 ? 0 : c >= kCells ? kCells - 1 : c;
}

template <int SOURCE>
__global__ void __launch_bounds__(kThreads) pair_buckets_kernel(BucketParams p) {
  using Value = std::conditional_t<SOURCE == MF_BUCKETS_OFFSET, int64_t, double>;
  __shared__ __attribute__((aligned(16))) float s_pos[3][kTile];
  __shared__ Value s_edges[MF_MAX_BUCKETS];
  __shared__ uint32_t s_cells[kCells / 4];
  __shared__ uint8_t tile[kTile][kTile + 4];
  __shared__ uint64_t s_key[4], s_qry[4];
  int64_t id = xcd_order(blockIdx.x, gridDim.x) + p.first;
  if (id >= p.tiles) return;
  int qt, kt;
  int64_t b;
  if (p.symmetric) {
    const int64_t per = int64_t(p.TK) * (p.TK + 1) / 2;
    b = id / per;
    const int64_t t = id - b * per;
    kt = int((sqrt(8.0 * double(t) + 1.0) - 1.0) * 0.5);
    while (int64_t(kt) * (kt + 1) / 2 > t) --kt;
    while (int64_t(kt + 1) * (kt + 2) / 2 <= t) ++kt;
    qt = int(t - int64_t(kt) * (kt + 1) / 2);
  } else {
    kt = int(id % p.TK);
    qt = int(id / p.TK % p.TQ);
    b = id / (int64_t(p.TK) * p.TQ);
  }
  const int tid = threadIdx.x, r = tid >> 2, c0 = (tid & 3) * 16;
  const int lane = tid & 63, wave = tid >> 6;
  const int i = qt * kTile + r;
  const int64_t S = (int64_t(p.Nk) + 63) / 64 * 64, St = (int64_t(p.Nq) + 63) / 64 * 64;

  if constexpr (SOURCE != MF_BUCKETS_INDEX) {
    s_cells[tid] = reinterpret_cast<const uint32_t*>(p.cells)[tid];
    if (tid < MF_MAX_BUCKETS) {
      const double e = p.edges[tid];
      if constexpr (SOURCE == MF_BUCKETS_OFFSET) s_edges[tid] = e == e ? int64_t(e) : INT64_MAX;
      else s_edges[tid] = e;
    }
  }
  if (SOURCE == MF_BUCKETS_DISTANCE && tid < 3 * kTile) {
    const int j = kt * kTile + tid / 3;
    s_pos[tid % 3][tid / 3] = j < p.Nk ? static_cast<const float*>(p.key_pos)[b * p.key_step + int64_t(kt) * (3 * kTile) + tid] : 0.0f;
  }
  const bool row_on = i < p.Nq && !(p.query_pad && p.query_pad[b * p.Nq + i]);
  // which of the tile's keys count: lane t's key t
  const int jl = kt * kTile + lane;
  const uint64_t keys = __ballot(jl < p.Nk && !(p.key_pad && p.key_pad[b * p.Nk + jl]));
  double qx = 0.0, qy = 0.0, qz = 0.0;
  int64_t qo = 0;
  if (i < p.Nq) {
    if constexpr (SOURCE == MF_BUCKETS_DISTANCE) {
      const float* c = static_cast<const float*>(p.query_pos) + b * p.query_step + int64_t(i) * 3;
      qx = c[0];
      qy = c[1];
      qz = c[2];
    } else if constexpr (SOURCE == MF_BUCKETS_OFFSET) {
      qo = static_cast<const int64_t*>(p.query_pos)[b * p.query_step + i];
    }
  }
  __syncthreads();
  uint32_t w[4] = {0x40404040u, 0x40404040u, 0x40404040u, 0x40404040u};  // kMasked
  const uint32_t mine = row_on ? uint32_t(keys >> c0) & 0xffffu : 0u;
  if (mine != 0) {
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      const int j = kt * kTile + c0 + t;
      const bool in = (mine >> t) & 1;
      unsigned code = kMasked;
      if constexpr (SOURCE == MF_BUCKETS_INDEX) {
        const int v = in ? static_cast<const int32_t*>(p.values)[(b * p.Nq + i) * p.Nk + j] : -1;
        if (v >= 0 && v < p.buckets) code = unsigned(v);
      } else {
        Value x;
        bool on = in;
        if constexpr (SOURCE == MF_BUCKETS_DISTANCE) {
          const double dx = qx - s_pos[0][c0 + t], dy = qy - s_pos[1][c0 + t], dz = qz - s_pos[2][c0 + t];
          x = (dx * dx + dy * dy) + dz * dz;
          on = on && !(p.cutoff >= 0.0 && x > p.cutoff);
        } else if constexpr (SOURCE == MF_BUCKETS_OFFSET) {
          x = (in ? static_cast<const int64_t*>(p.key_pos)[b * p.key_step + j] : 0) - qo;
          on = on && !(p.causal && x > 0);
        } else {
          x = in ? static_cast<const float*>(p.values)[(b * p.Nq + i) * p.Nk + j] : 0.0f;
          on = on && !(p.cutoff >= 0.0 && x > p.cutoff);
        }
        unsigned n = reinterpret_cast<const uint8_t*>(s_cells)[cell_of(float(x), p.base, p.shift)];
        if (x != x) n = 0;
        if constexpr (SOURCE == MF_BUCKETS_OFFSET) {
          while (n + 1 < unsigned(p.buckets) && x >= s_edges[n]) ++n;
        } else {
          while (x >= s_edges[n]) ++n;  // (not past the NaN at the end)
        }
        if (on) code = n;
      }
      w[t >> 2] = (w[t >> 2] & ~(255u << (8 * (t & 3)))) | code << (8 * (t & 3));
    }
  }
  const bool any = (w[0] & w[1] & w[2] & w[3]) != 0x40404040u;  // (a bucket has no bit 6)
#pragma unroll
  for (int t = 0; t < 4; ++t) *reinterpret_cast<uint32_t*>(&tile[r][c0 + 4 * t]) = w[t];
  if (i < p.Nq)
    *reinterpret_cast<uint4*>(p.index + (b * p.Nq + i) * S + kt * kTile + c0) = make_uint4(w[0], w[1], w[2], w[3]);
  __syncthreads();

  // the transposed tile: thread (key r, queries c0 ..)
  const int j = kt * kTile + r;
  uint32_t u[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int t = 0; t < 16; ++t) u[t >> 2] |= uint32_t(tile[c0 + t][r]) << (8 * (t & 3));
  const bool key_on = (u[0] & u[1] & u[2] & u[3]) != 0x40404040u;
  if (p.symmetric) {
    if (qt != kt && j < p.Nk)
      *reinterpret_cast<uint4*>(p.index + (b * p.Nk + j) * S + qt * kTile + c0) = make_uint4(u[0], u[1], u[2], u[3]);
  } else if (p.index_t && j < p.Nk) {
    *reinterpret_cast<uint4*>(p.index_t + (b * p.Nk + j) * St + qt * kTile + c0) = make_uint4(u[0], u[1], u[2], u[3]);
  }
  // bits 4 r' .. + 3 of a wave's ballot: the threads of row 16 wave + r'
  const uint64_t kb = __ballot(key_on), qb = __ballot(any);
  const bool kr = lane < 16 && ((kb >> (4 * lane)) & 15) != 0, qr = lane < 16 && ((qb >> (4 * lane)) & 15) != 0;
  const uint64_t km = __ballot(kr), qm = __ballot(qr);
  if (lane == 0) {
    s_key[wave] = km << (16 * wave);
    s_qry[wave] = qm << (16 * wave);
  }
  __syncthreads();
  if (tid == 0) {
    p.key_any[(b * p.TQ + qt) * p.TK + kt] = s_key[0] | s_key[1] | s_key[2] | s_key[3];
    // (symmetric: query_any is key_any, the other tile's word)
    if (!p.symmetric || qt != kt)
      p.query_any[(b * p.TK + kt) * p.TQ + qt] = s_qry[0] | s_qry[1] | s_qry[2] | s_qry[3];
  }
}

// -- the bias ----------------------------------------------------------------------------------------------------
struct BiasParams {
  const uint8_t* index;
  const void* table;
  void* bias;
  float* parts;        // gradient: [H, K, pieces]
  int64_t chunks;      // 16-key chunks of all rows
  int64_t rows_index;  // rows of the index (the rows of a batch of one, or all)
  int B, H, Nq, Nk, K, S, table_dtype;
  int head_step;       // heads of a workgroup
  int pieces;
};

template <typename T>
__device__ __forceinline__ float load_one(const void* p, int64_t at) {
  return float(static_cast<const T*>(p)[at]);
}

template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Wide {  // 16 bytes at any element
  T v[16 / sizeof(T)];
};

template <typename T>
__global__ void __launch_bounds__(kThreads) bucket_bias_kernel(BiasParams p) {
  extern __shared__ float s_table[];  // [head_step][kPitch]
  const int h0 = blockIdx.y * p.head_step, heads = min(p.head_step, p.H - h0);
  for (int n = threadIdx.x; n < heads * kPitch; n += kThreads) {
    const int h = n / kPitch, c = n - h * kPitch;
    float v = -INFINITY;
    if (c < p.K) {
      const int64_t at = int64_t(c) * p.H + h0 + h;
      v = p.table_dtype == MF_DTYPE_F32    ? load_one<float>(p.table, at)
          : p.table_dtype == MF_DTYPE_BF16 ? load_one<__bf16>(p.table, at)
                                           : load_one<_Float16>(p.table, at);
    }
    s_table[n] = v;
  }
  __syncthreads();
  const int64_t id = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (id >= p.chunks) return;
  const int per = (p.Nk + 15) / 16;
  const int64_t row = id / per;
  const int c = int(id - row * per), b = int(row / p.Nq), i = int(row - int64_t(b) * p.Nq);
  const uint4 packed = *reinterpret_cast<const uint4*>(p.index + (row % p.rows_index) * p.S + 16 * c);
  const uint32_t w[4] = {packed.x, packed.y, packed.z, packed.w};
  const int left = p.Nk - 16 * c;
  constexpr int V = 16 / sizeof(T);
  for (int h = 0; h < heads; ++h) {
    T* out = static_cast<T*>(p.bias) + ((int64_t(b) * p.H + h0 + h) * p.Nq + i) * p.Nk + 16 * c;
    const float* table = s_table + h * kPitch;
    if (left >= 16) {
#pragma unroll
      for (int u = 0; u < 16 / V; ++u) {
        Wide<T> x;
#pragma unroll
        for (int t = 0; t < V; ++t) x.v[t] = static_cast<T>(table[byte_of(w, V * u + t)]);
        *reinterpret_cast<Wide<T>*>(out + V * u) = x;
      }
    } else {
#pragma unroll
      for (int t = 0; t < 16; ++t)
        if (t < left) out[t] = static_cast<T>(table[byte_of(w, t)]);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) bucket_bias_bwd_kernel(BiasParams p) {
  extern __shared__ float s_bins[];  // [K + 1][kThreads]; the last one takes the masked pairs
  const int tid = threadIdx.x;
  for (int c = 0; c <= p.K; ++c) s_bins[c * kThreads + tid] = 0.0f;
  const int h = blockIdx.y;
  const int per = (p.Nk + 15) / 16;
  for (int64_t id = int64_t(blockIdx.x) * kThreads + tid; id < p.chunks; id += int64_t(p.pieces) * kThreads) {
    const int64_t row = id / per;
    const int c = int(id - row * per), b = int(row / p.Nq), i = int(row - int64_t(b) * p.Nq);
    const uint4 packed = *reinterpret_cast<const uint4*>(p.index + (row % p.rows_index) * p.S + 16 * c);
    const uint32_t w[4] = {packed.x, packed.y, packed.z, packed.w};
    const int left = p.Nk - 16 * c;
    const T* in = static_cast<const T*>(p.bias) + ((int64_t(b) * p.H + h) * p.Nq + i) * p.Nk + 16 * c;
    float x[16];
    if (left >= 16) {
      constexpr int V = 16 / sizeof(T);
#pragma unroll
      for (int u = 0; u < 16 / V; ++u) {
        const Wide<T> y = *reinterpret_cast<const Wide<T>*>(in + V * u);
#pragma unroll
        for (int t = 0; t < V; ++t) x[V * u + t] = float(y.v[t]);
      }
    } else {
#pragma unroll
      for (int t = 0; t < 16; ++t) x[t] = t < left ? float(in[t]) : 0.0f;
    }
#pragma unroll
    for (int t = 0; t < 16; ++t) s_bins[min(int(byte_of(w, t)), p.K) * kThreads + tid] += x[t];
  }
  __syncthreads();
  for (int c = tid >> 6; c < p.K; c += kThreads / 64) {
    const float* s = s_bins + c * kThreads + (tid & 63);
    const float v = wave_sum((s[0] + s[64]) + (s[128] + s[192]));
    if ((tid & 63) == 0) p.parts[(int64_t(h) * p.K + c) * p.pieces + blockIdx.x] = v;
  }
}

// dtable[c, h] from the pieces' sums [H, K, pieces], one workgroup each.
__global__ void __launch_bounds__(kThreads) table_sum_kernel(const float* parts, void* dtable, int H, int K, int pieces,
                                                             int dtype) {
  const int c = blockIdx.x % K, h = blockIdx.x / K;
  const float* in = parts + int64_t(blockIdx.x) * pieces;
  double v = 0.0;
  for (int n = threadIdx.x; n < pieces; n += kThreads) v += in[n];
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  __shared__ double s[4];
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    const float sum = float((s[0] + s[1]) + (s[2] + s[3]));
    const int64_t at = int64_t(c) * H + h;
    if (dtype == MF_DTYPE_F32) static_cast<float*>(dtable)[at] = sum;
    else if (dtype == MF_DTYPE_BF16) static_cast<__bf16*>(dtable)[at] = static_cast<__bf16>(sum);
    else static_cast<_Float16*>(dtable)[at] = static_cast<_Float16>(sum);
  }
}

int launch_table_sum(const float* parts, void* dtable, int heads, int buckets, int pieces, int dtype, hipStream_t s) {
  hipLaunchKernelGGL(table_sum_kernel, dim3(unsigned(heads * buckets)), dim3(kThreads), 0, s, parts, dtable, heads,
                     buckets, pieces, dtype);
  MF_HIP_CHECK(hipGetLastError());
  return MF_OK;
}

namespace {

bool dtype_ok(int d) { return d == MF_DTYPE_F32 || d == MF_DTYPE_F16 || d == MF_DTYPE_BF16; }

// 0, or the refusal of what the forward and the gradient share.
int check_bias(const mf_bucket_bias_args* a, const char* what) {
  const std::string name(what);
  if (a == nullptr) return fail(MF_ERR_INVALID_ARGUMENT, name + ": args is NULL");
  if (!a->index || !a->bias) return fail(MF_ERR_INVALID_ARGUMENT, name + ": index and bias must be non-NULL");
  if (a->batch < 0 || a->heads < 0 || a->queries < 0 || a->keys < 0)
    return fail(MF_ERR_INVALID_ARGUMENT, name + ": batch, heads, queries and keys must be non-negative");
  if (a->index_batch != 1 && a->index_batch != a->batch)
    return fail(MF_ERR_INVALID_ARGUMENT, name + ": index_batch must be 1 or batch");
  if (a->buckets < 1 || a->buckets > MF_MAX_BUCKETS)
    return fail(MF_ERR_UNSUPPORTED, name + ": buckets must be in [1, 64]");
  if (a->heads > 128) return fail(MF_ERR_UNSUPPORTED, name + ": heads must be <= 128");
  if (a->queries > (1 << 24) || a->keys > (1 << 24))
    return fail(MF_ERR_UNSUPPORTED, name + ": queries and keys must be <= 2^24");
  if (!dtype_ok(a->table_dtype) || !dtype_ok(a->bias_dtype))
    return fail(MF_ERR_UNSUPPORTED, name + ": only supports float32/float16/bfloat16");
  if (reinterpret_cast<uintptr_t>(a->index) % 16 != 0)
    return fail(MF_ERR_INVALID_ARGUMENT, name + ": index must be 16-byte aligned");
  return MF_OK;
}

BiasParams bias_params(const mf_bucket_bias_args* a) {
  BiasParams p = {};
  p.index = a->index;
  p.table = a->table;
  p.bias = a->bias;
  p.chunks = int64_t(a->batch) * a->queries * ((a->keys + 15) / 16);
  p.rows_index = int64_t(a->index_batch) * a->queries;
  p.B = a->batch;
  p.H = a->heads;
  p.Nq = a->queries;
  p.Nk = a->keys;
  p.K = a->buckets;
  p.S = (a->keys + 63) / 64 * 64;
  p.table_dtype = a->table_dtype;
  return p;
}

// Pieces a head's pairs are summed in: four chunks a thread and more, and no more workgroups than are resident at two a
// CU (66 KB of LDS each) twice over.
int bias_pieces(const mf_bucket_bias_args* a) {
  const int64_t chunks = int64_t(a->batch) * a->queries * ((a->keys + 15) / 16);
  return int(std::max<int64_t>(1, std::min<int64_t>((chunks + 4 * kThreads - 1) / (4 * kThreads),
                                                    std::max(1, 1024 / std::max(1, a->heads)))));
}

}  // namespace
}  // namespace bucket
}  // namespace mf

extern "C" int mf_pair_buckets(const mf_pair_buckets_args* a, void* stream) {
  using namespace mf;
  using namespace mf::bucket;
  if (a == nullptr) return fail(MF_ERR_INVALID_ARGUMENT, "mf_pair_buckets: args is NULL");
  if (a->source < MF_BUCKETS_DISTANCE || a->source > MF_BUCKETS_INDEX)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_pair_buckets: source must be one of MF_BUCKETS_*");
  const bool positions = a->source == MF_BUCKETS_DISTANCE || a->source == MF_BUCKETS_OFFSET;
  if (positions ? !a->query_pos || !a->key_pos : !a->values)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_pair_buckets: the source's positions or values must be non-NULL");
  if (!a->index || !a->key_any || !a->query_any)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_pair_buckets: index, key_any and query_any must be non-NULL");
  if (a->batch < 0 || a->queries < 0 || a->keys < 0)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_pair_buckets: batch, queries and keys must be non-negative");
  if ((a->index_t == a->index || a->query_any == a->key_any) &&
      (a->index_t != a->index || a->source != MF_BUCKETS_DISTANCE || a->query_pos != a->key_pos || a->query_pad != a->key_pad ||
       a->query_step != a->key_step || a->queries != a->keys || a->query_any != a->key_any))
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_pair_buckets: index_t may equal index for the distances of one set of atoms only");
  if (a->buckets < 1 || a->buckets > MF_MAX_BUCKETS)
    return fail(MF_ERR_UNSUPPORTED, "mf_pair_buckets: buckets must be in [1, 64]");
  if (a->source != MF_BUCKETS_INDEX) {
    if (a->num_edges != a->buckets - 1 || (a->num_edges > 0 && !a->edges))
      return fail(MF_ERR_INVALID_ARGUMENT, "mf_pair_buckets: edges must be buckets - 1 numbers");
    for (int e = 0; e < a->num_edges; ++e) {
      if (!std::isfinite(a->edges[e]) || (e > 0 && !(a->edges[e] > a->edges[e - 1])))
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_pair_buckets: edges must be finite and rise");
      if (a->source == MF_BUCKETS_DISTANCE && a->edges[e] < 0.0)
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_pair_buckets: edges of distances must not be negative");
      if (std::fabs(a->edges[e]) > (a->source == MF_BUCKETS_OFFSET ? 9007199254740992.0 : 3.5e38))
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_pair_buckets: edges out of range");
    }
  }
  if (std::isnan(a->cutoff)) return fail(MF_ERR_INVALID_ARGUMENT, "mf_pair_buckets: cutoff must not be NaN");
  if (a->queries > (1 << 24) || a->keys > (1 << 24))
    return fail(MF_ERR_UNSUPPORTED, "mf_pair_buckets: queries and keys must be <= 2^24");
  for (const void* ptr : {static_cast<const void*>(a->index), static_cast<const void*>(a->index_t)})
    if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0)
      return fail(MF_ERR_INVALID_ARGUMENT, "mf_pair_buckets: index and index_t must be 16-byte aligned");
  if (a->batch == 0 || a->queries == 0 || a->keys == 0) return MF_OK;
  BucketParams p = {};
  p.query_pos = a->query_pos;
  p.key_pos = a->key_pos;
  p.values = a->values;
  p.query_pad = a->query_pad;
  p.key_pad = a->key_pad;
  p.index = a->index;
  p.index_t = a->index_t;
  p.key_any = a->key_any;
  p.query_any = a->query_any;
  p.query_step = a->query_step;
  p.key_step = a->key_step;
  p.symmetric = a->index_t == a->index;
  p.buckets = a->buckets;
  p.causal = a->causal;
  p.Nq = a->queries;
  p.Nk = a->keys;
  p.TQ = (a->queries + kTile - 1) / kTile;
  p.TK = (a->keys + kTile - 1) / kTile;
  const bool squares = a->source == MF_BUCKETS_DISTANCE;
  const int num = a->source == MF_BUCKETS_INDEX ? 0 : a->num_edges;
  p.cutoff = a->cutoff < 0.0 ? -1.0 : squares ? a->cutoff * a->cutoff : a->cutoff;
  for (int e = 0; e < MF_MAX_BUCKETS; ++e)
    p.edges[e] = e >= num ? std::nan("") : squares ? a->edges[e] * a->edges[e] : a->edges[e];
  if (num > 0) {
    // (an edge whose square passes fp32 is in the cell of infinity, as the values there are)
    const int64_t low = ordered_bits(float(p.edges[0])), high = ordered_bits(float(p.edges[num - 1]));
    while (((high >> p.shift) - (low >> p.shift)) >= kCells) ++p.shift;
    p.base = int(low >> p.shift);
    for (int c = 0, e = 0; c < kCells; ++c) {
      while (e < num && cell_of(float(p.edges[e]), p.base, p.shift) < c) ++e;
      p.cells[c] = uint8_t(e);
    }
  }
  p.tiles = p.symmetric ? int64_t(a->batch) * p.TK * (p.TK + 1) / 2 : int64_t(a->batch) * p.TQ * p.TK;
  constexpr int64_t kMost = int64_t(1) << 23;  // workgroups of a launch
  for (p.first = 0; p.first < p.tiles; p.first += kMost) {
    const dim3 grid(unsigned((std::min(kMost, p.tiles - p.first) + 7) / 8 * 8));
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a->source == MF_BUCKETS_DISTANCE)
      hipLaunchKernelGGL(pair_buckets_kernel<MF_BUCKETS_DISTANCE>, grid, dim3(kThreads), 0, s, p);
    else if (a->source == MF_BUCKETS_OFFSET)
      hipLaunchKernelGGL(pair_buckets_kernel<MF_BUCKETS_OFFSET>, grid, dim3(kThreads), 0, s, p);
    else if (a->source == MF_BUCKETS_VALUE)
      hipLaunchKernelGGL(pair_buckets_kernel<MF_BUCKETS_VALUE>, grid, dim3(kThreads), 0, s, p);
    else
      hipLaunchKernelGGL(pair_buckets_kernel<MF_BUCKETS_INDEX>, grid, dim3(kThreads), 0, s, p);
    MF_HIP_CHECK(hipGetLastError());
  }
  return MF_OK;
}

extern "C" int mf_bucket_bias(const mf_bucket_bias_args* a, void* stream) {
  using namespace mf;
  using namespace mf::bucket;
  if (const int status = check_bias(a, "mf_bucket_bias")) return status;
  if (!a->table) return fail(MF_ERR_INVALID_ARGUMENT, "mf_bucket_bias: table must be non-NULL");
  if (a->batch == 0 || a->heads == 0 || a->queries == 0 || a->keys == 0) return MF_OK;
  BiasParams p = bias_params(a);
  const int64_t blocks = (p.chunks + kThreads - 1) / kThreads;
  if (blocks * kThreads > 0xffffffffLL) return fail(MF_ERR_UNSUPPORTED, "mf_bucket_bias: batch * queries * keys too large");
  // a workgroup takes all heads (one read of the index) unless that leaves less than eight workgroups a CU
  const int parts = int(std::min<int64_t>(a->heads, std::max<int64_t>(1, (2048 + blocks - 1) / blocks)));
  p.head_step = (a->heads + parts - 1) / parts;
  const dim3 grid(unsigned(blocks), unsigned((a->heads + p.head_step - 1) / p.head_step));
  const unsigned lds = unsigned(p.head_step * kPitch * sizeof(float));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->bias_dtype == MF_DTYPE_F32) hipLaunchKernelGGL(bucket_bias_kernel<float>, grid, dim3(kThreads), lds, s, p);
  else if (a->bias_dtype == MF_DTYPE_BF16) hipLaunchKernelGGL(bucket_bias_kernel<__bf16>, grid, dim3(kThreads), lds, s, p);
  else hipLaunchKernelGGL(bucket_bias_kernel<_Float16>, grid, dim3(kThreads), lds, s, p);
  MF_HIP_CHECK(hipGetLastError());
  return MF_OK;
}

extern "C" uint64_t mf_bucket_bias_bwd_workspace_size(const mf_bucket_bias_args* a) {
  if (a == nullptr || a->batch <= 0 || a->heads <= 0 || a->queries <= 0 || a->keys <= 0 || a->buckets <= 0) return 0;
  return uint64_t(a->heads) * a->buckets * mf::bucket::bias_pieces(a) * sizeof(float);
}

extern "C" int mf_bucket_bias_bwd(const mf_bucket_bias_args* a, void* stream) {
  using namespace mf;
  using namespace mf::bucket;
  if (const int status = check_bias(a, "mf_bucket_bias_bwd")) return status;
  if (!a->dtable) return fail(MF_ERR_INVALID_ARGUMENT, "mf_bucket_bias_bwd: dtable must be non-NULL");
  if (a->heads == 0) return MF_OK;
  BiasParams p = bias_params(a);
  hipStream_t s = static_cast<hipStream_t>(stream);
  // without a pair the sums are empty, and zero
  if (p.chunks == 0) return launch_table_sum(nullptr, a->dtable, a->heads, a->buckets, 0, a->table_dtype, s);
  if (!a->workspace || a->workspace_bytes < mf_bucket_bias_bwd_workspace_size(a) ||
      reinterpret_cast<uintptr_t>(a->workspace) % 16 != 0)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_bucket_bias_bwd: the workspace must be 16-byte aligned and hold "
                                         "mf_bucket_bias_bwd_workspace_size bytes");
  p.pieces = bias_pieces(a);
  p.parts = static_cast<float*>(a->workspace);
  const dim3 grid(unsigned(p.pieces), unsigned(a->heads));
  const int lds = (a->buckets + 1) * kThreads * int(sizeof(float));
  const void* fn = a->bias_dtype == MF_DTYPE_F32    ? reinterpret_cast<const void*>(bucket_bias_bwd_kernel<float>)
                   : a->bias_dtype == MF_DTYPE_BF16 ? reinterpret_cast<const void*>(bucket_bias_bwd_kernel<__bf16>)
                                                    : reinterpret_cast<const void*>(bucket_bias_bwd_kernel<_Float16>);
  if (const int status = ensure_dynamic_lds(fn, (MF_MAX_BUCKETS + 1) * kThreads * int(sizeof(float)))) return status;
  if (a->bias_dtype == MF_DTYPE_F32)
    hipLaunchKernelGGL(bucket_bias_bwd_kernel<float>, grid, dim3(kThreads), lds, s, p);
  else if (a->bias_dtype == MF_DTYPE_BF16)
    hipLaunchKernelGGL(bucket_bias_bwd_kernel<__bf16>, grid, dim3(kThreads), lds, s, p);
  else
    hipLaunchKernelGGL(bucket_bias_bwd_kernel<_Float16>, grid, dim3(kThreads), lds, s, p);
  MF_HIP_CHECK(hipGetLastError());
  return launch_table_sum(p.parts, a->dtable, a->heads, a->buckets, p.pieces, a->table_dtype, s);
}
