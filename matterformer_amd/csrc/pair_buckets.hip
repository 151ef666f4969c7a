// Buckets of the pairs of a batch and the learned bias they give, on gfx950
// (mf_pair_buckets, mf_bucket_bias, mf_bucket_bias_bwd).
//
// pair_buckets_kernel: bucket(i, j) = how many of the rising edges are at or
// below the pair's value (a distance, an offset, a given number).  A workgroup
// writes a tile of 64 queries by 64 keys, a thread 16 keys of one query, and
// through LDS the same tile transposed, with the words that say which of its
// keys and queries have a pair at all.  Distances are compared as squares, in
// fp64 without contraction, so that the bucket is that of the exact distance of
// the fp32 coordinates but for the roundings of fp64.  Bound by the vector
// instructions of distances (8 cells of 1997 atoms: 24 us), by the writes of
// offsets, most of whose tiles have one bucket (2 x 8192^2 in both layouts, 268 MB: 67).
//
// bucket_bias_kernel: a thread reads the buckets of 16 bytes of bias once and
// writes them for every head; the tables lie in LDS, one bank a bucket.  Bound
// by its writes (4 x 12 planes of 1997^2 in bf16, 383 MB: 69 us).
//
// bucket_bias_bwd_kernel: sums by bucket without atomics between lanes.  Every
// lane keeps a sum per bucket of its own in LDS ([bucket][thread]: one bank a
// lane whatever the buckets), to which it adds in the order of its pairs; then
// the threads' sums are joined in a fixed order, and table_sum_kernel joins the
// workgroups' in fp64.  Two calls give identical bits.  A sum is read, added to
// and written: 9 clocks a wave, where an fp32 atomic of LDS takes 193.  Bound by
// the time that takes at the nine waves a CU that the sums leave room for (bf16,
// same planes: 140 us; fp32, twice the bytes, 150).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "bucket_tiles.h"

namespace mf {
namespace bucket {

constexpr int kThreads = 256;
// Of bucket_bias_bwd_kernel: 50 KB of sums at 64 buckets, three workgroups and nine waves a CU.  (256, two and eight: bias and
// gradient of 4 x 12 x 1997^2 in bf16 209 us instead of 207.)
constexpr int kSumThreads = 192;

// Bucket of a value: a table by the leading bits of its fp32 rounding (an order-preserving integer) gives how many edges
// lie in lower cells; those in the value's own cell, mostly none or one, are compared with it.  1024 cells over the
// edges' range: 157 an octave for distances of 0.1 to 9, where a count of 32 compares takes four times as long.
constexpr int kCells = 1024;
constexpr int64_t kCounts = (int64_t(1) << 32) - 64;  // tiles of a call: they are counted in 32 bits

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
  uint32_t first, tiles;  // workgroups before this launch's, and in all
  uint32_t per;           // of a batch entry
  uint32_t grid;          // of this launch
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
// With shift 0 (edges within 1024 steps of fp32) the distance of a value of the other sign passes 32 bits: it saturates, in one
// instruction.  (Clamping to the cells' bits first, with two scalar operands: two orders of 8192 places 1.5 us longer.)
__host__ __device__ __forceinline__ int cell_of(float x, int base, int shift) {
  const int c = __builtin_elementwise_sub_sat(ordered_bits(x) >> shift, base);
  return c < 0 ? 0 : c >= kCells ? kCells - 1 : c;
}

// The least and the greatest of a wave's values.
template <bool LEAST>
__device__ __forceinline__ int wave_end(int v) {
  return wave_join(v, LEAST ? INT32_MAX : INT32_MIN, [](int a, int b) { return LEAST ? min(a, b) : max(a, b); });
}

// 16 bytes: a code where the mask has a bit, kMasked where not.
__device__ __forceinline__ uint4 masked_codes(uint32_t mask, uint32_t code) {
  uint32_t w[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const uint32_t on = (((mask >> (4 * t)) & 15u) * 0x00204081u & 0x01010101u) * 255u;
    w[t] = (on & (code * 0x01010101u)) | (~on & 0x40404040u);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int SOURCE>
__global__ void __launch_bounds__(kThreads) pair_buckets_kernel(BucketParams p) {
  using Value = std::conditional_t<SOURCE == MF_BUCKETS_OFFSET, int64_t, double>;
  __shared__ __attribute__((aligned(16))) float s_pos[3][kTile];
  __shared__ Value s_edges[MF_MAX_BUCKETS];
  __shared__ uint32_t s_cells[kCells / 4];
  __shared__ int64_t s_off[SOURCE == MF_BUCKETS_OFFSET ? kTile : 1];
  __shared__ int s_off32[SOURCE == MF_BUCKETS_OFFSET ? kTile : 1];
  __shared__ uint8_t tile[kTile][kTile + 4];
  __shared__ uint64_t s_key[4], s_qry[4];
  // (asked for together: one by one, each waits for its own line of the arguments)
  asm volatile("" ::"s"(p.index), "s"(p.key_pos), "s"(p.TK), "s"(p.base), "s"(p.tiles), "s"(p.grid), "s"(p.key_any));
  uint32_t cells_in = 0;
  double edge_in = 0.0;
  if constexpr (SOURCE == MF_BUCKETS_DISTANCE || SOURCE == MF_BUCKETS_VALUE) {
    cells_in = reinterpret_cast<const uint32_t*>(p.cells)[threadIdx.x];
    edge_in = p.edges[threadIdx.x & (MF_MAX_BUCKETS - 1)];
  }
  const uint32_t id = xcd_order(blockIdx.x, p.grid) + p.first;
  if (id >= p.tiles) return;
  uint32_t qt, kt;
  int64_t b;
  if (p.symmetric) {
    const uint32_t entry = id / p.per, t = id - entry * p.per;
    b = entry;
    kt = uint32_t((sqrtf(8.0f * float(t) + 1.0f) - 1.0f) * 0.5f);  // (off by one at most)
    if (kt * (kt + 1) / 2 > t) --kt;
    if ((kt + 1) * (kt + 2) / 2 <= t) ++kt;
    qt = t - kt * (kt + 1) / 2;
  } else {
    // two tiles by two follow one another: together they write whole lines of both layouts (two orders of 8192 places: 67 us;
    // by rows 81, eight by one 73)
    const uint32_t entry = id / p.per, in_entry = id - entry * p.per;
    const uint32_t pair = in_entry / (2 * uint32_t(p.TK)), in_pair = in_entry - pair * 2 * uint32_t(p.TK);
    const uint32_t both = 2 * pair + 1 < uint32_t(p.TQ);
    kt = in_pair >> both;
    qt = 2 * pair + (in_pair & both);
    b = entry;
  }
  const int tid = threadIdx.x, r = tid >> 2, c0 = (tid & 3) * 16;
  const int lane = tid & 63, wave = tid >> 6;
  const int i = qt * kTile + r;
  const int64_t S = (int64_t(p.Nk) + 63) / 64 * 64, St = (int64_t(p.Nq) + 63) / 64 * 64;

  // which of the tile's keys and queries count: lane t's key and query t
  const int jl = kt * kTile + lane, il = qt * kTile + lane;
  uint8_t key_out = jl >= p.Nk, query_out = il >= p.Nq;
  if (p.key_pad != nullptr && jl < p.Nk) key_out = p.key_pad[b * p.Nk + jl];
  if (p.query_pad != nullptr && il < p.Nq) query_out = p.query_pad[b * p.Nq + il];
  // OFFSET: positions relative to the tile's first key; where all are within 2^29 their differences are formed in 32 bits,
  // and if the least and the greatest of those that count have one bucket the tile has no other
  int64_t qo = 0;
  int q32 = 0;
  bool near = true;
  uint64_t keys, queries;
  if constexpr (SOURCE == MF_BUCKETS_OFFSET) {
    const int64_t* kp = static_cast<const int64_t*>(p.key_pos) + b * p.key_step;
    const int64_t* qp = static_cast<const int64_t*>(p.query_pos) + b * p.query_step;
    const int64_t base = kp[kt * kTile], key = jl < p.Nk ? kp[jl] : base, query = il < p.Nq ? qp[il] : base;
    keys = __ballot(key_out == 0);
    queries = __ballot(query_out == 0);
    const int64_t dk = key - base, dq = query - base;
    constexpr int64_t kNear = int64_t(1) << 29;
    near = !__any(!(dk > -kNear && dk < kNear && dq > -kNear && dq < kNear));
    if (near) {
      const bool key_in = (keys >> lane) & 1, query_in = (queries >> lane) & 1;
      const int low = wave_end<true>(key_in ? int(dk) : INT32_MAX), high = wave_end<false>(key_in ? int(dk) : INT32_MIN);
      const int qlow = wave_end<true>(query_in ? int(dq) : INT32_MAX), qhigh = wave_end<false>(query_in ? int(dq) : INT32_MIN);
      const bool none = keys == 0 || queries == 0 || (p.causal && low - qhigh > 0);  // no pair
      int code = kMasked;
      bool whole = none;
      if (!none && !(p.causal && high - qlow > 0)) {
        // (one value for the wave: its cell and edges come by scalar loads)
        const int cell = __builtin_amdgcn_readfirstlane(cell_of(float(low - qhigh), p.base, p.shift));
        code = (reinterpret_cast<const uint32_t*>(p.cells)[cell >> 2] >> (8 * (cell & 3))) & 255;
        while (double(low - qhigh) >= p.edges[code]) ++code;  // (not past the NaN at the end)
        whole = !(double(high - qlow) >= p.edges[code]);
      }
      if (whole) {
        const uint32_t row = (queries >> r) & 1 ? uint32_t(keys >> c0) & 0xffffu : 0u;
        const uint32_t column = (keys >> r) & 1 ? uint32_t(queries >> c0) & 0xffffu : 0u;
        const int j = kt * kTile + r;
        if (i < p.Nq) *reinterpret_cast<uint4*>(p.index + (b * p.Nq + i) * S + kt * kTile + c0) = masked_codes(row, code);
        if (p.index_t && j < p.Nk)
          *reinterpret_cast<uint4*>(p.index_t + (b * p.Nk + j) * St + qt * kTile + c0) = masked_codes(column, code);
        if (tid == 0) {
          p.key_any[(b * p.TQ + qt) * p.TK + kt] = none ? 0 : keys;
          p.query_any[(b * p.TK + kt) * p.TQ + qt] = none ? 0 : queries;
        }
        return;
      }
    }
    if (wave == 0) {
      s_off[lane] = key;
      s_off32[lane] = int(dk);  // (read where near)
    }
    if (near) q32 = __shfl(int(dq), r, 64);
    else if (i < p.Nq) qo = qp[i];
  }
  if constexpr (SOURCE != MF_BUCKETS_INDEX) {
    if constexpr (SOURCE == MF_BUCKETS_OFFSET) {
      cells_in = reinterpret_cast<const uint32_t*>(p.cells)[tid];
      edge_in = p.edges[tid & (MF_MAX_BUCKETS - 1)];
    }
    s_cells[tid] = cells_in;
    if (tid < MF_MAX_BUCKETS) {
      if constexpr (SOURCE == MF_BUCKETS_OFFSET) s_edges[tid] = edge_in == edge_in ? int64_t(edge_in) : INT64_MAX;
      else s_edges[tid] = edge_in;
    }
  }
  if (SOURCE == MF_BUCKETS_DISTANCE && tid < 3 * kTile) {
    const int j = kt * kTile + tid / 3;
    s_pos[tid % 3][tid / 3] = j < p.Nk ? static_cast<const float*>(p.key_pos)[b * p.key_step + int64_t(kt) * (3 * kTile) + tid] : 0.0f;
  }
  double qx = 0.0, qy = 0.0, qz = 0.0;
  if (SOURCE == MF_BUCKETS_DISTANCE && i < p.Nq) {
    const float* c = static_cast<const float*>(p.query_pos) + b * p.query_step + int64_t(i) * 3;
    qx = c[0];
    qy = c[1];
    qz = c[2];
  }
  if constexpr (SOURCE != MF_BUCKETS_OFFSET) {
    keys = __ballot(key_out == 0);
    queries = __ballot(query_out == 0);
  }
  __syncthreads();
  uint32_t w[4] = {0x40404040u, 0x40404040u, 0x40404040u, 0x40404040u};  // kMasked
  const uint32_t mine = (queries >> r) & 1 ? uint32_t(keys >> c0) & 0xffffu : 0u;
  if (mine != 0) {
    w[0] = w[1] = w[2] = w[3] = 0;
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      const int j = kt * kTile + c0 + t;
      const bool in = (mine >> t) & 1;
      unsigned code = kMasked;
      if constexpr (SOURCE == MF_BUCKETS_INDEX) {
        const int v = in ? static_cast<const int32_t*>(p.values)[(b * p.Nq + i) * p.Nk + j] : -1;
        if (v >= 0 && v < p.buckets) code = unsigned(v);
      } else if constexpr (SOURCE == MF_BUCKETS_OFFSET) {
        bool on = in;
        unsigned n;
        if (near) {
          const int x = s_off32[c0 + t] - q32;
          on = on && !(p.causal && x > 0);
          n = reinterpret_cast<const uint8_t*>(s_cells)[cell_of(float(x), p.base, p.shift)];
          while (int64_t(x) >= s_edges[n]) ++n;  // (not past the greatest at the end)
        } else {
          const int64_t x = s_off[c0 + t] - qo;
          on = on && !(p.causal && x > 0);
          n = reinterpret_cast<const uint8_t*>(s_cells)[cell_of(float(x), p.base, p.shift)];
          while (n + 1 < unsigned(p.buckets) && x >= s_edges[n]) ++n;
        }
        if (on) code = n;
      } else {
        double x;
        bool on = in;
        if constexpr (SOURCE == MF_BUCKETS_DISTANCE) {
          const double dx = qx - s_pos[0][c0 + t], dy = qy - s_pos[1][c0 + t], dz = qz - s_pos[2][c0 + t];
          x = (dx * dx + dy * dy) + dz * dz;
        } else {
          x = in ? static_cast<const float*>(p.values)[(b * p.Nq + i) * p.Nk + j] : 0.0f;
        }
        on = on && !(p.cutoff >= 0.0 && x > p.cutoff);
        // (a NaN has the first cell and passes no edge; squares are their own order)
        const float low = fmaxf(float(x), SOURCE == MF_BUCKETS_DISTANCE ? 0.0f : -INFINITY);
        const int cell = SOURCE == MF_BUCKETS_DISTANCE
                             ? min(max((__float_as_int(low) >> p.shift) - p.base, 0), kCells - 1)
                             : cell_of(low, p.base, p.shift);
        unsigned n = reinterpret_cast<const uint8_t*>(s_cells)[cell];
        while (x >= s_edges[n]) ++n;  // (not past the NaN at the end)
        if (on) code = n;
      }
      w[t >> 2] |= code << (8 * (t & 3));
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
// Both kernels walk a plane (one batch entry and head, Nq Nk entries) in its flat order, so that their accesses to the bias
// are 16 bytes and aligned whatever Nk is: where Nk is odd, planes and rows start off 16 bytes, and accesses that cross
// such a boundary cost the memory pipeline twice (by rows, 4 x 12 x 1997^2 in bf16: bias 114 us instead of 71, its
// gradient 180 instead of 163).  The buckets' rows are padded, so a run of them may have to be put
// together from the ends of two rows.
struct BiasParams {
  const uint8_t* index;
  const void* table;
  void* bias;
  float* parts;        // gradient: [H, K, pieces]
  int64_t plane;       // Nq Nk
  int64_t index_step;  // from one batch entry's buckets to the next (0: shared)
  int64_t first;       // bias: this launch's first chunk of a plane
  int64_t chunks;      // of a plane; bias: those of this launch
  int64_t total;       // gradient: chunks of all batch entries
  int64_t piece;       // gradient: chunks of a workgroup
  uint32_t threads;    // bias: of this launch
  int first_b;         // bias: this launch's first batch entry
  int H, Nq, Nk, K, S, table_dtype;
  int head_step;       // bias: heads of a workgroup
  int pieces;
};

template <typename T>
__device__ __forceinline__ float load_one(const void* p, int64_t at) {
  return float(static_cast<const T*>(p)[at]);
}

template <int N>
struct __attribute__((packed, aligned(1))) Words {  // at any byte
  uint32_t v[N];
};

__device__ __forceinline__ int64_t divide(int64_t x, int64_t by) {
  if (((x | by) >> 32) == 0) return uint32_t(x) / uint32_t(by);
  return x / by;
}

// 4 N bytes from byte `by` < 4 N on of two runs of words.
__device__ __forceinline__ uint32_t pick(bool second, uint32_t a, uint32_t b) { return second ? b : a; }
template <int N>
__device__ __forceinline__ void bytes_from(const uint32_t (&lo)[N], const uint32_t (&hi)[N], int by, uint32_t (&w)[N]) {
  const bool two = by & 8, one = by & 4;
  if constexpr (N == 4) {
    const uint32_t u0 = pick(two, lo[0], lo[2]), u1 = pick(two, lo[1], lo[3]), u2 = pick(two, lo[2], hi[0]),
                   u3 = pick(two, lo[3], hi[1]), u4 = pick(two, hi[0], hi[2]), u5 = pick(two, hi[1], hi[3]);
    const uint32_t v0 = pick(one, u0, u1), v1 = pick(one, u1, u2), v2 = pick(one, u2, u3), v3 = pick(one, u3, u4),
                   v4 = pick(one, u4, u5);
    w[0] = __builtin_amdgcn_alignbyte(v1, v0, by & 3);
    w[1] = __builtin_amdgcn_alignbyte(v2, v1, by & 3);
    w[2] = __builtin_amdgcn_alignbyte(v3, v2, by & 3);
    w[3] = __builtin_amdgcn_alignbyte(v4, v3, by & 3);
  } else {
    const uint32_t v0 = pick(one, lo[0], lo[1]), v1 = pick(one, lo[1], hi[0]), v2 = pick(one, hi[0], hi[1]);
    w[0] = __builtin_amdgcn_alignbyte(v1, v0, by & 3);
    w[1] = __builtin_amdgcn_alignbyte(v2, v1, by & 3);
  }
}

// Buckets one by one from (row, col) on of a batch entry; places before its first row or past its last are masked.
template <int N>
__device__ __forceinline__ void few_codes(const BiasParams& p, const uint8_t* in, int64_t row, int col, uint32_t (&w)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) w[n] = 0;
#pragma unroll
  for (int t = 0; t < 4 * N; ++t) {
    const uint32_t code = col >= 0 && row < p.Nq ? in[row * p.S + col] : uint32_t(kMasked);
    w[t >> 2] |= code << (8 * (t & 3));
    if (++col == p.Nk) {
      col = 0;
      ++row;
    }
  }
}

// A thread writes 16 aligned bytes of bias of every head from one window of buckets: head h's entries begin where its plane
// is at a multiple of 16 bytes, V - 1 entries into the window at most.
template <typename T>
__global__ void __launch_bounds__(kThreads) bucket_bias_kernel(BiasParams p) {
  extern __shared__ uint32_t s_table[];  // [head_step][kPitch]: entries in the bias's type, the others' bits zero
  constexpr int V = 16 / sizeof(T), N = V / 2;
  using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
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
    s_table[n] = __builtin_bit_cast(Bits, static_cast<T>(v));
  }
  __syncthreads();
  const uint32_t id = blockIdx.x * uint32_t(kThreads) + threadIdx.x;
  if (id >= p.threads) return;
  const uint32_t bl = id / uint32_t(p.chunks);
  const int64_t b = p.first_b + int64_t(bl), n = p.first + (id - bl * uint32_t(p.chunks)), from = n * V;
  const int64_t row = divide(from, p.Nk);
  const int col = int(from - row * p.Nk);
  const uint8_t* in = p.index + b * p.index_step;
  uint32_t w[N] = {};
  if (p.Nk % V == 0) {  // (every plane begins at a multiple of 16 bytes: the first V)
    const uint8_t* at = in + row * p.S + col;
#pragma unroll
    for (int t = 0; t < V / 4; ++t) w[t] = reinterpret_cast<const uint32_t*>(at)[t];
  } else if (p.Nk >= 2 * V) {
    const int start = min(col, p.Nk - 2 * V);
    const Words<N> lo = *reinterpret_cast<const Words<N>*>(in + row * p.S + start);
    uint32_t a[N], z[N];
#pragma unroll
    for (int t = 0; t < N; ++t) {
      w[t] = a[t] = lo.v[t];
      z[t] = 0x40404040u;
    }
    if (col != start) {
      if (row + 1 < p.Nq) {
        const Words<N> hi = *reinterpret_cast<const Words<N>*>(in + (row + 1) * p.S);
#pragma unroll
        for (int t = 0; t < N; ++t) z[t] = hi.v[t];
      }
      bytes_from<N>(a, z, col - start, w);
    }
  } else {
    few_codes<N>(p, in, row, col, w);
  }
  const int left = int(min(p.plane - from, int64_t(2 * V)));
  Bits* out = static_cast<Bits*>(p.bias) + (b * p.H + h0) * p.plane;
  unsigned begin = unsigned(b * p.H + h0) * unsigned(p.plane);  // of the plane, modulo V
  for (int h = 0; h < heads; ++h, out += p.plane, begin += unsigned(p.plane)) {
    const uint32_t* table = s_table + h * kPitch;
    const int a = int(-begin & (V - 1));
    uint32_t x[4] = {}, y[V];
    if constexpr (V == 8) {
      const uint32_t u0 = a & 4 ? w[1] : w[0], u1 = a & 4 ? w[2] : w[1], u2 = a & 4 ? w[3] : w[2];
      x[0] = __builtin_amdgcn_alignbyte(u1, u0, a & 3);
      x[1] = __builtin_amdgcn_alignbyte(u2, u1, a & 3);
    } else {
      x[0] = __builtin_amdgcn_alignbyte(w[1], w[0], a);
    }
#pragma unroll
    for (int t = 0; t < V; ++t) y[t] = table[byte_of(x, t)];
    if (a + V <= left) {
      *reinterpret_cast<uint4*>(out + from + a) =
          V == 4 ? make_uint4(y[0], y[1], y[2], y[3])
                 : make_uint4(y[0] | y[1] << 16, y[2] | y[3] << 16, y[V - 4] | y[V - 3] << 16, y[V - 2] | y[V - 1] << 16);
    } else {
#pragma unroll
      for (int t = 0; t < V - 1; ++t)
        if (a + t < left) out[from + a + t] = Bits(y[t]);
    }
    if (n == 0 && a > 0) {  // the entries before the plane's first multiple
#pragma unroll
      for (int t = 0; t < V - 1; ++t)
        if (t < a && t < left) out[t] = Bits(table[(w[t >> 2] >> (8 * (t & 3))) & 255u]);
    }
  }
}

// A workgroup sums a piece of one head's chunks, a thread 16 entries at a time, the next ones loaded while the last ones are
// added.
template <typename T>
__global__ void __launch_bounds__(kSumThreads) bucket_bias_bwd_kernel(BiasParams p) {
  extern __shared__ float s_bins[];  // [K + 1][kSumThreads]; the last one takes the masked pairs
  constexpr int V = 16 / sizeof(T), kKeys = 16;
  using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
  auto value = [](const uint32_t* words, int t) {
    return float(__builtin_bit_cast(T, Bits(sizeof(T) == 4 ? words[t] : words[t >> 1] >> (16 * (t & 1)))));
  };
  const int tid = threadIdx.x;
  for (int c = 0; c <= p.K; ++c) s_bins[c * kSumThreads + tid] = 0.0f;
  const int h = blockIdx.y;
  float* bins = s_bins + tid;

  // a plane's chunks begin at multiples of 16 bytes, the first one before the plane where that does not
  const int64_t end = min(p.total, (blockIdx.x + int64_t(1)) * p.piece);
  int64_t id = blockIdx.x * p.piece + tid, b = 0, n = id, from = 0, row = 0;
  int col = 0;
  auto enter = [&] {  // chunk n, past this batch entry's or the first
    const int64_t more = divide(n, p.chunks);
    b += more;
    n -= more * p.chunks;
    const int a = int(-(unsigned(b * p.H + h) * unsigned(p.plane)) & (V - 1));
    from = n * kKeys + (a ? a - kKeys : 0);
    row = from < 0 ? 0 : divide(from, p.Nk);
    col = int(from - row * p.Nk);
  };
  const int rows_on = kSumThreads * kKeys / p.Nk, cols_on = kSumThreads * kKeys - rows_on * p.Nk;
  auto advance = [&] {
    id += kSumThreads;
    n += kSumThreads;
    if (n >= p.chunks) {
      enter();
    } else {
      from += kSumThreads * kKeys;
      row += rows_on;
      col += cols_on;
      if (col >= p.Nk) {
        col -= p.Nk;
        ++row;
      }
      while (col < 0) {  // (from the chunk before the plane)
        col += p.Nk;
        --row;
      }
    }
  };
  uint32_t lo[4], hi[4];
  int by = 0;
  uint32_t x[kKeys / V * 4];  // (as words: halves would be taken apart, and waited for, where they are loaded)
  auto load = [&] {
    const uint8_t* in = p.index + b * p.index_step;
    const T* values = static_cast<const T*>(p.bias) + (b * p.H + h) * p.plane + from;
    by = 0;
    if (from >= 0 && from + kKeys <= p.plane && p.Nk >= kKeys) {
      const int start = min(col, p.Nk - kKeys);
      const Words<4> one = *reinterpret_cast<const Words<4>*>(in + row * p.S + start);
#pragma unroll
      for (int t = 0; t < 4; ++t) lo[t] = one.v[t];
      by = col - start;
      if (by != 0) {
        const uint4 two = *reinterpret_cast<const uint4*>(in + (row + 1) * p.S);
        hi[0] = two.x;
        hi[1] = two.y;
        hi[2] = two.z;
        hi[3] = two.w;
      }
#pragma unroll
      for (int u = 0; u < kKeys / V; ++u) {
        const uint4 one = reinterpret_cast<const uint4*>(values)[u];
        x[4 * u] = one.x;
        x[4 * u + 1] = one.y;
        x[4 * u + 2] = one.z;
        x[4 * u + 3] = one.w;
      }
    } else {
      few_codes<4>(p, in, row, col, lo);
#pragma unroll
      for (int t = 0; t < kKeys; ++t) {
        const uint32_t bits =
            from + t >= 0 && from + t < p.plane ? reinterpret_cast<const Bits*>(values)[t] : Bits(0);
        if (sizeof(T) == 4 || t % 2 == 0) x[t * sizeof(T) / 4] = bits;
        else x[t * sizeof(T) / 4] |= bits << 16;
      }
    }
  };
  bool more = id < end;
  if (more) {
    enter();
    load();
  }
  while (more) {
    uint32_t w[4] = {lo[0], lo[1], lo[2], lo[3]};
    if (by != 0) bytes_from<4>(lo, hi, by, w);
    uint32_t y[kKeys / V * 4];
#pragma unroll
    for (int u = 0; u < kKeys / V * 4; ++u) y[u] = x[u];
    advance();
    more = id < end;
    if (more) load();
    // two at a time: where both have one bucket the first takes both and the second adds to the masked pairs' row
#pragma unroll
    for (int t = 0; t < kKeys; t += 2) {
      const int c0 = min(int(byte_of(w, t)), p.K), c1 = min(int(byte_of(w, t + 1)), p.K);
      const float v0 = value(y, t), v1 = value(y, t + 1);
      const bool same = c0 == c1;
      float* b0 = bins + c0 * kSumThreads;
      float* b1 = bins + (same ? p.K : c1) * kSumThreads;
      const float s0 = *b0, s1 = *b1;
      *b0 = s0 + (same ? v0 + v1 : v0);
      *b1 = s1 + v1;
    }
  }
  __syncthreads();
  for (int n = tid >> 6; n < p.K; n += kSumThreads / 64) {
    const float* s = s_bins + n * kSumThreads + (tid & 63);
    const float v = wave_total((s[0] + s[64]) + s[128]);
    if ((tid & 63) == 0) p.parts[(int64_t(h) * p.K + n) * p.pieces + blockIdx.x] = v;
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
  if (int64_t(a->batch) * a->queries >= (int64_t(1) << 31))
    return fail(MF_ERR_UNSUPPORTED, name + ": batch * queries too large");
  if (reinterpret_cast<uintptr_t>(a->index) % 16 != 0 || reinterpret_cast<uintptr_t>(a->bias) % 16 != 0)
    return fail(MF_ERR_INVALID_ARGUMENT, name + ": index and bias must be 16-byte aligned");
  return MF_OK;
}

BiasParams bias_params(const mf_bucket_bias_args* a) {
  BiasParams p = {};
  p.index = a->index;
  p.table = a->table;
  p.bias = a->bias;
  p.H = a->heads;
  p.Nq = a->queries;
  p.Nk = a->keys;
  p.K = a->buckets;
  p.S = (a->keys + 63) / 64 * 64;
  p.plane = int64_t(a->queries) * a->keys;
  p.index_step = a->index_batch == 1 ? 0 : int64_t(a->queries) * p.S;
  p.table_dtype = a->table_dtype;
  return p;
}

// The chunks of 16 entries of a head, and how many of them a workgroup sums: four a thread and more, and no more workgroups
// than are resident at three a CU (50 KB of LDS each) twice over.
void bias_pieces(const mf_bucket_bias_args* a, BiasParams& p) {
  const int V = a->bias_dtype == MF_DTYPE_F32 ? 4 : 8;
  p.plane = int64_t(a->queries) * a->keys;
  p.chunks = (p.plane + 15) / 16 + (p.plane % V != 0);
  p.total = p.chunks * a->batch;
  const int64_t pieces = std::max<int64_t>(1, std::min<int64_t>((p.total + 4 * kSumThreads - 1) / (4 * kSumThreads),
                                                                std::max(1, 1536 / std::max(1, a->heads))));
  p.piece = ((p.total + pieces - 1) / pieces + kSumThreads - 1) / kSumThreads * kSumThreads;
  p.pieces = int((p.total + p.piece - 1) / p.piece);
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
      if (a->source == MF_BUCKETS_OFFSET && a->edges[e] != std::floor(a->edges[e]))  // (tiles compare them as integers)
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_pair_buckets: edges of offsets must be whole numbers");
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
  const int64_t per = p.symmetric ? int64_t(p.TK) * (p.TK + 1) / 2 : int64_t(p.TQ) * p.TK;
  if (per >= (int64_t(1) << 30) || a->batch * per >= kCounts)  // (bytes past 2^42, and 80 a tile and more)
    return fail(MF_ERR_UNSUPPORTED, "mf_pair_buckets: batch * queries * keys too large");
  const int64_t tiles = a->batch * per;
  p.tiles = uint32_t(tiles);
  p.per = uint32_t(per);
  constexpr int64_t kMost = int64_t(1) << 23;  // workgroups of a launch
  for (int64_t first = 0; first < tiles; first += kMost) {
    p.first = uint32_t(first);
    p.grid = unsigned((std::min(kMost, tiles - first) + 7) / 8 * 8);
    const dim3 grid(p.grid);
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
  const int V = a->bias_dtype == MF_DTYPE_F32 ? 4 : 8;
  const int64_t chunks = (p.plane + V - 1) / V;
  // a workgroup takes all heads (one read of the index) unless that leaves less than eight workgroups a CU
  const int64_t all = (chunks * a->batch + kThreads - 1) / kThreads;
  const int parts = int(std::min<int64_t>(a->heads, std::max<int64_t>(1, (2048 + all - 1) / all)));
  p.head_step = (a->heads + parts - 1) / parts;
  const unsigned lds = unsigned(p.head_step * kPitch * sizeof(float));
  hipStream_t s = static_cast<hipStream_t>(stream);
  constexpr int64_t kMost = int64_t(1) << 30;  // threads of a launch: whole batch entries, or a part of one
  const int64_t entries = std::max<int64_t>(1, kMost / chunks);
  for (int64_t b = 0; b < a->batch; b += entries)
    for (p.first = 0; p.first < chunks; p.first += kMost) {
      p.first_b = int(b);
      p.chunks = std::min(kMost, chunks - p.first);
      p.threads = uint32_t(p.chunks * std::min(entries, a->batch - b));
      const dim3 grid((p.threads + kThreads - 1) / kThreads, unsigned((a->heads + p.head_step - 1) / p.head_step));
      if (a->bias_dtype == MF_DTYPE_F32) hipLaunchKernelGGL(bucket_bias_kernel<float>, grid, dim3(kThreads), lds, s, p);
      else if (a->bias_dtype == MF_DTYPE_BF16) hipLaunchKernelGGL(bucket_bias_kernel<__bf16>, grid, dim3(kThreads), lds, s, p);
      else hipLaunchKernelGGL(bucket_bias_kernel<_Float16>, grid, dim3(kThreads), lds, s, p);
      MF_HIP_CHECK(hipGetLastError());
    }
  return MF_OK;
}

extern "C" uint64_t mf_bucket_bias_bwd_workspace_size(const mf_bucket_bias_args* a) {
  if (a == nullptr || a->batch <= 0 || a->heads <= 0 || a->queries <= 0 || a->keys <= 0 || a->buckets <= 0) return 0;
  mf::bucket::BiasParams p = {};
  mf::bucket::bias_pieces(a, p);
  return uint64_t(a->heads) * a->buckets * p.pieces * sizeof(float);
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
  if (a->batch == 0 || a->queries == 0 || a->keys == 0) return launch_table_sum(nullptr, a->dtable, a->heads, a->buckets, 0, a->table_dtype, s);
  if (!a->workspace || a->workspace_bytes < mf_bucket_bias_bwd_workspace_size(a) ||
      reinterpret_cast<uintptr_t>(a->workspace) % 16 != 0)
    return fail(MF_ERR_INVALID_ARGUMENT, "mf_bucket_bias_bwd: the workspace must be 16-byte aligned and hold "
                                         "mf_bucket_bias_bwd_workspace_size bytes");
  bias_pieces(a, p);
  p.parts = static_cast<float*>(a->workspace);
  const dim3 grid(unsigned(p.pieces), unsigned(a->heads));
  const int lds = (a->buckets + 1) * kSumThreads * int(sizeof(float));
  const void* fn = a->bias_dtype == MF_DTYPE_F32    ? reinterpret_cast<const void*>(bucket_bias_bwd_kernel<float>)
                   : a->bias_dtype == MF_DTYPE_BF16 ? reinterpret_cast<const void*>(bucket_bias_bwd_kernel<__bf16>)
                                                    : reinterpret_cast<const void*>(bucket_bias_bwd_kernel<_Float16>);
  if (const int status = ensure_dynamic_lds(fn, (MF_MAX_BUCKETS + 1) * kSumThreads * int(sizeof(float)))) return status;
  if (a->bias_dtype == MF_DTYPE_F32)
    hipLaunchKernelGGL(bucket_bias_bwd_kernel<float>, grid, dim3(kSumThreads), lds, s, p);
  else if (a->bias_dtype == MF_DTYPE_BF16)
    hipLaunchKernelGGL(bucket_bias_bwd_kernel<__bf16>, grid, dim3(kSumThreads), lds, s, p);
  else
    hipLaunchKernelGGL(bucket_bias_bwd_kernel<_Float16>, grid, dim3(kSumThreads), lds, s, p);
  MF_HIP_CHECK(hipGetLastError());
  return launch_table_sum(p.parts, a->dtable, a->heads, a->buckets, p.pieces, a->table_dtype, s);
}
