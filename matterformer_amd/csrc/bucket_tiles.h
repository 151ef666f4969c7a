// What the kernels of attention with a bias by buckets share (bucket_attn.hip, bucket_attn_bwd.hip): 64-row tiles of a
// head in LDS, products of 32 x 32, and the table of the bias.
//
// A product has rows (keys or queries, from LDS) and columns (32 a wave, one a lane and its partner 32 lanes on, in
// registers): C = A B with A = 32 rows x 16, B = 16 x 32 columns a step (MFMA 32x32x16).  Lane l holds column l & 31 and
// the accumulators' rows 8 (t >> 2) + 4 half + (t & 3), t = 0 .. 15, half = l >> 5.  The rows are taken from LDS in an
// order in which these are the 16 rows 16 half + t of the block: then a lane's buckets are 16 consecutive bytes, its
// row statistics 16 consecutive words, and the accumulators 8 s .. 8 s + 7, rounded, are the B operand of step s of the
// second product, whose A operand (the tile transposed) is read by transposing reads in the same order.  Nothing goes
// through LDS between the two products.
#pragma once

#include "mf_common.h"

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float mf_f32x16;

namespace mf {
namespace bucket {

constexpr int kTile = 64;    // rows of a staged tile, and of a tile of the buckets' tables
constexpr int kMasked = 64;  // the bucket of a pair that is left out; up to 64 buckets count
constexpr int kPitch = 65;   // floats between the tables of two heads

template <typename T>
struct Mma32;
template <>
struct Mma32<__bf16> {
  __device__ static __forceinline__ mf_f32x16 mma(mf_bf16x8 a, mf_bf16x8 b, mf_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma32<_Float16> {
  __device__ static __forceinline__ mf_f32x16 mma(mf_f16x8 a, mf_f16x8 b, mf_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

__device__ __forceinline__ mf_f32x16 zeros16() {
  mf_f32x16 z;
#pragma unroll
  for (int t = 0; t < 16; ++t) z[t] = 0.0f;
  return z;
}

// The other half's value, and the larger and the sum of both, of a column's two lanes.
__device__ __forceinline__ float pair_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// All lanes' values joined, in every lane; none: what joins to nothing.  Six instructions that hand values from lane to lane,
// where shuffles go through LDS one after the other (a wave's sum: about 60 clocks instead of 800).
template <typename Join>
__device__ __forceinline__ int wave_join(int v, int none, Join join) {
  v = join(v, __builtin_amdgcn_update_dpp(none, v, 0x111, 0xf, 0xf, false));  // rows of 16 lanes: 1, 2, 4, 8 further on
  v = join(v, __builtin_amdgcn_update_dpp(none, v, 0x112, 0xf, 0xf, false));
  v = join(v, __builtin_amdgcn_update_dpp(none, v, 0x114, 0xf, 0xf, false));
  v = join(v, __builtin_amdgcn_update_dpp(none, v, 0x118, 0xf, 0xf, false));
  v = join(v, __builtin_amdgcn_update_dpp(none, v, 0x142, 0xa, 0xf, false));  // a row's last lane to the next row
  v = join(v, __builtin_amdgcn_update_dpp(none, v, 0x143, 0xc, 0xf, false));  // the first half's to the second
  return __builtin_amdgcn_readlane(v, 63);
}
__device__ __forceinline__ float wave_total(float v) {
  return __int_as_float(wave_join(__float_as_int(v), 0, [](int a, int b) {
    return __float_as_int(__int_as_float(a) + __int_as_float(b));
  }));
}
// Of values that are not negative.
__device__ __forceinline__ float wave_peak(float v) {
  return __int_as_float(wave_join(__float_as_int(v), 0, [](int a, int b) {
    return __float_as_int(fmaxf(__int_as_float(a), __int_as_float(b)));
  }));
}

// Row of a 32-row block that lane m of an A operand stands for.
__device__ __forceinline__ int block_row(int m) { return 16 * ((m >> 2) & 1) + 4 * (m >> 3) + (m & 3); }

// Chunk swizzle of a staged row of DP entries (16-byte chunks).  The 16 rows that an access of 16 lanes reads at one
// chunk (rows 0 - 7 and 16 - 23 of a block, or 8 - 15 and 24 - 31) fall on different banks, and so do the four rows by
// four chunks of two transposing reads.
template <int DP>
__device__ __forceinline__ int swz(int row) {
  const int b0 = row & 1, b1 = (row >> 1) & 1, b2 = (row >> 2) & 1, b4 = (row >> 4) & 1;
  if constexpr (DP == 128) return b0 << 2 | b1 << 3 | b2 | b4 << 1;
  else if constexpr (DP == 64) return b1 << 2 | b2 | b4 << 1;
  else return b2 | b4 << 1;
}

// Copies the rows of a 64-row tile (those in a set; the others and the entries past D become zeros) into LDS.  W waves take
// part; stride: bytes between rows.
template <int DP, int W>
struct TileCopy {
  static constexpr int CPR = DP / 8, kLoads = CPR / W;
  static_assert(kLoads >= 1, "a wave copies at least one chunk a lane");
  unsigned off[kLoads];  // of the lane's chunks from the tile's first row

  __device__ __forceinline__ TileCopy(unsigned stride, int D, int wave, int lane) { start(stride, D, wave, lane); }
  __device__ __forceinline__ void start(unsigned stride, int D, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int q = (wave * kLoads + i) * 64 + lane, row = q / CPR, chunk = (q % CPR) ^ swz<DP>(row);
      off[i] = chunk * 8 < D ? unsigned(row) * stride + unsigned(chunk) * 16 : kLdsCopyOutside;
    }
  }
  __device__ __forceinline__ void copy(const char* base, uint64_t set, char* lds, int wave, int lane) const {
    const mf_i32x4 src = lds_copy_source(base);
    if (set == ~uint64_t(0)) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) lds_copy16(src, off[i], lds + (wave * kLoads + i) * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row = ((wave * kLoads + i) * 64 + lane) / CPR;
        const uint32_t word = row & 32 ? uint32_t(set >> 32) : uint32_t(set);
        lds_copy16(src, (word >> (row & 31)) & 1 ? off[i] : kLdsCopyOutside, lds + (wave * kLoads + i) * 1024);
      }
    }
  }
};

// Where a lane reads a staged tile: byte offsets that 32-row blocks and eight-row steps shift by constants (the swizzle
// takes no part of them).
template <typename T, int DP>
struct LaneReads {
  using Op = typename Elem<T>::Operand;
  int row;     // A operand: row block_row(lane & 31), chunk half; chunk 2 kk + half lies at row ^ (kk << 5)
  int lo, hi;  // transposed: rows 16 half + e and 4 further, the lane's four entries; 32 nd entries on at ^ (nd << 6)

  __device__ __forceinline__ explicit LaneReads(int lane) {
    const int half = lane >> 5, g = (lane >> 4) & 1, e = (lane >> 2) & 3, a = lane & 3;
    const int r = block_row(lane & 31);
    row = r * (DP * 2) + ((half ^ swz<DP>(r)) << 4);
    const int t = 16 * half + e, chunk = 2 * (a & 1) + g, sub = (a >> 1) * 8;
    lo = t * (DP * 2) + ((chunk ^ swz<DP>(t)) << 4) + sub;
    hi = (t + 4) * (DP * 2) + ((chunk ^ swz<DP>(t + 4)) << 4) + sub;
  }
  // The same `bytes` further on (a multiple of 256).
  __device__ __forceinline__ LaneReads shifted(int bytes) const {
    LaneReads r = *this;
    r.row += bytes;
    r.lo += bytes;
    r.hi += bytes;
    return r;
  }
  // A operand of block kb: entries 16 kk + 8 half .. + 7 of the lane's row.
  __device__ __forceinline__ Op rows(const char* lds, int kb, int kk) const {
    return *reinterpret_cast<const Op*>(lds + (row ^ (kk << 5)) + kb * (32 * DP * 2));
  }
  // A operand of the transposed tile: output rows 32 nd .. + 31 (lane m: entry 32 nd + block_row(m)), inputs the rows
  // 32 kb + 16 half + 8 s .. + 7.
  __device__ __forceinline__ Op columns(const char* lds, int kb, int s, int nd) const {
    const int at = (32 * kb + 8 * s) * (DP * 2);
    return __builtin_shufflevector(read_tr16(reinterpret_cast<const T*>(lds + (lo ^ (nd << 6)) + at)),
                                   read_tr16(reinterpret_cast<const T*>(lds + (hi ^ (nd << 6)) + at)), 0, 1, 2, 3, 4, 5, 6,
                                   7);
  }
};

// The tiles of a row of sets from `first` on, below `end`, whose set is not empty, in order, with their sets; 64 tiles'
// sets at a time in the lanes.  A second row of sets (or null) is joined to the first.
struct Tiles {
  const uint64_t* a;
  const uint64_t* b;
  int at, end;
  uint64_t active, sets;

  __device__ __forceinline__ Tiles(const uint64_t* a_, const uint64_t* b_, int first, int end_)
      : a(a_), b(b_), at(first - 64), end(end_), active(0), sets(0) {}

  __device__ __forceinline__ bool next(int& tile, uint64_t& set) {
    while (active == 0) {
      at += 64;
      if (at >= end) return false;
      const int t = at + (threadIdx.x & 63);
      sets = t < end ? a[t] : 0;
      if (b != nullptr && t < end) sets |= b[t];
      active = __ballot(sets != 0);
    }
    const int l = __builtin_ctzll(active);
    active &= active - 1;
    tile = at + l;
    set = uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(sets)), l))) |
          uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(sets >> 32)), l))) << 32;
    return true;
  }
};

// Which of the 64 rows of tile `column` have a partner in the tiles first .. end - 1: the union down a column of a table
// whose rows are `pitch` apart.
__device__ __forceinline__ uint64_t union_of(const uint64_t* table, int pitch, int column, int first, int end) {
  uint64_t u = 0;
  for (int t = first + int(threadIdx.x & 63); t < end; t += 64) u |= table[int64_t(t) * pitch + column];
  auto either = [](int a, int b) { return a | b; };
  return uint64_t(uint32_t(wave_join(int(uint32_t(u)), 0, either))) |
         uint64_t(uint32_t(wave_join(int(uint32_t(u >> 32)), 0, either))) << 32;
}

// The bias tables of `heads` heads from `first` on, in log2 units: entries past the buckets are -inf, and a finite entry
// stays finite, so that the lowest value of a type masks as it does in a softmax over it alone.
__device__ __forceinline__ void load_tables(float* lds, const void* table, int dtype, int buckets, int all_heads,
                                            int first, int heads, int threads) {
  for (int n = threadIdx.x; n < heads * kPitch; n += threads) {
    const int h = n / kPitch, c = n - h * kPitch;
    float v = -INFINITY;
    if (c < buckets) {
      const int64_t at = int64_t(c) * all_heads + first + h;
      if (dtype == MF_DTYPE_F32) v = static_cast<const float*>(table)[at];
      else if (dtype == MF_DTYPE_BF16) v = float(static_cast<const __bf16*>(table)[at]);
      else v = float(static_cast<const _Float16*>(table)[at]);
      if (fabsf(v) < INFINITY) v = fminf(fmaxf(v * kLog2e, -3.4028234e38f), 3.4028234e38f);
    }
    lds[n] = v;
  }
}

// Byte t of 16.
__device__ __forceinline__ unsigned byte_of(const uint32_t (&w)[4], int t) { return (w[t >> 2] >> (8 * (t & 3))) & 255u; }

// Workgroups of a launch in an order in which those that follow one another run on one XCD.  grid: a multiple of 8.
__device__ __forceinline__ uint32_t xcd_order(unsigned block, unsigned grid) {
  return (block & 7) * (grid >> 3) + (block >> 3);
}

// A unit is a tile of columns of a head.  In the order of units, eight key heads (with their query heads) take the same
// tile before they take the next, fewer where an XCD's share is fewer: the units of an XCD stream few heads' rows, and
// the tiles past a padded batch's last atoms, which have nothing to do, come in runs instead of at every second place,
// which the hardware's dealing of workgroups to CUs would turn into idle ones (64 x 181 atoms, 44 on average: 20.6 and
// 33.6 us against 17.0 and 29.0).  Where the work grows with the tile (earlier keys only: queries; for keys it falls), the
// units with the most come first, and where an XCD's share is less than a key head's units, the tiles come in eight
// sequences, so that each share has some of all.
struct Unit {
  int64_t b;
  int head, tile;  // head: of `heads`, `inside` of them to a key head
};
__device__ __forceinline__ Unit unit_of(uint32_t id, uint32_t batch, uint32_t heads, uint32_t inside, uint32_t tiles,
                                        bool rising) {
  const uint32_t key_heads = heads / inside, groups = batch * key_heads;
  const uint32_t block = groups >= 64 ? 8 : groups >= 8 ? groups >> 3 : 1;
  const uint32_t first = id / (block * tiles * inside) * block;
  const uint32_t r = id - first * tiles * inside, per = min(block, groups - first) * inside;
  const uint32_t i = r / per, in_tile = r - i * per;
  uint32_t n = i;
  if (groups < 8 && tiles > 8) {  // `longer` sequences of q + 1 tiles, the others of q
    const uint32_t q = tiles >> 3, longer = tiles & 7;
    if (i < longer * (q + 1)) {
      n = i / (q + 1);
      n += (i - n * (q + 1)) * 8;
    } else {
      const uint32_t j = i - longer * (q + 1);
      n = j / q;
      n += longer + (j - n * q) * 8;
    }
  }
  const uint32_t in_block = in_tile / inside, group = first + in_block, b = group / key_heads;
  Unit u;
  u.tile = int(rising ? n : tiles - 1 - n);
  u.head = int((group - b * key_heads) * inside + in_tile - in_block * inside);
  u.b = b;
  return u;
}

}  // namespace bucket
}  // namespace mf
