// What the attention kernels share: the rows of a key head, tiles in LDS, the matrix products'
// operands and the masks.
//
// Rows.  The G = H / Hk query heads of a key head are one problem of R = Tq G rows, row r being
// query t = r / G of head hk G + r % G: a few tokens still fill a tile, and dK and dV sum over a
// group's heads in the order of the rows.
//
// Products.  All are formed as 32 x 32 tiles with the softmax's axis down the accumulator and the
// kernel's own row (forward, dQ) or key (dK, dV) across it, in v_mfma_f32_32x32x16_{bf16,f16} or
// v_mfma_f32_32x32x2_f32:
//
//   forward, dQ   S^T = K Q^T      O^T  += V^T P^T     dP^T = V dO^T    dQ^T += K^T dS^T
//   dK, dV        S   = Q K^T      dV^T += dO^T P      dP   = dO V^T    dK^T += Q^T dS
//
// so that lane l holds, for its own column l % 32, the 16 entries 8 (i / 4) + 4 (l / 32) + i % 4
// of the other axis: a row's statistics are a lane's scalars (joined once between lanes l and
// l + 32), and the exponentials are the next product's right operand where they lie.  That
// product sums over the axis in the order in which the lanes hold it: its left operand, read
// transposed from LDS, takes the same order.
//
// Tiles.  Rows of DP elements, copied from memory to LDS by the buffer unit; 16-byte vectors
// XOR-swizzled by row.  Rows past the end, columns past D and keys that the mask drops come from
// beyond the buffer's bound, as zeros, or their results are replaced, not multiplied away.
#pragma once

#include "gemm_core.h"

namespace nf {
namespace attn {

using gemm::bf16x8;
using gemm::floatx16;
using gemm::lds_ptr_t;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s *lds_v4s;

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr uint32_t kOob = 0x80000000u;
constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;

// A tensor [B, T, heads, D] of unit last stride; strides in bytes.
struct View {
  const char *p;
  int64_t b, t, h;
};

struct Shape {
  int B, Tq, Tk, H, Hk, G, D;
  int R;          // rows of a key head: Tq G
  int nvec;       // 16-byte vectors of a row that hold columns
  int off;        // causal: row t sees keys up to t + off = t + Tk - Tq
  int causal;
  uint32_t ginv;  // ceil(2^32 / G), 0 for G = 1
  float c;        // |scale| log2(e)
  float scale;
  uint32_t flip;  // scale < 0: the sign bits of one operand of S are flipped
  const uint8_t *mask;  // [B, Tk], bytes: the keys that may be attended (not 0); null: all
  int64_t mask_b;       // from sample to sample
};

// x / G for the small x of a tile
__device__ __forceinline__ int div_g(const Shape &s, int x) {
  return s.ginv ? (int)__umulhi((uint32_t)x, s.ginv) : x;
}

// Block -> (key head of a sample, tile).  Blocks go to the 8 XCDs in turn; the tiles of a head stay
// on 8 / gcd(heads, 8) of them, so that its keys and values are in few L2s, dealt in turn, so that
// the long and the short tiles of a causal call are spread evenly.  False: no tile for the block.
__device__ __forceinline__ bool place(int heads, int tiles, int *head, int *tile) {
  const int i = blockIdx.x, xcd = i & 7;
  const int low = heads & -heads, g = low < 8 ? low : 8;  // gcd(heads, 8)
  const int64_t s = (int64_t)(i >> 3) * (8 / g) + xcd / g;
  if (s >= (int64_t)(heads / g) * tiles) return false;
  *head = xcd % g + g * (int)(s / tiles);
  *tile = (int)(s % tiles);
  return true;
}
inline int64_t place_grid(int64_t heads, int64_t tiles) {
  const int64_t low = heads & -heads, g = low < 8 ? low : 8;
  return (heads / g * tiles + 8 / g - 1) / (8 / g) * 8;
}

// ---------------------------------------------------------------------------
// tiles
// ---------------------------------------------------------------------------
template <typename T, int DP>
struct Tile {
  static constexpr int ROW = DP * (int)sizeof(T);  // bytes
  static constexpr int NV = ROW / 16;              // vectors of a row: 4, 8, 12, 16 or 32
  static constexpr int KS = ROW / 32;              // steps of a product over a row
  static constexpr int NB = DP / 32;               // 32-wide column blocks
  static constexpr int VE = 16 / (int)sizeof(T);
  // The 16 rows that 16 lanes read at one vector, and the 4 rows that a transposing read of 16
  // lanes covers 32 bytes of, lie in different banks (64 of 4 bytes).
  __device__ __forceinline__ static int swz(int row) {
    if constexpr (NV == 8)  // two rows to a bank cycle
      return ((row >> 1) & 1) << 2 | ((row >> 2) & 1) << 1 | ((row >> 3) & 1);
    else if constexpr (NV == 4 || NV == 12)  // rows lie 1/4 or 3/4 of a bank cycle apart
      return (row >> 2) & 3;
    else
      return (row & 3) << 2 | ((row >> 2) & 3);
  }
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const char *p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(p), (short)0, 0x7fffffff, 0x00020000);
}

// The byte offsets at which a lane's copies of a tile of ROWS rows read, and the copies themselves:
// 1 KB of the tile each.
template <typename T, int DP, int ROWS>
struct TileCopy {
  using C = Tile<T, DP>;
  static constexpr int CW = ROWS * C::NV / kThreads;
  static_assert(CW >= 1 && ROWS * C::NV % kThreads == 0, "a tile is whole 1 KB copies a wavefront");
  uint32_t off[CW];
  // the lane's row in copy c
  __device__ __forceinline__ static int row_of(int wave, int c) {
    const int l = threadIdx.x & 63;
    if constexpr (64 % C::NV == 0)
      return (wave * CW + c) * (64 / C::NV) + l / C::NV;
    else
      return ((wave * CW + c) * 64 + l) / C::NV;
  }
  // `at(row, &in)`: a row's byte offset and whether it exists
  template <class F>
  __device__ __forceinline__ void set(int nvec, int wave, F &&at) {
    const int l = threadIdx.x & 63;
#pragma unroll
    for (int c = 0; c < CW; ++c) {
      const int row = row_of(wave, c);
      const int vec = ((wave * CW + c) * 64 + l - row * C::NV) ^ C::swz(row);
      bool in = true;
      const uint32_t o = at(row, &in) + (uint32_t)vec * 16u;
      off[c] = in && vec < nvec ? o : kOob;
    }
  }
  __device__ __forceinline__ void issue(const char *p, char *lds, int wave) const {
    const auto rsrc = buffer(p);
#pragma unroll
    for (int c = 0; c < CW; ++c)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)(lds + (wave * CW + c) * 1024), 16,
                                               off[c], 0, 0, 0);
  }
};

// ---------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ floatx16 mma(const u32x4 &a, const u32x4 &b, floatx16 acc) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[e]), __uint_as_float(b[e]), acc,
                                                 0, 0, 0);
    return acc;
  } else if constexpr (__is_same(T, bf16)) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
  }
}

// One step's left operand of mma_rows, and of mma_cols in 16 bits (step j: rows 16 (j / NB) .. + 15,
// column block j % NB), for products that are placed one by one.
template <typename T, int DP>
__device__ __forceinline__ u32x4 row_frag(const char *tile, int kb, int k) {
  using C = Tile<T, DP>;
  const int l = threadIdx.x & 63, h = l >> 5, row = l & 31;
  return *reinterpret_cast<const u32x4 *>(tile + (kb * 32 + row) * C::ROW +
                                          ((2 * k + h) ^ C::swz(row)) * 16);
}
// A transposing read: of each 16 lanes, lane a + 4 q addresses row q at columns 4 a .. 4 a + 3
// and lane i receives column i of the four rows.
template <typename T, int DP>
__device__ __forceinline__ u32x4 col_frag(const char *tile, int kb, int step) {
  using C = Tile<T, DP>;
  static_assert(sizeof(T) == 2, "16-bit elements");
  const int l = threadIdx.x & 63, h = l >> 5, j = l & 15;
  const int vec = 4 * (step % C::NB) + 2 * ((l >> 4) & 1) + ((j & 3) >> 1), in = (j & 1) * 8;
  const int ra = 16 * (step / C::NB) + 4 * h + (j >> 2), rb = ra + 8;
  const char *p = tile + kb * 32 * C::ROW + in;
  const v4s u = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (lds_v4s)(p + ra * C::ROW + ((vec ^ C::swz(ra)) << 4)));
  const v4s w = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (lds_v4s)(p + rb * C::ROW + ((vec ^ C::swz(rb)) << 4)));
  return __builtin_bit_cast(u32x4, __builtin_shufflevector(u, w, 0, 1, 2, 3, 4, 5, 6, 7));
}
// What comes before stays before: the order in which the source places reads, products and
// vector operations is the order in which they issue.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

// acc += rows 32 kb .. + 31 of the tile times the columns held in b (one row of DP elements a lane:
// vector 2 k + lane / 32 of it at step k).
template <typename T, int DP>
__device__ __forceinline__ void mma_rows(const char *tile, int kb,
                                         const u32x4 (&b)[Tile<T, DP>::KS], floatx16 &acc) {
  using C = Tile<T, DP>;
  const int l = threadIdx.x & 63, h = l >> 5, row = l & 31;
  const char *p = tile + (kb * 32 + row) * C::ROW;
  const int sw = C::swz(row);
#pragma unroll
  for (int k = 0; k < C::KS; ++k) {
    const u32x4 a = *reinterpret_cast<const u32x4 *>(p + ((2 * k + h) ^ sw) * 16);
    acc = mma<T>(a, b[k], acc);
  }
}

// The 16 values of a lane as the right operand over their axis: two vectors of 8 in 16 bits.
template <typename T>
struct Packed {
  u32x4 v[2];
  __device__ __forceinline__ void set(const floatx16 &x) {
    typedef T t8 __attribute__((ext_vector_type(8)));
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      t8 y;
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = static_cast<T>(x[8 * s + i]);
      v[s] = __builtin_bit_cast(u32x4, y);
    }
  }
};
template <>
struct Packed<float> {
  floatx16 v;
  __device__ __forceinline__ void set(const floatx16 &x) { v = x; }
};
// In two terms, the second what the first's rounding left: no rounding to 16 bits is then felt.
// For the calls with few rows, which no matrix product bounds and whose results are sums of few
// such terms.
template <typename T>
struct Twice {
  Packed<T> hi, lo;
  __device__ __forceinline__ void set(const floatx16 &x) {
    floatx16 y;
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = x[i] - to_f32(from_f32<T>(x[i]));
    hi.set(x);
    lo.set(y);
  }
};
template <>
struct Twice<float> {
  Packed<float> hi;
  __device__ __forceinline__ void set(const floatx16 &x) { hi.set(x); }
};

// acc[nb] += (columns 32 nb .. + 31 of rows 32 kb .. + 31 of the tile)^T x, over those rows in the
// order in which the lanes hold x.
template <typename T, int DP>
__device__ __forceinline__ void mma_cols(const char *tile, int kb, const Packed<T> &x,
                                         floatx16 (&acc)[Tile<T, DP>::NB]) {
  using C = Tile<T, DP>;
  const int l = threadIdx.x & 63, h = l >> 5;
  const char *p = tile + kb * 32 * C::ROW;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = 8 * (i / 4) + 4 * h + i % 4;
#pragma unroll
      for (int nb = 0; nb < C::NB; ++nb) {
        const int vec = (8 * nb + (l & 31) / 4) ^ C::swz(row);
        const float a = *reinterpret_cast<const float *>(p + row * C::ROW + vec * 16 + (l & 3) * 4);
        acc[nb] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, x.v[i], acc[nb], 0, 0, 0);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 2 * C::NB; ++j) {
      const u32x4 a = col_frag<T, DP>(tile, kb, j);
      acc[j % C::NB] = mma<T>(a, x.v[j / C::NB], acc[j % C::NB]);
    }
  }
}

template <typename T, int DP>
__device__ __forceinline__ void mma_cols(const char *tile, int kb, const Twice<T> &x,
                                         floatx16 (&acc)[Tile<T, DP>::NB]) {
  using C = Tile<T, DP>;
  if constexpr (sizeof(T) == 4) {
    mma_cols<T, DP>(tile, kb, x.hi, acc);
  } else {
#pragma unroll
    for (int j = 0; j < 2 * C::NB; ++j) {
      const u32x4 a = col_frag<T, DP>(tile, kb, j);
      floatx16 &to = acc[j % C::NB];
      to = mma<T>(a, x.lo.v[j / C::NB], to);
      to = mma<T>(a, x.hi.v[j / C::NB], to);
    }
  }
}

// A row of a tensor as mma_rows' right operand: zeros past the row's vectors, or for no row.
template <typename T, int DP>
__device__ __forceinline__ void load_row(const char *p, bool in, int nvec, uint32_t flip,
                                         u32x4 (&v)[Tile<T, DP>::KS]) {
  const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int k = 0; k < Tile<T, DP>::KS; ++k) {
    u32x4 x = {0u, 0u, 0u, 0u};
    if (in && 2 * k + h < nvec) x = *reinterpret_cast<const u32x4 *>(p + (2 * k + h) * 16);
    v[k] = x ^ flip;
  }
}

// ---------------------------------------------------------------------------
// lanes l and l + 32
// ---------------------------------------------------------------------------
__device__ __forceinline__ float pair_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ floatx16 splat(float x) {
  floatx16 v;
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = x;
  return v;
}

// The other axis's index of entry i of a lane, within 32.
__device__ __forceinline__ int entry(int i) {
  return 8 * (i / 4) + 4 * ((threadIdx.x & 63) >> 5) + i % 4;
}

// ---------------------------------------------------------------------------
// tiles of keys
// ---------------------------------------------------------------------------
// The mask of a sample in words of 64 keys, 64 words at a time: lane i holds word i of the chunk.
// A word is read by readlane, and the next one that has a key found in the lanes' ballot.
struct MaskWords {
  const uint8_t *p;  // the sample's bytes
  int keys;
  int chunk;      // the one that is held
  uint64_t mine;  // the lane's word
  uint64_t some;  // the words that have a key

  // not 0 for each byte, as 4 bits
  __device__ __forceinline__ static uint32_t four(uint32_t x) {
    x |= x >> 4;
    x |= x >> 2;
    x |= x >> 1;
    return ((x & 0x01010101u) * 0x01020408u) >> 24 & 15u;
  }
  __device__ __forceinline__ void load(int c) {
    const int l = threadIdx.x & 63;
    mine = 0;
    if (keys < 64) {
      const uint64_t all = __ballot(l < keys && p[min(l, keys - 1)] != 0);
      if (l == 0) mine = all;
    } else {
      const int64_t at = ((int64_t)c * 64 + l) * 64;
      const int64_t from = at + 64 <= keys ? at : keys - 64;  // the last word: the last 64 bytes
      if (at < keys) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          u32x4 x;
          __builtin_memcpy(&x, p + from + 16 * i, 16);
#pragma unroll
          for (int j = 0; j < 4; ++j) mine |= (uint64_t)four(x[j]) << (16 * i + 4 * j);
        }
        mine >>= at - from;
      }
    }
    some = __ballot(mine != 0);
    chunk = c;
  }
  __device__ __forceinline__ uint64_t word(int w) {
    if (w >> 6 != chunk) load(w >> 6);
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), w & 63) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)mine, w & 63);
  }
  // the first word from w on that has a key, or `end`
  __device__ __forceinline__ int next(int w, int end) {
    while (w < end) {
      if (w >> 6 != chunk) load(w >> 6);
      const uint64_t from = some >> (w & 63);
      if (from) return w + __builtin_ctzll(from);
      w = (w | 63) + 1;
    }
    return end;
  }
};

// The keys of 32 that a lane's row may attend: those up to `last` (of the 32; negative: none) whose
// bit is in `word`, shifted so that entry i is bit 8 (i / 4) + i % 4 for every lane.
__device__ __forceinline__ uint32_t live32(int last, uint32_t word) {
  const uint32_t upto = last < 0 ? 0u : last >= 31 ? ~0u : (2u << last) - 1u;
  return (upto & word) >> (4 * ((threadIdx.x & 63) >> 5));
}
// x where entry i is live, else `other`.
__device__ __forceinline__ float keep(float x, uint32_t live, int i, uint32_t other) {
  const uint32_t m = (uint32_t)((int32_t)(live << (31 - (8 * (i / 4) + i % 4))) >> 31);
  return __uint_as_float((__float_as_uint(x) & m) | (other & ~m));
}
constexpr uint32_t kMinusInf = 0xff800000u;

// ---------------------------------------------------------------------------
// work split along the summed axis
// ---------------------------------------------------------------------------
// A block's `len` tiles are cut every c, the last part being c / 2 to 1.5 c: blocks of the same part
// go over the same tiles at the same time, which their L2 then holds.
__host__ __device__ __forceinline__ int parts_of(int len, int c) {
  const int n = (int)(((int64_t)len + c / 2) / c);
  return n > 1 ? n : 1;
}
constexpr int kMostParts = 128;

// Tiles of keys that rows [tile br, + br) go over.
template <int TK>
__device__ __forceinline__ int key_tiles(const Shape &s, int tile, int br) {
  const int64_t stop = (int64_t)tile * br + br;
  const int rows_end = stop < s.R ? (int)stop : s.R;
  const int last = s.causal ? (rows_end - 1) / s.G + s.off : s.Tk - 1;
  return last < 0 ? 0 : last / TK + 1;
}
// The first tile of TR rows that sees a key of keys [tile bk, + bk).
template <int TR>
__device__ __forceinline__ int first_row_tile(const Shape &s, int tile, int bk) {
  const int end = (s.R + TR - 1) / TR;
  const int64_t from = s.causal ? (int64_t)tile * bk - s.off : 0;
  const int64_t at = from > 0 ? from * s.G / TR : 0;
  return at < end ? (int)at : end;
}

// The part length for `tiles` blocks a head of up to `longest` tiles each, `slots` blocks at once on
// the chip.  Blocks of one length go in rounds: as many parts as take the least time, in tiles a
// block 1.5 beside its own, the join 4 and 1.2 for each part that a slot writes and reads.  A causal
// call's blocks fall from the longest to few and fill up what it leaves: two parts a slot (delta, dK
// and dV of 2 x 4096 tokens, 16 heads on 4 of 128: 366 us, in 3 parts a slot 392, in 4 409, in 8 461).
inline int part_length(int64_t heads, int64_t tiles, int64_t longest, bool causal, int slots) {
  const int64_t blocks = heads * tiles;
  if (blocks >= 4 * (int64_t)slots) return 1 << 28;
  if (causal && tiles > 1) {
    const int64_t c = (blocks * longest / 2 + 2 * slots) / (2 * slots);
    const int64_t least = c > 4 ? c : 4, most = (longest + kMostParts - 1) / kMostParts;
    return (int)(least > most ? least : most);
  }
  int best = 1 << 28;
  double time = 0.;
  for (int n = 1; n <= kMostParts && n <= longest; ++n) {
    const int64_t c = (longest + n - 1) / n, rounds = (blocks * n + slots - 1) / slots;
    const double t = (double)rounds * ((double)c + 1.5) +
                     (n > 1 ? 4. + 1.2 * n * (double)blocks / slots : 0.);
    if (n > 1 && t >= time) continue;
    time = t;
    best = n == 1 ? 1 << 28 : (int)c;
  }
  return best;
}

// A key head's keys and values, tile by tile of TK, into LDS: K, then V.  MASKED: with the sample's
// mask words; tiles without a key are passed over.
template <typename T, int DP, int TK, bool MASKED>
struct KeyTiles {
  static constexpr int TILE = TK * Tile<T, DP>::ROW;
  static constexpr int N = MASKED ? (TK + 63) / 64 : 0;
  struct Bits {
    uint64_t w[N ? N : 1];
    // the 32 of them from key 32 i of the tile
    __device__ __forceinline__ uint32_t half(int i) const {
      if constexpr (!MASKED) return ~0u;
      uint64_t x = w[0];
      if constexpr (N == 2) x = i >= 2 ? w[1] : w[0];
      return (uint32_t)(x >> (32 * (i & 1)));
    }
    __device__ __forceinline__ bool all() const {
      if constexpr (!MASKED) return true;
      uint64_t x = w[0];
      if constexpr (N == 2) x &= w[1];
      return (TK == 32 ? x | ~0xffffffffull : x) == ~0ull;
    }
  };
  using Copy = TileCopy<T, DP, TK>;
  const Shape &s;
  const char *k, *v;
  int64_t kt, vt;  // bytes from key to key
  MaskWords mask;
  int end;  // the first tile that is not wanted
  int wave;
  Copy kc, vc;  // of a whole tile

  __device__ __forceinline__ KeyTiles(const Shape &s_, const View &kv, const View &vv, int b,
                                      int hk, int end_, int wave_)
      : s(s_), k(kv.p + b * kv.b + hk * kv.h), v(vv.p + b * vv.b + hk * vv.h), kt(kv.t), vt(vv.t),
        end(end_), wave(wave_) {
    if constexpr (MASKED) {
      mask.p = s.mask + b * s.mask_b;
      mask.keys = s.Tk;
      mask.chunk = -1;
    }
    kc.set(s.nvec, wave, [&](int row, bool *) { return (uint32_t)row * (uint32_t)kt; });
    vc.set(s.nvec, wave, [&](int row, bool *) { return (uint32_t)row * (uint32_t)vt; });
  }

  // the first tile from i on that has keys, and its bits
  __device__ __forceinline__ int seek(int i, Bits &x) {
    if constexpr (MASKED) {
      const int stop = (s.Tk + 63) / 64;  // words
      if constexpr (TK == 32) {
        while (i < end) {
          const int w = mask.next(i >> 1, stop);
          if (w >= stop) return end;
          if (i < 2 * w) i = 2 * w;
          x.w[0] = mask.word(w) >> (32 * (i & 1)) & 0xffffffffull;
          if (x.w[0]) break;
          ++i;
        }
      } else {
        const int w = mask.next(i * N, stop);
        if (w >= stop) return end;
        i = w / N;
        if (i < end) {
#pragma unroll
          for (int j = 0; j < N; ++j) x.w[j] = i * N + j < stop ? mask.word(i * N + j) : 0ull;
        }
      }
      if (i > end) i = end;
    }
    return i;
  }
  // zero: the keys that the mask drops arrive as zeros; without, as they lie, for an operand of a
  // product whose results for them are replaced
  __device__ __forceinline__ void copy_one(const char *p, int64_t step, const Copy &whole, int i,
                                           const Bits &x, char *lds, bool zero) const {
    const int left = s.Tk - i * TK;
    const char *at = p + (int64_t)i * TK * step;
    if (left >= TK && (!(MASKED && zero) || x.all())) return whole.issue(at, lds, wave);
    Copy c = whole;
    if constexpr (64 % Tile<T, DP>::NV == 0) {
      constexpr int PER = 64 / Tile<T, DP>::NV, ROWS = Copy::CW * PER;  // rows of a copy, a wavefront
      static_assert(ROWS <= 32, "a wavefront's rows are in one half of a word");
      const int row0 = Copy::row_of(wave, 0);
      uint32_t live = ~0u;
      if (MASKED && zero) {
        uint64_t w = x.w[0];
        if constexpr (N == 2) w = wave >= kWaves / 2 ? x.w[1] : x.w[0];
        live = (uint32_t)(w >> (row0 & 63));
      }
      const int rows = left - row0;  // from the lane's first on
      if (rows < 32) live &= rows > 0 ? (1u << rows) - 1u : 0u;
#pragma unroll
      for (int j = 0; j < Copy::CW; ++j)
        if (!(live & (1u << (j * PER)))) c.off[j] = kOob;
    } else {
#pragma unroll
      for (int j = 0; j < Copy::CW; ++j) {
        const int row = Copy::row_of(wave, j);
        bool in = row < left;
        if (MASKED && zero) {
          uint64_t w = x.w[0];
          if constexpr (N == 2) w = row >= 64 ? x.w[1] : x.w[0];
          in = in && (w >> (row & 63) & 1);
        }
        if (!in) c.off[j] = kOob;
      }
    }
    c.issue(at, lds, wave);
  }
  __device__ __forceinline__ void copy_k(int i, const Bits &x, char *lds, bool zero) const {
    copy_one(k, kt, kc, i, x, lds, zero);
  }
  __device__ __forceinline__ void copy_v(int i, const Bits &x, char *lds, bool zero) const {
    copy_one(v, vt, vc, i, x, lds + TILE, zero);
  }
};

// A key head's rows of q or dout, tile by tile of TR, into LDS; those before `first` and past the
// last arrive as zeros.
template <typename T, int DP, int TR>
struct RowTiles {
  using Copy = TileCopy<T, DP, TR>;
  const Shape &s;
  const char *p;
  int64_t t, h;  // bytes from token to token, head to head
  int wave, first;
  // the tiles that begin with a token's first row and have every row
  int whole_from;
  uint32_t whole_count;
  Copy whole;

  __device__ __forceinline__ RowTiles(const Shape &s_, const View &v, int b, int hk, int wave_,
                                      int first_)
      : s(s_), p(v.p + b * v.b + (int64_t)hk * s_.G * v.h), t(v.t), h(v.h), wave(wave_),
        first(first_), whole_from((first_ + TR - 1) / TR),
        whole_count(TR % s_.G == 0 ? (uint32_t)max(s_.R / TR - whole_from, 0) : 0u) {
    set(whole, 0, 0, TR);
  }
  __device__ __forceinline__ void set(Copy &c, int g0, int from, int to) const {
    c.set(s.nvec, wave, [&](int row, bool *in) {
      *in = row >= from && row < to;
      const int x = g0 + row, dt = div_g(s, x), g = x - dt * s.G;
      return (uint32_t)dt * (uint32_t)t + (uint32_t)g * (uint32_t)h;
    });
  }
  __device__ __forceinline__ void copy(int tile, char *lds) const {
    const int row0 = tile * TR, t0 = row0 / s.G;
    const char *at = p + (int64_t)t0 * t;
    if ((uint32_t)(tile - whole_from) < whole_count) return whole.issue(at, lds, wave);
    Copy c;
    set(c, row0 - t0 * s.G, first - row0, s.R - row0);
    c.issue(at, lds, wave);
  }
};

// ---------------------------------------------------------------------------
// results
// ---------------------------------------------------------------------------
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Accumulated columns through LDS, so that memory is written a row at a time: a wavefront's 32 rows
// of DP floats, 16-byte vectors XOR-swizzled by row.
template <int DP>
struct Turned {
  static constexpr int BYTES = 32 * DP * 4;
  static constexpr int V = DP / 4;  // vectors of a row
  __device__ __forceinline__ static int at(int row, int v) {
    return row * DP * 4 + ((v ^ (row & (V % 16 == 0 ? V - 1 : 7) & 31)) << 4);
  }
  __device__ __forceinline__ static void put(char *lds, const floatx16 (&acc)[DP / 32], float f) {
    const int row = threadIdx.x & 31;
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        f32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = acc[n][4 * e4 + i] * f;
        *reinterpret_cast<f32x4 *>(lds + at(row, (32 * n + entry(4 * e4)) / 4)) = x;
      }
  }
  __device__ __forceinline__ static f32x4 get(const char *lds, int row, int v) {
    return *reinterpret_cast<const f32x4 *>(lds + at(row, v));
  }
};

// Columns d .. d + 3 of a row p of D elements.
template <typename T>
__device__ __forceinline__ void store_quad(T *p, int d, int D, const f32x4 &v) {
  if (d + 4 <= D) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = from_f32<T>(v[i]);
    __builtin_memcpy(p + d, &x, sizeof(x));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < D) p[d + i] = from_f32<T>(v[i]);
  }
}

// What other lanes of the wavefront wrote to LDS before this is seen after it, and what they read
// before it is not overwritten by what comes after.  A wavefront's LDS operations go in order, so it
// is no instruction (the forward's code is the same with it; dK and dV of 2 x 4096 rows, 16 heads of
// 128: 582 us without and with); but without it nothing holds the compiler to that order.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// A wavefront's 32 rows (KW = 1), or a block's 32 rows in four parts that are summed (KW = 4; barriers
// around it are the caller's), as `put` left them: each vector to store(row, column, values).
template <int DP, int KW, class F>
__device__ __forceinline__ void each_vector(const char *smem, int wave, F &&store) {
  using U = Turned<DP>;
  constexpr int PER = KW == 4 ? kThreads : 64;
  const int first = KW == 4 ? (int)threadIdx.x : (int)(threadIdx.x & 63);
  if (KW == 1) wave_order();
#pragma unroll
  for (int i = 0; i < 32 * U::V / PER; ++i) {
    const int x = i * PER + first, row = x / U::V, v = x % U::V;
    f32x4 y;
    if constexpr (KW == 4)
      y = ((U::get(smem, row, v) + U::get(smem + U::BYTES, row, v)) +
           U::get(smem + 2 * U::BYTES, row, v)) + U::get(smem + 3 * U::BYTES, row, v);
    else
      y = U::get(smem + wave * U::BYTES, row, v);
    store(row, 4 * v, y);
  }
  if (KW == 1) wave_order();  // the next `put` goes to the same place
}

// a lane's 64-bit value, from every lane
__device__ __forceinline__ int64_t from_lane(int64_t x, int lane) {
  const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)x, lane);
  return (int64_t)__shfl((int)(x >> 32), lane) << 32 | lo;
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
struct Sizes {  // what a call is about, as its entry points take it
  int64_t B, Tq, Tk, H, Hk, D;
  int dtype;
  int es() const { return dtype == NF_DTYPE_F32 ? 4 : 2; }
  int64_t rows() const { return Tq * (H / Hk); }
  // columns of a tile; fp32 rows of 96 would not swizzle
  int dp() const {
    return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 && dtype != NF_DTYPE_F32 ? 96 : 128;
  }
};
// NF_OK, or the error that is set
int check_sizes(const char *op, const Sizes &z);
int make_view(const char *op, const char *name, const void *p, int64_t sb, int64_t st, int64_t sh,
              const Sizes &z, int64_t group, View *v);
Shape make_shape(const Sizes &z, int causal, float scale, const uint8_t *mask, int64_t mask_b);

struct FwdArgs {
  Shape s;
  View q, k, v;
  char *out;     // [B, Tq, H, D]
  char *low;     // what out's rounding left, the same layout; null: not kept
  float *lse;    // [B Hk, R] in powers of two; null: not kept
  float *part;   // rows in parts: O [most][B Hk R][DP], then (m, l) pairs
  int length, most, tiles;  // parts of about `length` tiles, at most `most`
};

struct BwdArgs {
  Shape s;
  View q, k, v, dout;
  const char *out, *low;
  const float *lse;
  float *ndelta;  // [B Hk, R]: -delta
  char *dq, *dk, *dv;
  // rows, or keys, in parts: dQ [most][B Hk R][DP], dK and dV [most][B Hk Tk][2][DP]
  float *part;
  int tiles, length, most;
};

struct Plan {
  int kw, tiles, length, most;
  size_t bytes;  // of the parts
};
Plan fwd_plan(const Sizes &z, bool causal);
Plan dq_plan(const Sizes &z, bool causal);
Plan dkv_plan(const Sizes &z, bool causal);
// one translation unit for each type has their kernels
template <typename T>
int launch_fwd(const FwdArgs &a, const Sizes &z, hipStream_t st);
template <typename T>
int launch_bwd(const BwdArgs &a, const Sizes &z, hipStream_t st);

// The state's parts, in bytes from its start: log-sum-exps, what out's rounding left.
struct State {
  size_t low, total;
};
State state_of(const Sizes &z);
// Whether the wavefronts of a block share its 32 rows (or keys) and split the other axis: `own` rows
// or keys a head.  Wavefronts with 32 of their own read a tile once for 128; where the blocks of
// 128 are fewer than fill the chip, four times the blocks are the faster.
bool shared_blocks(const Sizes &z, int64_t own);

}  // namespace attn
}  // namespace nf
