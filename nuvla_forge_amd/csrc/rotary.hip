// Rotary positions over several axes: pair j of every head of q and k turns by
// pos[token, axis(j)] * freq(j).
//
// A block takes a few tokens of a sample, forms their cosines and sines once (P a token) in LDS,
// and turns every head with them.  Angles are kept in turns: the product of position and frequency
// and its fraction in 64 bits, so that angles of up to about 2^27 turns lose nothing (in 32 bits a
// position of 10^6 would be off by 0.06 radians; in 64, farther ones by 2^-52 of theirs), then sine and cosine of the fraction in 32 bits.  The frequencies
// come as kernel arguments, made in 64 bits on the host: no table in memory, no upload.
//
// A thread turns two pieces of 16 bytes at a time, one in each half of a head, at any alignment, with
// the lanes of a head side by side in both: the two elements of a pair where those lie half a head
// apart, two runs of pairs where they are neighbours.  Pieces of 8 elements, alone where
// neighbours pair, took 136 us (now 133: halves, the shape below), 153 (131: neighbours) and 143
// (126: fp32, 32768 tokens).
//
// What bounds it: memory (bf16, 20 heads of 128, 65536 tokens: 133 us, 5.06 TB/s, neighbours paired
// 131; fp32 at half the tokens 126, 5.3; a copy of 1 GiB runs at 5.10).  Rows that are no whole cache
// lines reach less: 3.1 TB/s at 12 heads of 123, 3.4 at 100.
#include <math.h>

#include "nf_device.h"

namespace nf {
namespace {

constexpr int kBlock = 256;
constexpr int kMaxPairs = 256, kMaxAxes = 4;
constexpr int kTable = 2048;  // (cos, sin) pairs of a block: 16 KB
// Stores take the non-temporal hint where a launch reads and writes more than the Infinity Cache
// holds: bf16, 20 heads of 128, 65536 tokens (671 MB) 141.8 us plain, 135.1 hinted, 32768 74.1 and
// 55.7; 16384 (168 MB) 30.6 and 30.4, where the attention that follows finds them cached.
constexpr int64_t kNtMinBytes = (int64_t)256 << 20;

struct RotaryArgs {
  const void *x[2];  // q, k (k may be absent: heads[1] = 0)
  void *out[2];      // [B, T, heads, D]
  int64_t sb[2], st[2], sh[2];
  int heads[2];
  int T, D, P, axes, tiles, tokens;  // tokens of a block
  int chunks, turned;                // items of a head, of those turned
  uint32_t heads_inv;                // ceil(2^32 / heads), 0: one
  const void *pos;                   // [B or 1, T, axes]
  int64_t pos_b;                     // elements between samples, 0: shared
  int pos_kind;                      // 0 int64, 1 int32, 2 fp32
  float sign;
  int first[kMaxAxes];               // an axis's first pair
  double turns[kMaxPairs];           // frequency / 2 pi
};

// 16 bytes at any alignment, or the first of them.  The sums below are written as fmaf, not left to
// the compiler: an element that two pieces share comes out alike in both.
template <typename T>
struct Piece {
  static constexpr int kSize = 16 / (int)sizeof(T);
  T v[kSize];
  __device__ __forceinline__ void load(const T *p, int valid) {
    if (valid >= kSize) {
      __builtin_memcpy(v, p, 16);
    } else {
#pragma unroll
      for (int i = 0; i < kSize; ++i) v[i] = i < valid ? p[i] : static_cast<T>(0.f);
    }
  }
  template <bool NT>
  __device__ __forceinline__ void store(T *p, int valid) const {
    if (valid >= kSize) {
      u32x4 a;
      __builtin_memcpy(&a, v, 16);
      u32x4_any *q = reinterpret_cast<u32x4_any *>(p);
      if constexpr (NT)
        __builtin_nontemporal_store(a, q);
      else
        *q = a;
    } else {
#pragma unroll
      for (int i = 0; i < kSize; ++i)
        if (i < valid) p[i] = v[i];
    }
  }
};

template <typename T>
__device__ __forceinline__ void turn_neighbours(Piece<T> &u, const float *cs, const float *sn) {
  constexpr int H = Piece<T>::kSize / 2;
  float c[H], s[H];
  __builtin_memcpy(c, cs, sizeof(c));
  __builtin_memcpy(s, sn, sizeof(s));
#pragma unroll
  for (int k = 0; k < H; ++k) {
    const float e = to_f32(u.v[2 * k]), f = to_f32(u.v[2 * k + 1]);
    u.v[2 * k] = from_f32<T>(fmaf(e, c[k], -(f * s[k])));
    u.v[2 * k + 1] = from_f32<T>(fmaf(e, s[k], f * c[k]));
  }
}

template <typename T, bool INTER, bool NT>
__global__ __launch_bounds__(kBlock) void rotary_kernel(RotaryArgs a) {
  constexpr int E = Piece<T>::kSize;
  __shared__ __attribute__((aligned(16))) float cs[kTable], sn[kTable];
  const int b = blockIdx.x / a.tiles, t0 = (blockIdx.x - b * a.tiles) * a.tokens;
  const int n = min(a.tokens, a.T - t0);
  const int pitch = (a.P + 7) & ~7;
  for (int i = threadIdx.x; i < n * a.P; i += kBlock) {
    const int t = i / a.P, j = i - t * a.P;
    int axis = 0;
#pragma unroll
    for (int x = 1; x < kMaxAxes; ++x) axis += x < a.axes && j >= a.first[x];
    const int64_t at = b * a.pos_b + (int64_t)(t0 + t) * a.axes + axis;
    const double pos = a.pos_kind == 0   ? (double)static_cast<const int64_t *>(a.pos)[at]
                       : a.pos_kind == 1 ? (double)static_cast<const int32_t *>(a.pos)[at]
                                         : (double)static_cast<const float *>(a.pos)[at];
    const double turn = pos * a.turns[j];
    float s, c;
    sincospif(2.f * (float)(turn - rint(turn)), &s, &c);
    cs[t * pitch + j] = c;
    sn[t * pitch + j] = s * a.sign;
  }
  __syncthreads();
  const int slot = threadIdx.x / a.chunks, chunk = threadIdx.x - slot * a.chunks;
  const int step = kBlock / a.chunks, all = a.heads[0] + a.heads[1];
  if (slot >= step) return;
  for (int i = slot; i < n * all; i += step) {
    const int t = a.heads_inv ? (int)__umulhi((uint32_t)i, a.heads_inv) : i;
    const int hh = i - t * all, which = hh >= a.heads[0], h = which ? hh - a.heads[0] : hh;
    const T *x = static_cast<const T *>(a.x[which]) + b * a.sb[which] +
                 (t0 + t) * a.st[which] + h * a.sh[which];
    T *y = static_cast<T *>(a.out[which]) +
           (((int64_t)b * a.T + t0 + t) * a.heads[which] + h) * a.D;
    // An item is two pieces of 16 bytes, one in each half of its run (the turned elements or the
    // rest), so that lanes lie side by side in both.  A piece that would pass the run's end ends
    // with it: what it shares with the piece before it is formed twice, to the same bits.
    const bool turn = chunk < a.turned;
    const int run = turn ? 2 * a.P : a.D - 2 * a.P, items = turn ? a.turned : a.chunks - a.turned;
    const int first = turn ? 0 : 2 * a.P;
    const int c0 = (turn ? chunk : chunk - a.turned) * E;
    const bool halves = turn && !INTER;  // the second half is pair j's other element
    const int size = halves ? a.P : run;
    const bool whole = size >= E;
    const int e0 = whole ? min(c0, size - E) : c0;
    const int e1 = halves ? a.P + e0 : whole ? min(items * E + c0, size - E) : items * E + c0;
    const int left0 = size - c0, left1 = halves ? left0 : size - items * E - c0;
    Piece<T> u, v;
    u.load(x + first + e0, whole ? E : left0);
    v.load(x + first + e1, whole ? E : left1);
    if (halves) {
      float c[E], s[E];
      __builtin_memcpy(c, cs + t * pitch + e0, sizeof(c));
      __builtin_memcpy(s, sn + t * pitch + e0, sizeof(s));
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const float e = to_f32(u.v[k]), f = to_f32(v.v[k]);
        u.v[k] = from_f32<T>(fmaf(e, c[k], -(f * s[k])));
        v.v[k] = from_f32<T>(fmaf(e, s[k], f * c[k]));
      }
    } else if (turn) {
      turn_neighbours(u, cs + t * pitch + e0 / 2, sn + t * pitch + e0 / 2);
      turn_neighbours(v, cs + t * pitch + e1 / 2, sn + t * pitch + e1 / 2);
    }
    u.template store<NT>(y + first + e0, whole ? E : left0);
    v.template store<NT>(y + first + e1, whole ? E : left1);
  }
}

template <typename T>
int launch(const RotaryArgs &a, int64_t grid, bool inter, bool nt, hipStream_t s) {
#define NF_ROTARY(I, N) rotary_kernel<T, I, N><<<(unsigned)grid, kBlock, 0, s>>>(a)
  if (inter && nt)
    NF_ROTARY(true, true);
  else if (inter)
    NF_ROTARY(true, false);
  else if (nt)
    NF_ROTARY(false, true);
  else
    NF_ROTARY(false, false);
#undef NF_ROTARY
  return check_launch("nf_rotary");
}

}  // namespace
}  // namespace nf

using namespace nf;

extern "C" int nf_rotary(const void *q, int64_t q_b, int64_t q_t, int64_t q_h, void *q_out,
                         int64_t H, const void *k, int64_t k_b, int64_t k_t, int64_t k_h,
                         void *k_out, int64_t Hk, const void *positions, int64_t pos_b,
                         int pos_kind, int64_t B, int64_t T, int64_t D, const int32_t *sections,
                         int axes, double base, int joint, int interleaved, int inverse, int dtype,
                         void *stream) {
  const char *op = "nf_rotary";
  if (!is_dtype(dtype)) return set_error(NF_ERR_DTYPE, "%s: dtype %d", op, dtype);
  if (pos_kind < 0 || pos_kind > 2) return set_error(NF_ERR_DTYPE, "%s: pos_kind %d", op, pos_kind);
  if (B < 0 || T < 0 || H < 0 || Hk < 0 || D <= 0)
    return set_error(NF_ERR_ARG, "%s: B=%lld T=%lld H=%lld Hk=%lld D=%lld", op, (long long)B,
                     (long long)T, (long long)H, (long long)Hk, (long long)D);
  if (axes < 1 || axes > kMaxAxes || !sections)
    return set_error(NF_ERR_ARG, "%s: %d axes outside [1, %d]", op, axes, kMaxAxes);
  RotaryArgs a = {};
  int64_t pairs = 0;
  for (int i = 0; i < axes; ++i) {
    if (sections[i] < 0 || sections[i] > kMaxPairs)
      return set_error(NF_ERR_ARG, "%s: section %d", op, (int)sections[i]);
    a.first[i] = (int)pairs;
    pairs += sections[i];
  }
  if (pairs < 1 || pairs > kMaxPairs || 2 * pairs > D || D > 8 * kBlock / 2)
    return set_error(NF_ERR_ARG, "%s: %lld pairs in rows of %lld (at most %d pairs, %d elements)",
                     op, (long long)pairs, (long long)D, kMaxPairs, 4 * kBlock);
  if (!(base > 0.0) || !isfinite(base)) return set_error(NF_ERR_ARG, "%s: base %g", op, base);
  if (B == 0 || T == 0 || H + Hk == 0) return NF_OK;
  if ((H && (!q || !q_out)) || (Hk && (!k || !k_out)) || !positions)
    return set_error(NF_ERR_ARG, "%s: null pointer", op);
  if (H + Hk > 65536 || T > (int64_t)1 << 30)
    return set_error(NF_ERR_ARG, "%s: T=%lld, %lld heads too large", op, (long long)T,
                     (long long)(H + Hk));
  const int P = (int)pairs;
  for (int i = 0, at = 0; i < axes; ++i)
    for (int j = 0; j < sections[i]; ++j, ++at) {
      const double e = joint ? (double)at / P : (double)j / sections[i];
      a.turns[at] = pow(base, -e) / 6.283185307179586476925286766559;
    }
  a.x[0] = q;
  a.x[1] = k;
  a.out[0] = q_out;
  a.out[1] = k_out;
  a.sb[0] = q_b, a.st[0] = q_t, a.sh[0] = q_h;
  a.sb[1] = k_b, a.st[1] = k_t, a.sh[1] = k_h;
  a.heads[0] = (int)H;
  a.heads[1] = (int)Hk;
  a.T = (int)T;
  a.D = (int)D;
  a.P = P;
  a.axes = axes;
  const int es = dtype == NF_DTYPE_F32 ? 4 : 2, e = 16 / es;
  a.turned = (P + e - 1) / e;
  a.chunks = a.turned + (int)((D - 2 * P + 2 * e - 1) / (2 * e));
  const int all = (int)(H + Hk);
  a.heads_inv = all == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + all - 1) / all);
  a.pos = positions;
  a.pos_b = pos_b;
  a.pos_kind = pos_kind;
  a.sign = inverse ? -1.f : 1.f;
  // tokens of a block: about 8 pieces a thread, but no fewer blocks than fill the chip twice, and
  // no more than the table holds
  const int64_t per_token = (int64_t)all * a.chunks;
  int64_t n = 8 * kBlock / per_token;
  if (n > B * T / 512) n = B * T / 512;
  if (n > kTable / ((P + 7) & ~7)) n = kTable / ((P + 7) & ~7);
  if (n > T) n = T;
  if (n < 1) n = 1;
  a.tokens = (int)n;
  a.tiles = (int)((T + n - 1) / n);
  const int64_t grid = B * a.tiles;
  if (grid > kMaxLaunchThreads / kBlock)
    return set_error(NF_ERR_ARG, "%s: B=%lld T=%lld too large", op, (long long)B, (long long)T);
  const bool nt = 2 * B * T * all * D * es > kNtMinBytes;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == NF_DTYPE_F32) return launch<float>(a, grid, interleaved, nt, s);
  if (dtype == NF_DTYPE_BF16) return launch<bf16>(a, grid, interleaved, nt, s);
  return launch<f16>(a, grid, interleaved, nt, s);
}
