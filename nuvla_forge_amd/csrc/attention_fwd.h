// Attention, forward: out = softmax(scale q k^T over the keys that may be attended) v.
//
// One pass over the keys with a running maximum m and sum l: with c = |scale| log2(e) and S the
// bare products, p = 2^(c S - m), l += sum p, O += p v; where m grows, O and l are scaled by
// 2^(m_old - m_new); out = O / l, and the row's log-sum-exp is m + log2(l).
//
// What bounds it.  Heads of 128: the matrix pipe is busy for half of the cycles and the vector unit
// (16 lanes: four operations and a 16-cycle exponential for each logit) for the other half, two
// wavefronts a SIMD overlapping them in part, at a clock that the power limit holds near 1.9 GHz:
// 2 x 4096 tokens, 16 heads 265 us (1.04 PFLOP/s); 16384 causal tokens on 4 key heads 1.02 ms.
// Heads of 64: the exponentials (160 us, 0.86).  Few rows: reading K and V (65536 keys of 4 heads
// of 128, one token: 25 us, 5.4 TB/s).  fp32 runs on the fp32 matrix instructions (157 TFLOP/s).
// Under a key mask every tile is tested entry by entry, whole ones too: 2 x 4096 causal tokens, 16
// heads on 4, 153 us, with lengths between half and full 183 (dQ 198 and 227).
#pragma once

#include <type_traits>

#include "attention.h"

namespace nf {
namespace attn {

// m is raised only when a logit passes it by kSlack (in powers of two): p is then at most
// 2^(kSlack + kBias), 2^15 in fp16, which every type holds, and most tiles leave O as it is.
constexpr float kSlack = 8.f;
// fp16 ends at 2^-24: p carries a factor 2^7, so that it is normal down to 2^-21 of the largest.
template <typename T>
constexpr float kBias = __is_same(T, f16) ? 7.f : 0.f;

// KW = 1: a wavefront has 32 rows of its own, a block 128, and the next tile is copied under this
// one's products.  KW = 4: a block has 32 rows, and a wavefront a quarter of each tile's keys; one
// tile in LDS, so that two blocks share a CU and one's copy runs under the other's products (one
// token for 8 caches of up to 4096 keys 13.7 us, 16.0 with two tiles and one block).  Tiles of 128
// keys there, so that a wavefront has a product's 32; of 64 where rows are a wavefront's own, and 32
// in fp32 rows of 512 bytes, which leave two blocks their LDS.
template <typename T, int DP, int KW, bool MASKED>
struct Fwd {
  using C = Tile<T, DP>;
  static constexpr int BR = KW == 1 ? 32 * kWaves : 32;                // rows of a block
  static constexpr int TK = KW == 4 ? 128 : (C::ROW > 256 ? 32 : 64);  // keys of a tile
  static constexpr int NK = KW == 4 ? 1 : TK / 32;                     // of those, 32s of a wavefront
  using Keys = KeyTiles<T, DP, TK, MASKED>;
  static constexpr int TILE = Keys::TILE;
  static constexpr int STAGES = KW == 1 && 4 * TILE <= 128 * 1024 ? 2 : 1;
  static constexpr int END = kWaves * Turned<DP>::BYTES + (KW == 4 ? 1024 : 0);
  static constexpr int LDS = STAGES * 2 * TILE > END ? STAGES * 2 * TILE : END;
};

template <typename T, int DP, int KW, bool MASKED>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 || (KW == 4 && DP <= 64) ? 2 : 1) void attn_fwd_kernel(
    FwdArgs a) {
  using F = Fwd<T, DP, KW, MASKED>;
  using C = Tile<T, DP>;
  __shared__ __attribute__((aligned(16))) char smem[F::LDS];
  const Shape &s = a.s;
  int bh, job;
  if (!place(s.B * s.Hk, a.tiles * a.most, &bh, &job)) return;
  const int part = job / a.tiles;
  const int tile = a.tiles - 1 - (job - part * a.tiles);  // causal: the longest first
  const int len = key_tiles<F::TK>(s, tile, F::BR), parts = parts_of(len, a.length);
  if (part >= parts) return;
  const int b = bh / s.Hk, hk = bh % s.Hk;
  const int l = threadIdx.x & 63, h = l >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r0 = tile * F::BR + (KW == 1 ? 32 * wave : 0);  // the wavefront's first row

  // the lane's row
  const int r = r0 + (l & 31);
  const int rc = min(r, s.R - 1), t = rc / s.G, g = rc - t * s.G;
  u32x4 q[C::KS];
  load_row<T, DP>(a.q.p + b * a.q.b + t * a.q.t + (int64_t)(hk * s.G + g) * a.q.h, r < s.R, s.nvec,
                  s.flip, q);
  const int last = s.causal ? t + s.off : s.Tk - 1;  // the lane's last key
  const int block_least = s.causal ? tile * F::BR / s.G + s.off : s.Tk - 1;  // its first row's
  int at = part * a.length;
  const int end = part + 1 < parts ? at + a.length : len;
  // every row of the block sees every key of the tiles before this one
  const int full = MASKED ? 0 : min(end, max(block_least + 1, 0) / F::TK);

  floatx16 o[C::NB];
#pragma unroll
  for (int n = 0; n < C::NB; ++n) o[n] = splat(0.f);
  float m = -kInf, sum = 0.f;  // sum: of the lane's own entries

  typename F::Keys keys(s, a.k, a.v, b, hk, end, wave);
  typename F::Keys::Bits cur, nxt;
  auto copy = [&](int i, const typename F::Keys::Bits &x, char *lds) {
    keys.copy_k(i, x, lds, false);  // a dropped key's logit is replaced
    keys.copy_v(i, x, lds, true);   // its value is multiplied by 0
  };
  at = keys.seek(at, cur);
  if (at < end) copy(at, cur, smem);
  auto step = [&](auto edge, int buf) {
    constexpr bool EDGE = decltype(edge)::value;
    const int next = keys.seek(at + 1, nxt);
    gemm::wait_vm_barrier<0>();
    if (F::STAGES == 2 && next < end) copy(next, nxt, smem + (buf ^ 1) * 2 * F::TILE);
    const char *kt = smem + buf * 2 * F::TILE, *vt = kt + F::TILE;
    const int kb0 = KW == 4 ? wave : 0;
    floatx16 p[F::NK];
#pragma unroll
    for (int i = 0; i < F::NK; ++i) {
      floatx16 acc = splat(0.f);
      mma_rows<T, DP>(kt, kb0 + i, q, acc);
      p[i] = acc;
      if constexpr (EDGE) {
        const uint32_t live = live32(last - (at * F::TK + 32 * (kb0 + i)), cur.half(kb0 + i));
#pragma unroll
        for (int e = 0; e < 16; ++e) p[i][e] = keep(p[i][e], live, e, kMinusInf);
      }
    }
    float top = p[0][0];
#pragma unroll
    for (int i = 0; i < F::NK; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, p[i][e]);
    top = pair_max(top) * s.c - kBias<T>;
    if (__any(top > m + kSlack)) {
      const float up = fmaxf(m, top);
      const float f = exp2_(m - (up == -kInf ? 0.f : up));
      m = up;
      sum *= f;
#pragma unroll
      for (int n = 0; n < C::NB; ++n) o[n] *= f;
    }
    const float base = m == -kInf ? 0.f : m;
#pragma unroll
    for (int i = 0; i < F::NK; ++i) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        p[i][e] = exp2_(fmaf(p[i][e], s.c, -base));
        sum += p[i][e];
      }
      if constexpr (KW == 4) {
        Twice<T> x;
        x.set(p[i]);
        mma_cols<T, DP>(vt, kb0 + i, x, o);
      } else {
        Packed<T> x;
        x.set(p[i]);
        mma_cols<T, DP>(vt, kb0 + i, x, o);
      }
    }
    if (F::STAGES == 1) {
      __syncthreads();
      if (next < end) copy(next, nxt, smem);
    }
    at = next;
    cur = nxt;
  };
  // tiles that every row sees whole, in pairs, so that the buffers' addresses are constants
  while (at + 1 < full) {
    step(std::false_type{}, 0);
    step(std::false_type{}, F::STAGES - 1);
  }
  int buf = 0;
  while (at < end) {
    step(std::true_type{}, buf);
    buf ^= F::STAGES - 1;
  }
  sum = pair_sum(sum);

  __syncthreads();
  float f = 1.f;
  if constexpr (KW == 4) {  // the four wavefronts' parts of the same rows
    float *stat = reinterpret_cast<float *>(smem + kWaves * Turned<DP>::BYTES);  // [4][2][32]
    if (h == 0) {
      stat[wave * 64 + l] = m;
      stat[wave * 64 + 32 + l] = sum;
    }
    __syncthreads();
    float top = -kInf, total = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, stat[w * 64 + (l & 31)]);
    const float base = top == -kInf ? 0.f : top;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      total += stat[w * 64 + 32 + (l & 31)] * exp2_(stat[w * 64 + (l & 31)] - base);
    f = exp2_(m - base);
    m = top;
    sum = total;
  }
  if (parts == 1) f *= sum == 0.f ? 0.f : 1.f / sum;  // no key: 0; a NaN stays one
  Turned<DP>::put(smem + wave * Turned<DP>::BYTES, o, f);
  if (KW == 4) __syncthreads();
  const int64_t row = (int64_t)bh * s.R + r;  // the lane's
  const bool lead = r < s.R && h == 0 && (KW == 1 || wave == 0);
  if (parts > 1) {
    const int64_t rows = (int64_t)s.B * s.Hk * s.R;
    float *op = a.part + ((int64_t)part * rows + (int64_t)bh * s.R + r0) * DP;
    each_vector<DP, KW>(smem, wave, [&](int i, int d, const f32x4 &x) {
      if (r0 + i < s.R) store_quad<float>(op + i * DP, d, DP, x);
    });
    if (lead) {
      float *ml = a.part + (int64_t)a.most * rows * DP + ((int64_t)part * rows + row) * 2;
      ml[0] = m;
      ml[1] = sum;
    }
    return;
  }
  const int64_t to = (((int64_t)b * s.Tq + t) * s.H + hk * s.G + g) * s.D;
  each_vector<DP, KW>(smem, wave, [&](int i, int d, const f32x4 &x) {
    const int64_t at_ = from_lane(to, i);
    if (r0 + i >= s.R) return;
    store_quad<T>(reinterpret_cast<T *>(a.out) + at_, d, s.D, x);
    if (a.low) {
      f32x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = x[e] - to_f32(from_f32<T>(x[e]));
      store_quad<T>(reinterpret_cast<T *>(a.low) + at_, d, s.D, y);
    }
  });
  if (a.lse && lead) a.lse[row] = sum == 0.f ? kInf : m + __log2f(sum);
}

// Joins the parts of a row, in a fixed order: W wavefronts a row, every W-th part each.
template <typename T, int DP, int KW, int W>
__global__ __launch_bounds__(kThreads) void attn_join_kernel(FwdArgs a) {
  using F = Fwd<T, DP, KW, false>;
  __shared__ float sums[kWaves][(DP + 63) / 64 * 64];
  const Shape &s = a.s;
  const int64_t rows = (int64_t)s.B * s.Hk * s.R;
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * (kWaves / W) + wave / W;
  if (row >= rows) return;
  const int64_t bh = row / s.R;
  const int r = (int)(row - bh * s.R);
  const int n = parts_of(key_tiles<F::TK>(s, r / F::BR, F::BR), a.length);
  if (n == 1) return;  // the row is written
  const float *ml = a.part + (int64_t)a.most * rows * DP + row * 2;
  float m[2], sum = 0.f, top = -kInf;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    m[j] = l + 64 * j < n ? ml[(l + 64 * j) * rows * 2] : -kInf;
    top = fmaxf(top, m[j]);
  }
  top = wave_max(top);
  const float base = top == -kInf ? 0.f : top;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    m[j] = exp2_(m[j] - base);
    if (l + 64 * j < n) sum += ml[(l + 64 * j) * rows * 2 + 1] * m[j];
  }
  sum = wave_sum(sum);
  constexpr int NJ = (DP + 63) / 64;
  float o[NJ] = {};
  auto add = [&](int i) {
    const float f = __shfl(i < 64 ? m[0] : m[1], i & 63);
    const float *p = a.part + (i * rows + row) * DP;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      if (l + 64 * j < DP) o[j] = fmaf(p[l + 64 * j], f, o[j]);
  };
  int i = wave % W;
  for (; i + 3 * W < n; i += 4 * W) {
    add(i);
    add(i + W);
    add(i + 2 * W);
    add(i + 3 * W);
  }
  for (; i < n; i += W) add(i);
  if constexpr (W > 1) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) sums[wave][l + 64 * j] = o[j];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      o[j] = ((sums[0][l + 64 * j] + sums[1][l + 64 * j]) + sums[2][l + 64 * j]) +
             sums[3][l + 64 * j];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t b = bh / s.Hk, hk = bh % s.Hk, t = r / s.G, g = r % s.G;
  const int64_t to = ((b * s.Tq + t) * s.H + hk * s.G + g) * s.D;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int d = l + 64 * j;
    if (d >= s.D) continue;
    const float x = o[j] * inv;
    reinterpret_cast<T *>(a.out)[to + d] = from_f32<T>(x);
    if (a.low) reinterpret_cast<T *>(a.low)[to + d] = from_f32<T>(x - to_f32(from_f32<T>(x)));
  }
  if (a.lse && l == 0) a.lse[row] = sum == 0.f ? kInf : top + __log2f(sum);
}

template <typename T, int DP, int KW>
void join(const FwdArgs &a, hipStream_t st) {
  const int64_t rows = (int64_t)a.s.B * a.s.Hk * a.s.R;
  if (a.most > 8)
    attn_join_kernel<T, DP, KW, kWaves><<<(unsigned)rows, kThreads, 0, st>>>(a);
  else
    attn_join_kernel<T, DP, KW, 1>
        <<<(unsigned)((rows + kWaves - 1) / kWaves), kThreads, 0, st>>>(a);
}

template <typename T, int DP>
int launch_fwd_dp(FwdArgs a, const Plan &p, hipStream_t st) {
  a.length = p.length;
  a.most = p.most;
  a.tiles = p.tiles;
  const unsigned grid =
      (unsigned)place_grid((int64_t)a.s.B * a.s.Hk, (int64_t)p.tiles * p.most);
  if (p.kw == 4 && a.s.mask)
    attn_fwd_kernel<T, DP, 4, true><<<grid, kThreads, 0, st>>>(a);
  else if (p.kw == 4)
    attn_fwd_kernel<T, DP, 4, false><<<grid, kThreads, 0, st>>>(a);
  else if (a.s.mask)
    attn_fwd_kernel<T, DP, 1, true><<<grid, kThreads, 0, st>>>(a);
  else
    attn_fwd_kernel<T, DP, 1, false><<<grid, kThreads, 0, st>>>(a);
  if (p.most > 1 && p.kw == 4)
    join<T, DP, 4>(a, st);
  else if (p.most > 1)
    join<T, DP, 1>(a, st);
  return check_launch("nf_attention_fwd");
}

template <typename T>
int launch_fwd(const FwdArgs &a, const Sizes &z, hipStream_t st) {
  switch (z.dp()) {
    case 32: return launch_fwd_dp<T, 32>(a, fwd_plan(z, a.s.causal), st);
    case 64: return launch_fwd_dp<T, 64>(a, fwd_plan(z, a.s.causal), st);
    case 96:
      if constexpr (sizeof(T) == 2) return launch_fwd_dp<T, 96>(a, fwd_plan(z, a.s.causal), st);
      [[fallthrough]];
    default: return launch_fwd_dp<T, 128>(a, fwd_plan(z, a.s.causal), st);
  }
}

}  // namespace attn
}  // namespace nf
