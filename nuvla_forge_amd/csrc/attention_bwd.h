// Attention, backward: the probabilities are formed again from the row's log-sum-exp L,
//
//   P = 2^(c S - L),  delta = rowsum(dO O),  dS = P (dP - delta)  with  dP = dO V^T
//   dV = P^T dO,  dQ = scale dS K,  dK = scale dS^T Q,
//
// in two launches: one over tiles of rows for delta and dQ, one over tiles of keys for dK and dV.
// Each sums in an order of its own that no other block takes part in (no atomics: the same bits
// every run), at the price of S and dP formed twice (seven products of a tile where five would do).
// delta is formed from O's two parts, rounded and left over: out of the rounded part alone it would
// be the largest error of dS where a row attends few keys.
//
// P and dS are rounded to the inputs' 16 bits for their products, as the matrix instructions take
// them: results are then off by about 1.45 times what their own last rounding costs.  Where few
// rows or keys share a block both go in two terms, and the last rounding is all that is left.
//
// What bounds it: as the forward, with the exponentials a smaller share: 2 x 4096 tokens, 16 heads of
// 128: dQ 358 us (1.15 PFLOP/s of its three products), dK and dV 570 (0.96 of four; a wavefront
// alone on its SIMD); of 64 208 and 284.
//
// What does not fit its registers: dQ in bf16, 96 columns, rows of a wavefront's own, unmasked keeps 10
// of them (44 bytes a lane) in scratch memory; dK and dV in fp16, 128 columns, 4 to 10 in accumulation
// registers; dK and dV in fp32, 128 columns, shared (calls of up to 32 keys) 608 bytes a lane in scratch.
#pragma once

#include <type_traits>

#include "attention.h"

namespace nf {
namespace attn {

// fp16 holds 2^-24 to 65504, and gradients may lie anywhere: dS is scaled by a power of two of its
// column's own (a row's in dQ, a key's in dK), chosen so that its largest entry so far is about
// 2^kTop; a larger one scales what is accumulated.  Other types take dS as it is.
constexpr int kTop = 12;
template <typename T, int NB>
struct Ranged {
  __device__ __forceinline__ void fit(floatx16 &, floatx16 (&)[NB]) {}
  __device__ __forceinline__ float undo() const { return 1.f; }
};
template <int NB>
struct Ranged<f16, NB> {
  int e = -1000;  // entries are below 2^e; none so far
  __device__ __forceinline__ void fit(floatx16 &x, floatx16 (&acc)[NB]) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(x[i]));
    top = pair_max(top);
    const bool real = top > 0.f && top < kInf;
    const int now = real ? __builtin_amdgcn_frexp_expf(top) : -1000;
    if (__any(now > e + 2)) {
      const int up = now > e ? now : e;
      const float f = e == -1000 ? 0.f : ldexpf(1.f, e - up);
#pragma unroll
      for (int n = 0; n < NB; ++n)
        if (e != up) acc[n] *= f;
      e = up;
    }
    const int by = e == -1000 ? 0 : kTop - e;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = ldexpf(x[i], by);
  }
  // what the accumulated sum is to be multiplied by
  __device__ __forceinline__ float undo() const { return e == -1000 ? 1.f : ldexpf(1.f, e - kTop); }
};
// fp16: P carries a factor 2^kPExp into dV's product
template <typename T>
constexpr float kPExp = __is_same(T, f16) ? 15.f : 0.f;

// KW as in the forward: 1, a wavefront has 32 rows of its own; 4, the wavefronts share a block's 32
// rows and take a quarter of each tile's keys.
template <typename T, int DP, int KW, bool MASKED>
struct Dq {
  using C = Tile<T, DP>;
  static constexpr int BR = KW == 1 ? 32 * kWaves : 32;
  static constexpr int TK = KW == 4 ? 128 : (C::ROW > 256 ? 32 : 64);
  static constexpr int NK = KW == 4 ? 1 : TK / 32;
  using Keys = KeyTiles<T, DP, TK, MASKED>;
  static constexpr int TILE = Keys::TILE;
  static constexpr int STAGES = KW == 1 && 4 * TILE <= 128 * 1024 ? 2 : 1;
  static constexpr int END = kWaves * Turned<DP>::BYTES;
  static constexpr int LDS = STAGES * 2 * TILE > END ? STAGES * 2 * TILE : END;
};

template <typename T, int DP, int KW, bool MASKED>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 || (KW == 4 && DP <= 64) ? 2 : 1) void attn_dq_kernel(
    BwdArgs a) {
  using F = Dq<T, DP, KW, MASKED>;
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
  const int r0 = tile * F::BR + (KW == 1 ? 32 * wave : 0);

  const int r = r0 + (l & 31);
  const int rc = min(r, s.R - 1), t = rc / s.G, g = rc - t * s.G;
  const int64_t row = (int64_t)bh * s.R + rc;
  const int64_t at_out = (((int64_t)b * s.Tq + t) * s.H + hk * s.G + g) * s.D;
  u32x4 q[C::KS], dout[C::KS];
  load_row<T, DP>(a.dout.p + b * a.dout.b + t * a.dout.t + (int64_t)(hk * s.G + g) * a.dout.h,
                  r < s.R, s.nvec, 0u, dout);
  const float lse = a.lse[row];
  float nd = 0.f;  // -delta: the lane's half of the columns, then both
  {
    const T *out = reinterpret_cast<const T *>(a.out) + at_out;
    const T *low = a.low ? reinterpret_cast<const T *>(a.low) + at_out : nullptr;
#pragma unroll
    for (int k = 0; k < C::KS; ++k) {
      const int col = (2 * k + h) * C::VE;
      const int valid = min(max(s.D - col, 0), C::VE);
      T d[C::VE], o[C::VE] = {}, w[C::VE] = {};
      __builtin_memcpy(d, &dout[k], 16);
      if (valid == C::VE) {
        __builtin_memcpy(o, out + col, 16);
        if (low) __builtin_memcpy(w, low + col, 16);
      } else {
#pragma unroll
        for (int i = 0; i < C::VE; ++i) {
          if (i < valid) o[i] = out[col + i];
          if (i < valid && low) w[i] = low[col + i];
        }
      }
#pragma unroll
      for (int i = 0; i < C::VE; ++i)
        nd = fmaf(-to_f32(d[i]), to_f32(o[i]) + to_f32(w[i]), nd);
    }
    nd = pair_sum(nd);
    if (lse == kInf) nd = 0.f;  // no key: whatever dO holds
    if (r < s.R && h == 0 && (KW == 1 || wave == 0) && part == 0) a.ndelta[row] = nd;
  }
  if (!a.dq) return;  // the call is for delta alone
  load_row<T, DP>(a.q.p + b * a.q.b + t * a.q.t + (int64_t)(hk * s.G + g) * a.q.h, r < s.R, s.nvec,
                  s.flip, q);
  const int last = s.causal ? t + s.off : s.Tk - 1;
  const int block_least = s.causal ? tile * F::BR / s.G + s.off : s.Tk - 1;
  const int begin = part * a.length, end = part + 1 < parts ? begin + a.length : len;
  const int full = MASKED ? 0 : min(end, max(block_least + 1, 0) / F::TK);

  floatx16 dq[C::NB];
#pragma unroll
  for (int n = 0; n < C::NB; ++n) dq[n] = splat(0.f);
  Ranged<T, C::NB> range;

  typename F::Keys keys(s, a.k, a.v, b, hk, end, wave);
  typename F::Keys::Bits cur, nxt;
  auto copy = [&](int i, const typename F::Keys::Bits &x, char *lds) {
    keys.copy_k(i, x, lds, true);   // a dropped key is multiplied by 0
    keys.copy_v(i, x, lds, false);  // its value gives dS alone, which is replaced
  };
  int at = keys.seek(begin, cur);
  if (at < end) copy(at, cur, smem);
  auto step = [&](auto edge, int buf) {
    constexpr bool EDGE = decltype(edge)::value;
    const int next = keys.seek(at + 1, nxt);
    gemm::wait_vm_barrier<0>();
    if (F::STAGES == 2 && next < end) copy(next, nxt, smem + (buf ^ 1) * 2 * F::TILE);
    const char *kt = smem + buf * 2 * F::TILE, *vt = kt + F::TILE;
    const int kb0 = KW == 4 ? wave : 0;
#pragma unroll
    for (int i = 0; i < F::NK; ++i) {
      floatx16 p = splat(0.f), dp = splat(nd);
      mma_rows<T, DP>(kt, kb0 + i, q, p);
      mma_rows<T, DP>(vt, kb0 + i, dout, dp);
#pragma unroll
      for (int e = 0; e < 16; ++e) dp[e] *= exp2_(fmaf(p[e], s.c, -lse));
      if constexpr (EDGE) {
        const uint32_t live = live32(last - (at * F::TK + 32 * (kb0 + i)), cur.half(kb0 + i));
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] = keep(dp[e], live, e, 0u);
      }
      range.fit(dp, dq);
      if constexpr (KW == 4) {
        Twice<T> x;
        x.set(dp);
        mma_cols<T, DP>(kt, kb0 + i, x, dq);
      } else {
        Packed<T> x;
        x.set(dp);
        mma_cols<T, DP>(kt, kb0 + i, x, dq);
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
  const float f = s.scale * range.undo();
  __syncthreads();
  Turned<DP>::put(smem + wave * Turned<DP>::BYTES, dq, f);
  if (KW == 4) __syncthreads();
  float *sums = a.part + ((int64_t)part * s.B * s.Hk * s.R + (int64_t)bh * s.R + r0) * DP;
  each_vector<DP, KW>(smem, wave, [&](int i, int d, const f32x4 &x) {
    const int64_t to = from_lane(at_out, i);
    if (r0 + i >= s.R) return;
    if (parts > 1)
      store_quad<float>(sums + i * DP, d, DP, x);
    else
      store_quad<T>(reinterpret_cast<T *>(a.dq) + to, d, s.D, x);
  });
}

// KW = 1: a block has 128 keys, a wavefront 32, and goes over the rows.  KW = 4: a block has 32 keys,
// and a wavefront a quarter of each tile's rows.
template <typename T, int DP, int KW>
struct Dkv {
  using C = Tile<T, DP>;
  static constexpr int BK = KW == 1 ? 32 * kWaves : 32;
  static constexpr int TR = KW == 4 ? 128 : C::ROW > 256 ? 32 : 64;  // rows of a tile
  static constexpr int NR = KW == 4 ? 1 : TR / 32;                   // of those, 32s of a wavefront
  static constexpr int TILE = TR * C::ROW;
  static constexpr int STAGE = 2 * TILE + 2 * 4 * (TR < 64 ? 64 : TR);  // q, dout, lse, -delta
  static constexpr bool TWO = DP <= 64 && sizeof(T) == 2;  // blocks on a CU
  static constexpr int STAGES = !(TWO && KW == 4) && 2 * STAGE <= 140 * 1024 ? 2 : 1;
  static constexpr int LDS = STAGES * STAGE;
  static_assert(LDS >= kWaves * Turned<DP>::BYTES, "the results turn in the tiles' place");
};

template <typename T, int DP, int KW>
__global__ __launch_bounds__(kThreads, (Dkv<T, DP, KW>::TWO ? 2 : 1)) void attn_dkv_kernel(
    BwdArgs a) {
  using F = Dkv<T, DP, KW>;
  using C = Tile<T, DP>;
  __shared__ __attribute__((aligned(16))) char smem[F::LDS];
  const Shape &s = a.s;
  int bh, job;
  if (!place(s.B * s.Hk, a.tiles * a.most, &bh, &job)) return;
  const int part = job / a.tiles, tile = job - part * a.tiles;  // causal: the first have most rows
  const int begin = first_row_tile<F::TR>(s, tile, F::BK), len = (s.R + F::TR - 1) / F::TR - begin;
  const int parts = parts_of(len, a.length);
  if (part >= parts) return;
  const int b = bh / s.Hk, hk = bh % s.Hk;
  const int l = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  const int key0 = tile * F::BK + (KW == 1 ? 32 * wave : 0);
  const int key = key0 + (l & 31);
  const bool live = key < s.Tk && (!s.mask || s.mask[b * s.mask_b + key]);
  u32x4 k[C::KS], v[C::KS];
  load_row<T, DP>(a.k.p + b * a.k.b + hk * a.k.h + key * a.k.t, live, s.nvec, s.flip, k);
  load_row<T, DP>(a.v.p + b * a.v.b + hk * a.v.h + key * a.v.t, live, s.nvec, 0u, v);
  // causal: row r sees the key from r = (key - off) G on
  const int from = s.causal ? max(key - s.off, 0) : 0;
  const int64_t rmin64 = (int64_t)from * s.G;
  const int rmin = (int)(rmin64 < s.R ? rmin64 : s.R);
  // Causal: the first row that may attend a key, the first one or, under a mask, the first that it
  // leaves the block.  The rows before it are not read: a NaN or an infinity there, in the query or dO
  // of a row without a key for one, would be one in the gradients too, multiplied by 0.  (What they
  // read as is 0; -delta is 0 and the log-sum-exp infinity for a row without a key.)
  int least = 0, row_first = 0;
  if (s.causal) {
    if (s.mask) {
      least = s.Tk;
#pragma unroll
      for (int i = F::BK / 32 - 1; i >= 0; --i) {  // lanes l and l + 32 ask for the same key
        const int j = tile * F::BK + 32 * i + (l & 31);
        const uint32_t some =
            (uint32_t)__ballot(KW == 4 ? live : j < s.Tk && s.mask[b * s.mask_b + j] != 0);
        if (some) least = tile * F::BK + 32 * i + __builtin_ctz(some);
      }
    }
    row_first = (int)min((int64_t)max(least - s.off, 0) * s.G, (int64_t)s.R);
  }
  const int end = begin + len - part * a.length;  // from the last row back
  int at = part + 1 < parts ? end - a.length : begin;
  at = least == s.Tk ? end : min(max(at, row_first / F::TR), end);  // no key: no row
  // from this tile on, every row sees every key of the block
  const int64_t every = s.causal ? (int64_t)max(tile * F::BK + F::BK - 1 - s.off, 0) * s.G : 0;
  const int full = (int)min((every + F::TR - 1) / F::TR, (int64_t)end);

  const char *lp = reinterpret_cast<const char *>(a.lse + (int64_t)bh * s.R);
  const char *np = reinterpret_cast<const char *>(a.ndelta + (int64_t)bh * s.R);
  const RowTiles<T, DP, F::TR> qs(s, a.q, b, hk, wave, row_first),
      dos(s, a.dout, b, hk, wave, row_first);
  auto copy = [&](int i, char *buf) {
    const int row0 = i * F::TR, left = s.R - row0;
    qs.copy(i, buf);
    dos.copy(i, buf + F::TILE);
    if (F::TR > 64 || wave < 2) {  // 64 values a wavefront: log-sum-exps, then -deltas
      constexpr int EACH = F::TR > 64 ? 2 : 1;
      const int at4 = (wave % EACH) * 64 + l;
      const auto rsrc = buffer((wave < EACH ? lp : np) + (int64_t)row0 * 4);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)(buf + 2 * F::TILE + 256 * wave), 4,
                                               at4 < left ? at4 * 4u : kOob, 0, 0, 0);
    }
  };

  floatx16 dk[C::NB], dv[C::NB];
#pragma unroll
  for (int n = 0; n < C::NB; ++n) dk[n] = dv[n] = splat(0.f);
  Ranged<T, C::NB> range;

  // The whole tiles that every row and key share come last, in pairs, so that the buffers' addresses
  // are constants; an odd one goes with the edge.
  const int pairs = max(end - max(at, full), 0) / 2, rest = end - 2 * pairs;
  int buf = (rest - at) & (F::STAGES - 1);
  if (at < end) copy(at, smem + buf * F::STAGE);
  auto step = [&](auto edge, int buf) {
    constexpr bool EDGE = decltype(edge)::value;
    gemm::wait_vm_barrier<0>();
    if (F::STAGES == 2 && at + 1 < end) copy(at + 1, smem + (buf ^ 1) * F::STAGE);
    const char *qt = smem + buf * F::STAGE, *dt = qt + F::TILE;
    const float *lse = reinterpret_cast<const float *>(qt + 2 * F::TILE);
    const float *nd = lse + (F::TR < 64 ? 64 : F::TR);
    if constexpr (sizeof(T) == 4 || KW == 4) {
#pragma unroll
      for (int n = 0; n < F::NR; ++n) {
        const int i = KW == 4 ? wave : n;
        floatx16 p = splat(0.f), ds;
#pragma unroll
        for (int e = 0; e < 16; ++e) ds[e] = nd[32 * i + entry(e)];
        mma_rows<T, DP>(qt, i, k, p);
        mma_rows<T, DP>(dt, i, v, ds);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          p[e] = exp2_(fmaf(p[e], s.c, kPExp<T> - lse[32 * i + entry(e)]));
        if constexpr (EDGE) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            p[e] = at * F::TR + 32 * i + entry(e) >= rmin ? p[e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) ds[e] *= p[e];
        Twice<T> x;
        x.set(p);
        mma_cols<T, DP>(dt, i, x, dv);
        range.fit(ds, dk);
        x.set(ds);
        mma_cols<T, DP>(qt, i, x, dk);
      }
    } else {
      // Four products of KS steps each, in an order that keeps the matrix pipe fed by a wavefront
      // alone on its SIMD: a product's operands are read under the one before it, the exponentials
      // form under dP and dS under dV.
      constexpr int KS = C::KS, PER = (16 + KS - 2) / (KS - 1);  // entries a step after the first
      static_assert(KS == 2 * C::NB, "as many steps along a row as down the columns");
      u32x4 fa[KS], fb[KS];
#pragma unroll
      for (int j = 0; j < KS; ++j) fa[j] = row_frag<T, DP>(qt, 0, j);
#pragma unroll
      for (int i = 0; i < F::TR / 32; ++i) {
        floatx16 p = splat(0.f), ds, ls;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          ds[e] = nd[32 * i + entry(e)];
          ls[e] = lse[32 * i + entry(e)];
        }
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          fb[j] = row_frag<T, DP>(dt, i, j);
          p = mma<T>(fa[j], k[j], p);
          in_order();
        }
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          fa[j] = col_frag<T, DP>(dt, i, j);
          ds = mma<T>(fb[j], v[j], ds);
#pragma unroll
          for (int e = (j - 1) * PER; e >= 0 && e < j * PER && e < 16; ++e) {
            p[e] = exp2_(fmaf(p[e], s.c, kPExp<T> - ls[e]));
            if constexpr (EDGE) p[e] = at * F::TR + 32 * i + entry(e) >= rmin ? p[e] : 0.f;
          }
          in_order();
        }
        Packed<T> x;
        x.set(p);
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          fb[j] = col_frag<T, DP>(qt, i, j);
          dv[j % C::NB] = mma<T>(fa[j], x.v[j / C::NB], dv[j % C::NB]);
#pragma unroll
          for (int e = (j - 1) * PER; e >= 0 && e < j * PER && e < 16; ++e) ds[e] *= p[e];
          in_order();
        }
        range.fit(ds, dk);
        x.set(ds);
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          if (i + 1 < F::TR / 32) fa[j] = row_frag<T, DP>(qt, i + 1, j);
          dk[j % C::NB] = mma<T>(fb[j], x.v[j / C::NB], dk[j % C::NB]);
          in_order();
        }
      }
    }
    ++at;
    if (F::STAGES == 1) {
      __syncthreads();
      if (at < end) copy(at, smem);
    }
  };
  while (at < rest) {
    step(std::true_type{}, buf);
    buf ^= F::STAGES - 1;
  }
  while (at < end) {
    step(std::false_type{}, 0);
    step(std::false_type{}, F::STAGES - 1);
  }
  __syncthreads();
  const float fv = exp2_(-kPExp<T>), fk = s.scale * exp2_(-kPExp<T>) * range.undo();
  char *turned = smem + wave * Turned<DP>::BYTES;
  const int64_t first = (int64_t)bh * s.Tk + key0;
  auto put = [&](const floatx16(&acc)[C::NB], float f, void *out, int which) {
    if (KW == 4) __syncthreads();
    Turned<DP>::put(turned, acc, f);
    if (KW == 4) __syncthreads();
    each_vector<DP, KW>(smem, wave, [&](int i, int d, const f32x4 &y) {
      // a key that is left out: zeros, whatever was formed
      const f32x4 x = __shfl((int)live, i) ? y : f32x4{0.f, 0.f, 0.f, 0.f};
      if (key0 + i >= s.Tk) return;
      if (parts > 1) {
        const int64_t rows = (int64_t)s.B * s.Hk * s.Tk;
        store_quad<float>(a.part + (((int64_t)part * rows + first + i) * 2 + which) * DP, d, DP, x);
      } else if (out) {
        T *to = static_cast<T *>(out) + (((int64_t)b * s.Tk + key0 + i) * s.Hk + hk) * s.D;
        store_quad<T>(to, d, s.D, x);
      }
    });
  };
  put(dk, fk, a.dk, 0);
  put(dv, fv, a.dv, 1);
}

// Sums the parts of a row of dQ, or of a key's dK and dV (KEYS), in their order: a wavefront a row.
// KW: as in the kernel that wrote them.
template <typename T, int DP, int KW, bool KEYS>
__global__ __launch_bounds__(kThreads) void attn_sum_kernel(BwdArgs a) {
  constexpr int W = KEYS ? 2 * DP : DP;  // of a row
  const Shape &s = a.s;
  const int per = KEYS ? s.Tk : s.R, l = threadIdx.x & 63;
  const int64_t rows = (int64_t)s.B * s.Hk * per;
  const int64_t row = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int64_t bh = row / per;
  const int r = (int)(row - bh * per);
  int len;
  if constexpr (!KEYS) {
    using F = Dq<T, DP, KW, false>;
    len = key_tiles<F::TK>(s, r / F::BR, F::BR);
  } else {
    using F = Dkv<T, DP, KW>;
    len = (s.R + F::TR - 1) / F::TR - first_row_tile<F::TR>(s, r / F::BK, F::BK);
  }
  const int n = parts_of(len, a.length);
  if (n == 1) return;  // the row is written
  constexpr int NJ = (W + 63) / 64;
  float x[NJ] = {};
  const float *p = a.part + row * W + l;
#pragma unroll 4
  for (int i = 0; i < n; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      if (l + 64 * j < W) x[j] += p[(int64_t)i * rows * W + 64 * j];
  const int64_t b = bh / s.Hk, hk = bh % s.Hk;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int c = l + 64 * j, d = c % DP;
    if (c >= W || d >= s.D) continue;
    if constexpr (!KEYS) {
      const int64_t t = r / s.G, g = r % s.G;
      reinterpret_cast<T *>(a.dq)[((b * s.Tq + t) * s.H + hk * s.G + g) * s.D + d] =
          from_f32<T>(x[j]);
    } else {
      T *to = reinterpret_cast<T *>(c < DP ? a.dk : a.dv);
      if (to) to[((b * s.Tk + r) * s.Hk + hk) * s.D + d] = from_f32<T>(x[j]);
    }
  }
}

template <typename T, int DP, int KW>
void launch_dq(BwdArgs &a, hipStream_t st) {
  const unsigned grid = (unsigned)place_grid((int64_t)a.s.B * a.s.Hk, (int64_t)a.tiles * a.most);
  if (a.s.mask)
    attn_dq_kernel<T, DP, KW, true><<<grid, kThreads, 0, st>>>(a);
  else
    attn_dq_kernel<T, DP, KW, false><<<grid, kThreads, 0, st>>>(a);
  if (a.most > 1 && a.dq) {
    const int64_t rows = (int64_t)a.s.B * a.s.Hk * a.s.R;
    attn_sum_kernel<T, DP, KW, false><<<(unsigned)((rows + kWaves - 1) / kWaves), kThreads, 0, st>>>(a);
  }
}

template <typename T, int DP, int KW>
void launch_dkv(BwdArgs &a, hipStream_t st) {
  attn_dkv_kernel<T, DP, KW>
      <<<(unsigned)place_grid((int64_t)a.s.B * a.s.Hk, (int64_t)a.tiles * a.most), kThreads, 0,
         st>>>(a);
  if (a.most > 1) {
    const int64_t rows = (int64_t)a.s.B * a.s.Hk * a.s.Tk;
    attn_sum_kernel<T, DP, KW, true>
        <<<(unsigned)((rows + kWaves - 1) / kWaves), kThreads, 0, st>>>(a);
  }
}

template <typename T, int DP>
int launch_bwd_dp(BwdArgs a, const Sizes &z, hipStream_t st) {
  auto take = [&](const Plan &p) {
    a.tiles = p.tiles;
    a.length = p.length;
    a.most = p.most;
    return p.kw;
  };
  const int kw = take(dq_plan(z, a.s.causal));
  if (!a.dq) a.most = 1, a.length = 1 << 28;  // for delta alone
  if (kw == 4)
    launch_dq<T, DP, 4>(a, st);
  else
    launch_dq<T, DP, 1>(a, st);
  if (a.dk || a.dv) {
    if (take(dkv_plan(z, a.s.causal)) == 4)
      launch_dkv<T, DP, 4>(a, st);
    else
      launch_dkv<T, DP, 1>(a, st);
  }
  return check_launch("nf_attention_bwd");
}

template <typename T>
int launch_bwd(const BwdArgs &a, const Sizes &z, hipStream_t st) {
  switch (z.dp()) {
    case 32: return launch_bwd_dp<T, 32>(a, z, st);
    case 64: return launch_bwd_dp<T, 64>(a, z, st);
    case 96:
      if constexpr (sizeof(T) == 2) return launch_bwd_dp<T, 96>(a, z, st);
      [[fallthrough]];
    default: return launch_bwd_dp<T, 128>(a, z, st);
  }
}

}  // namespace attn
}  // namespace nf
