// Token log probabilities on the language-model head: for every row m of hidden, with
// z = hidden[m] . weight^T,
//   lse = log sum exp z,   logprob = z[target] - lse,
//   entropy = -sum p (z - lse),  p = exp(z - lse),
//   and the top_k largest z with their columns (ties: the lower column first),
// and the gradient of logprob and entropy by hidden and weight.  lse is held as mx + ls, mx the
// row's largest logit and ls = log sum exp(z - mx), and z - lse formed as (z - mx) - ls: their sum
// rounded to fp32 would lose what of ls lies below half a step of mx (3e-5 at logits of 1000).
// The [M, V] logits are never held at once; all on the caller's stream, sums in fixed orders,
// no atomics.
//
// Only valid rows (target != ignore_index, inside [0, V)) do any work: they are compacted
// on the device and every later kernel sizes itself by the device count.
//
// Forward (nf_token_logprobs_fwd), more than 256 rows, or more than 64 over V > 32768:
//   1. ce_compact: the valid rows in order.  lp_gather: Hc = hidden[rows], and zeros (id
//      -1) into the outputs of the other rows.
//   2. per chunk of rows: lp_logits, the logits tile by tile, of which statistics and
//      records of strips are left; lp_finish: the row's values from those.
// Fewer: the same without the compaction, on smaller tiles (MidCfg); fp32 up to 32 rows:
// lp_skinny, one pass over weight, and lp_finish.
// Backward (nf_token_logprobs_bwd), with g and h the upstream gradients of a row's logprob
// and entropy H:
//   dz = g (onehot - p) - h p (z - lse + H)
//   dz is formed from what the forward kept of every logit (lp_from_kept), or from the
//   logits formed again tile by tile (lp_dz: W Hc^T, as in the cross entropy's logits), and
//   rounded once to the input type;
//   then the cross entropy's gradient products, dW (+)= dz^T Hc and dHc = dz W, and the
//   scatter of dHc to the hidden rows.
#include "lm_head.h"

namespace nf {
namespace lp {

using namespace gemm;
using ce::chunk_count;
using ce::log_f32;

constexpr int kMaxTop = 32;

// z - lse below this is as good as -inf: exp of it is zero in fp32
constexpr float kFar = -200.f;

// ---------------------------------------------------------------------------
// 1. Hc[r, :] = hidden[rows[r], :] for r < n, 0 for n <= r < M; rows m that are not
// valid get 0 in every output (id -1).  One wavefront per row.  lo0 > 0: Hc has 2 lo0 >= 2 M
// rows, the second lo0 as the first (see few_rows).
// ---------------------------------------------------------------------------
constexpr int kGatherThreads = 256;

struct RowOut {
  float *logprob, *entropy;  // [M]
  float *top_lp;             // [M, top_k]
  int64_t *top_id;
  int top_k;
};

template <typename T, bool VEC>
__global__ __launch_bounds__(kGatherThreads) void lp_gather_kernel(
    const T *__restrict__ H, int64_t D, const int *__restrict__ rows, const int *__restrict__ pos,
    const int *n_ptr, int64_t M, int64_t lo0, T *__restrict__ Hc, RowOut out) {
  constexpr int kWaves = kGatherThreads / 64;
  constexpr int VE = VEC ? 16 / (int)sizeof(T) : 1;
  const int64_t n = *n_ptr;
  const int l = threadIdx.x & 63;
  const int64_t R = lo0 > 0 ? lo0 : M;
  for (int64_t r = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6); r < R;
       r += (int64_t)gridDim.x * kWaves) {
    const T *h = r < n ? H + (int64_t)rows[r] * D : nullptr;
    for (int64_t c = (int64_t)l * VE; c < D; c += 64 * VE) {
      if constexpr (VEC) {
        u32x4 v = {0u, 0u, 0u, 0u};
        if (h) v = *reinterpret_cast<const u32x4 *>(h + c);
        *reinterpret_cast<u32x4 *>(Hc + r * D + c) = v;
        if (lo0 > 0) *reinterpret_cast<u32x4 *>(Hc + (lo0 + r) * D + c) = v;
      } else {
        const T v = h ? h[c] : static_cast<T>(0.f);
        Hc[r * D + c] = v;
        if (lo0 > 0) Hc[(lo0 + r) * D + c] = v;
      }
    }
    if (r < M && pos[r] < 0) {
      if (l == 0) {
        out.logprob[r] = 0.f;
        out.entropy[r] = 0.f;
      }
      if (l < out.top_k) {
        out.top_lp[r * out.top_k + l] = 0.f;
        out.top_id[r * out.top_k + l] = -1;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// 2. The logits, never stored.  What a pass leaves of a token's logits, strip by strip of
// the vocabulary:
//   Stat, per statistics strip: the maximum mx, S = sum exp(z - mx) and
//     T = sum (z - mx) exp(z - mx);
//   Rec (with top_k), per strip of 32 logits: the largest (the first of equals), its place
//     in the strip, and the second largest, rounded up to 16 bits.
// A strip's 32 columns are column(strip, c), c = 0 .. 31, rising in c.  The top_k largest
// logits of a row lie in the top_k strips whose largest come first; a second largest that
// could be among them makes lp_finish form that strip's logits again, in the same order of
// sums and so to the same bits.
// ---------------------------------------------------------------------------
struct __attribute__((aligned(16))) Stat {
  float mx, s, t, pad;
};
struct __attribute__((aligned(8))) Rec {
  float first;
  uint32_t rest;  // bits 31..16: the second largest as the top half of an fp32; 5..0: place
};
constexpr uint32_t kNoPlace = 63;  // no logit of the strip compares (all NaN)

// The least bf16 value >= x, as bits 31..16 (what is left of a NaN does not matter).
__device__ __forceinline__ uint32_t bf16_up(float x) {
  const uint32_t u = __float_as_uint(x);
  return (u >> 31 ? u : u + 0xffffu) & 0xffff0000u;
}

// The columns of a strip.  Pass over block tiles (2^lw strips to a statistics strip, which is
// a wavefront's 32 << lw rows): a strip is 32 of the logits that one lane holds for a token, two
// 32-row MFMA tiles of its half of the lanes; skinny pass (lw 0): 32 columns in a row.
struct Strips {
  int lw;
  __host__ __device__ int per_stat() const { return 1 << lw; }
  __device__ __forceinline__ int column(int strip, int c) const {
    if (!lw) return strip * 32 + c;
    const int stat = strip >> lw, k = strip & ((1 << lw) - 1);  // k = half << (lw - 1) | q
    const int half = k >> (lw - 1), q = k & ((1 << (lw - 1)) - 1);
    return (stat << (lw + 5)) + (2 * q + (c >> 4)) * 32 + 8 * ((c & 15) >> 2) + 4 * half + (c & 3);
  }
};

// A row's target as the call gives it: its column, or -1 where the row does not count.
__device__ __forceinline__ int target_column(const int64_t *targets, int64_t m, int64_t V,
                                             int64_t ignore_index) {
  const int64_t t = targets[m];
  return t != ignore_index && t >= 0 && t < V ? (int)t : -1;
}

constexpr float kKeptScale = 32768.f;

// One block tile: acc = W_tile Hc_tile^T (rows: vocabulary, columns: tokens), so a lane
// holds 16 TM logits of each of its TN tokens and the strip's values are reductions in
// registers.  What bounds it: the products at D 2048 (bf16, 3686 rows, V 32000: 455 us, 1.06
// PFLOP/s); at D 384 the epilogue, which nothing overlaps (11920 rows, V 50001: 570 us for 458
// GFLOP, 665 with the records: their stores ~50, the places ~30, the second largest ~20).
// Two blocks of half the token columns a CU, 32 k a stage, to overlap it: level without records
// (613 us against 608), 766 against 788 with them, and 20% slower at D 2048.
// stats [crows, nstat], recs [crows, nstat * WTM / 32], tgt [crows].
// KEEP (16-bit inputs): kKeptScale exp(z - mx), mx the strip's maximum, is kept for the backward
// in fp16, E [crows, ldp]: half a step of 2^-11 of each down to 2^-29 of the strip's largest (20
// nats below it), half of 2^-39 of the largest of what is below that.  With bf16, 2^-8, its
// rounding would add to dz's own; the scale, a power of two, puts the largest at the upper end of
// fp16's range.  Blocks past the tiles run the transposes of `tp`.  `targets`: Hc is hidden as it
// lies, all crows rows of it (a middling number of rows, which are not compacted).
template <class C, bool BUF, bool SB, bool TOP, bool KEEP>
__global__ NF_GEMM_BOUNDS(C) void lp_logits_kernel(
    const typename C::TI *W, const typename C::TI *Hc, int64_t V, int64_t D, int64_t j0,
    int64_t crows, const int *n_ptr, const int *tcol, const int64_t *targets,
    int64_t ignore_index, Stat *stats, int nstat, Rec *recs, float *tgt, f16 *E, int64_t ldp,
    int vtiles, int ttiles, gemm::TpJobs tp) {
  __shared__ __attribute__((aligned(16))) char smem[C::LDS_BYTES];
  if constexpr (KEEP) {
    static_assert(C::LDS_BYTES >= gemm::kTpRegionRows * gemm::kTpRegionPitch * 2,
                  "transpose region does not fit the LDS");
    const int q = (int)blockIdx.x - vtiles * ttiles;
    if (q >= 0) {
      if (q < tp.n) gemm::tp_jobs_run<C::NT>(tp, q, reinterpret_cast<uint16_t *>(smem));
      return;
    }
  }
  int vt, tt;
  gemm::group_tile(gemm::xcd_order(blockIdx.x, vtiles * ttiles), vtiles, ttiles,
                   gemm::kTileGroup, vt, tt);
  const int64_t cnt = targets ? crows : chunk_count(n_ptr, j0, crows);
  const int64_t v0 = (int64_t)vt * C::BM;
  const int64_t t0 = (int64_t)tt * C::BN;
  if (t0 >= cnt) return;
  floatx16 acc[C::TM][C::TN];
  gemm::mainloop<C, BUF>(W, D, Hc + j0 * D, D, V, cnt, D, v0, t0, smem, acc);

  const int l = threadIdx.x & 63, half = l >> 5;
  const int w = threadIdx.x >> 6, wm = w / C::WN, wn = w % C::WN;
  const int64_t vtile0 = v0 + wm * C::WTM;
  const int64_t crow0 = vtile0 + 4 * half;
  const int stat = vt * C::WM + wm;
  // rows past the vocabulary: -inf, which adds nothing and comes after any logit
  if (vtile0 + C::WTM > V) {
    const int vlim = (int)(V - crow0 < C::WTM ? V - crow0 : C::WTM);
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int j = 0; j < C::TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (i * 32 + 8 * (r >> 2) + (r & 3) >= vlim) acc[i][j][r] = -INFINITY;
  }
  constexpr int NS = C::TM / 2;  // strips of a lane and token
  using TS = typename std::conditional<KEEP, f16, typename C::TI>::type;
  ce::EStore<C, SB, TS> store;
  if constexpr (KEEP) store.init(E, ldp, nullptr, 0, V, crows, v0, t0, cnt, smem);
#pragma unroll
  for (int j = 0; j < C::TN; ++j) {
    const int64_t tok = t0 + wn * C::WTN + j * 32 + (l & 31);
    float mx = -INFINITY;
    if constexpr (TOP) {
      float first[NS], second[NS];
      uint32_t place[NS];
#pragma unroll
      for (int q = 0; q < NS; ++q) {
        first[q] = second[q] = -INFINITY;
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const float x = acc[2 * q + (c >> 4)][j][c & 15];
          second[q] = __builtin_amdgcn_fmed3f(first[q], second[q], x);
          first[q] = fmaxf(first[q], x);
        }
        place[q] = kNoPlace;
#pragma unroll
        for (int c = 31; c >= 0; --c)
          place[q] = acc[2 * q + (c >> 4)][j][c & 15] == first[q] ? (uint32_t)c : place[q];
        mx = fmaxf(mx, first[q]);
      }
      if (tok < cnt) {
        Rec *dst = recs + (tok * nstat + stat) * (2 * NS) + half * NS;
#pragma unroll
        for (int q = 0; q < NS; ++q) dst[q] = Rec{first[q], bf16_up(second[q]) | place[q]};
      }
    } else {
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, acc[i][j][r]);
    }
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    if (tok < cnt) {  // the target logit, from the one lane that holds it
      const int col = targets ? target_column(targets, tok, V, ignore_index) : tcol[j0 + tok];
      const int64_t loc64 = (int64_t)col - vtile0;
      const int loc = (int)(loc64 >= 0 && loc64 < C::WTM ? loc64 : -1);
      if (loc >= 0 && ((loc >> 2) & 1) == half) {
        const int want = ((loc >> 5) << 4) | (((loc & 31) >> 3) << 2) | (loc & 3);
        float z = 0.f;
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) z = (i * 16 + r == want) ? acc[i][j][r] : z;
        tgt[tok] = z;
      }
    }
    float s = 0.f, t = 0.f;
    const float base = mx == -INFINITY ? 0.f : mx;  // a strip of -inf (and NaN) alone
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float x = acc[i][j][r] - base;
        const float e = exp_f32(x);
        s += e;
        t += (KEEP ? fmaxf(x, kFar) : x) * e;
        acc[i][j][r] = KEEP ? e * kKeptScale : x;
      }
    // -inf * 0 is a NaN: without KEEP, where x is still there, a strip with a logit of -inf (or
    // past the vocabulary) and no NaN is summed again with x bounded.  Bounding every x costs 4%
    // of the tall head (12289 rows, D 384, V 50001, 20 alternatives 756 us against 728).
    if constexpr (!KEEP) {
      if (t != t && s == s) {
        t = 0.f;
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float x = acc[i][j][r];
            t += fmaxf(x, kFar) * exp_f32(x);
          }
      }
    }
    s += __shfl_xor(s, 32);
    t += __shfl_xor(t, 32);
    if (half == 0 && tok < cnt) stats[tok * nstat + stat] = Stat{mx, s, t, 0.f};
    if constexpr (KEEP) store.column(j, acc);
  }
  if constexpr (KEEP) store.finish();
}

// A row of at most 16 tokens against 16 vocabulary rows, k in order in steps of 32, as the
// block tiles' K loop takes them: a: rows of W, b: rows of H.  The lane supplies and k-vectors
// are those of v_mfma_f32_16x16x32_bf16: row lane % 16, k 8 (lane / 16) .. + 7.
template <typename TI>
struct Dot16;
template <>
struct Dot16<bf16> {
  floatx4 acc = {0.f, 0.f, 0.f, 0.f};
  struct Frag {
    u32x4 v;
  };
  // `p`: the lane's row; rows that do not exist are null (zeros)
  template <bool VK>
  __device__ __forceinline__ static Frag load(const bf16 *p, int64_t k, int64_t D) {
    return Frag{load_vec<bf16, VK>(p, 0, p ? 0 : 1, 1, k + 8 * ((threadIdx.x & 63) >> 4), D)};
  }
  __device__ __forceinline__ void add(const Frag &a, const Frag &b) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.v),
                                                  __builtin_bit_cast(bf16x8, b.v), acc, 0, 0, 0);
  }
  __device__ __forceinline__ floatx4 done() const { return acc; }
};
template <>
struct Dot16<float> {  // the products of mainloop_split, in its order
  floatx4 acc = {0.f, 0.f, 0.f, 0.f}, low = {0.f, 0.f, 0.f, 0.f};
  struct Frag {
    u32x4 part[3];
  };
  template <bool VK>
  __device__ __forceinline__ static Frag load(const float *p, int64_t k, int64_t D) {
    u32x4 x[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      x[h] = load_vec<float, VK>(p, 0, p ? 0 : 1, 1, k + 8 * ((threadIdx.x & 63) >> 4) + 4 * h, D);
    Frag f;
    split8(x, f.part);
    return f;
  }
  __device__ __forceinline__ static floatx4 mul(const u32x4 &a, const u32x4 &b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  __device__ __forceinline__ void add(const Frag &a, const Frag &b) {
    acc = mul(a.part[0], b.part[0], acc);
    low = mul(a.part[1], b.part[0], low);
    low = mul(a.part[2], b.part[0], low);
    low = mul(a.part[0], b.part[1], low);
    low = mul(a.part[1], b.part[1], low);
    low = mul(a.part[0], b.part[2], low);
  }
  __device__ __forceinline__ floatx4 done() const {
    floatx4 r;
#pragma unroll
    for (int q = 0; q < 4; ++q) r[q] = __builtin_isfinite(acc[q]) ? acc[q] + low[q] : acc[q];
    return r;
  }
};

// The logits of at most 16 NT rows of fp32, hidden used as it lies (no compaction).  What bounds
// it is reading W once: a wavefront streams 32 rows of W past the matrix pipe straight from
// memory, two steps of 32 k at a time, and the hidden rows come from the caches.  A wavefront's
// 32 columns are one strip: for token lane % 16 (+ 16 nt) a lane has columns 16 h +
// 4 (lane / 16) + q, joined over the four lane groups.  V 32000, with lp_finish, in a graph,
// against the tiles of MidCfg (which split 128 rows for every block): D 2048, 16 rows 66 us
// against 116, 32 rows 80 against 116, 64 rows 117 against 116; D 384 24, 28 and 39 against
// 31, 32 and 32.  In bf16 the tiles are the faster from 8 rows on (D 2048 26.6 us against 31.2, 64
// rows 27.9 against 55).
constexpr int kSkinnyThreads = 256;
template <typename TI>
constexpr int64_t kSkinnyRows = sizeof(TI) == 4 ? 32 : 0;

template <typename TI, int NT, bool VK>
__global__ __launch_bounds__(kSkinnyThreads) void lp_skinny_kernel(
    const TI *__restrict__ W, const TI *__restrict__ H, const int64_t *__restrict__ targets,
    int64_t M, int64_t V, int64_t D, int64_t ignore_index, Stat *__restrict__ stats, int nstat,
    Rec *__restrict__ recs, float *__restrict__ tgt) {
  using Frag = typename Dot16<TI>::Frag;
  const int l = threadIdx.x & 63;
  const int64_t strip = (int64_t)blockIdx.x * (kSkinnyThreads / 64) + (threadIdx.x >> 6);
  const int64_t v0 = strip * 32;
  if (v0 >= V) return;
  const TI *wrow[2], *hrow[NT];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t v = v0 + 16 * h + (l & 15);
    wrow[h] = v < V ? W + v * D : nullptr;
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int64_t m = 16 * n + (l & 15);
    hrow[n] = m < M ? H + m * D : nullptr;
  }
  Dot16<TI> acc[2][NT];
  constexpr int kDepth = 2;
  for (int64_t k0 = 0; k0 < D; k0 += 32 * kDepth) {
    Frag a[kDepth][2], b[kDepth][NT];
#pragma unroll
    for (int u = 0; u < kDepth; ++u) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        a[u][h] = Dot16<TI>::template load<VK>(wrow[h], k0 + 32 * u, D);
#pragma unroll
      for (int n = 0; n < NT; ++n)
        b[u][n] = Dot16<TI>::template load<VK>(hrow[n], k0 + 32 * u, D);
    }
#pragma unroll
    for (int u = 0; u < kDepth; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[h][n].add(a[u][h], b[u][n]);
  }
  const int grp = l >> 4;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int64_t tok = 16 * n + (l & 15);
    float z[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const floatx4 d = acc[h][n].done();
#pragma unroll
      for (int q = 0; q < 4; ++q)
        z[4 * h + q] = v0 + 16 * h + 4 * grp + q < V ? d[q] : -INFINITY;
    }
    float first = -INFINITY, second = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      second = __builtin_amdgcn_fmed3f(first, second, z[e]);
      first = fmaxf(first, z[e]);
    }
    int place = (int)kNoPlace;
#pragma unroll
    for (int e = 7; e >= 0; --e)
      place = z[e] == first ? 16 * (e >> 2) + 4 * grp + (e & 3) : place;
#pragma unroll
    for (int d = 16; d < 64; d <<= 1) {
      const float of = __shfl_xor(first, d), os = __shfl_xor(second, d);
      const int op = __shfl_xor(place, d);
      second = fmaxf(fminf(first, of), fmaxf(second, os));
      place = of > first || (of == first && op < place) ? op : place;
      first = fmaxf(first, of);
    }
    const float base = first == -INFINITY ? 0.f : first;
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = z[e] - base;
      const float ex = exp_f32(x);
      s += ex;
      t += fmaxf(x, kFar) * ex;
    }
    s += __shfl_xor(s, 16);
    t += __shfl_xor(t, 16);
    s += __shfl_xor(s, 32);
    t += __shfl_xor(t, 32);
    if (tok >= M) continue;
    if (grp == 0) {
      stats[tok * nstat + strip] = Stat{first, s, t, 0.f};
      if (recs) recs[tok * nstat + strip] = Rec{first, bf16_up(second) | (uint32_t)place};
    }
    const int64_t loc = (int64_t)target_column(targets, tok, V, ignore_index) - v0;
    if (loc >= 0 && loc < 32 && ((loc & 15) >> 2) == grp) {
      const int want = 4 * (int)(loc >> 4) + (int)(loc & 3);
      float x = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) x = e == want ? z[e] : x;
      tgt[tok] = x;
    }
  }
}

// ---------------------------------------------------------------------------
// 3. a row's outputs, one wavefront a row: the statistics joined in a fixed order
// (log p and the entropy follow: lse = mx + log S, H = log S - T / S), then the
// alternatives from the strips' records.  Its time is latency: 8 rows, V 32000, 8 alternatives
// 8 us, 3686 rows 28 us, of which the strips formed again (D 2048, at most a few a row) are most.
// ---------------------------------------------------------------------------
constexpr int kFinishThreads = 256;

__device__ __forceinline__ Stat join(const Stat &a, const Stat &b) {
  const float m = fmaxf(a.mx, b.mx), base = m == -INFINITY ? 0.f : m;
  const float xa = fmaxf(a.mx - base, kFar), xb = fmaxf(b.mx - base, kFar);
  const float ea = exp_f32(a.mx - base), eb = exp_f32(b.mx - base);
  return Stat{m, a.s * ea + b.s * eb, (a.t + a.s * xa) * ea + (b.t + b.s * xb) * eb, 0.f};
}

// (va, column ia) comes before (vb, ib): the larger value, of equals the lower column
__device__ __forceinline__ bool before(float va, int ia, float vb, int ib) {
  return va > vb || (va == vb && ia < ib);
}

// the wavefront's first (v, i) in that order, in every lane; `tag` goes with it
__device__ __forceinline__ void wave_first(float &v, int &i, int &tag) {
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const float ov = __shfl_xor(v, d);
    const int oi = __shfl_xor(i, d), ot = __shfl_xor(tag, d);
    if (before(ov, oi, v, i)) {
      v = ov;
      i = oi;
      tag = ot;
    }
  }
}

// A row's chosen strips, in the order of their first logits, and the logits that can be among
// its top_k: the firsts of strips that have no other, all of those that were formed again.
struct Chosen {
  float v[kMaxTop];
  int strip[kMaxTop];
  float cand_v[kMaxTop * 32];
  int cand_col[kMaxTop * 32];
  float again[32];  // a strip's logits
};

// A wavefront's own LDS writes are done before its later reads.
__device__ __forceinline__ void wave_lds_fence() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  asm volatile("" ::: "memory");
}

// The strips whose first logits come first among those after (pv, pi), from entry `found` on;
// how many there are then.  Every round reads the records again.
__device__ __forceinline__ int choose_slow(const Rec *rc, int nrec, const Strips &strips,
                                           int64_t V, int K, Chosen &ch, int found, float pv,
                                           int pi) {
  const int l = threadIdx.x & 63;
  for (; found < K; ++found) {
    float bv = -INFINITY;
    int bi = 0x7fffffff, bs = -1;
    for (int q = l; q < nrec; q += 64) {
      const Rec r = rc[q];
      const uint32_t place = r.rest & 63u;
      if (place == kNoPlace) continue;
      const int col = strips.column(q, (int)place);
      if (col < V && before(pv, pi, r.first, col) && before(r.first, col, bv, bi)) {
        bv = r.first;
        bi = col;
        bs = q;
      }
    }
    wave_first(bv, bi, bs);
    if (bs < 0) break;  // the same in every lane
    if (l == 0) {
      ch.v[found] = bv;
      ch.strip[found] = bs;
    }
    pv = bv;
    pi = bi;
  }
  return found;
}

// The same with the first logits in registers, NR a lane (lane l: strips l, l + 64, ...).
//
// From kRankedTop alternatives on: the K-th largest of the 64 lanes' maxima bounds what can be
// among them from below, and what is left by it, about 64 log(64 / (64 - K)) strips, is ranked.
// Forward in a graph against the rounds below, bf16: D 384, 12289 rows, V 50001, 20 alternatives
// 714 us against 767, 8 699 against 716, 4 level, 2 690 against 688; 4096 rows, V 5000, 8 61
// against 66; 8 rows, D 2048, V 32000, 32 49 against 62, 8 29.8 against 31.7, 1 29.5 against 28.6.
//
// Fewer, or more than 64 left (equal logits), or less than K lanes with a logit above -inf: in
// rounds.  Each lane keeps its maximum; a round takes the wavefront's and clears the register
// that held it.  Of equal values the lower column: within a lane the earlier register (64 strips
// are whole statistics strips), between lanes by the records.  Ends at logits of -inf, which
// choose_slow orders.
constexpr int kRankedTop = 4;
template <int NR>
__device__ __forceinline__ int choose(const Rec *rc, int nrec, const Strips &strips, int64_t V,
                                      int K, Chosen &ch) {
  const int l = threadIdx.x & 63;
  float v[NR], best = -INFINITY;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int q = l + 64 * i;
    v[i] = q < nrec ? rc[q].first : -INFINITY;
    best = fmaxf(best, v[i]);
  }
  auto column_of = [&](int strip) { return strips.column(strip, (int)(rc[strip].rest & 63u)); };
  if (K >= kRankedTop) {
    // `last`: the K-th largest of the lanes' maxima, equal ones counted; K firsts are no less
    int above = 0;
#pragma unroll
    for (int j = 0; j < 64; ++j)
      above += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(best), j)) > best ? 1 : 0;
    const float last = -wave_max(above < K ? -best : -INFINITY);
    int n = 0;
    if (last > -INFINITY) {
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const uint64_t may = __ballot(v[i] >= last);
        if (!may) continue;
        const int q = n + __popcll(may & ((1ull << l) - 1ull));
        if (((may >> l) & 1) && q < 64) {
          ch.cand_v[q] = v[i];
          ch.cand_col[q] = l + 64 * i;
        }
        n += __popcll(may);
      }
    }
    if (n > 0 && n <= 64) {
      wave_lds_fence();
      const float x = l < n ? ch.cand_v[l] : -INFINITY;
      const int strip = l < n ? ch.cand_col[l] : 0;
      const int col = column_of(strip);
      int place = 0;
      for (int j = 0; j < n; ++j)
        place += before(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), j)),
                        __builtin_amdgcn_readlane(col, j), x, col)
                     ? 1
                     : 0;
      if (l < n && place < K) {
        ch.v[place] = x;
        ch.strip[place] = strip;
      }
      return K;
    }
  }
  int found = 0, pi = -1;
  float pv = INFINITY;
  while (found < K) {
    const float mx = wave_max(best);
    if (mx == -INFINITY) break;
    const uint64_t held = __ballot(best == mx);
    // the register that holds it, in every lane that has it
    int at = 0;
#pragma unroll
    for (int i = NR - 1; i >= 0; --i) at = v[i] == mx ? i : at;
    int win = __ffsll((unsigned long long)held) - 1;
    if (held & (held - 1)) {  // more than one lane: seldom
      int col = (held >> l) & 1 ? column_of(l + 64 * at) : 0x7fffffff, tag = l;
      float same = 0.f;
      wave_first(same, col, tag);
      win = __builtin_amdgcn_readfirstlane(tag);
    }
    const int slot = __builtin_amdgcn_readlane(at, win), strip = win + 64 * slot;
    if (l == 0) {
      ch.v[found] = mx;
      ch.strip[found] = strip;
    }
    ++found;
    pv = mx;
    pi = strip;  // its column is looked up below, if need be
    best = -INFINITY;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      v[i] = l == win && i == slot ? -INFINITY : v[i];
      best = fmaxf(best, v[i]);
    }
  }
  if (found == K) return K;
  return choose_slow(rc, nrec, strips, V, K, ch, found, pv, found ? column_of(pi) : -1);
}

// NR: records in a lane's registers (0: more than fit, read in every round).  `targets`: the
// pass whose rows are not compacted: rows that do not count get their zeros here, and the state
// is written for the backward (Hc null: none will come).
template <typename TI, bool VK, int NR>
__global__ __launch_bounds__(kFinishThreads) void lp_finish_kernel(
    const TI *W, const TI *H, int64_t V, int64_t D, const Stat *__restrict__ stats, int nstat,
    const Rec *__restrict__ recs, Strips strips, const float *__restrict__ tgt, int64_t j0,
    int64_t crows, int *n_ptr, int *rows, int *tcol, int *pos, TI *Hc, int64_t lo0,
    const int64_t *__restrict__ targets, int64_t ignore_index, float *__restrict__ mx_out,
    float *__restrict__ ls_out, float *__restrict__ ent_out, float *__restrict__ lp_out,
    RowOut out) {
  constexpr int kWaves = kFinishThreads / 64;
  __shared__ Chosen chosen_w[kWaves];
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t row = (int64_t)blockIdx.x * kWaves + w;
  const int K = out.top_k;
  int64_t m;
  const TI *hrow;
  if (targets) {
    if (row >= (lo0 > 0 ? lo0 : crows)) return;
    m = row;
    hrow = H + row * D;
    const int tc = row < crows ? target_column(targets, row, V, ignore_index) : -1;
    constexpr int VE = VK ? 16 / (int)sizeof(TI) : 1;
    for (int64_t c = (int64_t)l * VE; Hc && c < D; c += 64 * VE) {
      if constexpr (VK) {
        u32x4 x = {0u, 0u, 0u, 0u};
        if (tc >= 0) x = *reinterpret_cast<const u32x4 *>(hrow + c);
        *reinterpret_cast<u32x4 *>(Hc + row * D + c) = x;
        if (lo0 > 0) *reinterpret_cast<u32x4 *>(Hc + (lo0 + row) * D + c) = x;
      } else {
        const TI x = tc >= 0 ? hrow[c] : static_cast<TI>(0.f);
        Hc[row * D + c] = x;
        if (lo0 > 0) Hc[(lo0 + row) * D + c] = x;
      }
    }
    if (row >= crows) return;  // padding of the two copies
    if (l == 0) {
      rows[row] = (int)row;
      pos[row] = (int)row;
      tcol[row] = tc;
      if (row == 0) *n_ptr = (int)crows;
    }
    if (tc < 0) {
      if (l == 0) {
        mx_out[row] = 0.f;
        ls_out[row] = 0.f;
        ent_out[row] = 0.f;
        out.logprob[row] = 0.f;
        out.entropy[row] = 0.f;
      }
      if (l < K) {
        out.top_lp[row * K + l] = 0.f;
        out.top_id[row * K + l] = -1;
      }
      return;
    }
  } else {
    if (row >= chunk_count(n_ptr, j0, crows)) return;
    m = rows[j0 + row];
    hrow = H + (j0 + row) * D;
  }
  const Stat *st = stats + row * nstat;
  Stat a{-INFINITY, 0.f, 0.f, 0.f};
  for (int k = l; k < nstat; k += 64) a = join(a, st[k]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1)
    a = join(a, Stat{__shfl_xor(a.mx, d), __shfl_xor(a.s, d), __shfl_xor(a.t, d), 0.f});
  const float ls = log_f32(a.s), ent = ls - a.t / a.s;
  auto logprob = [&](float z) { return (z - a.mx) - ls; };
  if (l == 0) {
    mx_out[j0 + row] = a.mx;
    ls_out[j0 + row] = ls;
    ent_out[j0 + row] = ent;
    lp_out[j0 + row] = logprob(tgt[row]);
    out.logprob[m] = logprob(tgt[row]);
    out.entropy[m] = ent;
  }
  if (K == 0) return;
  Chosen &ch = chosen_w[w];
  const int nrec = nstat * strips.per_stat();
  const Rec *rc = recs + row * nrec;
  int found;
  if constexpr (NR > 0)
    found = choose<NR>(rc, nrec, strips, V, K, ch);
  else
    found = choose_slow(rc, nrec, strips, V, K, ch, 0, INFINITY, -1);
  wave_lds_fence();  // lane 0 wrote `ch` for all
  // a strip whose second logit may come before the last of them is formed again; with fewer
  // than K strips every strip is among them, and each is formed again
  const float last = found < K ? -INFINITY : ch.v[K - 1];
  bool need = false;
  int col = -1;
  float val = 0.f;
  if (l < found) {
    const uint32_t rest = rc[ch.strip[l]].rest;
    need = __uint_as_float(rest & 0xffff0000u) >= last;
    col = strips.column(ch.strip[l], (int)(rest & 63u));
    val = ch.v[l];
  }
  const uint64_t redo = __ballot(need);
  if (redo == 0) {  // the first logits of the chosen strips are the row's K first
    if (l < K) {
      out.top_lp[m * K + l] = l < found ? logprob(val) : __builtin_nanf("");
      out.top_id[m * K + l] = l < found ? col : -1;
    }
    return;
  }
  const uint64_t alone = __ballot(l < found && !need);
  int n = __popcll(alone);  // candidates
  if ((alone >> l) & 1) {
    const int q = __popcll(alone & ((1ull << l) - 1ull));
    ch.cand_v[q] = val;
    ch.cand_col[q] = col;
  }
  for (uint64_t todo = redo; todo; todo &= todo - 1) {
    const int strip = ch.strip[__ffsll((unsigned long long)todo) - 1];
    Dot16<TI> acc[2];
    const TI *wrow[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = strips.column(strip, 16 * h + (l & 15));
      wrow[h] = c < V ? W + (int64_t)c * D : nullptr;
    }
    constexpr int kDepth = sizeof(TI) == 2 ? 8 : 2;
    for (int64_t k0 = 0; k0 < D; k0 += 32 * kDepth) {
      typename Dot16<TI>::Frag fa[kDepth][2], fb[kDepth];
#pragma unroll
      for (int u = 0; u < kDepth; ++u) {
        fb[u] = Dot16<TI>::template load<VK>(hrow, k0 + 32 * u, D);
#pragma unroll
        for (int h = 0; h < 2; ++h)
          fa[u][h] = Dot16<TI>::template load<VK>(wrow[h], k0 + 32 * u, D);
      }
#pragma unroll
      for (int u = 0; u < kDepth; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) acc[h].add(fa[u][h], fb[u]);
    }
    // every column of the product is this token: lane l has places 4 (l / 16) .. + 3
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const floatx4 z = acc[h].done();
      if ((l & 15) == 0)
#pragma unroll
        for (int q = 0; q < 4; ++q) ch.again[16 * h + 4 * (l >> 4) + q] = z[q];
    }
    wave_lds_fence();
    // those that do not come after the last of the chosen strips' firsts (NaN: none)
    const float x = ch.again[l & 31];
    const int c = strips.column(strip, l & 31);
    const uint64_t may = __ballot(l < 32 && c < V && x >= last);
    if ((may >> l) & 1) {
      const int q = n + __popcll(may & ((1ull << l) - 1ull));
      ch.cand_v[q] = x;
      ch.cand_col[q] = c;
    }
    n += __popcll(may);
    wave_lds_fence();
  }
  wave_lds_fence();
  // a candidate's place is the number of those before it
  for (int q0 = 0; q0 < n; q0 += 64) {
    const int q = q0 + l;
    const float x = q < n ? ch.cand_v[q] : 0.f;
    const int c = q < n ? ch.cand_col[q] : 0;
    int place = 0;
    for (int j0 = 0; j0 < n; j0 += 64) {
      const float y = j0 + l < n ? ch.cand_v[j0 + l] : 0.f;
      const int d = j0 + l < n ? ch.cand_col[j0 + l] : 0;
      const int m0 = n - j0 < 64 ? n - j0 : 64;
      for (int j = 0; j < m0; ++j)
        place += before(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(y), j)),
                        __builtin_amdgcn_readlane(d, j), x, c)
                     ? 1
                     : 0;
    }
    if (q < n && place < K) {
      out.top_lp[m * K + place] = logprob(x);
      out.top_id[m * K + place] = c;
    }
  }
  if (l >= n && l < K) {  // none left that compares
    out.top_lp[m * K + l] = __builtin_nanf("");
    out.top_id[m * K + l] = -1;
  }
}

// ---------------------------------------------------------------------------
// backward: dz of one chunk, in the layouts of ce::EStore, the logits formed again.  Bound as
// lp_logits: fp32, 439 rows, D 384, V 32000 92 us where lp_logits takes 77.
// ---------------------------------------------------------------------------
struct RowIn {
  const int *n, *rows, *tcol;        // compacted rows
  const float *mx, *ls, *ent, *lp;   // per compacted row: lse = mx + ls
  const float *g, *h;                // upstream, per row of hidden; either may be null
};

// With few rows one entry of dz can make up most of a gradient, and its one rounding to 16
// bits all of the gradient's error (up to 2^-8, measured 3.8e-3 where 1.7e-3 is what the
// output's own rounding leaves; over many rows the roundings average out).  Up to kFewRows
// rows dz is therefore held as two 16-bit terms, dz = hi + lo: row r of the products is hi,
// row lo0 + r is lo, on a second copy of the hidden row.  The rows come free: the tiles have
// 256 of them.
constexpr int64_t kFewRows = 128;
template <typename TI>
int64_t few_rows(int64_t M) {  // lo0; 0: dz is one term
  return sizeof(TI) == 2 && M <= kFewRows ? round_up(M, 8) : 0;
}

template <class C, bool BUF, bool SB>
__global__ NF_GEMM_BOUNDS(C) void lp_dz_kernel(
    const typename C::TI *W, const typename C::TI *Hc, int64_t V, int64_t D, int64_t j0,
    int64_t crows, RowIn in, int64_t lo0, int *two, float *ones, typename C::TI *E, int64_t ldp,
    typename C::TI *ET, int64_t ldet, int vtiles, int ttiles, gemm::TpJobs tp) {
  using TI = typename C::TI;
  constexpr int ES = (int)sizeof(TI);
  __shared__ __attribute__((aligned(16))) char smem[C::LDS_BYTES];
  if constexpr (ES == 2) {
    static_assert(C::LDS_BYTES >= gemm::kTpRegionRows * gemm::kTpRegionPitch * 2,
                  "transpose region does not fit the LDS");
    const int q = (int)blockIdx.x - vtiles * ttiles;
    if (q >= 0) {
      if (q < tp.n) gemm::tp_jobs_run<C::NT>(tp, q, reinterpret_cast<uint16_t *>(smem));
      return;
    }
  }
  int vt, tt;
  gemm::group_tile(gemm::xcd_order(blockIdx.x, vtiles * ttiles), vtiles, ttiles,
                   gemm::kTileGroup, vt, tt);
  const int64_t live = chunk_count(in.n, j0, crows);
  const int64_t cnt = lo0 > 0 ? 2 * lo0 : live;
  const int64_t v0 = (int64_t)vt * C::BM;
  const int64_t t0 = (int64_t)tt * C::BN;
  if (t0 >= cnt) return;
  if (lo0 > 0 && blockIdx.x == 0 && threadIdx.x == 0) *two = (int)cnt;
  // the gradient products' row factor is one: dz carries every factor
  if (vt == 0 && threadIdx.x < C::BN && t0 + threadIdx.x < cnt) ones[j0 + t0 + threadIdx.x] = 1.f;
  floatx16 acc[C::TM][C::TN];
  gemm::mainloop<C, BUF>(W, D, Hc + j0 * D, D, V, cnt, D, v0, t0, smem, acc);

  const int l = threadIdx.x & 63, half = l >> 5;
  const int w = threadIdx.x >> 6, wm = w / C::WN, wn = w % C::WN;
  const int64_t vtile0 = v0 + wm * C::WTM;
  const int64_t crow0 = vtile0 + 4 * half;
  // rows past the vocabulary: -inf, whose dz is 0
  if (vtile0 + C::WTM > V) {
    const int vlim = (int)(V - crow0 < C::WTM ? V - crow0 : C::WTM);
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int j = 0; j < C::TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (i * 32 + 8 * (r >> 2) + (r & 3) >= vlim) acc[i][j][r] = -INFINITY;
  }
  ce::EStore<C, SB> store;
  store.init(E, ldp, ET, ldet, V, crows, v0, t0, cnt, smem);
#pragma unroll
  for (int j = 0; j < C::TN; ++j) {
    const int64_t tok = t0 + wn * C::WTN + j * 32 + (l & 31);
    float g = 0.f, h = 0.f, mx = 0.f, ls = 0.f, ent = 0.f;
    int want = -1;  // the register that holds the target, if this lane does
    const bool low = lo0 > 0 && tok >= lo0;
    const int64_t row = j0 + (low ? tok - lo0 : tok);
    bool counts = false;
    if (row - j0 < live) {
      const int64_t m = in.rows[row];
      const int tc = in.tcol[row];
      counts = tc >= 0;
      if (counts) {
        g = in.g ? in.g[m] : 0.f;
        h = in.h ? in.h[m] : 0.f;
      }
      mx = in.mx[row];
      ls = in.ls[row];
      ent = in.ent[row];
      const int64_t loc64 = (int64_t)tc - vtile0;
      const int loc = (int)(loc64 >= 0 && loc64 < C::WTM ? loc64 : -1);
      if (loc >= 0 && ((loc >> 2) & 1) == half)
        want = ((loc >> 5) << 4) | (((loc & 31) >> 3) << 2) | (loc & 3);
    }
    // a row that does not count, or of the padding: its hidden row is zero here, but an
    // infinity in weight makes a NaN of its logits
    if (!counts) {
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    }
    const float a = -(g + h * ent);
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float x = (acc[i][j][r] - mx) - ls;
        // exp is 0 where x is -inf, and a NaN where it is one
        const float dz = exp_f32(x) * (a - h * fmaxf(x, kFar));
        acc[i][j][r] = i * 16 + r == want ? dz + g : dz;
        if constexpr (ES == 2)
          if (low) acc[i][j][r] -= static_cast<float>(static_cast<TI>(acc[i][j][r]));
      }
    store.column(j, acc);
  }
  store.finish();
}

// dz of one chunk from what the forward kept, E [crows, ldp] in fp16: with mx the strip's
// maximum and e = E / kKeptScale, p = e exp(mx - lse) and z - lse = log e + mx - lse.  The
// target's own entry is formed from the row's logprob, an fp32 value: 1 - p of a sure token would
// be lost in E's rounding.  A thread takes 8 columns of a row (they lie in one strip).
constexpr int kKeptThreads = 256;
constexpr int64_t kKeptCols = (int64_t)1 << 26;  // the grid's second extent ends at 65535 blocks
constexpr int64_t kKeptRows = kMaxLaunchThreads / kKeptThreads - 8;  // and its first

template <int WTM>
__global__ __launch_bounds__(kKeptThreads) void lp_from_kept_kernel(
    const f16 *__restrict__ E, bf16 *__restrict__ dz, int64_t ldp, int64_t V,
    const Stat *__restrict__ stats, int nstat, RowIn in, float *__restrict__ ones) {
  const int64_t row = blockIdx.x, live = *in.n;
  if (row >= (live + 7) / 8 * 8) return;
  const int64_t c = ((int64_t)blockIdx.y * kKeptThreads + threadIdx.x) * 8;
  if (c >= ldp) return;
  float v[8];
  if (row >= live) {  // the products' K padding
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
    Chunk8<bf16>::store(dz + row * ldp + c, v);
    return;
  }
  const int64_t m = in.rows[row];
  const float g = in.g ? in.g[m] : 0.f, h = in.h ? in.h[m] : 0.f;
  const float mx = in.mx[row], ls = in.ls[row], ent = in.ent[row], a = -(g + h * ent);
  if (c == 0) ones[row] = 1.f;
  Chunk8<f16>::load(E + row * ldp + c, v);
  if (c < V) {
    const float o = (stats[row * nstat + c / WTM].mx - mx) - ls;
    const float f = exp_f32(o);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] *= 1.f / kKeptScale;
      // log 0 = -inf goes with p = 0; a NaN stays one through p
      const float x = h != 0.f ? fmaxf(log_f32(v[i]) + o, kFar) : 0.f;
      v[i] = v[i] * f * (a - h * x);
    }
    const int64_t t = in.tcol[row] - c;
    if (t >= 0 && t < 8) {
      const float lp = in.lp[row];
      const float own = exp_f32(lp) * (a - h * fmaxf(lp, kFar)) + g;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i == t ? own : v[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
  }
  Chunk8<bf16>::store(dz + row * ldp + c, v);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// Whether the dH product of M rows reads weight as it lies (its K loop over an N-major operand
// is the slower one, 1.9 against 1.65 us a stage, and there are M / 256 rows of tiles) and not
// a transpose made for it (which moves V D twice).  bf16, V 32000, forward and backward: D 2048,
// 5 rows 157 us against 220, 300 rows 232 against 282, 512 rows 276 against 328, 768 rows 413
// against 414; D 384 62 against 73, 88 against 94, 112 against 107, 131 against 136.
inline bool weight_as_is(int64_t M, int64_t D, int64_t V) {
  return M <= 256 + D / 4 && D % 8 == 0 && sb_ok(V * D * (int64_t)sizeof(bf16));
}

// The tiling for `rows` rows, as MidCfg names them, or -1: the main tiles, which are also the
// better ones where the smaller ones' 128 rows make more than a block a CU, from 256 * 128 =
// 32768 tokens on (V 43813, D 304, 178 rows, forward and backward: 91 us against 109; V 128256,
// D 1024, 128 rows, forward 180 against 188; the fp32 backward, V 85667, D 1432, 47 rows, with
// the forward 1176 against 1233, V 50001, D 384, 33 rows 200 against 217; that forward takes
// Tall64).  bf16 of up to 64 rows gains from its 64 columns at every V.
template <typename TI>
int mid_form(int64_t rows, int64_t V) {
  if (rows <= 64 && (sizeof(TI) == 2 || V <= 32768)) return 64;
  if (rows > 256 || V > 32768) return -1;
  return rows <= 128 ? 128 : 256;
}

template <typename TI>
ce::Plan grad_plan(int64_t M, int64_t D, int64_t V, int64_t chunk_rows) {
  const int64_t lo0 = few_rows<TI>(M);
  return ce::make_plan<TI, false>(lo0 > 0 ? 2 * lo0 : M, D, V, chunk_rows);
}

// What the forward keeps for the backward: the rows, and, with `keep`, where one chunk takes
// every row (by chunk_rows' bound on memory), exp(z - mx) of every logit with the strips'
// statistics and the transposes of weight and of the rows that the products read: the
// backward then forms dz in one pass over it instead of forming the logits again.  M 4096,
// D 2048, V 32000, 10% left out: forward and backward 1513 us, against 1828 with the logits
// formed twice (the kernel lp_from_kept takes 96 us, 5.5 TB/s, in the place of 528 of lp_dz;
// keeping costs lp_logits 60).  178 rows, D 1024: 123 us against 129; with a narrower D forming
// them again on MidCfg's tiles is the faster (D 384: 73 against 75).
struct State {
  bool kept, as_is;  // as_is: no transpose of weight among it
  int nstat;
  int64_t lo0;
  size_t scal, rows, tcol, pos, mx, ls, ent, lp, hc, e, stats, wt, hct, total;
};
template <typename TI>
State state_layout(int64_t M, int64_t D, int64_t V, int64_t chunk_rows, bool keep) {
  using C = MainCfg<TI>;
  State s{};
  s.lo0 = few_rows<TI>(M);
  size_t o = 0;
  auto take = [&](size_t bytes) { const size_t at = o; o = align256(o + bytes); return at; };
  s.scal = take(64);
  s.rows = take((size_t)M * sizeof(int));
  s.tcol = take((size_t)M * sizeof(int));
  s.pos = take((size_t)M * sizeof(int));
  s.mx = take((size_t)M * sizeof(float));
  s.ls = take((size_t)M * sizeof(float));
  s.ent = take((size_t)M * sizeof(float));
  s.lp = take((size_t)M * sizeof(float));
  s.hc = take((size_t)(s.lo0 > 0 ? 2 * s.lo0 : M) * D * sizeof(TI));
  if (sizeof(TI) == 2 && keep && M > kFewRows && M <= kKeptRows && V <= kKeptCols &&
      (D >= 1024 || mid_form<TI>(M, V) < 0)) {
    const ce::Plan L = grad_plan<TI>(M, D, V, chunk_rows);
    if (L.nch == 1) {
      s.kept = true;
      s.nstat = (int)((V + C::BM - 1) / C::BM) * C::WM;
      s.e = take((size_t)L.crows * L.ldp * sizeof(f16));
      s.stats = take((size_t)L.crows * s.nstat * sizeof(Stat));
      s.as_is = weight_as_is(M, D, V);
      s.wt = take(s.as_is ? 0 : (size_t)D * L.ldwt * sizeof(TI));
      s.hct = take((size_t)D * L.ldht * sizeof(TI));
    }
  }
  s.total = o;
  return s;
}
template <typename TI>
struct View {
  int *n;
  float *inv;
  int *rows, *tcol, *pos;
  float *mx, *ls, *ent, *lp;
  TI *Hc, *Wt, *Hct;
  f16 *E;
  Stat *stats;
  View(const State &L, char *s)
      : n(reinterpret_cast<int *>(s + L.scal)),
        inv(reinterpret_cast<float *>(s + L.scal + 16)),
        rows(reinterpret_cast<int *>(s + L.rows)),
        tcol(reinterpret_cast<int *>(s + L.tcol)),
        pos(reinterpret_cast<int *>(s + L.pos)),
        mx(reinterpret_cast<float *>(s + L.mx)),
        ls(reinterpret_cast<float *>(s + L.ls)),
        ent(reinterpret_cast<float *>(s + L.ent)),
        lp(reinterpret_cast<float *>(s + L.lp)),
        Hc(reinterpret_cast<TI *>(s + L.hc)),
        Wt(reinterpret_cast<TI *>(s + L.wt)),
        Hct(reinterpret_cast<TI *>(s + L.hct)),
        E(reinterpret_cast<f16 *>(s + L.e)),
        stats(reinterpret_cast<Stat *>(s + L.stats)) {}
};

// W^T (the dH product's B operand) and Hc^T (the dW product's), both zero-padded: as extra
// blocks (`tp`) of a launch of tiles where their rows are whole 16-byte vectors of 16-bit
// elements, else by launches of their own.
template <typename TI>
int transposes(const TI *W, const TI *Hc, int64_t Mb, int64_t D, int64_t V, const ce::Plan &L,
               TI *Wt, TI *Hct, gemm::TpJobs &tp, hipStream_t s) {  // Wt null: Hc^T alone
  using U = typename std::conditional<sizeof(TI) == 2, uint16_t, uint32_t>::type;
  tp = gemm::TpJobs{};
  if (sizeof(TI) == 2 && D % 8 == 0 && aligned16(W)) {
    auto add = [&](int j, const TI *in, int64_t R, TI *out, int64_t ldo) {
      tp.in[j] = reinterpret_cast<const uint16_t *>(in);
      tp.out[j] = reinterpret_cast<uint16_t *>(out);
      tp.R[j] = R;
      tp.Cn[j] = D;
      tp.ldi[j] = D;
      tp.ldo[j] = ldo;
      tp.rb[j] = (int)((ldo + gemm::kTpRegionRows - 1) / gemm::kTpRegionRows);
      tp.cb[j] = (int)((D + gemm::kTpRegionCols - 1) / gemm::kTpRegionCols);
      tp.n += tp.rb[j] * tp.cb[j];
    };
    add(0, Hc, Mb, Hct, L.ldht);
    if (Wt) add(1, W, V, Wt, L.ldwt);
    return NF_OK;
  }
  if (Wt)
    if (int e = launch_transpose<U>(W, V, D, D, Wt, L.ldwt, s)) return e;
  return launch_transpose<U>(Hc, Mb, D, D, Hct, L.ldht, s);
}

// Tilings for up to 64, 128 and 256 rows, where the cross entropy's tile of 256 x 256 leaves
// half of the CUs without a block and most of its token columns empty: 128 rows of W a block
// (V 32000 is a block a CU) and more stages.  What bounds them is reading W once.  bf16, V
// 32000, forward in a graph, against the main tiles after a compaction: D 2048, 8 rows 26.6 us
// (the 131 MB of W partly in the Infinity Cache) against 59, 128 rows 36.9 against 60, 256 rows
// 43 against 61; D 384 12.1 against 25, 15.3 against 25, 17.8 against 26.  fp32, 128 rows: D
// 2048 130 us against 161, D 384 33 against 45.
// Tall64: fp32 of 33 to 64 rows where the 128 rows of W would make more than a block a CU, with no
// empty token columns: 64 rows, V 85667, D 1024 158 us against 178 on the main tiles, V 33000 70
// against 89, V 128256, D 2048 320 against 356, D 256 57 against 69.
template <typename TI>
struct MidCfg;
template <>
struct MidCfg<bf16> {
  using T64 = DCfg<128, 64, 2, 2, 4, 64>;
  using T128 = DCfg<128, 128, 2, 2, 4, 64>;
  using T256 = DCfg<128, 256, 2, 4, 3, 64>;
};
template <>
struct MidCfg<float> {
  using T64 = SplitCfg<128, 128, 2, 2>;
  using T128 = T64;
  using T256 = SplitCfg<256, 128, 4, 2>;
  using Tall64 = SplitCfg<256, 64, 4, 1>;
};

// A chunk's statistics and records take 3/8 V bytes a row (fp32: 1/2 V) against the 4 V of
// the logits that chunk_rows bounds, so a chunk has up to 8 chunk_rows rows.
struct FwdPlan {
  // 0: the skinny pass; 64, 128, 256: MidCfg's tiles; kTall64: Tall64; -1: the main ones, compacted
  int form;
  int64_t crows;
  int nstat, vtiles, ttiles;
  Strips strips;
  size_t stats, recs, tgt, total;
};
constexpr int kTall64 = 63;
template <class C>
void tile_plan(FwdPlan &p, int64_t V) {
  static_assert(C::WTM == 128 || C::WTM == 64, "strips of a wavefront's tile");
  p.vtiles = (int)((V + C::BM - 1) / C::BM);
  p.ttiles = (int)((p.crows + C::BN - 1) / C::BN);
  p.nstat = p.vtiles * C::WM;
  p.strips = Strips{C::WTM == 128 ? 2 : 1};
}
template <typename TI>
FwdPlan fwd_plan(int64_t M, int64_t V, int64_t chunk_rows, int top_k, bool kept) {
  FwdPlan p{};
  const int64_t mcap = round_up(M, 256);
  p.form = M <= kSkinnyRows<TI> ? 0 : kept ? -1 : mid_form<TI>(M, V);
  if (sizeof(TI) == 4 && p.form < 0 && M <= 64) p.form = kTall64;
  p.crows = p.form >= 0 ? M
            : chunk_rows < mcap / 8 && !kept ? round_up(8 * chunk_rows, 256)
                                             : mcap;
  if (p.form < 0 && !kept) {
    // what one launch takes: 64 logits a thread or more, and in lp_finish 64 threads a row
    int64_t most = kMaxLaunchThreads / round_up(V, 256) * 64;
    if (most > kMaxLaunchThreads / 64) most = kMaxLaunchThreads / 64;
    most = most < 256 ? 256 : most / 256 * 256;
    if (p.crows > most) p.crows = most;
  }
  using F = MidCfg<TI>;
  if (p.form == 64)
    tile_plan<typename F::T64>(p, V);
  else if (p.form == 128)
    tile_plan<typename F::T128>(p, V);
  else if (p.form == 256)
    tile_plan<typename F::T256>(p, V);
  else if (p.form < 0)
    tile_plan<MainCfg<TI>>(p, V);
  if constexpr (sizeof(TI) == 4) {
    if (p.form == kTall64) tile_plan<typename F::Tall64>(p, V);
  }
  if (p.form == 0) {
    p.nstat = (int)((V + 31) / 32);
    p.strips = Strips{0};
  }
  size_t o = 0;
  auto take = [&](size_t bytes) { const size_t at = o; o = align256(o + bytes); return at; };
  p.stats = take(kept ? 0 : (size_t)p.crows * p.nstat * sizeof(Stat));
  p.recs = take(top_k ? (size_t)p.crows * p.nstat * p.strips.per_stat() * sizeof(Rec) : 0);
  p.tgt = take((size_t)p.crows * sizeof(float));
  p.total = o;
  return p;
}

// Enough for either form: a state that is kept takes every row in one chunk, on the main tiles.
template <typename TI>
size_t fwd_bytes(int64_t M, int64_t D, int64_t V, int64_t chunk_rows, int top_k) {
  const size_t plain = fwd_plan<TI>(M, V, chunk_rows, top_k, false).total;
  if (!state_layout<TI>(M, D, V, chunk_rows, true).kept) return plain;
  const size_t kept = fwd_plan<TI>(M, V, chunk_rows, top_k, true).total;
  return kept > plain ? kept : plain;
}

// The records of a row in a lane's registers, up to 64 (V 131072 at 32 logits a record) and where
// the strips formed again load in vectors; else every round over the alternatives reads them from
// memory.  Forward in a graph, bf16, D 256, V 130000, 8 alternatives: 8 rows 43 us against 182 by
// rounds, 1024 rows 138 against 351, 20 alternatives 47 against 385 and 139 against 687; V 32000
// 19 against 56 and 54 against 91.  V 140000 is by rounds: 200, 375, 416 and 720.
template <typename TI>
int launch_finish(const TI *W, const TI *H, int64_t V, int64_t D, const FwdPlan &P,
                  const Stat *stats, const Rec *recs, const float *tgt, int64_t j0, int64_t rows,
                  const View<TI> &S, TI *hc, int64_t lo0, const int64_t *targets,
                  int64_t ignore_index, const RowOut &out, hipStream_t s) {
  const bool vk = D % (16 / (int64_t)sizeof(TI)) == 0 && aligned16(W) && aligned16(H);
  const int64_t waves = targets && lo0 > 0 ? lo0 : rows;
  const unsigned grid = (unsigned)((waves + kFinishThreads / 64 - 1) / (kFinishThreads / 64));
  const int nrec = P.nstat * P.strips.per_stat();
#define NF_LP_FINISH(VK, NR)                                                                   \
  lp_finish_kernel<TI, VK, NR><<<grid, kFinishThreads, 0, s>>>(                                \
      W, H, V, D, stats, P.nstat, recs, P.strips, tgt, j0, rows, S.n, S.rows, S.tcol, S.pos,   \
      hc, lo0, targets, ignore_index, S.mx, S.ls, S.ent, S.lp, out)
  if (vk && nrec <= 64 * 16)
    NF_LP_FINISH(true, 16);
  else if (vk && nrec <= 64 * 32)
    NF_LP_FINISH(true, 32);
  else if (vk && nrec <= 64 * 64)
    NF_LP_FINISH(true, 64);
  else if (vk)
    NF_LP_FINISH(true, 0);
  else
    NF_LP_FINISH(false, 0);
#undef NF_LP_FINISH
  return check_launch("lp_finish");
}

template <typename TI>
int fwd_run(const TI *H, const TI *W, const int64_t *targets, int64_t M, int64_t D, int64_t V,
            int64_t ignore_index, int64_t chunk_rows, bool keep, const RowOut &out, char *state,
            char *ws, hipStream_t s) {
  using C = MainCfg<TI>;
  const State L = state_layout<TI>(M, D, V, chunk_rows, keep);
  const View<TI> S(L, state);
  const FwdPlan P = fwd_plan<TI>(M, V, chunk_rows, out.top_k, L.kept);
  Stat *stats = L.kept ? S.stats : reinterpret_cast<Stat *>(ws + P.stats);
  Rec *recs = out.top_k ? reinterpret_cast<Rec *>(ws + P.recs) : nullptr;
  float *tgt = reinterpret_cast<float *>(ws + P.tgt);
  const int64_t VE = 16 / (int64_t)sizeof(TI);
  int e;
  if constexpr (kSkinnyRows<TI> > 0) {
    if (P.form == 0) {
      const bool vk = D % VE == 0 && aligned16(H) && aligned16(W);
      const unsigned grid = (unsigned)((V + 127) / 128);
#define NF_LP_SKINNY(NT, VK)                                                                   \
  lp_skinny_kernel<TI, NT, VK><<<grid, kSkinnyThreads, 0, s>>>(W, H, targets, M, V, D,         \
                                                               ignore_index, stats, P.nstat,   \
                                                               recs, tgt)
      if (vk && M <= 16)
        NF_LP_SKINNY(1, true);
      else if (vk)
        NF_LP_SKINNY(2, true);
      else
        NF_LP_SKINNY(2, false);
#undef NF_LP_SKINNY
      if ((e = check_launch("lp_skinny"))) return e;
      return launch_finish<TI>(W, H, V, D, P, stats, recs, tgt, 0, M, S, keep ? S.Hc : nullptr,
                               keep ? L.lo0 : 0, targets, ignore_index, out, s);
    }
  }
  if (P.form > 0) {
    const bool vk = buf_ok<TI>(H, D, M, D) && buf_ok<TI>(W, D, V, D);
    const unsigned grid = (unsigned)(P.vtiles * P.ttiles);
    const gemm::TpJobs none{};
#define NF_LP_MID(T, BUF, TOP)                                                                 \
  lp_logits_kernel<typename MidCfg<TI>::T, BUF, false, TOP, false>                             \
      <<<grid, MidCfg<TI>::T::NT, 0, s>>>(W, H, V, D, 0, M, nullptr, nullptr, targets,         \
                                          ignore_index, stats, P.nstat, recs, tgt, nullptr, 0, \
                                          P.vtiles, P.ttiles, none)
#define NF_LP_MID_T(T)                 \
  do {                                 \
    if (vk && recs)                    \
      NF_LP_MID(T, true, true);        \
    else if (vk)                       \
      NF_LP_MID(T, true, false);       \
    else if (recs)                     \
      NF_LP_MID(T, false, true);       \
    else                               \
      NF_LP_MID(T, false, false);      \
  } while (0)
    if (P.form == 64)
      NF_LP_MID_T(T64);
    else if (P.form == 128)
      NF_LP_MID_T(T128);
    else if (P.form == 256)
      NF_LP_MID_T(T256);
    if constexpr (sizeof(TI) == 4) {
      if (P.form == kTall64) NF_LP_MID_T(Tall64);
    }
#undef NF_LP_MID_T
#undef NF_LP_MID
    if ((e = check_launch("lp_logits"))) return e;
    return launch_finish<TI>(W, H, V, D, P, stats, recs, tgt, 0, M, S, keep ? S.Hc : nullptr,
                             keep ? L.lo0 : 0, targets, ignore_index, out, s);
  }
  ce::ce_compact_kernel<<<1, ce::kCompactThreads, 0, s>>>(targets, M, V, ignore_index, S.rows,
                                                          S.tcol, S.pos, S.n, S.inv, nullptr);
  if ((e = check_launch("ce_compact"))) return e;
  const bool vec = D % VE == 0 && aligned16(H) && aligned16(S.Hc);
  int64_t blocks = (M + 3) / 4;
  if (blocks > 4096) blocks = 4096;
  if (vec)
    lp_gather_kernel<TI, true><<<(unsigned)blocks, kGatherThreads, 0, s>>>(
        H, D, S.rows, S.pos, S.n, M, L.lo0, S.Hc, out);
  else
    lp_gather_kernel<TI, false><<<(unsigned)blocks, kGatherThreads, 0, s>>>(
        H, D, S.rows, S.pos, S.n, M, L.lo0, S.Hc, out);
  if ((e = check_launch("lp_gather"))) return e;
  const bool vk = buf_ok<TI>(S.Hc, D, M, D) && buf_ok<TI>(W, D, V, D);
  gemm::TpJobs tp{};
  int64_t ldp = 0;
  bool sb = false;
  if (L.kept) {
    const ce::Plan G = grad_plan<TI>(M, D, V, chunk_rows);
    ldp = G.ldp;
    sb = sb_ok(G.crows * ldp * (int64_t)sizeof(f16));
    if ((e = transposes<TI>(W, S.Hc, M, D, V, G, L.as_is ? nullptr : S.Wt, S.Hct, tp, s)))
      return e;
  }
  for (int64_t j0 = 0; j0 < M; j0 += P.crows) {
    const int64_t rows = M - j0 < P.crows ? M - j0 : P.crows;
    const int ttiles = (int)((rows + C::BN - 1) / C::BN);
    const unsigned grid = (unsigned)(P.vtiles * ttiles + tp.n);
    // kept: the chunk is every row, and E's extent that of its buffer
#define NF_LP_LOGITS(BUF, SB, TOP, KEEP)                                                      \
  lp_logits_kernel<C, BUF, SB, TOP, KEEP><<<grid, C::NT, 0, s>>>(                             \
      W, S.Hc, V, D, j0, P.crows, S.n, S.tcol, nullptr, 0, stats, P.nstat, recs, tgt, S.E,    \
      ldp, P.vtiles, ttiles, tp)
    bool launched = false;
    if constexpr (sizeof(TI) == 2) {
      launched = L.kept;
      if (L.kept && vk && sb && out.top_k)
        NF_LP_LOGITS(true, true, true, true);
      else if (L.kept && vk && sb)
        NF_LP_LOGITS(true, true, false, true);
      else if (L.kept && vk && out.top_k)
        NF_LP_LOGITS(true, false, true, true);
      else if (L.kept && vk)
        NF_LP_LOGITS(true, false, false, true);
      else if (L.kept && out.top_k)
        NF_LP_LOGITS(false, false, true, true);
      else if (L.kept)
        NF_LP_LOGITS(false, false, false, true);
    }
    if (launched)
      ;
    else if (vk && out.top_k)
      NF_LP_LOGITS(true, false, true, false);
    else if (vk)
      NF_LP_LOGITS(true, false, false, false);
    else if (out.top_k)
      NF_LP_LOGITS(false, false, true, false);
    else
      NF_LP_LOGITS(false, false, false, false);
#undef NF_LP_LOGITS
    if ((e = check_launch("lp_logits"))) return e;
    if ((e = launch_finish<TI>(W, S.Hc, V, D, P, stats, recs, tgt, j0, rows, S, S.Hc, L.lo0, nullptr,
                               ignore_index, out, s)))
      return e;
  }
  return NF_OK;
}

// The backward's plan and workspace: the cross entropy's, without the room for transposes that the
// call does not make (weight's where it is read as it lies; both where the state was kept).
template <typename TI>
ce::Plan bwd_plan(int64_t M, int64_t D, int64_t V, int64_t chunk_rows, const State &s) {
  ce::Plan L = grad_plan<TI>(M, D, V, chunk_rows);
  const size_t wt = L.s_hct - L.s_wt, hct = L.s_p - L.s_hct;
  const int64_t Mb = s.lo0 > 0 ? 2 * s.lo0 : M;
  const bool no_wt = s.kept || (sizeof(TI) == 2 && weight_as_is(Mb, D, V));
  const size_t less = (no_wt ? wt : 0) + (s.kept ? hct : 0);
  if (no_wt) L.s_hct -= wt;
  for (size_t *at : {&L.s_p, &L.s_pt, &L.s_dhc, &L.s_dwacc, &L.s_total}) *at -= less;
  return L;
}
template <typename TI>
size_t bwd_bytes(int64_t M, int64_t D, int64_t V, int64_t chunk_rows) {
  const ce::Plan L =
      bwd_plan<TI>(M, D, V, chunk_rows, state_layout<TI>(M, D, V, chunk_rows, true));
  return L.s_total + L.b_total + 256;
}

template <typename TI>
int bwd_run(const TI *W, int64_t M, int64_t D, int64_t V, int64_t chunk_rows, bool keep,
            char *state, const float *g, const float *h, void *dH, int dt_h, void *dW, int dt_w,
            char *ws, hipStream_t s) {
  using C = MainCfg<TI>;
  const State KL = state_layout<TI>(M, D, V, chunk_rows, keep);
  const View<TI> K(KL, state);
  const int64_t lo0 = KL.lo0, Mb = lo0 > 0 ? 2 * lo0 : M;  // rows of the products
  const ce::Plan L = bwd_plan<TI>(M, D, V, chunk_rows, KL);
  ce::StateView<TI> S(L, ws);
  int *const two = S.n;
  if (lo0 == 0) S.n = K.n;  // else *two, by lp_dz
  float *part = reinterpret_cast<float *>(ws + L.s_total);
  const RowIn in{K.n, K.rows, K.tcol, K.mx, K.ls, K.ent, K.lp, g, h};
  TI *const PT = L.single ? nullptr : S.PT;
  gemm::TpJobs tp{};
  const gemm::TpJobs none{};
  int e;
  const TI *Wn = nullptr;
  if (KL.kept) {
    S.Wt = K.Wt;
    S.Hct = K.Hct;
    Wn = KL.as_is ? W : nullptr;
  } else {
    Wn = sizeof(TI) == 2 && weight_as_is(Mb, D, V) ? W : nullptr;
    if ((e = transposes<TI>(W, K.Hc, Mb, D, V, L, Wn || !dH ? nullptr : S.Wt, S.Hct, tp, s)))
      return e;
  }
  const bool vk = buf_ok<TI>(K.Hc, D, Mb, D) && buf_ok<TI>(W, D, V, D);
  const bool sb = sb_ok(L.crows * L.ldp * (int64_t)sizeof(TI)) &&
                  (L.single || sb_ok(V * L.crows * (int64_t)sizeof(TI)));
  for (int64_t c = 0; c < L.nch; ++c) {
    const int64_t j0 = c * L.crows;
    const gemm::TpJobs &tj = c == 0 ? tp : none;
#define NF_LP_DZ(CFG, BUF, SB)                                                                 \
  do {                                                                                         \
    const int vt = (int)((V + CFG::BM - 1) / CFG::BM), tt = (int)((cap + CFG::BN - 1) / CFG::BN); \
    lp_dz_kernel<CFG, BUF, SB><<<(unsigned)(vt * tt + tj.n), CFG::NT, 0, s>>>(                 \
        W, K.Hc, V, D, j0, L.crows, in, lo0, two, S.cfac, S.P, L.ldp, PT, L.crows, vt, tt, tj); \
  } while (0)
    // rows of the chunk, padding included (the products read up to 7 rows past them)
    const int64_t cap = Mb - j0 < L.crows ? round_up(Mb - j0, 8) : L.crows;
    const int form = mid_form<TI>(Mb, V);
    using F = MidCfg<TI>;
    using T64 = typename F::T64;
    using T128 = typename F::T128;
    using T256 = typename F::T256;
    bool formed = false;
    if constexpr (sizeof(TI) == 2) {
      formed = KL.kept;
      if (KL.kept) {
        const dim3 kg((unsigned)round_up(M, 8),
                      (unsigned)((L.ldp / 8 + kKeptThreads - 1) / kKeptThreads));
        lp_from_kept_kernel<C::WTM><<<kg, kKeptThreads, 0, s>>>(K.E, S.P, L.ldp, V, K.stats,
                                                                KL.nstat, in, S.cfac);
      }
    }
    if (formed)
      ;
    else if (vk && sb && form == 64)
      NF_LP_DZ(T64, true, true);
    else if (vk && sb && form == 128)
      NF_LP_DZ(T128, true, true);
    else if (vk && sb && form == 256)
      NF_LP_DZ(T256, true, true);
    else if (vk && sb)
      NF_LP_DZ(C, true, true);
    else if (vk)
      NF_LP_DZ(C, true, false);
    else
      NF_LP_DZ(C, false, false);
#undef NF_LP_DZ
    if ((e = check_launch(formed ? "lp_from_kept" : "lp_dz"))) return e;
    const bool last = c + 1 == L.nch;
    if ((e = ce::launch_grads<TI>(L, S, c, D, V, c > 0 ? S.dWacc : nullptr,
                                  last ? dW : S.dWacc, last ? dt_w : NF_DTYPE_F32, nullptr, part,
                                  s, /*final_dw=*/last, /*reduce_dh=*/!last, dW != nullptr,
                                  dH != nullptr, Wn)))
      return e;
  }
  if (!dH) return NF_OK;
  const ce::SplitRows sp{part, L.split.S, (L.nch - 1) * L.crows, L.crows, S.cfac, lo0};
  const bool vec = D % 4 == 0;
  int64_t blocks = (M * (vec ? D / 4 : D) + 255) / 256;
  if (blocks > 4096) blocks = 4096;
  if (vec)
    ce::ce_scatter_dh_kernel<4><<<(unsigned)blocks, 256, 0, s>>>(S.dHc, D, K.pos, M, nullptr, dH,
                                                                 dt_h, sp);
  else
    ce::ce_scatter_dh_kernel<1><<<(unsigned)blocks, 256, 0, s>>>(S.dHc, D, K.pos, M, nullptr, dH,
                                                                 dt_h, sp);
  return check_launch("ce_scatter_dh");
}

}  // namespace lp
}  // namespace nf

using namespace nf;
using namespace nf::lp;
using ce::ce_check_dtype;
using ce::dtype_ok;

namespace {
// Columns are ints, padded to whole block tiles: V at most 2^30.
constexpr int64_t kMaxCols = (int64_t)1 << 30;
bool sizes_ok(int64_t M, int64_t D, int64_t V) { return ce::ce_sizes_ok(M, D, V) && V <= kMaxCols; }
int check_shape(const char *fn, int64_t M, int64_t D, int64_t V) {
  if (int e = ce::ce_check_shape(fn, M, D, V)) return e;
  if (V > kMaxCols) return set_error(NF_ERR_ARG, "%s: V exceeds 2^30", fn);
  return NF_OK;
}
}  // namespace

extern "C" size_t nf_token_logprobs_state_bytes(int64_t M, int64_t D, int64_t V,
                                                int64_t chunk_rows, int keep, int dtype) {
  if (!sizes_ok(M, D, V) || chunk_rows <= 0 || !dtype_ok(dtype)) return 0;
  return dtype == NF_DTYPE_BF16 ? state_layout<bf16>(M, D, V, chunk_rows, keep != 0).total
                                : state_layout<float>(M, D, V, chunk_rows, keep != 0).total;
}

extern "C" size_t nf_token_logprobs_fwd_workspace(int64_t M, int64_t D, int64_t V,
                                                  int64_t chunk_rows, int top_k, int dtype) {
  if (!sizes_ok(M, D, V) || chunk_rows <= 0 || !dtype_ok(dtype) || top_k < 0 ||
      top_k > kMaxTop || top_k > V)
    return 0;
  return dtype == NF_DTYPE_BF16 ? fwd_bytes<bf16>(M, D, V, chunk_rows, top_k)
                                : fwd_bytes<float>(M, D, V, chunk_rows, top_k);
}

extern "C" size_t nf_token_logprobs_bwd_workspace(int64_t M, int64_t D, int64_t V,
                                                  int64_t chunk_rows, int dtype) {
  if (!sizes_ok(M, D, V) || chunk_rows <= 0 || !dtype_ok(dtype)) return 0;
  return dtype == NF_DTYPE_BF16 ? bwd_bytes<bf16>(M, D, V, chunk_rows)
                                : bwd_bytes<float>(M, D, V, chunk_rows);
}

extern "C" int nf_token_logprobs_fwd(const void *hidden, const void *weight,
                                     const int64_t *targets, int64_t M, int64_t D, int64_t V,
                                     int64_t ignore_index, int64_t chunk_rows, int top_k,
                                     int keep, int dtype, float *logprobs, float *entropy,
                                     float *top_logprobs, int64_t *top_ids, void *state,
                                     size_t state_bytes, void *workspace,
                                     size_t workspace_bytes, void *stream) {
  const char *fn = "nf_token_logprobs_fwd";
  if (int e = check_shape(fn, M, D, V)) return e;
  if (chunk_rows <= 0) return set_error(NF_ERR_ARG, "%s: chunk_rows must be > 0", fn);
  if (top_k < 0 || top_k > kMaxTop || top_k > V)
    return set_error(NF_ERR_ARG, "%s: top_k=%d outside [0, min(%d, V)]", fn, top_k, kMaxTop);
  if (!hidden || !weight || !targets || !logprobs || !entropy || !state ||
      (top_k > 0 && (!top_logprobs || !top_ids)))
    return set_error(NF_ERR_ARG, "%s: null pointer", fn);
  if (int e = ce_check_dtype(fn, dtype)) return e;
  const size_t sb = nf_token_logprobs_state_bytes(M, D, V, chunk_rows, keep, dtype);
  if (state_bytes < sb || !aligned16(state))
    return set_error(NF_ERR_WORKSPACE, "%s: state %zu bytes < required %zu", fn, state_bytes, sb);
  const size_t wb = nf_token_logprobs_fwd_workspace(M, D, V, chunk_rows, top_k, dtype);
  if (!workspace || workspace_bytes < wb || !aligned16(workspace))
    return set_error(NF_ERR_WORKSPACE, "%s: workspace %zu bytes < required %zu", fn,
                     workspace_bytes, wb);
  hipStream_t s = static_cast<hipStream_t>(stream);
  char *st = static_cast<char *>(state), *ws = static_cast<char *>(workspace);
  const RowOut out{logprobs, entropy, top_logprobs, top_ids, top_k};
  if (dtype == NF_DTYPE_BF16)
    return fwd_run<bf16>((const bf16 *)hidden, (const bf16 *)weight, targets, M, D, V,
                         ignore_index, chunk_rows, keep != 0, out, st, ws, s);
  return fwd_run<float>((const float *)hidden, (const float *)weight, targets, M, D, V,
                        ignore_index, chunk_rows, keep != 0, out, st, ws, s);
}

extern "C" int nf_token_logprobs_bwd(const void *weight, int64_t M, int64_t D, int64_t V,
                                     int64_t chunk_rows, int keep, int dtype, void *state,
                                     size_t state_bytes, const float *g_logprobs,
                                     const float *g_entropy, void *dhidden, int dt_hidden,
                                     void *dweight, int dt_weight, void *workspace,
                                     size_t workspace_bytes, void *stream) {
  const char *fn = "nf_token_logprobs_bwd";
  if (int e = check_shape(fn, M, D, V)) return e;
  if (chunk_rows <= 0) return set_error(NF_ERR_ARG, "%s: chunk_rows must be > 0", fn);
  if (!weight || !state) return set_error(NF_ERR_ARG, "%s: null pointer", fn);
  if (!keep)  // few rows are then left where they lie, and the state has none of them
    return set_error(NF_ERR_ARG, "%s: a state made without keep serves no backward", fn);
  if (int e = ce_check_dtype(fn, dtype)) return e;
  if ((dhidden && !is_dtype(dt_hidden)) || (dweight && !is_dtype(dt_weight)))
    return set_error(NF_ERR_DTYPE, "%s: gradient dtypes %d, %d", fn, dt_hidden, dt_weight);
  const size_t sb = nf_token_logprobs_state_bytes(M, D, V, chunk_rows, keep, dtype);
  if (state_bytes < sb || !aligned16(state))
    return set_error(NF_ERR_WORKSPACE, "%s: state %zu bytes < required %zu", fn, state_bytes, sb);
  const size_t wb = nf_token_logprobs_bwd_workspace(M, D, V, chunk_rows, dtype);
  if (!workspace || workspace_bytes < wb || !aligned16(workspace))
    return set_error(NF_ERR_WORKSPACE, "%s: workspace %zu bytes < required %zu", fn,
                     workspace_bytes, wb);
  if (!dhidden && !dweight) return NF_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  char *st = static_cast<char *>(state), *ws = static_cast<char *>(workspace);
  if (dtype == NF_DTYPE_BF16)
    return bwd_run<bf16>((const bf16 *)weight, M, D, V, chunk_rows, keep != 0, st, g_logprobs, g_entropy,
                         dhidden, dt_hidden, dweight, dt_weight, ws, s);
  return bwd_run<float>((const float *)weight, M, D, V, chunk_rows, keep != 0, st, g_logprobs, g_entropy,
                        dhidden, dt_hidden, dweight, dt_weight, ws, s);
}
