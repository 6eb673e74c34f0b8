// Chunked cross entropy on the MFMA GEMM core of gemm_core.h and the parts of
// lm_head.h, in two calls,
// all on the caller's stream with fixed reduction orders (no atomics).
//
// Only valid rows (target != ignore_index, inside [0, V)) do any work: the
// forward compacts them on the device (no count reaches the host), and every
// later kernel sizes itself by that device count.  The logits are formed once
// per row (6 * n_valid * V * D flops in all: logits, dH, dW), never twice.
//
// Forward (nf_ce_fwd):
//   1. ce_compact: the valid rows in order -> rows[], their target columns,
//      pos[m] (compacted index or -1), n_valid, inv = 1 / max(n_valid, 1).
//   2. ce_gather: Hc = H[rows] ([M, D], zero past n_valid) and each valid
//      row's target logit mref = Hc[r] . W[target], the row's reference.
//      Wt = W^T [D, V] (zero-padded; the dH product's K-contiguous B
//      operand) is formed by the first logits launch's last blocks (16-bit
//      inputs) or by a transpose launch here (fp32).
//   3. per chunk of `crows` compacted rows:
//      ce_logits: S = Hc_c W^T tile by tile (formed transposed, W Hc_c^T, so a
//                 lane holds each token's logits along the vocabulary); per
//                 (vocabulary tile of WTM rows, token) the max and the sum of
//                 exp(S - max), the target logit, and E = exp(S - mref) in
//                 the input type, row-major [crows, ldp] and (unless E is
//                 held once: "single", see Plan) transposed [V, crows];
//      ce_lse:    lse per row from the tile statistics (fixed order), the
//                 row's loss lse - S[target], the row factor cfac =
//                 exp(mref - lse) / n, and the one-hot term folded into E's
//                 target entry, so cfac * E = (softmax - onehot) / n; rows
//                 whose maximum lies far above mref are rescaled to it;
//      ce_scale_hct: Hct = (cfac * Hc_c)^T, the dW product's B operand; in
//                 the last chunk's launch, also the mean loss;
//      gradient products of every chunk but the last (one launch):
//                 dW_acc (+)= E^T_c Hct_c^T  (fp32 [V, D], K = the chunk's rows;
//                             single: dW_acc^T (+)= Hct_c E_c, fp32 [D, V],
//                             E read N-major)
//                 dHc_c   = cfac * (E_c Wt^T) (fp32, K = V, split along K)
// Backward (nf_ce_bwd, with the loss's grad_output g): the last chunk's
// products, dW = g * (dW_acc + E^T Hct^T) written in dweight's type (single:
// formed transposed and stored through LDS as [V, D]), and the scatter of
// dHc back to the hidden rows as g * dH (0 for ignored rows).
//
// Memory: the state kept between the calls holds one chunk's E (once, for
// twice the rows, when single), W^T, the scaled Hc^T and the fp32 dH rows,
// plus the fp32 dW accumulator when there is more than one chunk; E and the
// accumulator stay within the bytes the reference's chunk loop holds for
// them (see make_plan), so E covers every row at once only where that fits.

#include "lm_head.h"

namespace nf {
namespace ce {

__device__ __forceinline__ float2 combine_stats(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  if (m == -INFINITY) return make_float2(m, 0.f);
  return make_float2(m, a.y * exp_f32(a.x - m) + b.y * exp_f32(b.x - m));
}

// ---------------------------------------------------------------------------
// 2. Hc[r, :] = H[rows[r], :] for r < n_valid, 0 for n_valid <= r < R, and
// the row's reference logit mref[r] = H[rows[r], :] . W[tcol[r], :] (fp32, a
// fixed-order sum; 0 past n_valid).  One wavefront per row.  E is stored
// relative to mref (exp(S - mref)), so mref needs only to lie within the
// exponent range of the row's largest logit; the target logit does for every
// row whose loss is below ~50 nats, and for any other row the logits pass
// keeps E in range and the statistics pass rescales it (ce_lse_kernel).
// VEC: 16-byte vectors
// (D a multiple of the vector width, aligned rows).
// ---------------------------------------------------------------------------
constexpr int kGatherThreads = 256;

template <typename T, bool VEC>
__global__ __launch_bounds__(kGatherThreads) void ce_gather_kernel(
    const T *__restrict__ H, const T *__restrict__ W, int64_t D, const int *__restrict__ rows,
    const int *__restrict__ tcol, const int *n_ptr, int64_t R, T *__restrict__ Hc,
    float *__restrict__ mref) {
  constexpr int kWaves = kGatherThreads / 64;
  const int64_t n = *n_ptr;
  constexpr int VE = VEC ? 16 / (int)sizeof(T) : 1;
  const int l = threadIdx.x & 63;
  for (int64_t r = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6); r < R;
       r += (int64_t)gridDim.x * kWaves) {
    const bool live = r < n;
    const T *h = live ? H + (int64_t)rows[r] * D : nullptr;
    const T *w = live ? W + (int64_t)tcol[r] * D : nullptr;
    float dot = 0.f;
    for (int64_t c = (int64_t)l * VE; c < D; c += 64 * VE) {
      if constexpr (VEC) {
        u32x4 hv = {0u, 0u, 0u, 0u}, wv = {0u, 0u, 0u, 0u};
        if (live) {
          hv = *reinterpret_cast<const u32x4 *>(h + c);
          wv = *reinterpret_cast<const u32x4 *>(w + c);
        }
        *reinterpret_cast<u32x4 *>(Hc + r * D + c) = hv;
        T he[VE], we[VE];
        __builtin_memcpy(he, &hv, 16);
        __builtin_memcpy(we, &wv, 16);
#pragma unroll
        for (int q = 0; q < VE; ++q) dot += static_cast<float>(he[q]) * static_cast<float>(we[q]);
      } else {
        const T hv = live ? h[c] : static_cast<T>(0.f);
        Hc[r * D + c] = hv;
        if (live) dot += static_cast<float>(hv) * static_cast<float>(w[c]);
      }
    }
    dot = wave_sum(dot);
    if (l == 0) mref[r] = live ? dot : 0.f;
  }
}

// ---------------------------------------------------------------------------
// 3. logits of one chunk, their tile statistics and E = exp(S - mref) in the
// input type, row-major and transposed.  The product is formed transposed,
// acc = W_tile Hc_tile^T (rows: vocabulary entries, columns: tokens), so each
// lane holds 16 * TM logits of each of its TN tokens: a wavefront's max and
// sum of exp over its WTM vocabulary rows are reductions in registers plus
// one exchange between the lane halves.  Statistics tile t covers vocabulary
// rows [t * WTM, (t + 1) * WTM): stats[t * crows + token] = (max, sum
// exp(S - max)), taken from the sum of E (see the epilogue).  The target
// logit comes from the one lane holding it.  E = exp(S - mref) goes out in the
// layouts of EStore (columns V..ldp zero: exp(-inf)).  With a row
// factor P = inv * exp(mref - lse) (ce_lse_kernel), P * E is the softmax.
// ---------------------------------------------------------------------------
constexpr float kStatsGap = 64.f;  // exp(-64) of a row maximum is below fp32 resolution
// E entries relative to mref stay below exp(kBaseGap): a wavefront whose
// maximum for a token lies further above mref stores that token's E relative
// to its own maximum instead (see the epilogue)
constexpr float kBaseGap = 60.f;

// Blocks past the vtiles x ttiles logits tiles run the transpose regions of
// `tp` (16-bit inputs only): dispatched last, they fill the CUs that the
// final partial wave of tiles leaves idle.
template <class C, bool BUF, bool SB>
__global__ NF_GEMM_BOUNDS(C) void ce_logits_kernel(
    const typename C::TI *W, const typename C::TI *Hc, int64_t V, int64_t D, int64_t j0,
    int64_t crows, const int *n_ptr, const int *tcol, const float *mref, float2 *stats,
    float *tgt, typename C::TI *E, int64_t ldp, typename C::TI *ET, int64_t ldet, int vtiles,
    int ttiles, gemm::TpJobs tp) {
  using TI = typename C::TI;
  constexpr int ES = (int)sizeof(TI);
  // one LDS buffer only: a second __shared__ object makes the compiler wait
  // for every direct-to-LDS copy in flight before each operand read of the
  // K loop; the E staging and the transposes reuse the operand stages
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
  const int64_t cnt = chunk_count(n_ptr, j0, crows);
  const int64_t v0 = (int64_t)vt * C::BM;
  const int64_t t0 = (int64_t)tt * C::BN;  // first token of the tile, chunk-local
  if (t0 >= cnt) return;
  floatx16 acc[C::TM][C::TN];
  gemm::mainloop<C, BUF>(W, D, Hc + j0 * D, D, V, cnt, D, v0, t0, smem, acc);

  const int l = threadIdx.x & 63, half = l >> 5;
  const int w = threadIdx.x >> 6, wm = w / C::WN, wn = w % C::WN;
  const int64_t vtile0 = v0 + wm * C::WTM;      // first vocabulary row of this wavefront
  const int64_t crow0 = vtile0 + 4 * half;      // vocabulary row of (i = 0, r = 0)
  const int stile = vt * C::WM + wm;            // statistics tile
  // Rows past the vocabulary (only in a wavefront whose rows reach V) are set
  // to -inf once, so the max, the sum and E need no per-element masks.
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
  EStore<C, SB> store;
  store.init(E, ldp, ET, ldet, V, crows, v0, t0, cnt, smem);
#pragma unroll
  for (int j = 0; j < C::TN; ++j) {
    const int tl = wn * C::WTN + j * 32 + (l & 31);  // token within the tile
    const int64_t tok = t0 + tl;                     // token within the chunk
    const float mr = tok < cnt ? mref[j0 + tok] : 0.f;  // the row's reference
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, acc[i][j][r]);
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    // the target logit, from the one lane that holds it (before the exp)
    if (tok < cnt) {
      const int64_t loc64 = (int64_t)tcol[j0 + tok] - vtile0;
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
    // E = exp(S - mref) relative to the row's reference (rows past V are -inf
    // and give 0; S - mref is exact where S is near mref, so the target's own
    // entry is exactly 1).  The tile's statistics
    // follow from its sum: s = sum exp(S - mx) = sum E / exp(mx - mref), the
    // divisor being the largest entry as formed (a lone entry gives 1).  A
    // tile more than kStatsGap below mref keeps s = 1: its share of the row
    // total, below exp(-kStatsGap) of the row maximum's, is under fp32
    // resolution.  Where the maximum lies more than kBaseGap above mref (a
    // row far from its reference), E = exp(S - mx) instead, so no entry
    // leaves the exponent range, and s = sum E is stored negated: the
    // statistics pass then rescales the row to its maximum.  A wavefront
    // with no row inside the vocabulary keeps (-inf, 0).
    const bool own = mx - mr > kBaseGap;
    const float base = own ? mx : mr;
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = exp_f32(acc[i][j][r] - base);
    float se = 0.f;
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) se += acc[i][j][r];
    se += __shfl_xor(se, 32);
    const float s = mx == -INFINITY ? 0.f
                    : own           ? -se
                    : (mr - mx > kStatsGap ? 1.f : se / exp_f32(mx - mr));
    if (half == 0 && tok < cnt) stats[(int64_t)stile * crows + tok] = make_float2(mx, s);
    store.column(j, acc);
  }
  store.finish();
}

// ---------------------------------------------------------------------------
// 4. lse per row of a chunk: a block takes 16 rows and 16 parts; part q
// combines statistics tiles q, q + 16, q + 32, ... of its row in that order
// (sixteen tiles' loads issued before their combines: one round of loads for
// vocabularies up to 32768), then the first part
// combines the 16 partial results in order.  A row of 16 tokens is 128
// contiguous bytes of the [ntiles][crows] statistics.
// ---------------------------------------------------------------------------
// The row factor cfac = inv * exp(mref - lse), so that cfac * E is the
// softmax over the row scaled by 1 / n.  The one-hot term goes into E itself:
// the target entry becomes exp(z - mref) - exp(lse - mref), so cfac * E is
// (softmax - onehot) / n, the gradient of the mean loss by the logits.
// The fast path holds while (lse - mref) + ln n <= kFactorGap: cfac (which
// multiplies Hc into the dW product's operand, rounded to the input type)
// then stays above exp(-kFactorGap), far inside the normal range of bf16 and
// fp32, and every E entry below exp(kFactorGap), far from overflow in the
// products' sums (lse is at least the row's largest logit).  Any other row
// (a loss above kFactorGap - ln n nats, ~52 at n = 4096, which includes every
// row with a tile stored relative to its own maximum; also a NaN / inf row)
// is rescaled by its block to the row's maximum M: each entry of statistics
// tile t is multiplied by exp(base_t - M), base_t being the reference that
// tile's E was formed with (mref, or the tile's maximum where its sum is
// negated), and the target entry becomes exp(z - M) - exp(lse - M); both
// layouts are rewritten, and mref becomes M (cfac is then at least
// 1 / (n V)).  No E entry left the exponent range in the logits pass, so
// nothing is lost but one rounding of the rescaled entries.
constexpr float kFactorGap = 60.f;
static_assert(kBaseGap <= kFactorGap, "a row with a tile of its own base must take the rescale");
constexpr int kLseRows = 16, kLseParts = 16, kLseThreads = kLseRows * kLseParts;

template <typename TI>
__global__ __launch_bounds__(kLseThreads) void ce_lse_kernel(
    const float2 *__restrict__ stats, int ntiles, int wtm, int64_t crows, const float *tgt,
    const int *n_ptr, int64_t j0, const float *inv_ptr, const int *__restrict__ tcol,
    float *__restrict__ mref, float *__restrict__ cfac, float *loss_row, TI *P, int64_t ldp,
    TI *PT, int64_t ldet, int64_t V) {
  __shared__ float2 part[kLseParts][kLseRows];
  __shared__ int own[kLseParts][kLseRows];
  __shared__ int redo[kLseRows];
  __shared__ float2 rowst[kLseRows];
  __shared__ float mold[kLseRows];  // mref as the logits pass used it
  const int64_t cnt = chunk_count(n_ptr, j0, crows);
  const int rl = threadIdx.x % kLseRows, q = threadIdx.x / kLseRows;
  const int64_t row = (int64_t)blockIdx.x * kLseRows + rl;
  if ((int64_t)blockIdx.x * kLseRows >= cnt) return;  // the whole block is past the chunk
  float2 a = make_float2(-INFINITY, 0.f);
  int flag = 0;
  if (row < cnt) {
    constexpr int kBatch = 16;
    for (int t0 = q; t0 < ntiles; t0 += kLseParts * kBatch) {
      float2 v[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int t = t0 + u * kLseParts;
        v[u] = t < ntiles ? stats[(int64_t)t * crows + row] : make_float2(-INFINITY, 0.f);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        flag |= v[u].y < 0.f;
        a = combine_stats(a, make_float2(v[u].x, fabsf(v[u].y)));
      }
    }
  }
  part[q][rl] = a;
  own[q][rl] = flag;
  __syncthreads();
  const float inv = *inv_ptr;
  if (q == 0) {
    int again = 0;
    if (row < cnt) {
#pragma unroll
      for (int k = 1; k < kLseParts; ++k) {
        a = combine_stats(a, part[k][rl]);
        flag |= own[k][rl];
      }
      const float ls = a.x + log_f32(a.y);
      const float z = tgt[row];
      loss_row[j0 + row] = ls - z;
      const float m = mref[j0 + row];
      again = flag || !(ls - m - log_f32(inv) <= kFactorGap);  // also for a NaN / inf row
      if (!again) {
        cfac[j0 + row] = inv * exp_f32(m - ls);
        const int64_t tc = tcol[j0 + row];
        const TI e = static_cast<TI>(exp_f32(z - m) - exp_f32(ls - m));
        P[row * ldp + tc] = e;
        if (PT) PT[tc * ldet + row] = e;
      }
    }
    redo[rl] = again;
    rowst[rl] = a;
    mold[rl] = row < cnt ? mref[j0 + row] : 0.f;
  }
  __syncthreads();
  // The rows outside the reference's range (rare), all of the block's rows
  // together: a thread takes 8 entries (ldp and wtm are multiples of 8, so
  // the eight lie in one statistics tile; rows of P are 16-byte aligned) of
  // each row and rescales those of the rows off the fast path.  With E also
  // held transposed it then writes the block's 16 columns of E^T for those 8
  // vocabulary entries from all 16 rows (the other rows' entries are final
  // and go back unchanged; rows past the chunk's count give zeros, the K
  // padding of the dW product).
  int any = 0;
#pragma unroll
  for (int k = 0; k < kLseRows; ++k) any |= redo[k];
  if (!any) return;  // uniform across the block
  constexpr int kVec = 8, kWords = kVec * (int)sizeof(TI) / 16;
  constexpr int kColWords = kLseRows * (int)sizeof(TI) / 16;
  const int64_t r0 = (int64_t)blockIdx.x * kLseRows;
  for (int64_t v0 = (int64_t)threadIdx.x * kVec; v0 < ldp; v0 += (int64_t)kLseThreads * kVec) {
    TI ev[kLseRows][kVec];
#pragma unroll
    for (int k = 0; k < kLseRows; ++k) {
      if ((redo[k] || PT) && r0 + k < cnt) {
        u32x4 raw[kWords];
#pragma unroll
        for (int w = 0; w < kWords; ++w)
          raw[w] = reinterpret_cast<const u32x4 *>(P + (r0 + k) * ldp + v0)[w];
        __builtin_memcpy(ev[k], raw, sizeof(ev[k]));
      } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) ev[k][i] = static_cast<TI>(0.f);
      }
    }
#pragma unroll
    for (int k = 0; k < kLseRows; ++k) {
      if (!redo[k]) continue;
      const int64_t r = r0 + k;
      const float mx = rowst[k].x, ls = rowst[k].x + log_f32(rowst[k].y);
      float f = 0.f;
      if (v0 < V) {
        const float2 ts = stats[(v0 / wtm) * crows + r];
        f = exp_f32((ts.y < 0.f ? ts.x : mold[k]) - mx);
      }
      const int64_t tc = tcol[j0 + r];
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const int64_t v = v0 + i;
        const float e = v >= V   ? 0.f
                        : v == tc ? exp_f32(tgt[r] - mx) - exp_f32(ls - mx)
                                  : static_cast<float>(ev[k][i]) * f;
        ev[k][i] = static_cast<TI>(e);
      }
      u32x4 raw[kWords];
      __builtin_memcpy(raw, ev[k], sizeof(ev[k]));
#pragma unroll
      for (int w = 0; w < kWords; ++w) reinterpret_cast<u32x4 *>(P + r * ldp + v0)[w] = raw[w];
    }
    if (PT) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        if (v0 + i >= V) break;
        TI col[kLseRows];
#pragma unroll
        for (int k = 0; k < kLseRows; ++k) col[k] = ev[k][i];
        u32x4 raw[kColWords];
        __builtin_memcpy(raw, col, sizeof(col));
#pragma unroll
        for (int w = 0; w < kColWords; ++w)
          reinterpret_cast<u32x4 *>(PT + (v0 + i) * ldet + r0)[w] = raw[w];
      }
    }
  }
  if (threadIdx.x < kLseRows && redo[threadIdx.x]) {
    const int k = threadIdx.x;
    const float mx = rowst[k].x, ls = rowst[k].x + log_f32(rowst[k].y);
    mref[j0 + r0 + k] = mx;
    cfac[j0 + r0 + k] = inv * exp_f32(mx - ls);
  }
}

// ---------------------------------------------------------------------------
// 5. The dW product's B operand for a chunk: Hct[d, j0 + r] = cfac[j0 + r] *
// Hc[j0 + r, d] in the input type for r < count, 0 for count <= r <
// round_up(count, 8) (the product's K padding): the row factor enters the
// product over the rows through this operand.  64 x 64 tiles through LDS;
// VEC: 16-byte row vectors in and column vectors out (D a multiple of the
// vector width), else one element per access.
// With `loss` set (the last chunk's launch, when every row's loss is known),
// block (0, 0) first writes the mean loss: each thread sums a strided share
// of the n valid rows' losses, each wavefront reduces its lanes (fixed
// butterfly), and thread 0 adds the 4 wavefront sums in order.  This saves
// the launch a one-block loss kernel would cost.
// ---------------------------------------------------------------------------
constexpr int kPrepThreads = 256;

template <typename TI, bool VEC>
__global__ __launch_bounds__(kPrepThreads) void ce_scale_hct_kernel(
    const TI *__restrict__ Hc, int64_t D, const float *__restrict__ cfac,
    const int *n_ptr, int64_t j0, int64_t crows, TI *__restrict__ Hct, int64_t ldht,
    const float *__restrict__ loss_row, const float *inv_ptr, float *loss) {
  using U = typename std::conditional<sizeof(TI) == 2, uint16_t, uint32_t>::type;
  constexpr int VE = VEC ? 16 / (int)sizeof(TI) : 1;  // elements per access
  constexpr int PITCH = 64 + (sizeof(TI) == 2 ? 2 : 1);
  __shared__ U tile[64 * PITCH];
  if (loss != nullptr && blockIdx.x == 0 && blockIdx.y == 0) {
    __shared__ float sl[kPrepThreads / 64];
    const int64_t n = *n_ptr;
    float a = 0.f;
    for (int64_t i = threadIdx.x; i < n; i += kPrepThreads) a += loss_row[i];
    a = wave_sum(a);
    if ((threadIdx.x & 63) == 0) sl[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x == 0) {
      float tl = 0.f;
      for (int k = 0; k < kPrepThreads / 64; ++k) tl += sl[k];
      *loss = tl * *inv_ptr;
    }
  }
  const int64_t cnt = chunk_count(n_ptr, j0, crows);
  const int64_t cnt8 = (cnt + 7) / 8 * 8;
  const int64_t r0 = (int64_t)blockIdx.x * 64, d0 = (int64_t)blockIdx.y * 64;
  if (r0 >= cnt8) return;
  const int t = threadIdx.x;
  constexpr int VPR = 64 / VE;  // accesses per 64-element tile row
  for (int idx = t; idx < 64 * VPR; idx += kPrepThreads) {
    const int rr = idx / VPR, cv = idx % VPR;
    const int64_t r = r0 + rr, d = d0 + (int64_t)cv * VE;
    TI e[VE];
    const float f = r < cnt ? cfac[j0 + r] : 0.f;
    if constexpr (VEC) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (r < cnt && d < D) v = *reinterpret_cast<const u32x4 *>(Hc + (j0 + r) * D + d);
      __builtin_memcpy(e, &v, 16);
    } else {
      e[0] = (r < cnt && d < D) ? Hc[(j0 + r) * D + d] : static_cast<TI>(0.f);
    }
#pragma unroll
    for (int q = 0; q < VE; ++q) {
      const TI sc = static_cast<TI>(static_cast<float>(e[q]) * f);
      U bits;
      __builtin_memcpy(&bits, &sc, sizeof(U));
      tile[rr * PITCH + cv * VE + q] = bits;
    }
  }
  __syncthreads();
  for (int idx = t; idx < 64 * VPR; idx += kPrepThreads) {
    const int dc = idx / VPR, rv = idx % VPR;  // output row (d), row vector
    const int64_t d = d0 + dc, r = r0 + (int64_t)rv * VE;
    if (d >= D || r >= cnt8) continue;  // cnt8 is a multiple of VE
    U e[VE];
#pragma unroll
    for (int q = 0; q < VE; ++q) e[q] = tile[(rv * VE + q) * PITCH + dc];
    if constexpr (VEC) {
      *reinterpret_cast<u32x4 *>(Hct + d * ldht + j0 + r) = *reinterpret_cast<const u32x4 *>(e);
    } else {
      __builtin_memcpy(Hct + d * ldht + j0 + r, e, sizeof(U));
    }
  }
}


template <typename TI>
int ce_fwd_run(const TI *H, const TI *W, const int64_t *targets, int64_t M, int64_t D,
               int64_t V, int64_t ignore_index, int64_t chunk_rows, float *loss, int32_t *bad,
               char *state, char *ws, hipStream_t s) {
  using C = MainCfg<TI>;
  using U = typename std::conditional<sizeof(TI) == 2, uint16_t, uint32_t>::type;
  const Plan L = make_plan<TI>(M, D, V, chunk_rows);
  const StateView<TI> S(L, state);
  TI *Hc = reinterpret_cast<TI *>(ws + L.f_hc);
  int *rows = reinterpret_cast<int *>(ws + L.f_rows);
  int *tcol = reinterpret_cast<int *>(ws + L.f_tcol);
  float2 *stats = reinterpret_cast<float2 *>(ws + L.f_stats);
  float *tgt = reinterpret_cast<float *>(ws + L.f_tgt);
  float *mref = reinterpret_cast<float *>(ws + L.f_mref);
  float *loss_row = reinterpret_cast<float *>(ws + L.f_loss);
  float *part = reinterpret_cast<float *>(ws + L.f_part);
  int e;

  ce_compact_kernel<<<1, kCompactThreads, 0, s>>>(targets, M, V, ignore_index, rows, tcol,
                                                  S.pos, S.n, S.inv, bad);
  if ((e = check_launch("ce_compact"))) return e;
  const bool vec = D % (16 / (int64_t)sizeof(TI)) == 0 && aligned16(H) && aligned16(W) &&
                   aligned16(Hc);
  {
    constexpr int kRowsPerBlock = kGatherThreads / 64;
    int64_t blocks = (M + kRowsPerBlock - 1) / kRowsPerBlock;
    if (blocks > 4096) blocks = 4096;
    if (vec)
      ce_gather_kernel<TI, true><<<(unsigned)blocks, kGatherThreads, 0, s>>>(
          H, W, D, rows, tcol, S.n, M, Hc, mref);
    else
      ce_gather_kernel<TI, false><<<(unsigned)blocks, kGatherThreads, 0, s>>>(
          H, W, D, rows, tcol, S.n, M, Hc, mref);
    if ((e = check_launch("ce_gather"))) return e;
  }
  // W^T is only read by the dH product: with 16-bit elements and 16-byte
  // rows it is formed by extra blocks at the end of the first logits launch,
  // otherwise by its own launch here
  gemm::TpJobs tp{};
  const bool fold = sizeof(TI) == 2 && D % 8 == 0 && L.ldwt % 8 == 0 && aligned16(W) &&
                    aligned16(S.Wt);
  if (fold) {
    tp.in[0] = reinterpret_cast<const uint16_t *>(W);
    tp.out[0] = reinterpret_cast<uint16_t *>(S.Wt);
    tp.R[0] = V;
    tp.Cn[0] = D;
    tp.ldi[0] = D;
    tp.ldo[0] = L.ldwt;
    tp.rb[0] = (int)((L.ldwt + gemm::kTpRegionRows - 1) / gemm::kTpRegionRows);
    tp.cb[0] = (int)((D + gemm::kTpRegionCols - 1) / gemm::kTpRegionCols);
    tp.n = tp.rb[0] * tp.cb[0];
  } else if ((e = launch_transpose<U>(W, V, D, D, S.Wt, L.ldwt, s))) {
    return e;
  }
  const gemm::TpJobs none{};

  const bool vk = buf_ok<TI>(Hc, D, M, D) && buf_ok<TI>(W, D, V, D);
  const bool sb = sb_ok(L.crows * L.ldp * (int64_t)sizeof(TI));
  const unsigned glog = (unsigned)(L.vtiles * L.ttiles);
  TI *const PT = L.single ? nullptr : S.PT;
  const dim3 gprep((unsigned)(L.crows / 64), (unsigned)((D + 63) / 64));
  for (int64_t c = 0; c < L.nch; ++c) {
    const int64_t j0 = c * L.crows;
    const gemm::TpJobs &tj = c == 0 ? tp : none;
    const unsigned grid = glog + (unsigned)tj.n;
    if (vk && sb)
      ce_logits_kernel<C, true, true><<<grid, C::NT, 0, s>>>(
          W, Hc, V, D, j0, L.crows, S.n, tcol, mref, stats, tgt, S.P, L.ldp, PT, L.crows,
          L.vtiles, L.ttiles, tj);
    else if (vk)
      ce_logits_kernel<C, true, false><<<grid, C::NT, 0, s>>>(
          W, Hc, V, D, j0, L.crows, S.n, tcol, mref, stats, tgt, S.P, L.ldp, PT, L.crows,
          L.vtiles, L.ttiles, tj);
    else
      ce_logits_kernel<C, false, false><<<grid, C::NT, 0, s>>>(
          W, Hc, V, D, j0, L.crows, S.n, tcol, mref, stats, tgt, S.P, L.ldp, PT, L.crows,
          L.vtiles, L.ttiles, tj);
    if ((e = check_launch("ce_logits"))) return e;
    ce_lse_kernel<TI><<<(unsigned)(L.crows / kLseRows), kLseThreads, 0, s>>>(
        stats, L.ntiles, L.wtm, L.crows, tgt, S.n, j0, S.inv, tcol, mref, S.cfac, loss_row, S.P,
        L.ldp, PT, L.crows, V);
    if ((e = check_launch("ce_lse"))) return e;
    const bool last = c + 1 == L.nch;  // the mean loss comes with the last chunk's launch
    if (vec)
      ce_scale_hct_kernel<TI, true><<<gprep, kPrepThreads, 0, s>>>(
          Hc, D, S.cfac, S.n, j0, L.crows, S.Hct, L.ldht, loss_row, S.inv, last ? loss : nullptr);
    else
      ce_scale_hct_kernel<TI, false><<<gprep, kPrepThreads, 0, s>>>(
          Hc, D, S.cfac, S.n, j0, L.crows, S.Hct, L.ldht, loss_row, S.inv, last ? loss : nullptr);
    if ((e = check_launch("ce_scale_hct"))) return e;
    if (!last &&
        (e = launch_grads<TI>(L, S, c, D, V, c > 0 ? S.dWacc : nullptr, S.dWacc, NF_DTYPE_F32,
                              nullptr, part, s, /*final_dw=*/false)))
      return e;
  }
  return NF_OK;
}

template <typename TI>
int ce_bwd_run(int64_t M, int64_t D, int64_t V, int64_t chunk_rows, char *state,
               const float *g, void *dH, int dt_h, void *dW, int dt_w, char *ws, hipStream_t s) {
  const Plan L = make_plan<TI>(M, D, V, chunk_rows);
  const StateView<TI> S(L, state);
  float *part = reinterpret_cast<float *>(ws + L.b_part);
  int e;
  // the last chunk's split dH slices are added by the scatter below
  if ((e = launch_grads<TI>(L, S, L.nch - 1, D, V, L.nch > 1 ? S.dWacc : nullptr, dW, dt_w, g,
                            part, s, /*final_dw=*/true, /*reduce_dh=*/false)))
    return e;
  const SplitRows sp{part, L.split.S, (L.nch - 1) * L.crows, L.crows, S.cfac};
  const bool vec = D % 4 == 0;  // dHc rows and slices are then 16-byte aligned
  int64_t blocks = (M * (vec ? D / 4 : D) + 255) / 256;
  if (blocks > 4096) blocks = 4096;
  if (vec)
    ce_scatter_dh_kernel<4><<<(unsigned)blocks, 256, 0, s>>>(S.dHc, D, S.pos, M, g, dH, dt_h,
                                                             sp);
  else
    ce_scatter_dh_kernel<1><<<(unsigned)blocks, 256, 0, s>>>(S.dHc, D, S.pos, M, g, dH, dt_h,
                                                             sp);
  return check_launch("ce_scatter_dh");
}

}  // namespace ce
}  // namespace nf

using namespace nf;
using namespace nf::ce;

extern "C" size_t nf_ce_state_bytes(int64_t M, int64_t D, int64_t V, int64_t chunk_rows,
                                    int dtype) {
  if (!ce_sizes_ok(M, D, V) || chunk_rows <= 0 || !dtype_ok(dtype)) return 0;
  return plan_of(M, D, V, chunk_rows, dtype).s_total;
}

extern "C" size_t nf_ce_fwd_workspace(int64_t M, int64_t D, int64_t V, int64_t chunk_rows,
                                      int dtype) {
  if (!ce_sizes_ok(M, D, V) || chunk_rows <= 0 || !dtype_ok(dtype)) return 0;
  return plan_of(M, D, V, chunk_rows, dtype).f_total;
}

extern "C" size_t nf_ce_bwd_workspace(int64_t M, int64_t D, int64_t V, int64_t chunk_rows,
                                      int dtype) {
  if (!ce_sizes_ok(M, D, V) || chunk_rows <= 0 || !dtype_ok(dtype)) return 0;
  const size_t b = plan_of(M, D, V, chunk_rows, dtype).b_total;
  return b > 0 ? b : 256;  // never 0 for a valid shape (0 marks a refusal)
}

extern "C" int nf_ce_fwd(const void *hidden, const void *weight, const int64_t *targets,
                         int64_t M, int64_t D, int64_t V, int64_t ignore_index,
                         int64_t chunk_rows, int dtype, float *loss, int32_t *bad_targets,
                         void *state, size_t state_bytes, void *workspace,
                         size_t workspace_bytes, void *stream) {
  if (int e = ce_check_shape("nf_ce_fwd", M, D, V)) return e;
  if (chunk_rows <= 0) return set_error(NF_ERR_ARG, "nf_ce_fwd: chunk_rows must be > 0");
  if (!hidden || !weight || !targets || !loss || !state)
    return set_error(NF_ERR_ARG, "nf_ce_fwd: null pointer");
  if (int e = ce_check_dtype("nf_ce_fwd", dtype)) return e;
  const Plan L = plan_of(M, D, V, chunk_rows, dtype);
  if (state_bytes < L.s_total || !aligned16(state))
    return set_error(NF_ERR_WORKSPACE, "nf_ce_fwd: state %zu bytes < required %zu",
                     state_bytes, L.s_total);
  if (!workspace || workspace_bytes < L.f_total || !aligned16(workspace))
    return set_error(NF_ERR_WORKSPACE, "nf_ce_fwd: workspace %zu bytes < required %zu",
                     workspace_bytes, L.f_total);
  hipStream_t s = static_cast<hipStream_t>(stream);
  char *st = static_cast<char *>(state), *ws = static_cast<char *>(workspace);
  if (dtype == NF_DTYPE_BF16)
    return ce_fwd_run<bf16>((const bf16 *)hidden, (const bf16 *)weight, targets, M, D, V,
                            ignore_index, chunk_rows, loss, bad_targets, st, ws, s);
  return ce_fwd_run<float>((const float *)hidden, (const float *)weight, targets, M, D, V,
                           ignore_index, chunk_rows, loss, bad_targets, st, ws, s);
}

extern "C" int nf_ce_bwd(int64_t M, int64_t D, int64_t V, int64_t chunk_rows, int dtype,
                         void *state, size_t state_bytes, const float *grad_output,
                         void *dhidden, int dt_hidden, void *dweight, int dt_weight,
                         void *workspace, size_t workspace_bytes, void *stream) {
  if (int e = ce_check_shape("nf_ce_bwd", M, D, V)) return e;
  if (chunk_rows <= 0) return set_error(NF_ERR_ARG, "nf_ce_bwd: chunk_rows must be > 0");
  if (!state || !dhidden || !dweight) return set_error(NF_ERR_ARG, "nf_ce_bwd: null pointer");
  if (int e = ce_check_dtype("nf_ce_bwd", dtype)) return e;
  if (!is_dtype(dt_hidden) || !is_dtype(dt_weight))
    return set_error(NF_ERR_DTYPE, "nf_ce_bwd: gradient dtypes %d, %d", dt_hidden, dt_weight);
  const Plan L = plan_of(M, D, V, chunk_rows, dtype);
  if (state_bytes < L.s_total || !aligned16(state))
    return set_error(NF_ERR_WORKSPACE, "nf_ce_bwd: state %zu bytes < required %zu",
                     state_bytes, L.s_total);
  const size_t need = nf_ce_bwd_workspace(M, D, V, chunk_rows, dtype);
  if (!workspace || workspace_bytes < need || !aligned16(workspace))
    return set_error(NF_ERR_WORKSPACE, "nf_ce_bwd: workspace %zu bytes < required %zu",
                     workspace_bytes, need);
  hipStream_t s = static_cast<hipStream_t>(stream);
  char *st = static_cast<char *>(state), *ws = static_cast<char *>(workspace);
  if (dtype == NF_DTYPE_BF16)
    return ce_bwd_run<bf16>(M, D, V, chunk_rows, st, grad_output, dhidden, dt_hidden, dweight,
                            dt_weight, ws, s);
  return ce_bwd_run<float>(M, D, V, chunk_rows, st, grad_output, dhidden, dt_hidden, dweight,
                           dt_weight, ws, s);
}

// one call: [state | forward and backward scratch, overlapped]
extern "C" size_t nf_ce_workspace(int64_t M, int64_t D, int64_t V, int64_t chunk_rows,
                                  int dtype) {
  const size_t st = nf_ce_state_bytes(M, D, V, chunk_rows, dtype);
  const size_t f = nf_ce_fwd_workspace(M, D, V, chunk_rows, dtype);
  const size_t b = nf_ce_bwd_workspace(M, D, V, chunk_rows, dtype);
  if (!st || !f || !b) return 0;
  return st + (f > b ? f : b);
}

extern "C" int nf_ce_fwd_bwd(const void *hidden, const void *weight, const int64_t *targets,
                             int64_t M, int64_t D, int64_t V, int64_t ignore_index,
                             int64_t chunk_rows, int dtype, float *loss, float *dhidden,
                             float *dweight, int32_t *bad_targets, void *workspace,
                             size_t workspace_bytes, void *stream) {
  if (int e = ce_check_shape("nf_ce_fwd_bwd", M, D, V)) return e;
  if (chunk_rows <= 0) return set_error(NF_ERR_ARG, "nf_ce_fwd_bwd: chunk_rows must be > 0");
  if (!hidden || !weight || !targets || !loss || !dhidden || !dweight)
    return set_error(NF_ERR_ARG, "nf_ce_fwd_bwd: null pointer");
  if (int e = ce_check_dtype("nf_ce_fwd_bwd", dtype)) return e;
  const size_t need = nf_ce_workspace(M, D, V, chunk_rows, dtype);
  if (!workspace || workspace_bytes < need || !aligned16(workspace))
    return set_error(NF_ERR_WORKSPACE, "nf_ce_fwd_bwd: workspace %zu bytes < required %zu",
                     workspace_bytes, need);
  const size_t sb = nf_ce_state_bytes(M, D, V, chunk_rows, dtype);
  char *ws = static_cast<char *>(workspace);
  if (int e = nf_ce_fwd(hidden, weight, targets, M, D, V, ignore_index, chunk_rows, dtype, loss,
                        bad_targets, ws, sb, ws + sb, workspace_bytes - sb, stream))
    return e;
  return nf_ce_bwd(M, D, V, chunk_rows, dtype, ws, sb, nullptr, dhidden, NF_DTYPE_F32, dweight,
                   NF_DTYPE_F32, ws + sb, workspace_bytes - sb, stream);
}
