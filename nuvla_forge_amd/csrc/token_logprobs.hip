// Token log probabilities on the language-model head: for every row m of hidden, with
// z = hidden[m] . weight^T,
//   lse = log sum exp z,   logprob = z[target] - lse,
//   entropy = -sum p (z - lse),  p = exp(z - lse),
//   and the top_k largest z with their columns (ties: the lower column first),
// and the gradient of logprob and entropy by hidden and weight.  The [M, V] logits are
// never held at once; all on the caller's stream, sums in fixed orders, no atomics.
//
// Only valid rows (target != ignore_index, inside [0, V)) do any work: they are compacted
// on the device and every later kernel sizes itself by the device count.
//
// Forward (nf_token_logprobs_fwd):
//   1. ce_compact: the valid rows in order.  lp_gather: Hc = hidden[rows], and zeros (id
//      -1) into the outputs of the other rows.
//   2. per chunk of rows: the logits, then lp_rows: a block per row.
// Backward (nf_token_logprobs_bwd), with g and h the upstream gradients of a row's logprob
// and entropy H:
//   dz = g (onehot - p) - h p (z - lse + H)
//   lp_dz:  z formed again tile by tile (W Hc^T, as in the cross entropy's logits) and
//           turned into dz in the accumulators; one rounding to the input type;
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
// valid get 0 in every output (id -1).  One wavefront per row.
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
    const int *n_ptr, int64_t M, T *__restrict__ Hc, RowOut out) {
  constexpr int kWaves = kGatherThreads / 64;
  constexpr int VE = VEC ? 16 / (int)sizeof(T) : 1;
  const int64_t n = *n_ptr;
  const int l = threadIdx.x & 63;
  for (int64_t r = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6); r < M;
       r += (int64_t)gridDim.x * kWaves) {
    const T *h = r < n ? H + (int64_t)rows[r] * D : nullptr;
    for (int64_t c = (int64_t)l * VE; c < D; c += 64 * VE) {
      if constexpr (VEC) {
        u32x4 v = {0u, 0u, 0u, 0u};
        if (h) v = *reinterpret_cast<const u32x4 *>(h + c);
        *reinterpret_cast<u32x4 *>(Hc + r * D + c) = v;
      } else {
        Hc[r * D + c] = h ? h[c] : static_cast<T>(0.f);
      }
    }
    if (pos[r] < 0) {
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
// 2. a row's outputs from its logits: the maximum, then S = sum exp(z - max) and
// T = sum (z - max) exp(z - max) (log p and the entropy follow: lse = max + log S,
// H = log S - T / S), then the top_k largest, each the largest entry after the one
// before it in the order (value down, column up).
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 256;

__device__ __forceinline__ bool before(float va, int ia, float vb, int ib) {
  return va > vb || (va == vb && ia < ib);
}

template <typename F>
__device__ __forceinline__ float block_reduce(float v, float *sh, F op) {
  for (int d = 32; d; d >>= 1) v = op(v, __shfl_xor(v, d));
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
  for (int k = 1; k < kRowThreads / 64; ++k) v = op(v, sh[k]);
  __syncthreads();
  return v;
}

__global__ __launch_bounds__(kRowThreads) void lp_rows_kernel(
    const float *__restrict__ Z, int64_t ldz, int64_t V, const int *n_ptr, int64_t j0,
    int64_t crows, const int *__restrict__ rows, const int *__restrict__ tcol,
    float *__restrict__ lse_out, float *__restrict__ ent_out, RowOut out) {
  __shared__ float sh[kRowThreads / 64];
  __shared__ float sv[kRowThreads / 64];
  __shared__ int si[kRowThreads / 64];
  const int64_t row = blockIdx.x;
  if (row >= chunk_count(n_ptr, j0, crows)) return;
  const float *z = Z + row * ldz;
  float mx = -INFINITY;
  for (int64_t c = threadIdx.x; c < V; c += kRowThreads) mx = fmaxf(mx, z[c]);
  mx = block_reduce(mx, sh, [](float a, float b) { return fmaxf(a, b); });
  float s = 0.f, t = 0.f;
  for (int64_t c = threadIdx.x; c < V; c += kRowThreads) {
    const float x = z[c] - mx;
    const float e = exp_f32(x);
    s += e;
    t += x < kFar ? 0.f : x * e;
  }
  auto add = [](float a, float b) { return a + b; };
  s = block_reduce(s, sh, add);
  t = block_reduce(t, sh, add);
  const float ls = log_f32(s), lse = mx + ls, ent = ls - t / s;
  const int64_t m = rows[j0 + row];
  if (threadIdx.x == 0) {
    lse_out[j0 + row] = lse;
    ent_out[j0 + row] = ent;
    out.logprob[m] = z[tcol[j0 + row]] - lse;
    out.entropy[m] = ent;
  }
  float pv = INFINITY;
  int pi = -1;
  for (int k = 0; k < out.top_k; ++k) {
    float bv = -INFINITY;
    int bi = 0x7fffffff;
    for (int64_t c = threadIdx.x; c < V; c += kRowThreads) {
      const float v = z[c];
      if (before(pv, pi, v, (int)c) && before(v, (int)c, bv, bi)) {
        bv = v;
        bi = (int)c;
      }
    }
    for (int d = 32; d; d >>= 1) {
      const float ov = __shfl_xor(bv, d);
      const int oi = __shfl_xor(bi, d);
      if (before(ov, oi, bv, bi)) {
        bv = ov;
        bi = oi;
      }
    }
    if ((threadIdx.x & 63) == 0) {
      sv[threadIdx.x >> 6] = bv;
      si[threadIdx.x >> 6] = bi;
    }
    __syncthreads();
    for (int q = 0; q < kRowThreads / 64; ++q)
      if (before(sv[q], si[q], bv, bi)) {
        bv = sv[q];
        bi = si[q];
      }
    __syncthreads();
    if (threadIdx.x == 0) {
      out.top_lp[m * out.top_k + k] = bi < V ? bv - lse : __builtin_nanf("");
      out.top_id[m * out.top_k + k] = bi < V ? bi : -1;
    }
    pv = bv;
    pi = bi;
  }
}

// ---------------------------------------------------------------------------
// backward: dz of one chunk, in the layouts of ce::EStore
// ---------------------------------------------------------------------------
struct RowIn {
  const int *n, *rows, *tcol;       // compacted rows
  const float *lse, *ent;           // per compacted row
  const float *g, *h;               // upstream, per row of hidden; either may be null
};

template <class C, bool BUF, bool SB>
__global__ NF_GEMM_BOUNDS(C) void lp_dz_kernel(
    const typename C::TI *W, const typename C::TI *Hc, int64_t V, int64_t D, int64_t j0,
    int64_t crows, RowIn in, float *ones, typename C::TI *E, int64_t ldp, typename C::TI *ET,
    int64_t ldet, int vtiles, int ttiles, gemm::TpJobs tp) {
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
  const int64_t cnt = chunk_count(in.n, j0, crows);
  const int64_t v0 = (int64_t)vt * C::BM;
  const int64_t t0 = (int64_t)tt * C::BN;
  if (t0 >= cnt) return;
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
    float g = 0.f, h = 0.f, lse = 0.f, ent = 0.f;
    int want = -1;  // the register that holds the target, if this lane does
    if (tok < cnt) {
      const int64_t m = in.rows[j0 + tok];
      g = in.g ? in.g[m] : 0.f;
      h = in.h ? in.h[m] : 0.f;
      lse = in.lse[j0 + tok];
      ent = in.ent[j0 + tok];
      const int64_t loc64 = (int64_t)in.tcol[j0 + tok] - vtile0;
      const int loc = (int)(loc64 >= 0 && loc64 < C::WTM ? loc64 : -1);
      if (loc >= 0 && ((loc >> 2) & 1) == half)
        want = ((loc >> 5) << 4) | (((loc & 31) >> 3) << 2) | (loc & 3);
    }
    const float a = -(g + h * ent);
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float x = acc[i][j][r] - lse;
        x = x < kFar ? kFar : x;  // a NaN stays one
        const float dz = exp_f32(x) * (a - h * x);
        acc[i][j][r] = i * 16 + r == want ? dz + g : dz;
      }
    store.column(j, acc);
  }
  store.finish();
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// What the forward keeps for the backward.
struct State {
  size_t scal, rows, tcol, pos, lse, ent, hc, total;
};
template <typename TI>
State state_layout(int64_t M, int64_t D) {
  State s{};
  size_t o = 0;
  auto take = [&](size_t bytes) { const size_t at = o; o = align256(o + bytes); return at; };
  s.scal = take(64);
  s.rows = take((size_t)M * sizeof(int));
  s.tcol = take((size_t)M * sizeof(int));
  s.pos = take((size_t)M * sizeof(int));
  s.lse = take((size_t)M * sizeof(float));
  s.ent = take((size_t)M * sizeof(float));
  s.hc = take((size_t)M * D * sizeof(TI));
  s.total = o;
  return s;
}
template <typename TI>
struct View {
  int *n;
  float *inv;
  int *rows, *tcol, *pos;
  float *lse, *ent;
  TI *Hc;
  View(const State &L, char *s)
      : n(reinterpret_cast<int *>(s + L.scal)),
        inv(reinterpret_cast<float *>(s + L.scal + 16)),
        rows(reinterpret_cast<int *>(s + L.rows)),
        tcol(reinterpret_cast<int *>(s + L.tcol)),
        pos(reinterpret_cast<int *>(s + L.pos)),
        lse(reinterpret_cast<float *>(s + L.lse)),
        ent(reinterpret_cast<float *>(s + L.ent)),
        Hc(reinterpret_cast<TI *>(s + L.hc)) {}
};

struct FwdPlan {
  int64_t crows, ldz;
  size_t z, total;
};
template <typename TI>
FwdPlan fwd_plan(int64_t M, int64_t V, int64_t chunk_rows) {
  FwdPlan p{};
  const int64_t mcap = round_up(M, 256);
  p.crows = chunk_rows < mcap ? round_up(chunk_rows, 256) : mcap;
  p.ldz = round_up(V, 8);
  p.z = 0;
  p.total = align256((size_t)p.crows * p.ldz * sizeof(float));
  return p;
}

template <typename TI>
int fwd_run(const TI *H, const TI *W, const int64_t *targets, int64_t M, int64_t D, int64_t V,
            int64_t ignore_index, int64_t chunk_rows, const RowOut &out, char *state, char *ws,
            hipStream_t s) {
  using C = MainCfg<TI>;
  const View<TI> S(state_layout<TI>(M, D), state);
  const FwdPlan P = fwd_plan<TI>(M, V, chunk_rows);
  float *Z = reinterpret_cast<float *>(ws + P.z);
  int e;
  ce::ce_compact_kernel<<<1, ce::kCompactThreads, 0, s>>>(targets, M, V, ignore_index, S.rows,
                                                          S.tcol, S.pos, S.n, S.inv, nullptr);
  if ((e = check_launch("ce_compact"))) return e;
  const bool vec = D % (16 / (int64_t)sizeof(TI)) == 0 && aligned16(H) && aligned16(S.Hc);
  int64_t blocks = (M + 3) / 4;
  if (blocks > 4096) blocks = 4096;
  if (vec)
    lp_gather_kernel<TI, true><<<(unsigned)blocks, kGatherThreads, 0, s>>>(H, D, S.rows, S.pos,
                                                                           S.n, M, S.Hc, out);
  else
    lp_gather_kernel<TI, false><<<(unsigned)blocks, kGatherThreads, 0, s>>>(H, D, S.rows, S.pos,
                                                                            S.n, M, S.Hc, out);
  if ((e = check_launch("lp_gather"))) return e;
  for (int64_t j0 = 0; j0 < M; j0 += P.crows) {
    const int64_t rows = M - j0 < P.crows ? M - j0 : P.crows;
    auto jz = make_job<C>(S.Hc + j0 * D, D, W, D, nullptr, Z, NF_DTYPE_F32, nullptr, P.ldz, rows,
                          V, D);
    jz.dyn = S.n;
    jz.dyn_base = j0;
    jz.dyn_rows = 1;
    auto none = jz;
    none.tiles = 0;
    if ((e = launch_gemm_store<C>(jz, none, s))) return e;
    lp_rows_kernel<<<(unsigned)rows, kRowThreads, 0, s>>>(Z, P.ldz, V, S.n, j0, rows, S.rows,
                                                          S.tcol, S.lse, S.ent, out);
    if ((e = check_launch("lp_rows"))) return e;
  }
  return NF_OK;
}

template <typename TI>
int bwd_run(const TI *W, int64_t M, int64_t D, int64_t V, int64_t chunk_rows, char *state,
            const float *g, const float *h, void *dH, int dt_h, void *dW, int dt_w, char *ws,
            hipStream_t s) {
  using C = MainCfg<TI>;
  using U = typename std::conditional<sizeof(TI) == 2, uint16_t, uint32_t>::type;
  const View<TI> K(state_layout<TI>(M, D), state);
  const ce::Plan L = ce::make_plan<TI>(M, D, V, chunk_rows);
  ce::StateView<TI> S(L, ws);
  S.n = K.n;
  S.pos = K.pos;
  float *part = reinterpret_cast<float *>(ws + L.s_total);
  int e;
  // W^T (the dH product's B operand) and Hc^T (the dW product's), both zero-padded: by
  // extra blocks of the first dz launch where their rows are whole 16-byte vectors of
  // 16-bit elements, else by launches of their own
  gemm::TpJobs tp{};
  const gemm::TpJobs none{};
  const bool fold = sizeof(TI) == 2 && D % 8 == 0 && aligned16(W);
  if (fold) {
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
    add(0, W, V, S.Wt, L.ldwt);
    add(1, K.Hc, M, S.Hct, L.ldht);
  } else {
    if ((e = launch_transpose<U>(W, V, D, D, S.Wt, L.ldwt, s))) return e;
    if ((e = launch_transpose<U>(K.Hc, M, D, D, S.Hct, L.ldht, s))) return e;
  }
  const bool vk = buf_ok<TI>(K.Hc, D, M, D) && buf_ok<TI>(W, D, V, D);
  const bool sb = sb_ok(L.crows * L.ldp * (int64_t)sizeof(TI)) &&
                  (L.single || sb_ok(V * L.crows * (int64_t)sizeof(TI)));
  const RowIn in{K.n, K.rows, K.tcol, K.lse, K.ent, g, h};
  TI *const PT = L.single ? nullptr : S.PT;
  for (int64_t c = 0; c < L.nch; ++c) {
    const int64_t j0 = c * L.crows;
    const gemm::TpJobs &tj = c == 0 ? tp : none;
    const unsigned grid = (unsigned)(L.vtiles * L.ttiles) + (unsigned)tj.n;
    if (vk && sb)
      lp_dz_kernel<C, true, true><<<grid, C::NT, 0, s>>>(W, K.Hc, V, D, j0, L.crows, in, S.cfac,
                                                         S.P, L.ldp, PT, L.crows, L.vtiles,
                                                         L.ttiles, tj);
    else if (vk)
      lp_dz_kernel<C, true, false><<<grid, C::NT, 0, s>>>(W, K.Hc, V, D, j0, L.crows, in, S.cfac,
                                                          S.P, L.ldp, PT, L.crows, L.vtiles,
                                                          L.ttiles, tj);
    else
      lp_dz_kernel<C, false, false><<<grid, C::NT, 0, s>>>(W, K.Hc, V, D, j0, L.crows, in,
                                                           S.cfac, S.P, L.ldp, PT, L.crows,
                                                           L.vtiles, L.ttiles, tj);
    if ((e = check_launch("lp_dz"))) return e;
    const bool last = c + 1 == L.nch;
    if ((e = ce::launch_grads<TI>(L, S, c, D, V, c > 0 ? S.dWacc : nullptr,
                                  last ? dW : S.dWacc, last ? dt_w : NF_DTYPE_F32, nullptr, part,
                                  s, /*final_dw=*/last, /*reduce_dh=*/!last, dW != nullptr,
                                  dH != nullptr)))
      return e;
  }
  if (!dH) return NF_OK;
  const ce::SplitRows sp{part, L.split.S, (L.nch - 1) * L.crows, L.crows, S.cfac};
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

template <typename TI>
size_t bwd_bytes(int64_t M, int64_t D, int64_t V, int64_t chunk_rows) {
  const ce::Plan L = ce::make_plan<TI>(M, D, V, chunk_rows);
  return L.s_total + L.b_total + 256;
}

}  // namespace lp
}  // namespace nf

using namespace nf;
using namespace nf::lp;
using ce::ce_check_dtype;
using ce::ce_check_shape;
using ce::ce_sizes_ok;
using ce::dtype_ok;

extern "C" size_t nf_token_logprobs_state_bytes(int64_t M, int64_t D, int64_t V, int dtype) {
  if (!ce_sizes_ok(M, D, V) || !dtype_ok(dtype)) return 0;
  return dtype == NF_DTYPE_BF16 ? state_layout<bf16>(M, D).total : state_layout<float>(M, D).total;
}

extern "C" size_t nf_token_logprobs_fwd_workspace(int64_t M, int64_t D, int64_t V,
                                                  int64_t chunk_rows, int top_k, int dtype) {
  if (!ce_sizes_ok(M, D, V) || chunk_rows <= 0 || !dtype_ok(dtype) || top_k < 0 ||
      top_k > kMaxTop || top_k > V)
    return 0;
  return dtype == NF_DTYPE_BF16 ? fwd_plan<bf16>(M, V, chunk_rows).total
                                : fwd_plan<float>(M, V, chunk_rows).total;
}

extern "C" size_t nf_token_logprobs_bwd_workspace(int64_t M, int64_t D, int64_t V,
                                                  int64_t chunk_rows, int dtype) {
  if (!ce_sizes_ok(M, D, V) || chunk_rows <= 0 || !dtype_ok(dtype)) return 0;
  return dtype == NF_DTYPE_BF16 ? bwd_bytes<bf16>(M, D, V, chunk_rows)
                                : bwd_bytes<float>(M, D, V, chunk_rows);
}

extern "C" int nf_token_logprobs_fwd(const void *hidden, const void *weight,
                                     const int64_t *targets, int64_t M, int64_t D, int64_t V,
                                     int64_t ignore_index, int64_t chunk_rows, int top_k,
                                     int dtype, float *logprobs, float *entropy,
                                     float *top_logprobs, int64_t *top_ids, void *state,
                                     size_t state_bytes, void *workspace,
                                     size_t workspace_bytes, void *stream) {
  const char *fn = "nf_token_logprobs_fwd";
  if (int e = ce_check_shape(fn, M, D, V)) return e;
  if (chunk_rows <= 0) return set_error(NF_ERR_ARG, "%s: chunk_rows must be > 0", fn);
  if (top_k < 0 || top_k > kMaxTop || top_k > V)
    return set_error(NF_ERR_ARG, "%s: top_k=%d outside [0, min(%d, V)]", fn, top_k, kMaxTop);
  if (!hidden || !weight || !targets || !logprobs || !entropy || !state ||
      (top_k > 0 && (!top_logprobs || !top_ids)))
    return set_error(NF_ERR_ARG, "%s: null pointer", fn);
  if (int e = ce_check_dtype(fn, dtype)) return e;
  const size_t sb = nf_token_logprobs_state_bytes(M, D, V, dtype);
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
                         ignore_index, chunk_rows, out, st, ws, s);
  return fwd_run<float>((const float *)hidden, (const float *)weight, targets, M, D, V,
                        ignore_index, chunk_rows, out, st, ws, s);
}

extern "C" int nf_token_logprobs_bwd(const void *weight, int64_t M, int64_t D, int64_t V,
                                     int64_t chunk_rows, int dtype, void *state,
                                     size_t state_bytes, const float *g_logprobs,
                                     const float *g_entropy, void *dhidden, int dt_hidden,
                                     void *dweight, int dt_weight, void *workspace,
                                     size_t workspace_bytes, void *stream) {
  const char *fn = "nf_token_logprobs_bwd";
  if (int e = ce_check_shape(fn, M, D, V)) return e;
  if (chunk_rows <= 0) return set_error(NF_ERR_ARG, "%s: chunk_rows must be > 0", fn);
  if (!weight || !state) return set_error(NF_ERR_ARG, "%s: null pointer", fn);
  if (int e = ce_check_dtype(fn, dtype)) return e;
  if ((dhidden && !is_dtype(dt_hidden)) || (dweight && !is_dtype(dt_weight)))
    return set_error(NF_ERR_DTYPE, "%s: gradient dtypes %d, %d", fn, dt_hidden, dt_weight);
  const size_t sb = nf_token_logprobs_state_bytes(M, D, V, dtype);
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
    return bwd_run<bf16>((const bf16 *)weight, M, D, V, chunk_rows, st, g_logprobs, g_entropy,
                         dhidden, dt_hidden, dweight, dt_weight, ws, s);
  return bwd_run<float>((const float *)weight, M, D, V, chunk_rows, st, g_logprobs, g_entropy,
                        dhidden, dt_hidden, dweight, dt_weight, ws, s);
}
