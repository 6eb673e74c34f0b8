// What the language-model head's kernels share (the cross entropy in ce.hip, the
// token log probabilities in token_logprobs.hip): the compaction of the rows that
// count, the store of a tile of per-logit values in the layouts that the gradient
// products read, the plan of a call, the gradient products and the scatter of the
// hidden rows' gradient.
#pragma once

#include <initializer_list>
#include <type_traits>

#include "gemm_store.h"

namespace nf {
namespace ce {

using namespace gemm;

__device__ __forceinline__ float log_f32(float x) {
  constexpr float kLn2 = 0.6931471805599453f;  // ln(2)
  return __builtin_amdgcn_logf(x) * kLn2;       // log2 on the hardware
}

__device__ __forceinline__ int64_t chunk_count(const int *n_ptr, int64_t j0, int64_t crows) {
  const int64_t c = (int64_t)__builtin_amdgcn_readfirstlane(*n_ptr) - j0;
  return c < 0 ? 0 : (c > crows ? crows : c);
}

// ---------------------------------------------------------------------------
// 1. compaction of the valid rows, in order.  One block; each round takes
// 4 x 1024 targets, each wavefront ranks its lanes by a ballot, and the
// per-wavefront counts are prefixed through LDS in wavefront order.
// ---------------------------------------------------------------------------
constexpr int kCompactThreads = 1024, kCompactSub = 4;

static __global__ __launch_bounds__(kCompactThreads) void ce_compact_kernel(
    const int64_t *__restrict__ targets, int64_t M, int64_t V, int64_t ignore_index,
    int *__restrict__ rows, int *__restrict__ tcol, int *__restrict__ pos, int *n_out,
    float *inv_out, int *bad_out) {
  constexpr int kWaves = kCompactThreads / 64;
  __shared__ int wsum[kCompactSub][kWaves];
  __shared__ int wbad[kCompactSub][kWaves];
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint64_t below = (1ull << l) - 1ull;
  int carry = 0, bad_total = 0;  // the same in every thread
  for (int64_t base = 0; base < M; base += kCompactThreads * kCompactSub) {
    int64_t tg[kCompactSub];
    bool valid[kCompactSub];
    int before[kCompactSub];
#pragma unroll
    for (int u = 0; u < kCompactSub; ++u) {
      const int64_t m = base + (int64_t)u * kCompactThreads + threadIdx.x;
      tg[u] = m < M ? targets[m] : ignore_index;
      const bool in_range = tg[u] >= 0 && tg[u] < V;
      valid[u] = m < M && tg[u] != ignore_index && in_range;
      const bool bad = m < M && tg[u] != ignore_index && !in_range;
      const uint64_t vm = __ballot(valid[u]);
      const uint64_t bm = __ballot(bad);
      before[u] = __popcll(vm & below);
      if (l == 0) {
        wsum[u][w] = __popcll(vm);
        wbad[u][w] = __popcll(bm);
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kCompactSub; ++u) {
      int off = carry, tot = 0, btot = 0;
      for (int k = 0; k < kWaves; ++k) {
        off += k < w ? wsum[u][k] : 0;
        tot += wsum[u][k];
        btot += wbad[u][k];
      }
      const int64_t m = base + (int64_t)u * kCompactThreads + threadIdx.x;
      if (m < M) {
        if (valid[u]) {
          const int idx = off + before[u];
          rows[idx] = (int)m;
          tcol[idx] = (int)tg[u];
          pos[m] = idx;
        } else {
          pos[m] = -1;
        }
      }
      carry += tot;
      bad_total += btot;
    }
    __syncthreads();  // wsum / wbad are rewritten by the next round
  }
  if (threadIdx.x == 0) {
    *n_out = carry;
    *inv_out = 1.f / (float)(carry > 1 ? carry : 1);
    if (bad_out) *bad_out = bad_total;
  }
}

// ---------------------------------------------------------------------------
// The store of a block tile of per-logit values E held in the accumulators of a
// product formed transposed (rows: vocabulary, columns: tokens): row-major [token,
// ldp] (columns V..ldp as the accumulators hold them, tokens past the chunk's rows
// zero up to a multiple of 8) and, when ET is given, transposed [V, ldet] (tokens
// past the chunk's rows zero up to a multiple of 8).  16-bit 256 x 256 tiles go
// through LDS (free once the K loop ends): element (t, c) at byte t * 512 + 2 *
// (c ^ e_swz(t)), the XOR moving whole 8-element vectors so rows still read as
// 16-byte vectors while the writes of a half-wave spread over the banks, and a
// column gathers its 8 tokens per vector from 8 rows; others straight from the
// accumulators.
// ---------------------------------------------------------------------------
__device__ __forceinline__ int e_swz(int t) { return 8 * (((t >> 3) ^ (t & 7)) & 31); }

// TS: the stored type (16 bits with a 16-bit C).
template <class C, bool SB, typename TS = typename C::TI>
struct EStore {
  using TI = TS;
  static_assert(sizeof(TS) == sizeof(typename C::TI), "as wide as the product's inputs");
  static constexpr int ES = (int)sizeof(TI);
  static constexpr bool kStaged = ES == 2 && C::BM == 256 && C::BN == 256 && C::NT == 512 &&
                                  C::LDS_BYTES >= 256 * 512;
  OutBuf<SB> eout, etout;
  char *smem;
  int64_t V, ldp, ldet, v0, t0, cnt, cnt8;
  bool both;

  __device__ __forceinline__ void init(TI *E, int64_t ldp_, TI *ET, int64_t ldet_, int64_t V_,
                                       int64_t crows, int64_t v0_, int64_t t0_, int64_t cnt_,
                                       char *smem_) {
    V = V_; ldp = ldp_; ldet = ldet_; v0 = v0_; t0 = t0_; cnt = cnt_; smem = smem_;
    both = ET != nullptr;
    eout.init(E, crows * ldp * ES);
    etout.init(ET, V * ldet * ES);
    cnt8 = (cnt + 7) / 8 * 8;
  }

  // token column j of the wavefront's tile, its values in acc[.][j]
  __device__ __forceinline__ void column(int j, const floatx16 (&acc)[C::TM][C::TN]) const {
    const int l = threadIdx.x & 63, half = l >> 5;
    const int w = threadIdx.x >> 6, wm = w / C::WN, wn = w % C::WN;
    const int tl = wn * C::WTN + j * 32 + (l & 31);  // token within the tile
    const int64_t tok = t0 + tl;                     // token within the chunk
    const int64_t crow0 = v0 + wm * C::WTM + 4 * half;  // vocabulary row of (i = 0, r = 0)
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int o = i * 32 + 8 * g;  // offset of r = 4g from crow0
        TI ev[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) ev[q] = static_cast<TI>(acc[i][j][4 * g + q]);
        if constexpr (kStaged) {
          const int cl = wm * C::WTM + 4 * half + o;  // tile column (vocabulary)
          u32x2 packed;
          __builtin_memcpy(&packed, ev, 8);
          *reinterpret_cast<u32x2 *>(smem + tl * 512 + 2 * (cl ^ e_swz(tl))) = packed;
        } else {
          // straight from the accumulators: E row-major and E^T (zero past
          // the chunk's rows, up to the K padding of the dW product)
          const int64_t c = crow0 + o;
          if constexpr (ES == 2) {
            // c and ldp are multiples of 4: the four entries are one 8-byte vector
            u32x2 pk = {0u, 0u};
            if (tok < cnt) __builtin_memcpy(&pk, ev, 8);
            eout.st64((tok * ldp + c) * ES, tok < cnt8 && c < ldp, pk);
            if (both)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const uint16_t bits = (uint16_t)(pk[q >> 1] >> (16 * (q & 1)));
                etout.st16(((c + q) * ldet + tok) * ES, c + q < V && tok < cnt8, bits);
              }
          } else {
            // c and ldp are multiples of 4: the four entries are one vector
            u32x4 pk;
            __builtin_memcpy(&pk, ev, 16);
            eout.st128((tok * ldp + c) * ES, tok < cnt && c < ldp, pk);
#pragma unroll
            for (int q = 0; q < 4; ++q)
              etout.st32(((c + q) * ldet + tok) * ES, c + q < V && tok < cnt8,
                         tok < cnt ? static_cast<float>(ev[q]) : 0.f);
          }
        }
      }
  }

  // After every column, by all threads of the block: the staged tile out of LDS.
  __device__ __forceinline__ void finish() const {
    if constexpr (!kStaged) return;
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    __syncthreads();
    // wavefront w stores tile rows (tokens) 32 w .. 32 w + 31, two per
    // instruction (one per half-wave), as 16-byte vectors; ldp is a multiple
    // of 8, so a vector is wholly inside or outside the row.  Rows from the
    // chunk's count up to a multiple of 8 are zero (K padding of the dW
    // product when it reads E N-major).
    const int hv = l >> 5, c8 = 8 * (l & 31);
#pragma unroll 4
    for (int it = 0; it < 16; ++it) {
      const int t = 32 * w + 2 * it + hv;
      const int64_t tok = t0 + t, c = v0 + c8;
      const u32x4 v = tok < cnt ? *reinterpret_cast<const u32x4 *>(smem + t * 512 +
                                                                    2 * (c8 ^ e_swz(t)))
                                : u32x4{0u, 0u, 0u, 0u};
      eout.st128((tok * ldp + c) * ES, tok < cnt8 && c < ldp, v);
    }
    if (!both) return;  // E held once (the dW product reads it N-major)
    // E^T through transposing LDS reads (ds_read_b64_tr_b16: in each 16-lane
    // group, lane i receives element i % 4 of the 8-byte chunks addressed by
    // lanes i / 4 + 4 q, q = 0..3).  Lane j of a group addresses token row
    // T + 8 (j % 4) + j / 4 (+ 4 for the second read) at tile columns c0 ..
    // c0 + 3, so lane i gets tokens T + 8 (i / 4) .. + 7 of column c0 + i % 4:
    // one 16-byte E^T vector.  A wavefront covers 16 columns x 32 tokens per
    // step, wavefront w columns 32 w .. 32 w + 31; tokens past the chunk's
    // rows are zero up to cnt8 (the dW product's K padding), none beyond.
    typedef short v4s __attribute__((ext_vector_type(4)));
    const int grp = l >> 4, j = l & 15;
#pragma unroll 2
    for (int k = 0; k < 16; ++k) {
      const int C0 = 32 * w + 16 * (k >> 3), T = 32 * (k & 7);
      const int c0 = C0 + 4 * grp;
      const int ra = T + 8 * (j & 3) + (j >> 2), rb = ra + 4;
      const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) v4s *)(smem + ra * 512 + 2 * (c0 ^ e_swz(ra))));
      const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) v4s *)(smem + rb * 512 + 2 * (c0 ^ e_swz(rb))));
      const int64_t v = v0 + c0 + (j & 3), tok = t0 + T + 8 * (j >> 2);
      uint16_t e[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        e[q] = tok + q < cnt ? (uint16_t)a[q] : (uint16_t)0;
        e[4 + q] = tok + 4 + q < cnt ? (uint16_t)b[q] : (uint16_t)0;
      }
      u32x4 pk;
      __builtin_memcpy(&pk, e, 16);
      etout.st128((v * ldet + tok) * ES, v < V && tok < cnt8, pk);
    }
  }
};

// ---------------------------------------------------------------------------
// 6. dH[m, :] = g * dHc[pos[m], :] in dH's type, 0 where pos[m] < 0.
// ---------------------------------------------------------------------------
// VE elements per thread step (4 when D is a multiple of 4: one 16-byte load).
// With sp.S > 1 the last chunk's dH product was left in S fp32 slices
// (`part`, [S, crows, D]): for its rows (compacted index >= sp.j0) the kernel
// forms (sum of the slices in order 0 .. S-1) * (cfac * 1) as
// splitk_reduce_kernel would have written to dHc, then scales by g: the same
// operations in the same order, so the same bits, with one launch and one
// fp32 pass over the rows fewer.
// second > 0: row p's gradient is the sum of compacted rows p and second + p (a dz held as two
// terms: see token_logprobs.hip).
struct SplitRows {
  const float *part;
  int S;
  int64_t j0, crows;
  const float *cfac;
  int64_t second = 0;
};
template <int VE>
__global__ __launch_bounds__(256) void ce_scatter_dh_kernel(const float *__restrict__ dHc,
                                                            int64_t D,
                                                            const int *__restrict__ pos,
                                                            int64_t M, const float *g_ptr,
                                                            void *dH, int dt, SplitRows sp) {
  const float g = g_ptr ? *g_ptr : 1.f;
  const int64_t dv = D / VE;
  const int64_t total = M * dv;
  const int64_t slice = sp.crows * D;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / dv, c = (i - m * dv) * VE;
    const int first = pos[m];
    float v[VE];
    auto take = [&](int64_t p, float (&v)[VE]) {
      if (sp.S > 1 && p >= sp.j0) {
        const float *src = sp.part + (p - sp.j0) * D + c;
        float a[VE];
#pragma unroll
        for (int k = 0; k < VE; ++k) a[k] = 0.f;
        // slices added in order, 8 loads in flight per batch
        constexpr int kBatch = 8;
        for (int q0 = 0; q0 < sp.S; q0 += kBatch) {
          float t[kBatch][VE];
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            if (q0 + u < sp.S) {
              if constexpr (VE == 4) {
                const float4 w = *reinterpret_cast<const float4 *>(src + (q0 + u) * slice);
                t[u][0] = w.x; t[u][1] = w.y; t[u][2] = w.z; t[u][3] = w.w;
              } else {
                t[u][0] = src[(q0 + u) * slice];
              }
            }
          }
#pragma unroll
          for (int u = 0; u < kBatch; ++u)
            if (q0 + u < sp.S)
#pragma unroll
              for (int k = 0; k < VE; ++k) a[k] += t[u][k];
        }
        const float f = sp.cfac[p] * 1.f;
#pragma unroll
        for (int k = 0; k < VE; ++k) v[k] = a[k] * f;
      } else if constexpr (VE == 4) {
        const float4 q = p >= 0 ? *reinterpret_cast<const float4 *>(dHc + p * D + c)
                                : make_float4(0.f, 0.f, 0.f, 0.f);
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
      } else {
        v[0] = p >= 0 ? dHc[p * D + c] : 0.f;
      }
    };
    take(first, v);
    if (sp.second > 0 && first >= 0) {
      float t[VE];
      take(sp.second + first, t);
#pragma unroll
      for (int k = 0; k < VE; ++k) v[k] += t[k];
    }
#pragma unroll
    for (int k = 0; k < VE; ++k) store_dyn(dH, dt, m * D + c + k, v[k] * g);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// K split of a chunk's dH product.  The launch holding a chunk's gradient
// products has the dW blocks (K = the chunk's rows) and the dH blocks
// (K = V, long); dH is split into S slices so that the two kinds of blocks
// fill the 256 CUs to the same end: S minimises the launch's makespan, plus
// the write and (partly hidden) read of the S fp32 slices (~5 TB/s).  Block times from
// timestamps in the launch (us): a 64-deep stage of a 256 x 256 or 256 x 192
// tile 1.3-1.8 with K-contiguous operands and 1.8-2.0 with the N-major E
// (single), a 32-deep stage of the fp32 256 x 128 tile ~2; on top of its stages
// ~12 for a dW block (the accumulator's rows read before, stored after) and ~8
// for a dH block.  dcols: tile extent along D (C::BN, or 192).
// Swept (forward + backward): M 12289 D 384 V 50001 2.35 ms with 8 slices (8 of
// the 392 dW blocks are left to a last round of their own), 2.29 with 7, 2.45
// with 12-16; M 300 D 1024 V 128256 557 us with 16, 578 with 14 or 18, 647 with
// 8; M 4096 D 2048 V 32000 1.39 ms unsplit, 1.41 with 2, 1.51 with 8.
// Over 353 bf16 and 108 fp32 shapes, each with every split, the choice is 1.1%
// and 2.5% off the best in the geometric mean; with 1.5 passes for bf16 too it was
// 1.3%, and too many slices where D is small: M 2048 D 256 V 50001 321 us with
// 46, 295 with 32; M 2048 D 512 V 32000 282 with 16, 262 with 8.
struct Split {
  int S;
  int64_t kslice;
};
template <class C>
inline Split dh_split(int64_t rows, int64_t D, int64_t V, int64_t ldp, bool single,
                      int64_t dcols) {
  const int64_t tn = (D + dcols - 1) / dcols;
  const int64_t nw = (V + C::BM - 1) / C::BM * tn;
  const int64_t nh = (rows + C::BM - 1) / C::BM * tn;
  const bool half = sizeof(typename C::TI) == 2;
  const double nt = half ? 1.65 : 2.0;
  const double slices = half ? 2.0 : 1.5;  // passes over the slices, by the sweep
  const double lw = (double)((rows + C::BK - 1) / C::BK) * (single ? 1.9 : nt) + 12.0;
  Split best{1, ldp};
  double best_t = -1.0;
  for (int S = 1; S <= 64; S += S < 16 ? 1 : 4) {
    const int64_t ks = round_up((ldp + S - 1) / S, C::BK);
    const int64_t se = (ldp + ks - 1) / ks;
    const double lh = (double)(ks / C::BK) * nt + 8.0;
    double t = lh >= lw ? two_job_makespan(nh * se, lh, nw, lw)
                        : two_job_makespan(nw, lw, nh * se, lh);
    // the XCDs take contiguous ranges of a job's blocks: slices that are not
    // whole ranges share no operands there
    if (se % 8 != 0 && 8 % se != 0) t *= 1.04;
    if (se > 1) t += slices * (double)(se * rows * D) * 4.0 / 5e12 * 1e6;
    if (best_t < 0 || t < best_t - 1e-9) {
      best_t = t;
      best = {(int)se, ks};
    }
  }
  return best;
}

struct Plan {
  int64_t crows, nch;     // compacted rows per chunk (a multiple of 256), chunks
  int64_t ldp, ldwt, ldht;
  int wtm, ntiles;        // statistics tile height and count
  int vtiles, ttiles;     // logits grid
  Split split;            // dH product's K split
  // single: E is held once, as P (16-bit inputs): the dW product reads it
  // N-major, so a chunk holds twice the rows of the two-layout form in the
  // same bytes, and the fp32 dW accumulator is kept transposed, [D, ldp]
  bool single;
  // d192: the gradient products' tiles take 192 of the D extent, not 256
  bool d192;
  // state (kept from nf_ce_fwd to nf_ce_bwd)
  size_t s_scal, s_pos, s_cfac, s_wt, s_hct, s_p, s_pt, s_dhc, s_dwacc, s_total;
  // forward scratch
  size_t f_hc, f_rows, f_tcol, f_mref, f_stats, f_tgt, f_loss, f_part, f_total;
  // backward scratch
  size_t b_part, b_total;
};

// Row stride, in elements of `es` bytes, of matrices whose rows are read in
// 128-byte K slices: whole 128-byte lines once that pads a row by less than
// 1.6%, so a slice is one line and not parts of two.  V 50001 and M 12289 at
// D 384, forward + backward: 2.39 ms with padded rows, 2.61 with rows of whole
// 16-byte vectors.  column_bytes: what a column takes in each of the matrices; a
// matrix that only the padding would take past the 2 GiB of buffer addressing
// (element-wise copies from there on) keeps rows of whole vectors.
inline int64_t line_stride(int64_t n, size_t es, std::initializer_list<int64_t> column_bytes) {
  const int64_t plain = round_up(n, 8);
  const int64_t lines = n < 4096 ? plain : round_up(n, 128 / (int64_t)es);
  for (int64_t b : column_bytes)
    if (sb_ok(plain * b) && !sb_ok(lines * b)) return plain;
  return lines;
}

// BOTH: 16-bit E may be held in both layouts where they fit (see below); else always once.
template <typename TI, bool BOTH>
inline Plan plan_shape(int64_t M, int64_t D, int64_t V, int64_t chunk_rows) {
  using C = MainCfg<TI>;
  const size_t es = sizeof(TI);
  Plan P{};
  const int64_t mcap = round_up(M, 256);
  const int64_t want = chunk_rows < 1 ? 1 : (chunk_rows > mcap ? mcap : chunk_rows);
  if (sizeof(TI) == 2) {
    // chunk_rows bounds E and the dW accumulator together by what the
    // reference's chunk loop holds for the same roles: an fp32
    // [chunk_rows, V] logits tile and an fp32 [V, D] dW accumulator, i.e.
    // 2 (chunk_rows + D) rows of 16-bit E.  The first form inside it of:
    //  * one chunk, E in both layouts (2 mcap rows), for D >= 2048 only:
    //    the dW product on K-contiguous operands (one chunk, V 32000, fwd+bwd:
    //    M4096 D4096 2.96 ms against 3.06 held once; M8192 D2048 3.02
    //    against 3.05; M4096 D2048 level);
    //  * one chunk, E held once (mcap rows), no accumulator pass (at D 384 -
    //    1024 also faster than both layouts: M4096 D384 0.52 ms against
    //    0.55, M2048 D384 0.28 against 0.30-0.32, M1024 D1024 0.31 against
    //    0.33; at cfg4, M4096 D2048 with 3687 valid rows, the accumulator
    //    alone is the bytes of E for every row, and chunk_size 1024 runs in
    //    1.41-1.46 ms against 1.64 in two chunks);
    //  * chunks of 2 chunk_rows rows held once, beside the fp32 accumulator.
    const int64_t budget = 2 * ((chunk_rows < M ? chunk_rows : M) + D);
    P.single = !BOTH || D < 2048 || 2 * mcap > budget;
    const int64_t cr = P.single && mcap > budget ? round_up(2 * want, 256) : mcap;
    P.crows = cr > mcap ? mcap : cr;
  } else {
    // fp32: chunks of chunk_rows rows in both layouts (E alone is the
    // reference's tile) with the fp32 accumulator between them
    P.single = false;
    const int64_t cr = round_up(want, 256);
    P.crows = cr > mcap ? mcap : cr;
  }
  P.nch = (M + P.crows - 1) / P.crows;
  const int64_t eb = (int64_t)es;
  P.ldp = line_stride(V, es, {P.crows * eb, D * eb, P.single && P.nch > 1 ? D * 4 : 0});
  P.ldwt = P.ldp;
  P.ldht = line_stride(M, es, {D * eb});
  P.wtm = C::WTM;
  P.vtiles = (int)((V + C::BM - 1) / C::BM);
  P.ntiles = P.vtiles * C::WM;
  P.ttiles = (int)(P.crows / C::BN);
  // With E held once D is a tile extent of both gradient products (rows of
  // dW^T, columns of dH); a 192 tile reads ~6% more operand per product.
  P.d192 = P.single && round_up(D, 192) * 1.06 < round_up(D, 256);
  P.split = dh_split<C>(P.crows < M ? P.crows : M, D, V, P.ldp, P.single, P.d192 ? 192 : C::BN);
  const size_t part = P.split.S > 1 ? (size_t)P.split.S * P.crows * D * sizeof(float) : 0;
  size_t o = 0;
  auto take = [&](size_t bytes) { const size_t at = o; o = align256(o + bytes); return at; };
  P.s_scal = take(64);  // n_valid (int), inv (float)
  P.s_pos = take((size_t)M * sizeof(int));
  P.s_cfac = take((size_t)M * sizeof(float));
  P.s_wt = take((size_t)D * P.ldwt * es);
  P.s_hct = take((size_t)D * P.ldht * es);
  P.s_p = take((size_t)P.crows * P.ldp * es);
  P.s_pt = take(P.single ? 0 : (size_t)V * P.crows * es);
  P.s_dhc = take((size_t)M * D * sizeof(float));
  P.s_dwacc = take(P.nch > 1 ? (size_t)(P.single ? D * P.ldp : V * D) * sizeof(float) : 0);
  P.s_total = o;
  o = 0;
  P.f_hc = take((size_t)M * D * es);
  P.f_rows = take((size_t)M * sizeof(int));
  P.f_tcol = take((size_t)M * sizeof(int));
  P.f_mref = take((size_t)M * sizeof(float));
  P.f_stats = take((size_t)P.ntiles * P.crows * sizeof(float2));
  P.f_tgt = take((size_t)P.crows * sizeof(float));
  P.f_loss = take((size_t)M * sizeof(float));
  P.f_part = take(P.nch > 1 ? part : 0);
  P.f_total = o;
  o = 0;
  P.b_part = take(part);
  P.b_total = o;
  return P;
}

// A thread keeps its last shape's plan: the size calls and the launches of
// every step ask for the same one.
template <typename TI, bool BOTH = true>
inline Plan make_plan(int64_t M, int64_t D, int64_t V, int64_t chunk_rows) {
  struct Kept {
    int64_t M, D, V, chunk_rows;
    Plan P;
  };
  static thread_local Kept kept{0, 0, 0, 0, {}};
  if (kept.M != M || kept.D != D || kept.V != V || kept.chunk_rows != chunk_rows)
    kept = {M, D, V, chunk_rows, plan_shape<TI, BOTH>(M, D, V, chunk_rows)};
  return kept.P;
}

// Pointers into the state.
template <typename TI>
struct StateView {
  int *n;
  float *inv;
  int *pos;
  float *cfac;  // per compacted row: inv * exp(mref - lse)
  TI *Wt, *Hct, *P, *PT;
  float *dHc, *dWacc;
  StateView(const Plan &L, char *s)
      : n(reinterpret_cast<int *>(s + L.s_scal)),
        inv(reinterpret_cast<float *>(s + L.s_scal + 16)),
        pos(reinterpret_cast<int *>(s + L.s_pos)),
        cfac(reinterpret_cast<float *>(s + L.s_cfac)),
        Wt(reinterpret_cast<TI *>(s + L.s_wt)),
        Hct(reinterpret_cast<TI *>(s + L.s_hct)),
        P(reinterpret_cast<TI *>(s + L.s_p)),
        PT(reinterpret_cast<TI *>(s + L.s_pt)),
        dHc(reinterpret_cast<float *>(s + L.s_dhc)),
        dWacc(reinterpret_cast<float *>(s + L.s_dwacc)) {}
};

// The gradient products of chunk c in one launch: dW (+)= E^T_c Hct_c^T (E^T
// in the PT buffer; Hct holding the chunk's rows already times their factor
// cfac) and dHc_c = cfac_c * (E_c Wt^T) (E in the P buffer; the factor per
// output row, split along K).  dW goes
// to `dw_out` (type dt_w, scaled by g when given) on top of `dw_in` when
// given.
// reduce_dh = false leaves a split dH's fp32 slices in `part` for the
// caller (the backward's scatter adds them).  want_w, want_h: the products that
// are formed (a gradient that nobody asked for costs nothing).
// C, CT: the tilings of the products with a K-contiguous and an N-major B.
// Wn: weight as it lies, [V, D], for the dH product in the place of its transpose (single).
template <typename TI, class C, class CT>
int launch_grads_tiled(const Plan &L, const StateView<TI> &S, int64_t c, int64_t D, int64_t V,
                 const float *dw_in, void *dw_out, int dt_w, const float *g, float *part,
                 hipStream_t s, bool final_dw, bool reduce_dh, bool want_w, bool want_h,
                 const TI *Wn) {
  const int64_t j0 = c * L.crows;
  // single: dW^T (+)= Hct_c P_c, [D, V], with P read N-major; the fp32
  // accumulator holds dW^T [D, ldp] and the final product stores dW [V, D]
  // transposed (final_dw: dw_out is the caller's gradient).
  auto jw = L.single ? make_job<CT>(S.Hct + j0, L.ldht, S.P, L.ldp, dw_in, dw_out, dt_w, g,
                                    final_dw ? D : L.ldp, D, V, L.crows)
                     : make_job<C>(S.PT, L.crows, S.Hct + j0, L.ldht, dw_in, dw_out, dt_w, g,
                                   D, V, D, L.crows);
  if (L.single) {
    jw.bt = 1;
    jw.ct = final_dw ? 1 : 0;
    jw.ldcin = L.ldp;
  }
  jw.dyn = S.n;
  jw.dyn_base = j0;
  jw.dyn_rows = 0;  // K: the chunk's rows
  auto jh = Wn ? make_job<CT>(S.P, L.ldp, Wn, D, nullptr, S.dHc + j0 * D, NF_DTYPE_F32, nullptr,
                              D, L.crows, D, V)
               : make_job<C>(S.P, L.ldp, S.Wt, L.ldwt, nullptr, S.dHc + j0 * D, NF_DTYPE_F32,
                             nullptr, D, L.crows, D, L.ldp);
  if (Wn) {
    jh.bt = 1;
    jh.a_zeros = 1;  // E's columns V .. ldp
  }
  jh.dyn = S.n;
  jh.dyn_base = j0;
  jh.dyn_rows = 1;  // M: the chunk's rows
  jh.row_scale = S.cfac + j0;
  if (L.split.S > 1) {
    jh.ksplit = L.split.S;
    jh.kslice = L.split.kslice;
    jh.part = part;
    jh.tiles *= L.split.S;
  }
  if (!want_w) jw.tiles = 0;
  if (!want_h) jh.tiles = 0;
  // the longest blocks go first (the dW job is never split)
  return L.split.kslice > L.crows ? launch_gemm_store<C, CT>(jh, jw, s, reduce_dh)
                                  : launch_gemm_store<C, CT>(jw, jh, s, reduce_dh);
}

template <typename TI>
int launch_grads(const Plan &L, const StateView<TI> &S, int64_t c, int64_t D, int64_t V,
                 const float *dw_in, void *dw_out, int dt_w, const float *g, float *part,
                 hipStream_t s, bool final_dw, bool reduce_dh = true, bool want_w = true,
                 bool want_h = true, const TI *Wn = nullptr) {
  using C = MainCfg<TI>;
  if constexpr (sizeof(TI) == 2) {
    if (L.d192)
      return launch_grads_tiled<TI, Cols192Cfg, Rows192Cfg>(L, S, c, D, V, dw_in, dw_out, dt_w, g,
                                                            part, s, final_dw, reduce_dh, want_w,
                                                            want_h, Wn);
  }
  return launch_grads_tiled<TI, C, C>(L, S, c, D, V, dw_in, dw_out, dt_w, g, part, s, final_dw,
                                      reduce_dh, want_w, want_h, Wn);
}

// Sizes whose buffers could exist: M, V, D within int32 and each operand
// under 2^40 elements, so every byte count below fits int64 / size_t.
inline bool ce_sizes_ok(int64_t M, int64_t D, int64_t V) {
  const int64_t i32 = 0x7fffffffLL, cap = (int64_t)1 << 40;
  return M > 0 && D > 0 && V > 0 && M <= i32 && V <= i32 && D <= i32 && M * D <= cap &&
         V * D <= cap && M * V <= cap;
}
inline int ce_check_shape(const char *fn, int64_t M, int64_t D, int64_t V) {
  if (M <= 0 || D <= 0 || V <= 0)
    return set_error(NF_ERR_ARG, "%s: bad shape M=%lld D=%lld V=%lld", fn, (long long)M,
                     (long long)D, (long long)V);
  if (!ce_sizes_ok(M, D, V))
    return set_error(NF_ERR_ARG, "%s: M, V or D exceeds int32, or an operand 2^40 elements",
                     fn);
  return NF_OK;
}
inline int ce_check_dtype(const char *fn, int dtype) {
  if (dtype != NF_DTYPE_BF16 && dtype != NF_DTYPE_F32)
    return set_error(NF_ERR_DTYPE, "%s: dtype %d unsupported (bf16 or f32)", fn, dtype);
  return NF_OK;
}
inline bool dtype_ok(int dtype) { return dtype == NF_DTYPE_BF16 || dtype == NF_DTYPE_F32; }
inline Plan plan_of(int64_t M, int64_t D, int64_t V, int64_t chunk_rows, int dtype) {
  return dtype == NF_DTYPE_BF16 ? make_plan<bf16>(M, D, V, chunk_rows)
                                : make_plan<float>(M, D, V, chunk_rows);
}

}  // namespace ce
}  // namespace nf
