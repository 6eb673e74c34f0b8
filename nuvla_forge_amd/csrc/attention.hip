// Attention: the plans, the checks of arguments and the C entries.  The kernels are in
// attention_fwd.h and attention_bwd.h, compiled for one type in each attention_{fwd,bwd}_*.hip.
#include <math.h>

#include <initializer_list>

#include "attention.h"

namespace nf {
namespace attn {

constexpr int64_t kMaxBlocks = (int64_t)1 << 23;
// div_g is exact while the rows of a tile and a group, times the group, are below 2^32
constexpr int64_t kMaxGroup = 1 << 15;

int check_sizes(const char *op, const Sizes &z) {
  if (!is_dtype(z.dtype)) return set_error(NF_ERR_DTYPE, "%s: dtype %d", op, z.dtype);
  if (z.B < 0 || z.Tq < 0 || z.Tk < 0 || z.H <= 0 || z.Hk <= 0 || z.H % z.Hk)
    return set_error(NF_ERR_ARG, "%s: B=%lld Tq=%lld Tk=%lld H=%lld Hk=%lld", op, (long long)z.B,
                     (long long)z.Tq, (long long)z.Tk, (long long)z.H, (long long)z.Hk);
  if (z.D <= 0 || z.D > 128)
    return set_error(NF_ERR_ARG, "%s: D=%lld outside [1, 128]", op, (long long)z.D);
  if (z.H / z.Hk > kMaxGroup)
    return set_error(NF_ERR_ARG, "%s: %lld query heads a key head; at most %lld", op,
                     (long long)(z.H / z.Hk), (long long)kMaxGroup);
  const int64_t most = (int64_t)1 << 30;
  if (z.B > most || z.H > most / 1024 || z.Tq > most || z.Tk > most || z.rows() > most ||
      z.B * z.Hk > most || z.B * z.Hk * ((z.rows() + 31) / 32 + 1) > kMaxBlocks ||
      z.B * z.Hk * ((z.Tk + 31) / 32 + 1) > kMaxBlocks)
    return set_error(NF_ERR_ARG, "%s: B=%lld Tq=%lld Tk=%lld H=%lld Hk=%lld too large", op,
                     (long long)z.B, (long long)z.Tq, (long long)z.Tk, (long long)z.H,
                     (long long)z.Hk);
  return NF_OK;
}

// times log2(e) it has to be an fp32 number
int check_scale(const char *op, float scale) {
  if (fabsf(scale) <= 0x1p127f) return NF_OK;
  return set_error(NF_ERR_ARG, "%s: scale %g is beyond 2^127", op, (double)scale);
}

// `group`: heads between the first and the last element that a tile of one key head reads.
int make_view(const char *op, const char *name, const void *p, int64_t sb, int64_t st, int64_t sh,
              const Sizes &z, int64_t group, View *v) {
  const int es = z.es();
  if (!p) return set_error(NF_ERR_ARG, "%s: %s is null", op, name);
  if (!aligned16(p) || sb * es % 16 || st * es % 16 || sh * es % 16 || sb < 0 || st < 0 || sh < 0)
    return set_error(NF_ERR_ARG, "%s: %s: rows of 16-byte vectors expected", op, name);
  // a tile's offsets, 128 rows and a group of heads, fit the buffer unit's 31 bits
  const int64_t most = (int64_t)1 << 30;
  if (st > most / 512 || sh > most || 130 * st * es + group * sh * es >= most)
    return set_error(NF_ERR_ARG, "%s: %s: strides too large", op, name);
  *v = View{static_cast<const char *>(p), sb * es, st * es, sh * es};
  return NF_OK;
}

// Small calls alone (a large one would read K and V four times as often and form half as many
// products again), by the three kernels' time, own rows in parts -> shared: 3 x 301 x 1003, 6 heads
// of 80 on 2, fp16 88 -> 72 us; 1024 tokens, 8 heads of 64 64 -> 44, 2048 105 -> 98; 512, 8 heads of
// 128 on 4 68 -> 50, 1500 causal, 4 heads of 128 79 -> 87.  fp32 rows of 512 bytes leave a CU one
// block: 900, 4 heads of 128 160 -> 271.
// (The two-term products of shared blocks round less, so that a sample's 16-bit results also depend,
// within those roundings, on how many others are in its call.)
bool shared_blocks(const Sizes &z, int64_t own) {
  if (own <= 32) return true;
  if (z.dp() * z.es() > 256 || z.B * z.Hk * ((own + 127) / 128) >= 256) return false;
  const double work = (double)(z.B * z.Hk) * (double)z.rows() * (double)z.Tk * z.dp();
  return work <= (z.dp() <= 64 ? 0x1p31 : 0x1p30);
}

Shape make_shape(const Sizes &z, int causal, float scale, const uint8_t *mask, int64_t mask_b) {
  Shape s;
  s.B = (int)z.B;
  s.Tq = (int)z.Tq;
  s.Tk = (int)z.Tk;
  s.H = (int)z.H;
  s.Hk = (int)z.Hk;
  s.G = (int)(z.H / z.Hk);
  s.D = (int)z.D;
  s.R = (int)z.rows();
  const int ve = 16 / z.es();
  s.nvec = (int)((z.D + ve - 1) / ve);
  s.off = (int)(z.Tk - z.Tq);
  s.causal = causal;
  s.ginv = s.G == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + s.G - 1) / s.G);
  // 0 times a barred key's -infinity would be no number: a scale that rounds every logit to 0
  s.c = fmaxf(fabsf(scale) * kLog2e, 1e-30f);
  s.scale = scale;
  s.flip = scale < 0.f ? (z.es() == 2 ? 0x80008000u : 0x80000000u) : 0u;
  s.mask = mask;
  s.mask_b = mask_b;
  return s;
}

State state_of(const Sizes &z) {
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  State t;
  t.low = up((size_t)(z.B * z.Hk * z.rows()) * 4);
  t.total = t.low + (z.es() == 2 ? up((size_t)(z.B * z.Tq * z.H * z.D) * 2) : 0);
  return t;
}

// The blocks that part_length counts as running at once: two a CU of those whose wavefronts share
// rows of up to `narrow` bytes, else one, although the 16-bit forward and dQ, and dK and dV of up to
// 64 columns, leave room for two.  Counted as two, causal calls are cut too finely (4096 tokens,
// 16 heads on 4 of 128: forward 105.5 -> 113.9 us, dQ 138.5 -> 151.5); without a causal line 264
// blocks are cut with nothing gained by it (3 x 1400, 8 heads of 128: 49.2 us uncut -> 63.6, dQ
// 62.7 -> 84.3), 288 in one sequence of 4600 133.5 against 130.8; others of 272 to 504 come out alike.
static int slots_of(int kw, const Sizes &z, int narrow) {
  return kw == 4 && z.dp() * z.es() <= narrow ? 512 : 256;
}

Plan fwd_plan(const Sizes &z, bool causal) {
  Plan p;
  const int64_t R = z.rows(), heads = z.B * z.Hk;
  const bool wide = z.dp() * z.es() > 256;
  p.kw = shared_blocks(z, R) ? 4 : 1;
  p.tiles = (int)((R + (p.kw == 4 ? 31 : 127)) / (p.kw == 4 ? 32 : 128));
  const int tk = p.kw == 4 ? 128 : wide ? 32 : 64;
  const int64_t longest = (z.Tk + tk - 1) / tk;
  p.length = part_length(heads, p.tiles, longest, causal, slots_of(p.kw, z, 256));
  p.most = parts_of((int)longest, p.length);
  p.bytes = p.most > 1 ? (size_t)p.most * (size_t)(heads * R) * (size_t)(z.dp() + 2) * 4 : 0;
  return p;
}

Plan dq_plan(const Sizes &z, bool causal) {
  const bool shared = shared_blocks(z, z.rows()), wide = z.dp() * z.es() > 256;
  const int br = shared ? 32 : 128, tk = shared ? 128 : wide ? 32 : 64;
  const int64_t heads = z.B * z.Hk, longest = (z.Tk + tk - 1) / tk;
  Plan p;
  p.kw = shared ? 4 : 1;
  p.tiles = (int)((z.rows() + br - 1) / br);
  p.length = part_length(heads, p.tiles, longest, causal, slots_of(p.kw, z, 256));
  p.most = parts_of((int)longest, p.length);
  p.bytes = p.most > 1 ? (size_t)p.most * (size_t)(heads * z.rows()) * (size_t)z.dp() * 4 : 0;
  return p;
}

Plan dkv_plan(const Sizes &z, bool causal) {
  const bool shared = shared_blocks(z, z.Tk);
  const int bk = shared ? 32 : 128, tr = shared ? 128 : z.dp() * z.es() > 256 ? 32 : 64;
  const int64_t heads = z.B * z.Hk, longest = (z.rows() + tr - 1) / tr;
  Plan p;
  p.kw = shared ? 4 : 1;
  p.tiles = (int)((z.Tk + bk - 1) / bk);
  p.length = part_length(heads, p.tiles, longest, causal, slots_of(p.kw, z, 128));
  p.most = parts_of((int)longest, p.length);
  p.bytes = p.most > 1 ? (size_t)p.most * (size_t)(heads * z.Tk) * (size_t)z.dp() * 8 : 0;
  return p;
}

__global__ __launch_bounds__(256) void attn_zero_kernel(uint16_t *p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    p[i] = 0;
}

// Gradients of keys that no row attends.  The workspace and the rows, which say nothing then, are
// not looked at; the memory is: a pointer that the runtime does not know is refused, and on a host
// without a device there is none to write.
int zero_gradients(const char *op, std::initializer_list<void *> grads, int64_t bytes,
                   hipStream_t st) {
  int devices = 0;
  if (hipGetDeviceCount(&devices) != hipSuccess || devices == 0) {
    (void)hipGetLastError();
    return NF_OK;
  }
  for (void *p : grads) {
    if (!p) continue;
    hipPointerAttribute_t at = {};
    if (hipPointerGetAttributes(&at, p) != hipSuccess || at.type == hipMemoryTypeUnregistered) {
      (void)hipGetLastError();
      return set_error(NF_ERR_ARG, "%s: a gradient is not in device memory", op);
    }
  }
  const int64_t n = bytes / 2, blocks = (n + 255) / 256;
  for (void *p : grads)
    if (p)
      attn_zero_kernel<<<(unsigned)(blocks < 1024 ? blocks : 1024), 256, 0, st>>>(
          static_cast<uint16_t *>(p), n);
  return check_launch(op);
}

size_t delta_bytes(const Sizes &z) {
  return ((size_t)(z.B * z.Hk * z.rows()) * 4 + 255) / 256 * 256;
}
size_t bwd_bytes(const Sizes &z, bool causal) {
  const size_t a = dq_plan(z, causal).bytes, b = dkv_plan(z, causal).bytes;
  return delta_bytes(z) + (a > b ? a : b);  // dQ's parts are summed before dK's are formed
}

}  // namespace attn
}  // namespace nf

using namespace nf;
using namespace nf::attn;

extern "C" size_t nf_attention_state_bytes(int64_t B, int64_t Tq, int64_t Tk, int64_t H, int64_t Hk,
                                           int64_t D, int dtype) {
  const Sizes z{B, Tq, Tk, H, Hk, D, dtype};
  return check_sizes("nf_attention_state_bytes", z) ? 0 : state_of(z).total;
}

extern "C" size_t nf_attention_fwd_workspace(int64_t B, int64_t Tq, int64_t Tk, int64_t H,
                                             int64_t Hk, int64_t D, int causal, int dtype) {
  const Sizes z{B, Tq, Tk, H, Hk, D, dtype};
  if (check_sizes("nf_attention_fwd_workspace", z) || B * Tq * Tk == 0) return 0;
  return fwd_plan(z, causal).bytes;
}

extern "C" int nf_attention_fwd(const void *q, int64_t q_b, int64_t q_t, int64_t q_h, const void *k,
                                int64_t k_b, int64_t k_t, int64_t k_h, const void *v, int64_t v_b,
                                int64_t v_t, int64_t v_h, const uint8_t *key_mask, int64_t mask_b,
                                int64_t B, int64_t Tq, int64_t Tk, int64_t H, int64_t Hk, int64_t D,
                                int causal, float scale, int dtype, void *out, void *state,
                                size_t state_bytes, void *workspace, size_t workspace_bytes,
                                void *stream) {
  const char *op = "nf_attention_fwd";
  const Sizes z{B, Tq, Tk, H, Hk, D, dtype};
  if (const int rc = check_sizes(op, z)) return rc;
  if (const int rc = check_scale(op, scale)) return rc;
  if (B == 0 || Tq == 0) return NF_OK;
  if (Tk == 0) return set_error(NF_ERR_ARG, "%s: Tk=0", op);
  if (key_mask && mask_b < 0) return set_error(NF_ERR_ARG, "%s: mask_b < 0", op);
  const State parts = state_of(z);
  if ((state && state_bytes < parts.total) || workspace_bytes < fwd_plan(z, causal).bytes)
    return set_error(NF_ERR_WORKSPACE, "%s: state %zu of %zu bytes, workspace %zu of %zu", op,
                     state_bytes, parts.total, workspace_bytes, fwd_plan(z, causal).bytes);
  if (!out || !aligned16(state) || (fwd_plan(z, causal).bytes && (!workspace || !aligned16(workspace))))
    return set_error(NF_ERR_ARG, "%s: null or unaligned pointer", op);
  FwdArgs a = {};
  if (const int rc = make_view(op, "q", q, q_b, q_t, q_h, z, H / Hk, &a.q)) return rc;
  if (const int rc = make_view(op, "k", k, k_b, k_t, k_h, z, 0, &a.k)) return rc;
  if (const int rc = make_view(op, "v", v, v_b, v_t, v_h, z, 0, &a.v)) return rc;
  char *st = static_cast<char *>(state);
  a.s = make_shape(z, causal, scale, key_mask, mask_b);
  a.out = static_cast<char *>(out);
  a.low = st && z.es() == 2 ? st + parts.low : nullptr;
  a.lse = reinterpret_cast<float *>(st);
  a.part = static_cast<float *>(workspace);
  hipStream_t hs = static_cast<hipStream_t>(stream);
  if (dtype == NF_DTYPE_BF16) return launch_fwd<bf16>(a, z, hs);
  if (dtype == NF_DTYPE_F16) return launch_fwd<f16>(a, z, hs);
  return launch_fwd<float>(a, z, hs);
}

extern "C" size_t nf_attention_bwd_workspace(int64_t B, int64_t Tq, int64_t Tk, int64_t H,
                                             int64_t Hk, int64_t D, int causal, int dtype) {
  const Sizes z{B, Tq, Tk, H, Hk, D, dtype};
  return check_sizes("nf_attention_bwd_workspace", z) ? 0 : bwd_bytes(z, causal);
}

extern "C" int nf_attention_bwd(const void *q, int64_t q_b, int64_t q_t, int64_t q_h, const void *k,
                                int64_t k_b, int64_t k_t, int64_t k_h, const void *v, int64_t v_b,
                                int64_t v_t, int64_t v_h, const uint8_t *key_mask, int64_t mask_b,
                                const void *out, const void *dout, int64_t g_b, int64_t g_t,
                                int64_t g_h, int64_t B, int64_t Tq, int64_t Tk, int64_t H,
                                int64_t Hk, int64_t D, int causal, float scale, int dtype,
                                const void *state, size_t state_bytes, void *dq, void *dk, void *dv,
                                void *workspace, size_t workspace_bytes, void *stream) {
  const char *op = "nf_attention_bwd";
  const Sizes z{B, Tq, Tk, H, Hk, D, dtype};
  if (const int rc = check_sizes(op, z)) return rc;
  if (const int rc = check_scale(op, scale)) return rc;
  if (B == 0 || (!dq && !dk && !dv)) return NF_OK;
  if (Tq == 0)  // dq is empty, dk and dv are empty sums
    return Tk == 0 || (!dk && !dv)
               ? NF_OK
               : zero_gradients(op, {dk, dv}, B * Tk * Hk * D * z.es(), static_cast<hipStream_t>(stream));
  if (Tk == 0) return set_error(NF_ERR_ARG, "%s: Tk=0", op);
  if (key_mask && mask_b < 0) return set_error(NF_ERR_ARG, "%s: mask_b < 0", op);
  const State parts = state_of(z);
  if (state_bytes < parts.total || workspace_bytes < bwd_bytes(z, causal))
    return set_error(NF_ERR_WORKSPACE, "%s: state %zu of %zu bytes, workspace %zu of %zu", op,
                     state_bytes, parts.total, workspace_bytes, bwd_bytes(z, causal));
  if (!out || !state || !aligned16(state) || !workspace || !aligned16(workspace))
    return set_error(NF_ERR_ARG, "%s: null or unaligned pointer", op);
  BwdArgs a = {};
  if (const int rc = make_view(op, "q", q, q_b, q_t, q_h, z, H / Hk, &a.q)) return rc;
  if (const int rc = make_view(op, "k", k, k_b, k_t, k_h, z, 0, &a.k)) return rc;
  if (const int rc = make_view(op, "v", v, v_b, v_t, v_h, z, 0, &a.v)) return rc;
  if (const int rc = make_view(op, "dout", dout, g_b, g_t, g_h, z, H / Hk, &a.dout)) return rc;
  const char *st = static_cast<const char *>(state);
  a.s = make_shape(z, causal, scale, key_mask, mask_b);
  a.out = static_cast<const char *>(out);
  a.low = z.es() == 2 ? st + parts.low : nullptr;
  a.lse = reinterpret_cast<const float *>(st);
  a.ndelta = static_cast<float *>(workspace);
  a.part = a.ndelta + delta_bytes(z) / 4;
  a.dq = static_cast<char *>(dq);
  a.dk = static_cast<char *>(dk);
  a.dv = static_cast<char *>(dv);
  hipStream_t hs = static_cast<hipStream_t>(stream);
  if (dtype == NF_DTYPE_BF16) return launch_bwd<bf16>(a, z, hs);
  if (dtype == NF_DTYPE_F16) return launch_bwd<f16>(a, z, hs);
  return launch_bwd<float>(a, z, hs);
}
