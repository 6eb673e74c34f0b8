// Dropout from a counter: out = residual + keep * x / (1 - p), the mask computed from
// the element's index and never stored, so the backward forms it again.
//
// Elements 8 b .. 8 b + 7 share one block of Philox4x32-10 (Salmon, Moraes, Dror and
// Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011): counter (b, offset), both
// 64 bits, key the 64-bit seed; element 8 b + j takes bits 16 j .. 16 j + 15 of the 128.
// It is kept where that part is at least `threshold` = round(65536 p), so p acts in
// steps of 2^-16 and a kept element is scaled by 65536 / (65536 - threshold), which
// keeps the mean exact.  32 bits an element would cost twice the generator.
//
// What bounds it: memory (bf16 [65536, 2048]: 131 us, 6.1 TB/s, with a residual, 85 us, 6.3,
// without, where a copy of 1 GiB runs at 5.1), with the generator's ten rounds for eight
// elements (20 products at a quarter of the rate) close behind.
//
// A chunk of 8 elements is a thread's 16-byte vector (bf16, fp16) or two (fp32), at any
// alignment, fp32 arithmetic, one rounding at the store.  A dropped element gives the residual
// exactly, whatever x holds there (infinities and NaN too).
#include "nf_device.h"

namespace nf {
namespace {

constexpr int kBlock = 64;
// Stores take the non-temporal hint where a launch moves more than the Infinity Cache holds:
// bf16 [65536, 2048] with a residual (805 MB) 136.3 us plain, 130.9 hinted, without one (537
// MB) 86.6 and 84.9; fp32 [16384, 2048] without (268 MB) 50.7 and 51.5, bf16 [8192, 1024] with
// (50 MB) 9.3 and 9.5.
constexpr int64_t kNtStoreMinBytes = (int64_t)320 << 20;

// The eight 16-bit parts of block (b, offset) under `seed`.
__device__ __forceinline__ void philox8(uint64_t seed, uint64_t b, uint64_t offset,
                                        uint32_t (&word)[4]) {
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
  uint32_t c0 = (uint32_t)b, c1 = (uint32_t)(b >> 32);
  uint32_t c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t u = (uint64_t)c0 * 0xD2511F53u, v = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(v >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)v;
    c2 = (uint32_t)(u >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)u;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  word[0] = c0;
  word[1] = c1;
  word[2] = c2;
  word[3] = c3;
}

// I: x's type; O: the residual's and out's.
template <typename I, typename O, bool RES, bool NT>
__global__ __launch_bounds__(kBlock) void dropout_kernel(
    const I *__restrict__ x, const O *__restrict__ res, O *__restrict__ out, int64_t n,
    uint32_t threshold, float scale, const int64_t *__restrict__ seed_ptr, int64_t seed,
    int64_t offset) {
  const int64_t c = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (c * 8 >= n) return;
  const int64_t rem = n - c * 8;
  const int valid = rem >= 8 ? 8 : (int)rem;
  Any8<I> xv;
  Any8<O> rv;
  xv.load(x + c * 8, valid);
  if constexpr (RES) rv.load(res + c * 8, valid);
  uint32_t word[4];
  philox8((uint64_t)(seed_ptr ? *seed_ptr : seed), (uint64_t)c, (uint64_t)offset, word);
  float out8[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t part = (word[j >> 1] >> (16 * (j & 1))) & 0xffffu;
    const float y = part >= threshold ? to_f32(xv.v[j]) * scale : 0.f;
    out8[j] = RES ? y + to_f32(rv.v[j]) : y;
  }
  rv.set(out8);
  rv.template store<NT>(out + c * 8, valid);
}

template <typename I, typename O>
int launch(const void *x, const void *res, void *out, int64_t n, uint32_t threshold,
           const int64_t *seed_ptr, int64_t seed, int64_t offset, hipStream_t s) {
  const float scale = threshold < 65536u ? 65536.f / (float)(65536u - threshold) : 0.f;
  const unsigned grid = (unsigned)(((n + 7) / 8 + kBlock - 1) / kBlock);
  const I *xp = static_cast<const I *>(x);
  const O *rp = static_cast<const O *>(res);
  O *op = static_cast<O *>(out);
  const int64_t bytes = n * (int64_t)(sizeof(I) + (res ? 2 : 1) * sizeof(O));
  const bool nt = bytes > kNtStoreMinBytes;
#define NF_DROPOUT_LAUNCH(RES, NT)                                                                \
  dropout_kernel<I, O, RES, NT><<<grid, kBlock, 0, s>>>(xp, rp, op, n, threshold, scale, seed_ptr, \
                                                        seed, offset)
  if (res && nt)
    NF_DROPOUT_LAUNCH(true, true);
  else if (res)
    NF_DROPOUT_LAUNCH(true, false);
  else if (nt)
    NF_DROPOUT_LAUNCH(false, true);
  else
    NF_DROPOUT_LAUNCH(false, false);
#undef NF_DROPOUT_LAUNCH
  return check_launch("nf_dropout");
}

}  // namespace
}  // namespace nf

using namespace nf;

extern "C" int nf_dropout(const void *x, const void *residual, void *out, int64_t n,
                          int32_t threshold, const int64_t *seed_ptr, int64_t seed,
                          int64_t offset, int dt_x, int dt_out, void *stream) {
  if (n < 0) return set_error(NF_ERR_ARG, "nf_dropout: n=%lld < 0", (long long)n);
  if (threshold < 0 || threshold > 65536)
    return set_error(NF_ERR_ARG, "nf_dropout: threshold %d outside [0, 65536]", (int)threshold);
  if (offset < 0) return set_error(NF_ERR_ARG, "nf_dropout: offset < 0");
  if (!is_dtype(dt_x) || !is_dtype(dt_out) ||
      (dt_x != dt_out && dt_x != NF_DTYPE_F32 && dt_out != NF_DTYPE_F32))
    return set_error(NF_ERR_DTYPE, "nf_dropout: dtypes %d -> %d", dt_x, dt_out);
  if (n == 0) return NF_OK;
  if (!x || !out) return set_error(NF_ERR_ARG, "nf_dropout: null pointer");
  if ((n + 7) / 8 > kMaxLaunchThreads - kBlock)
    return set_error(NF_ERR_ARG, "nf_dropout: n=%lld too large (at most about 2^35)", (long long)n);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const uint32_t t = (uint32_t)threshold;
#define NF_DROPOUT(CX, CO, I, O) \
  if (dt_x == CX && dt_out == CO) \
    return launch<I, O>(x, residual, out, n, t, seed_ptr, seed, offset, s);
  NF_DROPOUT(NF_DTYPE_F32, NF_DTYPE_F32, float, float)
  NF_DROPOUT(NF_DTYPE_BF16, NF_DTYPE_BF16, bf16, bf16)
  NF_DROPOUT(NF_DTYPE_F16, NF_DTYPE_F16, f16, f16)
  NF_DROPOUT(NF_DTYPE_BF16, NF_DTYPE_F32, bf16, float)
  NF_DROPOUT(NF_DTYPE_F16, NF_DTYPE_F32, f16, float)
  NF_DROPOUT(NF_DTYPE_F32, NF_DTYPE_BF16, float, bf16)
  NF_DROPOUT(NF_DTYPE_F32, NF_DTYPE_F16, float, f16)
#undef NF_DROPOUT
  return set_error(NF_ERR_DTYPE, "nf_dropout: dtypes %d -> %d", dt_x, dt_out);
}
