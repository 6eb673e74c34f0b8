// Embedding lookup, out[m] = scale * table[ids[m]], and its gradient,
// dtable[v] = scale * sum over the m with ids[m] = v of dout[m], by sorted tokens: no
// atomics on values, every sum in a fixed order, every row of dtable written once.
//
// An id outside [0, V) gives a row of zeros and no gradient; the padding id is looked
// up like any other and gives no gradient.
//
// The gradient of up to 1024 tokens is one launch (emb_few); of more, three:
//   emb_sort:   block b of nb (a power of two) owns the ids that are b modulo nb, so that
//               frequent ids next to each other fall to different blocks; the order of
//               the sort is by block, then by id.  It reads all M ids, counting its own
//               (per wavefront and id, in LDS) and those of the blocks before it, which
//               gives every id's first position without a word from another block; then
//               it places its tokens, in order.
//   emb_reduce: the sorted positions in spans, one wavefront a span (and 64 vectors of
//               columns): a run of one id that lies inside the span is summed and written;
//               a piece of a run that crosses a span's border goes to the workspace as an
//               fp32 partial row.  Among these blocks, others write zeros to the rows of
//               ids that no token holds: the sums wait for memory, the zeros only write.
//   emb_join:   the partial rows of each run that crosses borders, added in order.
// So the work of a token that holds half the batch is spread like any other.
#include "nf_device.h"

namespace nf {
namespace {

// Rows are taken in pieces of 8 columns, with 16-byte accesses whatever their alignment (an
// odd D starts rows on any element, and the device takes global accesses on any byte: D 1645,
// bf16, forward and backward, element by element took 104 us where this takes 54).  A last piece that would
// pass the row's end starts at D - 8 and repeats columns of the one before: the same values
// to the same places.  VEC: D >= 8; else a row is one piece of D elements.
template <bool VEC>
__device__ __forceinline__ int64_t piece(int64_t c, int64_t D) {
  return VEC && c > D - 8 ? D - 8 : c;
}

template <typename T>
struct Raw : Any8<T> {
  template <bool VEC>
  __device__ __forceinline__ void load(const T *p, int64_t D) {
    if constexpr (VEC)
      Any8<T>::load(p);
    else
      Any8<T>::load(p, (int)D);
  }
};
template <typename T, bool VEC, bool NT = false>
__device__ __forceinline__ void store8u(T *p, int64_t D, const float (&f)[8]) {
  Any8<T> r;
  r.set(f);
  if constexpr (VEC)
    r.template store<NT>(p);
  else
    r.store(p, (int)D);
}

// ---------------------------------------------------------------------------
// forward: a group of 2^glog lanes takes a row, 8 columns a lane and step.  What bounds it is
// memory: bf16, 65536 tokens by Zipf's law, V 128256, D 2048, back to back 61 us for the 268 MB
// written and as much read (a third of it from HBM), 78 without the non-temporal hint on the
// stores; 76-83 between training steps, which leave nothing of the table in the caches; 8192
// tokens, D 1024 6.0 us, 7.0 without.
// ---------------------------------------------------------------------------
constexpr int kFwdThreads = 256;

template <typename W, typename O, bool VEC>
__global__ __launch_bounds__(kFwdThreads) void emb_fwd_kernel(
    const int64_t *__restrict__ ids, const W *__restrict__ table, int64_t ldt, float scale,
    int64_t M, int64_t D, int64_t V, O *__restrict__ out, int glog) {
  const int g = threadIdx.x & ((1 << glog) - 1);
  const int64_t m = (int64_t)blockIdx.x * (kFwdThreads >> glog) + (threadIdx.x >> glog);
  if (m >= M) return;
  const int64_t id = ids[m];
  const bool live = id >= 0 && id < V;
  const W *src = table + (live ? id : 0) * ldt;
  O *dst = out + m * D;
  const int64_t step = (int64_t)8 << glog;
  constexpr int kUnroll = 4;
  for (int64_t c0 = (int64_t)g * 8; c0 < D; c0 += kUnroll * step) {
    Raw<W> r[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (c0 + u * step < D) r[u].template load<VEC>(src + piece<VEC>(c0 + u * step, D), D);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (c0 + u * step < D) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = live ? to_f32(r[u].v[i]) * scale : 0.f;
        store8u<O, VEC, true>(dst + piece<VEC>(c0 + u * step, D), D, v);
      }
  }
}

// ---------------------------------------------------------------------------
// gradient
// ---------------------------------------------------------------------------
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kMaxIds = 512;    // ids per block
constexpr int kListed = 512;    // tokens a wavefront notes in LDS
constexpr int kZeroIds = 64;    // ids a wavefront looks at for rows to clear
constexpr int kJoinThreads = 512, kJoinWaves = kJoinThreads / 64;

// The ids' places: block id % nb, and in it id / nb; R ids a block.
struct Order {
  int log_nb, R;
  __device__ __forceinline__ int64_t place(int64_t id) const {
    return (id & (((int64_t)1 << log_nb) - 1)) * R + (id >> log_nb);
  }
  __host__ __device__ int64_t places() const { return (int64_t)R << log_nb; }
};
struct Token {
  int m, id;
};

__device__ __forceinline__ int wave_inclusive_sum(int v) {
  const int l = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(v, d);
    if (l >= d) v += o;
  }
  return v;
}

// first[place]: the sorted position of that id's first token (first[places]: the number of
// tokens that count); sorted: the token and its id at each position.
//
// A block's time goes into reading the ids (M 65536: 0.5 MB a block from the L2s) and
// into placing its tokens, where most of them belong to a few blocks: 24 us for 65536 tokens
// by Zipf's law, V 128256.
__global__ __launch_bounds__(kSortThreads) void emb_sort_kernel(
    const int64_t *__restrict__ ids, int64_t M, int64_t V, int64_t pad, Order ord,
    int *__restrict__ first, Token *__restrict__ sorted) {
  __shared__ int hist[kSortWaves][kMaxIds];
  __shared__ int list_m[kSortWaves][kListed];
  __shared__ int list_key[kSortWaves][kListed];
  __shared__ int below_w[kSortWaves];
  __shared__ int scan_w[kSortWaves];
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int blk = blockIdx.x, mask = (1 << ord.log_nb) - 1, R = ord.R;
  const uint64_t lower = (1ull << l) - 1ull;
  for (int k = l; k < R; k += 64) hist[w][k] = 0;  // the wavefront's own row
  const int64_t seg = ((M + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
  const int64_t m0 = (int64_t)w * seg, m1 = m0 + seg < M ? m0 + seg : M;
  __syncthreads();
  // 64 tokens from m on: the key of those that are the block's, else -1; and how many
  // belong to blocks before it
  int below = 0, noted = 0;
  constexpr int kBatch = 8;
  for (int64_t b = m0; b < m1; b += 64 * kBatch) {
    int64_t id[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int64_t m = b + u * 64 + l;
      id[u] = m < m1 ? ids[m] : -1;
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const bool counts = id[u] >= 0 && id[u] < V && id[u] != pad;
      const int owner = (int)id[u] & mask;
      below += counts && owner < blk ? 1 : 0;
      const bool in = counts && owner == blk;
      const uint64_t ins = __ballot(in);
      if (!ins) continue;
      if (in) {
        const int key = (int)(id[u] >> ord.log_nb), at = noted + __popcll(ins & lower);
        atomicAdd(&hist[w][key], 1);
        if (at < kListed) {
          list_m[w][at] = (int)(b + u * 64 + l);
          list_key[w][at] = key;
        }
      }
      noted += __popcll(ins);
    }
  }
  below = wave_inclusive_sum(below);
  if (l == 63) below_w[w] = below;
  __syncthreads();
  // per id: the counts of the wavefronts before, and the total
  int mine = 0;
  if ((int)threadIdx.x < R) {
#pragma unroll
    for (int k = 0; k < kSortWaves; ++k) {
      const int h = hist[k][threadIdx.x];
      hist[k][threadIdx.x] = mine;
      mine += h;
    }
  }
  const int incl = wave_inclusive_sum(mine);
  if (l == 63) scan_w[w] = incl;
  __syncthreads();
  int start = incl - mine;
  for (int k = 0; k < kSortWaves; ++k) {
    start += below_w[k];
    start += k < w ? scan_w[k] : 0;
  }
  if ((int)threadIdx.x < R) {
#pragma unroll
    for (int k = 0; k < kSortWaves; ++k) hist[k][threadIdx.x] += start;
    first[(int64_t)blk * R + threadIdx.x] = start;
    if (blk == mask && (int)threadIdx.x == R - 1) first[ord.places()] = start + mine;
  }
  __syncthreads();
  // the block's tokens in order: a wavefront ranks 64 at a time, the lanes that share an id
  // found by one ballot a bit (a loop over the different ids took 430 of the 448 us that
  // 65536 tokens by Zipf's law cost here, V 128256)
  int bits = 0;
  while ((1 << bits) < R) ++bits;
  volatile int *next = hist[w];
  auto place = [&](bool in, int m, int key) {
    uint64_t same = __ballot(in);
    for (int k = 0; k < bits; ++k) {
      const uint64_t set = __ballot((key >> k) & 1);
      same &= (key >> k) & 1 ? set : ~set;
    }
    if (in) {
      const int at = next[key];
      sorted[at + __popcll(same & lower)] = Token{m, (key << ord.log_nb) | blk};
      if ((same & lower) == 0) next[key] = at + __popcll(same);
    }
  };
  if (noted <= kListed) {
    for (int q = 0; q < noted; q += 64) {
      const bool in = q + l < noted;
      place(in, in ? list_m[w][q + l] : 0, in ? list_key[w][q + l] : 0);
    }
    return;
  }
  for (int64_t b = m0; b < m1; b += 64 * kBatch) {  // more than were noted: once more over the ids
    int64_t id[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int64_t m = b + u * 64 + l;
      id[u] = m < m1 ? ids[m] : -1;
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const bool in =
          id[u] >= 0 && id[u] < V && id[u] != pad && ((int)id[u] & mask) == blk;
      if (__ballot(in)) place(in, (int)(b + u * 64 + l), in ? (int)(id[u] >> ord.log_nb) : 0);
    }
  }
}

// O: dout's type, W: dtable's.  Blocks [0, nsum) of the interleaved order sum, a wavefront a
// (span, column part), parts of a span next to each other so that a row of dout is read
// whole at one time; the other blocks clear.  part[2 s] is the head of span s (the end, or
// all, of a run begun before it), part[2 s + 1] its tail (the begin of a run that goes on).
// What bounds it is memory: bf16, 65536 tokens by Zipf's law, V 128256, D 2048 164 us for the
// 268 MB read and 525 MB written, 4.8 TB/s.
template <typename O, typename W, bool VEC>
__global__ __launch_bounds__(256) void emb_reduce_kernel(
    const O *__restrict__ dout, int64_t ldo, const int *__restrict__ first,
    const Token *__restrict__ sorted, Order ord, int64_t V, int64_t D, float scale, int span,
    int cols, int64_t nclear, W *__restrict__ dtable, float *__restrict__ part) {
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  // clearing blocks spread evenly among the others
  const int64_t b = blockIdx.x, blocks = gridDim.x;
  const int64_t before_b = b * nclear / blocks;
  if ((b + 1) * nclear / blocks != before_b) {
    const int64_t v0 = (before_b * 4 + w) * kZeroIds;
    const int64_t v = v0 + l;
    const int64_t at = ord.place(v < V ? v : 0);
    uint64_t empty = __ballot(v < V && first[at + 1] == first[at]);
    const float zero[8] = {};
    for (; empty; empty &= empty - 1) {
      W *row = dtable + (v0 + __ffsll((unsigned long long)empty) - 1) * D;
      for (int64_t c = (int64_t)l * 8; c < D; c += 512)
        store8u<W, VEC>(row + piece<VEC>(c, D), D, zero);
    }
    return;
  }
  const int n = first[ord.places()];
  const int64_t u = (b - before_b) * 4 + w, s = u / cols;
  const int64_t t0 = s * span;
  if (t0 >= n) return;
  const int cnt = n - t0 < span ? (int)(n - t0) : span;
  const int64_t c8 = ((u - s * cols) * 64 + l) * 8, c = piece<VEC>(c8, D);
  const bool cin = c8 < D;
  const Token own = l < cnt ? sorted[t0 + l] : Token{0, -1};
  const int tok = own.m, id = own.id;
  const int before = t0 > 0 ? sorted[t0 - 1].id : -1;
  const int after = t0 + cnt < n ? sorted[t0 + cnt].id : -1;
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  bool begun_before = before == __builtin_amdgcn_readlane(id, 0);
  constexpr int kBatch = 8;
  Raw<O> cur[kBatch], nxt[kBatch];
  auto fetch = [&](int j0, Raw<O> (&r)[kBatch]) {
#pragma unroll
    for (int q = 0; q < kBatch; ++q)
      if (j0 + q < cnt && cin)
        r[q].template load<VEC>(dout + (int64_t)__builtin_amdgcn_readlane(tok, j0 + q) * ldo + c,
                                D);
  };
  fetch(0, cur);
  for (int j0 = 0; j0 < cnt; j0 += kBatch) {
    fetch(j0 + kBatch, nxt);  // under way while this batch is added
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const int j = j0 + q;
      if (j >= cnt) break;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += to_f32(cur[q].v[i]);
      const int here = __builtin_amdgcn_readlane(id, j);
      const bool last = j + 1 == cnt;
      const int then = last ? after : __builtin_amdgcn_readlane(id, j + 1 < 64 ? j + 1 : 63);
      if (last || then != here) {
        const bool goes_on = then == here;
        if (cin) {
          if (begun_before || goes_on) {
            store8u<float, VEC>(part + (2 * s + (begun_before ? 0 : 1)) * D + c, D, acc);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] *= scale;
            store8u<W, VEC>(dtable + (int64_t)here * D + c, D, acc);
          }
        }
        begun_before = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = 0.f;
      }
    }
#pragma unroll
    for (int q = 0; q < kBatch; ++q) cur[q] = nxt[q];
  }
}

// Block (s, y): the run that begins in span s and goes on past it, if there is one: its
// tail there and the heads of the spans after it.  Wavefront k adds the pieces k, k + 8,
// k + 16, ... in that order, the first wavefront the 8 sums.  Its time is the latency of the
// longest run (24 us where one token holds a twelfth of 65536), which the 8 wavefronts share.
template <typename W, bool VEC>
__global__ __launch_bounds__(kJoinThreads) void emb_join_kernel(
    const int *__restrict__ first, const Token *__restrict__ sorted, Order ord, int64_t D,
    float scale, int span, const float *__restrict__ part, W *__restrict__ dtable) {
  __shared__ float sums[kJoinWaves][512];
  const int n = first[ord.places()];
  const int64_t s = blockIdx.x, end = (s + 1) * span;  // a border between two spans
  if (end >= n) return;
  const int id = sorted[end - 1].id;
  if (sorted[end].id != id) return;  // no run crosses
  const int64_t at = ord.place(id);
  if (first[at] < s * span) return;  // it began before
  const int64_t pieces = (first[at + 1] - 1) / span - s + 1;
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t c8 = ((int64_t)blockIdx.y * 64 + l) * 8, c = piece<VEC>(c8, D);
  const bool cin = c8 < D;
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  if (cin) {
    constexpr int kBatch = 8;
    for (int64_t p0 = w; p0 < pieces; p0 += kJoinWaves * kBatch) {
      Raw<float> v[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int64_t p = p0 + u * kJoinWaves;
        if (p < pieces)
          v[u].template load<VEC>(part + (2 * (s + p) + (p == 0 ? 1 : 0)) * D + c, D);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (p0 + u * kJoinWaves < pieces)
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[i] += v[u].v[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[w][l * 8 + i] = acc[i];
  __syncthreads();
  if (w == 0 && cin) {
    const int waves = pieces < kJoinWaves ? (int)pieces : kJoinWaves;
    for (int k = 1; k < waves; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += sums[k][l * 8 + i];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] *= scale;
    store8u<W, VEC>(dtable + (int64_t)id * D + c, D, acc);
  }
}

// Few tokens (at most kFewTokens): the whole gradient in one launch, without a workspace.
// Block b owns the ids that are b modulo the grid, as in emb_sort, a thread looks at one
// token, and the block sorts its own in LDS.  A wavefront takes an id: zeros to its row where
// it has no token, else the sum; on an id of more than kLongRun tokens all wavefronts sum a
// part each, and the parts are added in order.  V 32000, bf16, 1024 tokens, in a graph,
// against the three launches: D 384 8.8 us against 16.3 (tokens by Zipf's law 10.3 against
// 16.7, all the same 19.3 against 19.4), D 2048 23.8 against 27.7 (27.5 against 27.9; all the
// same, where one block reads every row, 67 against 33).
constexpr int kFewTokens = 1024, kLongRun = 32;
constexpr int kFewThreads = 1024, kFewWaves = kFewThreads / 64;

template <typename O, typename W, bool VEC>
__global__ __launch_bounds__(kFewThreads) void emb_few_kernel(
    const O *__restrict__ dout, const int64_t *__restrict__ ids, int M, int64_t V, int64_t D,
    int64_t pad, float scale, Order ord, W *__restrict__ dtable) {
  static_assert(kFewTokens == kFewThreads && kMaxIds <= kFewThreads, "a token, an id a thread");
  __shared__ int hist[kFewWaves][kMaxIds];
  __shared__ int start[kMaxIds + 1], tok[kFewTokens];  // an id's first place; the tokens by id
  __shared__ int scan_w[kFewWaves];
  __shared__ int long_n, long_id[kFewTokens / kLongRun];
  __shared__ float sums[kFewWaves][512];
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, R = ord.R;
  const int blk = blockIdx.x, mask = (1 << ord.log_nb) - 1;
  const uint64_t lower = (1ull << l) - 1ull;
  for (int k = l; k < R; k += 64) hist[w][k] = 0;  // the wavefront's own row
  if (threadIdx.x == 0) long_n = 0;
  const int64_t id = (int)threadIdx.x < M ? ids[threadIdx.x] : -1;
  const bool in = id >= 0 && id < V && id != pad && ((int)id & mask) == blk;
  const int key = in ? (int)(id >> ord.log_nb) : 0;
  uint64_t same = __ballot(in);  // the lanes with this lane's id
  if (same)
    for (int k = 0; (1 << k) < R; ++k) {
      const uint64_t set = __ballot((key >> k) & 1);
      same &= (key >> k) & 1 ? set : ~set;
    }
  if (in && (same & lower) == 0) hist[w][key] = __popcll(same);
  __syncthreads();
  int mine = 0;
  if ((int)threadIdx.x < R) {
#pragma unroll
    for (int k = 0; k < kFewWaves; ++k) {
      const int h = hist[k][threadIdx.x];
      hist[k][threadIdx.x] = mine;
      mine += h;
    }
    if (mine > kLongRun) long_id[atomicAdd(&long_n, 1)] = threadIdx.x;  // in any order
  }
  const int incl = wave_inclusive_sum(mine);
  if (l == 63) scan_w[w] = incl;
  __syncthreads();
  int at = incl - mine;
  for (int k = 0; k < w; ++k) at += scan_w[k];
  if ((int)threadIdx.x < R) start[threadIdx.x] = at;
  if ((int)threadIdx.x == R - 1) start[R] = at + mine;
  __syncthreads();
  if (in) tok[start[key] + hist[w][key] + __popcll(same & lower)] = threadIdx.x;
  __syncthreads();
  // tokens [a, b) of the sorted order at the lane's columns from c on
  auto sum = [&](int a, int b, int64_t c, float (&acc)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    constexpr int kBatch = 8;
    for (int j0 = a; j0 < b; j0 += kBatch) {
      Raw<O> r[kBatch];
#pragma unroll
      for (int q = 0; q < kBatch; ++q)
        if (j0 + q < b) r[q].template load<VEC>(dout + (int64_t)tok[j0 + q] * D + c, D);
#pragma unroll
      for (int q = 0; q < kBatch; ++q)
        if (j0 + q < b)
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[i] += to_f32(r[q].v[i]);
    }
  };
  auto put = [&](int k, int64_t c, float (&acc)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] *= scale;
    store8u<W, VEC>(dtable + (((int64_t)k << ord.log_nb) | blk) * D + c, D, acc);
  };
  for (int k = w; k < R; k += kFewWaves) {
    const int a = start[k], b = start[k + 1];
    if ((((int64_t)k << ord.log_nb) | blk) >= V || b - a > kLongRun) continue;
    for (int64_t c8 = (int64_t)l * 8; c8 < D; c8 += 512) {
      const int64_t c = piece<VEC>(c8, D);
      float acc[8];
      sum(a, b, c, acc);  // zeros where a == b
      put(k, c, acc);
    }
  }
  for (int q = 0; q < long_n; ++q) {
    const int k = long_id[q], a = start[k], b = start[k + 1];
    const int per = (b - a + kFewWaves - 1) / kFewWaves;
    const int pa = a + w * per < b ? a + w * per : b, pb = pa + per < b ? pa + per : b;
    for (int64_t c0 = 0; c0 < D; c0 += 512) {
      const int64_t c8 = c0 + (int64_t)l * 8, c = piece<VEC>(c8, D);
      float acc[8];
      if (c8 < D) {
        sum(pa, pb, c, acc);
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[w][l * 8 + i] = acc[i];
      }
      __syncthreads();
      if (w == 0 && c8 < D) {
        for (int p = 1; p < kFewWaves; ++p)
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[i] += sums[p][l * 8 + i];
        put(k, c, acc);
      }
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
template <typename W, typename O>
int run_fwd(const int64_t *ids, const W *table, int64_t ldt, float scale, int64_t M, int64_t D,
            int64_t V, O *out, hipStream_t s) {
  const int64_t pieces = (D + 7) / 8;
  int glog = 3;
  while (glog < 6 && ((int64_t)1 << glog) < pieces) ++glog;
  const int64_t rows = kFwdThreads >> glog;
  const int64_t blocks = (M + rows - 1) / rows;
  if (blocks * kFwdThreads > kMaxLaunchThreads)
    return set_error(NF_ERR_ARG, "nf_embedding_fwd: M=%lld too large (2^26 at D > 256, to 2^29 at "
                     "D <= 64)", (long long)M);
  const unsigned grid = (unsigned)blocks;
  if (D >= 8)
    emb_fwd_kernel<W, O, true><<<grid, kFwdThreads, 0, s>>>(ids, table, ldt, scale, M, D, V, out,
                                                            glog);
  else
    emb_fwd_kernel<W, O, false><<<grid, kFwdThreads, 0, s>>>(ids, table, ldt, scale, M, D, V, out,
                                                             glog);
  return check_launch("nf_embedding_fwd");
}

struct BwdPlan {
  Order ord;  // 2^log_nb blocks of emb_sort
  int span;   // sorted positions per wavefront of emb_reduce
  int64_t spans;
  size_t first, sorted, part, total;
};
BwdPlan bwd_plan(int64_t M, int64_t D, int64_t V) {
  auto align = [](size_t x) { return (x + 255) & ~(size_t)255; };
  BwdPlan p;
  int log_nb = 8;  // a block a CU, more where an id's counter would not fit the LDS
  while (((V - 1) >> log_nb) + 1 > kMaxIds) ++log_nb;
  p.ord = Order{log_nb, (int)(((V - 1) >> log_nb) + 1)};
  // spans of 32 positions where that leaves 8192 wavefronts (32 a CU) and more, else of 16
  // or 8: fewer positions end sooner, but leave more partial rows
  const int64_t cols = (D + 511) / 512;
  p.span = M * cols >= 32 * 8192 ? 32 : M * cols >= 16 * 8192 ? 16 : 8;
  p.spans = (M + p.span - 1) / p.span;
  size_t o = 0;
  p.first = o;
  o = align(o + (size_t)(p.ord.places() + 1) * sizeof(int));
  p.sorted = o;
  o = align(o + (size_t)M * sizeof(Token));
  p.part = o;
  o = align(o + (size_t)p.spans * 2 * (size_t)D * sizeof(float));
  p.total = o;
  return p;
}

template <typename O, typename W, bool VEC>
int launch_bwd(const O *dout, const int64_t *ids, int64_t pad, float scale, int64_t M, int64_t D,
               int64_t V, W *dtable, char *ws, hipStream_t s) {
  const BwdPlan p = bwd_plan(M, D, V);
  int *first = reinterpret_cast<int *>(ws + p.first);
  Token *sorted = reinterpret_cast<Token *>(ws + p.sorted);
  float *part = reinterpret_cast<float *>(ws + p.part);
  if (M <= kFewTokens) {
    emb_few_kernel<O, W, VEC><<<1u << p.ord.log_nb, kFewThreads, 0, s>>>(
        dout, ids, (int)M, V, D, pad, scale, p.ord, dtable);
    return check_launch("emb_few");
  }
  const unsigned cols = (unsigned)((D + 511) / 512);
  const int64_t nsum = (p.spans * cols + 3) / 4, nclear = (V + 4 * kZeroIds - 1) / (4 * kZeroIds);
  emb_sort_kernel<<<1u << p.ord.log_nb, kSortThreads, 0, s>>>(ids, M, V, pad, p.ord, first,
                                                              sorted);
  if (int e = check_launch("emb_sort")) return e;
  emb_reduce_kernel<O, W, VEC><<<(unsigned)(nsum + nclear), 256, 0, s>>>(
      dout, D, first, sorted, p.ord, V, D, scale, p.span, (int)cols, nclear, dtable, part);
  if (int e = check_launch("emb_reduce")) return e;
  emb_join_kernel<W, VEC><<<dim3((unsigned)(p.spans - 1), cols), kJoinThreads, 0, s>>>(
      first, sorted, p.ord, D, scale, p.span, part, dtable);
  return check_launch("emb_join");
}

template <typename O, typename W>
int run_bwd(const O *dout, const int64_t *ids, int64_t pad, float scale, int64_t M, int64_t D,
            int64_t V, W *dtable, char *ws, hipStream_t s) {
  return D >= 8 ? launch_bwd<O, W, true>(dout, ids, pad, scale, M, D, V, dtable, ws, s)
                : launch_bwd<O, W, false>(dout, ids, pad, scale, M, D, V, dtable, ws, s);
}

// The table's type and out's: equal, or an fp32 table with rows in 16 bits.
bool types_ok(int dt_table, int dt_out) {
  return is_dtype(dt_table) && is_dtype(dt_out) &&
         (dt_table == dt_out || dt_table == NF_DTYPE_F32);
}
bool sizes_ok(int64_t M, int64_t D, int64_t V) {
  // D: at most 65535 column blocks of 512 elements in a grid
  const int64_t i32 = 0x7fffffffLL, cap = (int64_t)1 << 40;
  return M >= 0 && D > 0 && V > 0 && M < i32 && D <= 65535 * 512 && V < i32 && V * D <= cap &&
         M * D <= cap;
}
// The gradient's: what its launches take, V blocks of the sort, the spans and cleared rows of the
// sums, the spans of the join.
bool bwd_sizes_ok(int64_t M, int64_t D, int64_t V) {
  if (!sizes_ok(M, D, V)) return false;
  const BwdPlan p = bwd_plan(M, D, V);
  const int64_t cols = (D + 511) / 512;
  const int64_t sums = (p.spans * cols + 3) / 4 + (V + 4 * kZeroIds - 1) / (4 * kZeroIds);
  return ((int64_t)kSortThreads << p.ord.log_nb) <= kMaxLaunchThreads &&
         sums * 256 <= kMaxLaunchThreads && p.spans * kJoinThreads <= kMaxLaunchThreads;
}

}  // namespace
}  // namespace nf

using namespace nf;

extern "C" int nf_embedding_fwd(const int64_t *ids, const void *table, int64_t ld_table,
                                float scale, int64_t M, int64_t D, int64_t V, void *out,
                                int dt_table, int dt_out, void *stream) {
  if (!sizes_ok(M, D, V) || ld_table < D)
    return set_error(NF_ERR_ARG, "nf_embedding_fwd: bad shape M=%lld D=%lld V=%lld ld=%lld",
                     (long long)M, (long long)D, (long long)V, (long long)ld_table);
  if (!types_ok(dt_table, dt_out))
    return set_error(NF_ERR_DTYPE, "nf_embedding_fwd: dtypes %d -> %d", dt_table, dt_out);
  if (M == 0) return NF_OK;
  if (!ids || !table || !out) return set_error(NF_ERR_ARG, "nf_embedding_fwd: null pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
#define NF_EMB(CW, CO, W, O)                                                                   \
  if (dt_table == CW && dt_out == CO)                                                          \
    return run_fwd<W, O>(ids, static_cast<const W *>(table), ld_table, scale, M, D, V,         \
                         static_cast<O *>(out), s);
  NF_EMB(NF_DTYPE_F32, NF_DTYPE_F32, float, float)
  NF_EMB(NF_DTYPE_BF16, NF_DTYPE_BF16, bf16, bf16)
  NF_EMB(NF_DTYPE_F16, NF_DTYPE_F16, f16, f16)
  NF_EMB(NF_DTYPE_F32, NF_DTYPE_BF16, float, bf16)
  NF_EMB(NF_DTYPE_F32, NF_DTYPE_F16, float, f16)
#undef NF_EMB
  return set_error(NF_ERR_DTYPE, "nf_embedding_fwd: dtypes %d -> %d", dt_table, dt_out);
}

extern "C" size_t nf_embedding_bwd_workspace(int64_t M, int64_t D, int64_t V) {
  if (!bwd_sizes_ok(M, D, V)) return 0;
  return bwd_plan(M, D, V).total;
}

extern "C" int nf_embedding_bwd(const void *dout, const int64_t *ids, int64_t padding_id,
                                float scale, int64_t M, int64_t D, int64_t V, void *dtable,
                                int dt_out, int dt_table, void *workspace,
                                size_t workspace_bytes, void *stream) {
  if (!bwd_sizes_ok(M, D, V))
    return set_error(NF_ERR_ARG, "nf_embedding_bwd: bad shape M=%lld D=%lld V=%lld",
                     (long long)M, (long long)D, (long long)V);
  if (!types_ok(dt_table, dt_out))
    return set_error(NF_ERR_DTYPE, "nf_embedding_bwd: dtypes %d -> %d", dt_out, dt_table);
  if (!dtable || (M > 0 && (!dout || !ids)))
    return set_error(NF_ERR_ARG, "nf_embedding_bwd: null pointer");
  const size_t need = nf_embedding_bwd_workspace(M, D, V);
  if (!workspace || workspace_bytes < need || !aligned16(workspace))
    return set_error(NF_ERR_WORKSPACE, "nf_embedding_bwd: workspace %zu bytes < required %zu",
                     workspace_bytes, need);
  hipStream_t s = static_cast<hipStream_t>(stream);
  char *ws = static_cast<char *>(workspace);
#define NF_EMB(CW, CO, W, O)                                                                 \
  if (dt_table == CW && dt_out == CO)                                                        \
    return run_bwd<O, W>(static_cast<const O *>(dout), ids, padding_id, scale, M, D, V,      \
                         static_cast<W *>(dtable), ws, s);
  NF_EMB(NF_DTYPE_F32, NF_DTYPE_F32, float, float)
  NF_EMB(NF_DTYPE_BF16, NF_DTYPE_BF16, bf16, bf16)
  NF_EMB(NF_DTYPE_F16, NF_DTYPE_F16, f16, f16)
  NF_EMB(NF_DTYPE_F32, NF_DTYPE_BF16, float, bf16)
  NF_EMB(NF_DTYPE_F32, NF_DTYPE_F16, float, f16)
#undef NF_EMB
  return set_error(NF_ERR_DTYPE, "nf_embedding_bwd: dtypes %d -> %d", dt_out, dt_table);
}
