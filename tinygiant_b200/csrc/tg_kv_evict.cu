// tg_kv_evict.cu — tg_cache_evict: a key/value cache cut down to a budget by
// the attention its keys have gathered.
//
// Of sequence b and key head h with n = lens[b] positions, m = min(n, keep)
// stay: the last r = min(recent, m) always, and of the n - r others the m - r
// of the largest weight, equal weights by the lower position.  What stays
// keeps its order.  Weights compare as numbers (-0 equals 0), NaN above all.
//
// select_kernel, a block per (sequence, key head), finds the threshold (the
// (m - r)-th largest weight) by radix passes of 11, 11 and 10 bits over the
// weights' order-preserving integers, kept in shared memory where they fit,
// then numbers what stays in position order: counts by ballot for every 32
// positions, one prefix sum over the warps.  gather_kernel moves the rows:
// bound by HBM, 2 rows read and written per position.
#include <algorithm>

#include "../../include/tinygiant.h"
#include "tg_attn_tc.cuh"

namespace tg {

constexpr int EV_THREADS = 1024;
constexpr int EV_WARPS = EV_THREADS / 32;
constexpr int EV_CACHED = 40960;   // weights of a row kept in shared memory, at most (160 KB); longer rows are read again each pass

struct EvictArgs {
  const uint4 *k, *v;
  const float* w;
  const int* lens;
  uint4 *ko, *vo;
  float* wo;
  int *lens_out, *idx;
  int B, KH, cap, keep, recent, row16;        // row16: 16-byte words per row
  long long sk[3], sv[3], sw[2];              // sk, sv in 16-byte words
};

// Integers in the order of the weights: NaN above +inf, -0 = 0.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive prefix sum of v over the block; *total gets the sum.  red: one
// int per warp.
__device__ __forceinline__ int block_excl_sum(int v, int* red, int* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int x = v;
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) red[w] = x;
  __syncthreads();
  const int mine = red[lane];   // EV_WARPS = 32
  const int base = __reduce_add_sync(~0u, lane < w ? mine : 0);
  *total = __reduce_add_sync(~0u, mine);
  return base + x - v;
}

// 18 us for 256 rows of 8,192 (41 us with a block scan for every 512
// positions and the weights read again each pass).
__global__ void __launch_bounds__(EV_THREADS) select_kernel(const EvictArgs a, int cached) {
  static_assert(EV_WARPS == 32, "block_excl_sum");
  extern __shared__ uint32_t sk[];
  __shared__ int hist[2048];
  __shared__ int red[EV_WARPS];
  __shared__ uint32_t s_bin;
  __shared__ int s_need;
  pdl_wait();
  pdl_trigger();
  const int t = threadIdx.x, lane = t & 31, wp = t >> 5, b = blockIdx.x / a.KH, h = blockIdx.x % a.KH;
  const int n = min(max(a.lens[b], 0), a.cap), m = min(n, a.keep), r = min(a.recent, m);
  const float* w = a.w + b * a.sw[0] + h * a.sw[1];
  int* idx = a.idx + (size_t)blockIdx.x * a.keep;
  float* wo = a.wo + (size_t)blockIdx.x * a.keep;
  if (h == 0 && t == 0) a.lens_out[b] = m;
  const int cand = n - r, want = m - r;       // want <= cand
  for (int i = t; i < r; i += EV_THREADS) {
    idx[want + i] = cand + i;
    wo[want + i] = w[cand + i];
  }
  for (int i = m + t; i < a.keep; i += EV_THREADS) {
    idx[i] = -1;
    wo[i] = 0.f;
  }
  if (want == 0) return;
  if (want == cand) {   // all of them
    for (int i = t; i < cand; i += EV_THREADS) {
      idx[i] = i;
      wo[i] = w[i];
    }
    return;
  }
  auto key = [&](int i) { return cached ? sk[i] : order_key(w[i]); };
  uint32_t thr = 0;                           // keys above thr stay, and need of those equal to it
  int need = want, shift = 32;
  for (int pass = 0; pass < 3; pass++) {
    const int bits = pass < 2 ? 11 : 10;
    shift -= bits;
    for (int i = t; i < 2048; i += EV_THREADS) hist[i] = 0;
    __syncthreads();
#pragma unroll 4
    for (int i = t; i < cand; i += EV_THREADS) {
      uint32_t u;
      if (pass == 0) {
        u = order_key(w[i]);
        if (cached) sk[i] = u;
      } else {
        u = key(i);
      }
      if (pass == 0 || (u >> (shift + bits)) == (thr >> (shift + bits))) atomicAdd(&hist[(u >> shift) & ((1 << bits) - 1)], 1);
    }
    __syncthreads();
    // the bin, from the top, in which the need-th key lies
    const int nb = 1 << bits, per = nb / EV_THREADS;   // 2 bins a thread, or 1
    int c = 0;
    for (int i = 0; i < per; i++) c += hist[nb - 1 - (t * per + i)];
    int total;
    int above = block_excl_sum(c, red, &total);
    if (above < need && above + c >= need)
      for (int i = 0; i < per; i++) {
        const int bin = nb - 1 - (t * per + i);
        if (above + hist[bin] >= need) {
          s_bin = bin;
          s_need = need - above;
          break;
        }
        above += hist[bin];
      }
    __syncthreads();
    thr |= s_bin << shift;
    need = s_need;
  }
  // Each warp has a run of whole 32s; the numbers of kept keys before it, and
  // of keys equal to the threshold, whose first `need` stay, by prefix sums.
  const int groups = (cand + 31) / 32, per = (groups + EV_WARPS - 1) / EV_WARPS;
  const int g0 = min(groups, wp * per), g1 = min(groups, g0 + per);
  int above = 0, equal = 0;
  for (int g = g0; g < g1; g++) {
    const int i = g * 32 + lane;
    const uint32_t u = i < cand ? key(i) : 0;
    above += __popc(__ballot_sync(~0u, i < cand && u > thr));
    equal += __popc(__ballot_sync(~0u, i < cand && u == thr));
  }
  int total;
  const int eq0 = __shfl_sync(~0u, block_excl_sum(lane == 0 ? equal : 0, red, &total), 0);
  const int ab0 = __shfl_sync(~0u, block_excl_sum(lane == 0 ? above : 0, red, &total), 0);
  int at = ab0 + min(eq0, need), eqs = eq0;   // kept before this warp's run; equal ones before it
  for (int g = g0; g < g1; g++) {
    const int i = g * 32 + lane;
    const uint32_t u = i < cand ? key(i) : 0;
    const unsigned before = (1u << lane) - 1, em = __ballot_sync(~0u, i < cand && u == thr);
    const bool stay = i < cand && (u > thr || (u == thr && eqs + __popc(em & before) < need));
    const unsigned sm = __ballot_sync(~0u, stay);
    if (stay) {
      const int o = at + __popc(sm & before);
      idx[o] = i;
      wo[o] = w[i];
    }
    at += __popc(sm);
    eqs += __popc(em);
  }
}

// 78 us for 551 MB (256 rows of 2,048 of 8,192, 256 bytes): the rate of a copy.
// Rows of one (sequence, key head): word c of output row j from row idx[j],
// zeros behind the sequence's end.
__global__ void __launch_bounds__(256) gather_kernel(const EvictArgs a) {
  pdl_wait();   // the choice
  const int bh = blockIdx.y, b = bh / a.KH, h = bh % a.KH;
  const uint4* k = a.k + b * a.sk[0] + h * a.sk[1];
  const uint4* v = a.v + b * a.sv[0] + h * a.sv[1];
  const size_t o = (size_t)bh * a.keep * a.row16;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < a.keep * a.row16; i += gridDim.x * 256) {
    const int j = i / a.row16, c = i % a.row16, src = a.idx[(size_t)bh * a.keep + j];
    uint4 x = make_uint4(0, 0, 0, 0), y = x;
    if (src >= 0) {
      x = k[src * a.sk[2] + c];
      y = v[src * a.sv[2] + c];
    }
    a.ko[o + i] = x;
    a.vo[o + i] = y;
  }
}

}  // namespace tg

using namespace tg;

extern "C" int tg_cache_evict(const void* k, const void* v, const float* weights, const int* lens, void* k_out,
                              void* v_out, float* weights_out, int* lens_out, int* indices, int batch, int cap,
                              int n_kv_heads, int head_dim, const int64_t* strides, int keep, int recent,
                              void* stream) {
  ArgCheck c("tg_cache_evict");
  c.need(batch >= 0 && cap > 0 && n_kv_heads > 0, "cap and n_kv_heads must be positive, batch not negative");
  c.need(keep > 0 && keep <= cap && recent >= 0 && recent <= keep, "need 0 < keep <= cap and 0 <= recent <= keep");
  c.need(head_dim > 0 && head_dim % 8 == 0 && head_dim <= ATTN_MAX_HD, "head_dim must be a multiple of 8, at most 128");
  c.need(strides != nullptr, "strides is null");
  if (c.rc) return c.rc;
  const long long n3[3] = {batch, n_kv_heads, cap};
  long long t[6];
  for (int i = 0; i < 6; i++) t[i] = c.stride(strides[i], n3[i % 3]);
  c.need(strides[6] > 0 && strides[7] > 0, "strides of weights must be positive");
  c.need((long long)batch * n_kv_heads <= 65535, "batch x n_kv_heads is at most 65535");
  c.need((long long)keep * head_dim < (1ll << 31), "keep x head_dim must be below 2^31");
  if (c.rc || batch == 0) return c.rc;
  if (!c.device()) return c.rc;
  c.ptr(k, 16, "k"), c.ptr(v, 16, "v"), c.ptr(weights, 4, "weights"), c.ptr(lens, 4, "lens");
  c.ptr(k_out, 16, "k_out"), c.ptr(v_out, 16, "v_out"), c.ptr(weights_out, 4, "weights_out");
  c.ptr(lens_out, 4, "lens_out"), c.ptr(indices, 4, "indices");
  c.need(k_out != k && k_out != v && v_out != v && v_out != k && weights_out != weights && lens_out != lens,
         "the outputs must not overlap the inputs");
  if (c.rc) return c.rc;
  EvictArgs a{(const uint4*)k, (const uint4*)v, weights, lens, (uint4*)k_out, (uint4*)v_out, weights_out, lens_out,
              indices, batch, n_kv_heads, cap, keep, recent, head_dim / 8,
              {t[0] / 8, t[1] / 8, t[2] / 8}, {t[3] / 8, t[4] / 8, t[5] / 8}, {strides[6], strides[7]}};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int bh = batch * n_kv_heads, words = keep * (head_dim / 8);
  const int cached = cap <= EV_CACHED;
  const size_t smem = cached ? 4 * (size_t)cap : 0;
  static std::atomic<unsigned long long> set{0};
  cudaError_t e = attn_smem(select_kernel, 4 * EV_CACHED, set);
  if (e == cudaSuccess) e = launch_pdl(select_kernel, dim3(bh), EV_THREADS, smem, s, a, cached);
  if (e == cudaSuccess) e = launch_pdl(gather_kernel, dim3(std::min(64, (words + 255) / 256), bh), 256, 0, s, a);
  count_launches(2);
  return c.done(e);
}
