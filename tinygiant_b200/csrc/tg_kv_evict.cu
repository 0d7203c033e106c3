// tg_kv_evict.cu — tg_cache_evict: a key/value cache cut down to a budget by
// the attention its keys have gathered.
//
// Of sequence b and key head h with n = lens[b] positions, m = min(n, keep)
// stay: the last r = min(recent, m) always, and of the n - r others the m - r
// of the largest weight, equal weights by the lower position.  What stays
// keeps its order.  Weights compare as numbers (-0 equals 0), NaN above all.
//
// select_kernel, a block per (sequence, key head), finds the threshold (the
// (m - r)-th largest weight) by three radix passes of 11, 11 and 10 bits over
// the weights' order-preserving integers, then one pass in position order
// that numbers what stays.  gather_kernel moves the rows.
#include <algorithm>

#include "../../include/tinygiant.h"
#include "tg_attn.h"

namespace tg {

constexpr int EV_THREADS = 512;

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
  int base = 0, sum = 0;
  for (int i = 0; i < EV_THREADS / 32; i++) {
    if (i < w) base += red[i];
    sum += red[i];
  }
  *total = sum;
  return base + x - v;
}

__global__ void __launch_bounds__(EV_THREADS) select_kernel(const EvictArgs a) {
  __shared__ int hist[2048];
  __shared__ int red[EV_THREADS / 32];
  __shared__ uint32_t s_bin;
  __shared__ int s_need;
  const int t = threadIdx.x, b = blockIdx.x / a.KH, h = blockIdx.x % a.KH;
  const int n = min(max(a.lens[b], 0), a.cap), m = min(n, a.keep), r = min(a.recent, m);
  const float* w = a.w + b * a.sw[0] + h * a.sw[1];
  int* idx = a.idx + (size_t)blockIdx.x * a.keep;
  float* wo = a.wo + (size_t)blockIdx.x * a.keep;
  if (h == 0 && t == 0) a.lens_out[b] = m;
  const int cand = n - r, want = m - r;       // want <= cand
  uint32_t thr = 0;                           // keys above thr stay, and need of those equal to it
  int need = want;
  if (want > 0 && want < cand) {
    int shift = 32;
    for (int pass = 0; pass < 3; pass++) {
      const int bits = pass < 2 ? 11 : 10;
      shift -= bits;
      for (int i = t; i < 2048; i += EV_THREADS) hist[i] = 0;
      __syncthreads();
      for (int i = t; i < cand; i += EV_THREADS) {
        const uint32_t u = order_key(w[i]);
        if (pass == 0 || (u >> (shift + bits)) == (thr >> (shift + bits))) atomicAdd(&hist[(u >> shift) & ((1 << bits) - 1)], 1);
      }
      __syncthreads();
      // the bin, from the top, in which the need-th key lies
      const int nb = 1 << bits, per = nb / EV_THREADS;   // 4 or 2 bins a thread
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
      __syncthreads();
    }
  }
  int kept = 0, equal = 0;
  for (int i0 = 0; i0 < cand && want > 0; i0 += EV_THREADS) {
    const int i = i0 + t;
    const float x = i < cand ? w[i] : 0.f;
    const uint32_t u = order_key(x);
    int eq = want < cand && i < cand && u == thr, sum;
    const int er = equal + block_excl_sum(eq, red, &sum);
    equal += sum;
    const int stay = i < cand && (want == cand || u > thr || (eq && er < need));
    const int at = kept + block_excl_sum(stay, red, &sum);
    kept += sum;
    if (stay) {
      idx[at] = i;
      wo[at] = x;
    }
  }
  for (int i = t; i < r; i += EV_THREADS) {
    idx[want + i] = cand + i;
    wo[want + i] = w[cand + i];
  }
  for (int i = m + t; i < a.keep; i += EV_THREADS) {
    idx[i] = -1;
    wo[i] = 0.f;
  }
}

// Rows of one (sequence, key head): word c of output row j from row idx[j],
// zeros behind the sequence's end.
__global__ void __launch_bounds__(256) gather_kernel(const EvictArgs a) {
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
  select_kernel<<<bh, EV_THREADS, 0, s>>>(a);
  gather_kernel<<<dim3(std::min(64, (words + 255) / 256), bh), 256, 0, s>>>(a);
  count_launches(2);
  return c.done(cudaGetLastError());
}
