// tg_attn_prompt.cu — tg_attention_prompt: causal attention of packed prompts
// with grouped query heads, a sliding window, per-head sink logits and keys
// that precede a sequence's queries.
//
// Sequence s has the query rows [cu_q[s], cu_q[s+1]) and the keys
// [cu_k[s], cu_k[s+1]), nq and nk of them.  Its row i is at position
// p = nk - nq + i and attends to K = {j : 0 <= j <= p, j > p - window}
// (window 0: no lower bound) with x_j = scale q_i . k_j:
//   o_i = sum_K e^(x_j) v_j / (sum_K e^(x_j) + e^sink).
// Rows without a key give zeros.
//
// A warp per (row, query head): lanes take 32 keys at a time, a running
// maximum m, sum l and accumulator; one pass over the keys.
#include "../../include/tinygiant.h"
#include "tg_attn.h"

namespace tg {

struct PromptArgs {
  const void *q, *k, *v;
  void* out;
  const int *cu_q, *cu_k;
  const float* sinks;
  int n_seqs, total_q, total_k, H, KH, hd, window;
  long long sq[2], sk[2], sv[2], so[2];   // token and head strides, in elements
  float scale;
};

template <typename T>
__global__ void __launch_bounds__(128) prompt_rows_kernel(const PromptArgs a) {
  __shared__ float qs[4][ATTN_MAX_HD];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const long long item = (long long)blockIdx.x * 4 + w;
  if (item >= (long long)a.total_q * a.H) return;
  const int row = (int)(item / a.H), h = (int)(item % a.H), kh = h / (a.H / a.KH);
  int s = 0;
  while (s < a.n_seqs && a.cu_q[s + 1] <= row) s++;
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  if (s < a.n_seqs && a.cu_q[s] <= row) {
    const int k0 = max(0, a.cu_k[s]), nk = min(a.total_k, a.cu_k[s + 1]) - k0;
    const int p = nk - (a.cu_q[s + 1] - row);
    const int lo = a.window > 0 ? max(0, p - a.window + 1) : 0;
    const T* q = (const T*)a.q + row * a.sq[0] + h * a.sq[1];
    for (int d = lane; d < a.hd; d += 32) qs[w][d] = to_f32(q[d]);
    __syncwarp();
    for (int j0 = lo; j0 <= p; j0 += 32) {
      const int j = j0 + lane;
      float x = -INFINITY;
      if (j <= p) {
        const T* k = (const T*)a.k + (long long)(k0 + j) * a.sk[0] + kh * a.sk[1];
        x = 0.f;
        for (int d = 0; d < a.hd; d++) x = fmaf(qs[w][d], to_f32(k[d]), x);
        x *= a.scale;
      }
      float t = x;
      for (int o = 16; o; o >>= 1) t = fmaxf(t, __shfl_xor_sync(~0u, t, o));
      const float mn = fmaxf(m, t), m0 = mn == -INFINITY ? 0.f : mn, c = expf(m - m0);
      const float e = expf(x - m0);
      float sum = e;
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
      l = l * c + sum;
      m = mn;
      for (int r = 0; r < 4; r++) acc[r] *= c;
      for (int i = 0; i < 32 && j0 + i <= p; i++) {
        const float ei = __shfl_sync(~0u, e, i);
        const T* v = (const T*)a.v + (long long)(k0 + j0 + i) * a.sv[0] + kh * a.sv[1];
        for (int r = 0; r < 4; r++)
          if (lane + 32 * r < a.hd) acc[r] = fmaf(ei, to_f32(v[lane + 32 * r]), acc[r]);
      }
    }
    if (a.sinks) {
      const float sk = a.sinks[h], mn = fmaxf(m, sk), c = expf(m - mn);
      if (m != -INFINITY) {
        l = l * c + expf(sk - mn);
        for (int r = 0; r < 4; r++) acc[r] *= c;
      }
    }
  }
  T* o = (T*)a.out + row * a.so[0] + h * a.so[1];
  for (int r = 0; r < 4; r++)
    if (lane + 32 * r < a.hd) o[lane + 32 * r] = from_f32<T>(l > 0.f ? acc[r] / l : 0.f);
}

}  // namespace tg

using namespace tg;

extern "C" size_t tg_attention_prompt_workspace(int n_seqs, int total_q, int max_k, int n_heads, int n_kv_heads,
                                                int head_dim) {
  return 0;
}

extern "C" int tg_attention_prompt(int dtype, const void* q, const void* k, const void* v, void* out, const int* cu_q,
                                   const int* cu_k, const float* sinks, int n_seqs, int total_q, int total_k,
                                   int max_k, int n_heads, int n_kv_heads, int head_dim, const int64_t* strides,
                                   int window, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  ArgCheck c("tg_attention_prompt");
  c.need(dtype == ATTN_BF16 || dtype == ATTN_FP16, "dtype must be 0 (bf16) or 1 (fp16)");
  c.need(n_seqs >= 0 && total_q >= 0 && total_k >= 0 && max_k >= 0 && window >= 0, "counts must not be negative");
  c.need(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && n_heads / n_kv_heads <= 128,
         "n_heads must be a multiple of n_kv_heads, at most 128 times it");
  c.need(head_dim > 0 && head_dim % 8 == 0 && head_dim <= ATTN_MAX_HD, "head_dim must be a multiple of 8, at most 128");
  c.need(std::isfinite(scale) && scale > 0.f, "scale must be finite and positive");
  c.need(strides != nullptr, "strides is null");
  if (c.rc || !c.strides(strides, 8)) return c.rc;
  if (total_q == 0) return 0;
  c.need(n_seqs > 0, "rows without a sequence");
  if (!c.device()) return c.rc;
  c.ptr(q, 16, "q"), c.ptr(out, 16, "out"), c.ptr(cu_q, 4, "cu_q"), c.ptr(cu_k, 4, "cu_k");
  if (total_k > 0) c.ptr(k, 16, "k"), c.ptr(v, 16, "v");
  if (sinks) c.ptr(sinks, 4, "sinks");
  if (c.rc) return c.rc;
  PromptArgs a{q, k, v, out, cu_q, cu_k, sinks, n_seqs, total_q, total_k, n_heads, n_kv_heads, head_dim, window,
               {strides[0], strides[1]}, {strides[2], strides[3]}, {strides[4], strides[5]}, {strides[6], strides[7]},
               scale};
  const long long items = (long long)total_q * n_heads, grid = (items + 3) / 4;
  c.need(grid < (1ll << 31), "too many rows");
  if (c.rc) return c.rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == ATTN_BF16)
    prompt_rows_kernel<__nv_bfloat16><<<(unsigned)grid, 128, 0, s>>>(a);
  else
    prompt_rows_kernel<__half><<<(unsigned)grid, 128, 0, s>>>(a);
  count_launches(1);
  return c.done(cudaGetLastError());
}
