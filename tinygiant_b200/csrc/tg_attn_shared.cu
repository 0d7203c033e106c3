// tg_attn_shared.cu — tg_attention_shared: one new token of each sequence of a
// batch attends to a prefix that all sequences share and to the sequence's
// own cached keys.
//
// Sequence b has len = lens[b] own positions (its newest token's key is the
// last of them), at the positions P .. P + len - 1 behind the prefix; its
// query is at e = P + len - 1 and attends to the keys j <= e, j > e - window
// (window 0: all).  With x_j = scale q . k_j:
//   o = sum e^(x_j) v_j / (sum e^(x_j) + e^sink),
//   weights[b][kh][j] += sum over the query heads of kh of their softmax
//                        weight of own position j.
// A sequence without a key gives zeros.
//
// A warp per (sequence, query head) with a running maximum, sum and
// accumulator; one warp adds a key head's weights in a second pass.
#include "../../include/tinygiant.h"
#include "tg_attn.h"

namespace tg {

struct SharedArgs {
  const void *q, *pk, *pv, *k, *v;
  void* out;
  const int* lens;
  const float* sinks;
  float* weights;
  int B, P, max_len, H, KH, hd, window;
  long long sq[2], spk[2], spv[2], sk[3], sv[3], so[2], sw[2];
  float scale;
};

template <typename T>
__device__ __forceinline__ float row_dot(const float* q, const T* k, int hd) {
  float x = 0.f;
  for (int d = 0; d < hd; d++) x = fmaf(q[d], to_f32(k[d]), x);
  return x;
}

// A block per (sequence, key head), a warp at a time per query head.
template <typename T>
__global__ void __launch_bounds__(32) shared_rows_kernel(const SharedArgs a) {
  __shared__ float qs[ATTN_MAX_HD];
  const int lane = threadIdx.x, b = blockIdx.x / a.KH, kh = blockIdx.x % a.KH, G = a.H / a.KH;
  const int len = min(max(a.lens[b], 0), a.max_len), n = a.P + len, lo = a.window > 0 ? max(0, n - a.window) : 0;
  auto kp = [&](int j) {
    return j < a.P ? (const T*)a.pk + j * a.spk[1] + kh * a.spk[0]
                   : (const T*)a.k + b * a.sk[0] + kh * a.sk[1] + (j - a.P) * a.sk[2];
  };
  auto vp = [&](int j) {
    return j < a.P ? (const T*)a.pv + j * a.spv[1] + kh * a.spv[0]
                   : (const T*)a.v + b * a.sv[0] + kh * a.sv[1] + (j - a.P) * a.sv[2];
  };
  for (int g = 0; g < G; g++) {
    const int h = kh * G + g;
    const T* q = (const T*)a.q + b * a.sq[0] + h * a.sq[1];
    __syncwarp();
    for (int d = lane; d < a.hd; d += 32) qs[d] = to_f32(q[d]);
    __syncwarp();
    float acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
    for (int j0 = lo; j0 < n; j0 += 32) {
      const int j = j0 + lane;
      const float x = j < n ? row_dot(qs, kp(j), a.hd) * a.scale : -INFINITY;
      float t = x;
      for (int o = 16; o; o >>= 1) t = fmaxf(t, __shfl_xor_sync(~0u, t, o));
      const float mn = fmaxf(m, t), m0 = mn == -INFINITY ? 0.f : mn, c = expf(m - m0), e = expf(x - m0);
      float sum = e;
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
      l = l * c + sum;
      m = mn;
      for (int r = 0; r < 4; r++) acc[r] *= c;
      for (int i = 0; i < 32 && j0 + i < n; i++) {
        const float ei = __shfl_sync(~0u, e, i);
        const T* v = vp(j0 + i);
        for (int r = 0; r < 4; r++)
          if (lane + 32 * r < a.hd) acc[r] = fmaf(ei, to_f32(v[lane + 32 * r]), acc[r]);
      }
    }
    if (a.sinks && m != -INFINITY) {
      const float sk = a.sinks[h], mn = fmaxf(m, sk), c = expf(m - mn);
      l = l * c + expf(sk - mn);
      m = mn;
      for (int r = 0; r < 4; r++) acc[r] *= c;
    }
    T* o = (T*)a.out + b * a.so[0] + h * a.so[1];
    for (int r = 0; r < 4; r++)
      if (lane + 32 * r < a.hd) o[lane + 32 * r] = from_f32<T>(l > 0.f ? acc[r] / l : 0.f);
    if (a.weights)
      for (int j = max(lo, a.P) + lane; j < n; j += 32)
        a.weights[b * a.sw[0] + kh * a.sw[1] + (j - a.P)] += expf(row_dot(qs, kp(j), a.hd) * a.scale - m) / l;
  }
}

}  // namespace tg

using namespace tg;

extern "C" size_t tg_attention_shared_workspace(int batch, int prefix_len, int max_len, int n_heads, int n_kv_heads,
                                                int head_dim, int with_weights) {
  return 0;
}

extern "C" int tg_attention_shared(int dtype, const void* q, const void* prefix_k, const void* prefix_v, const void* k,
                                   const void* v, void* out, const int* lens, const float* sinks, float* weights,
                                   int batch, int prefix_len, int cap, int max_len, int n_heads, int n_kv_heads,
                                   int head_dim, const int64_t* strides, int window, float scale, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  ArgCheck c("tg_attention_shared");
  c.need(dtype == ATTN_BF16 || dtype == ATTN_FP16, "dtype must be 0 (bf16) or 1 (fp16)");
  c.need(batch >= 0 && prefix_len >= 0 && cap >= 0 && max_len >= 0 && max_len <= cap && window >= 0,
         "counts and window must not be negative, and max_len at most cap");
  c.need(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && n_heads / n_kv_heads <= 128,
         "n_heads must be a multiple of n_kv_heads, at most 128 times it");
  c.need(head_dim > 0 && head_dim % 8 == 0 && head_dim <= ATTN_MAX_HD, "head_dim must be a multiple of 8, at most 128");
  c.need(std::isfinite(scale) && scale > 0.f, "scale must be finite and positive");
  c.need(strides != nullptr, "strides is null");
  if (c.rc) return c.rc;
  const long long n5[5] = {batch, n_heads, n_kv_heads, prefix_len, cap};
  const int dim[14] = {0, 1, 2, 3, 2, 3, 0, 2, 4, 0, 2, 4, 0, 1};
  long long t[14];
  for (int i = 0; i < 14; i++) t[i] = c.stride(strides[i], n5[dim[i]]);
  c.need(!weights || (strides[14] > 0 && strides[15] > 0), "strides of weights must be positive");
  if (c.rc || batch == 0) return c.rc;
  if (!c.device()) return c.rc;
  c.ptr(q, 16, "q"), c.ptr(out, 16, "out"), c.ptr(lens, 4, "lens");
  if (prefix_len > 0) c.ptr(prefix_k, 16, "prefix_k"), c.ptr(prefix_v, 16, "prefix_v");
  if (cap > 0) c.ptr(k, 16, "k"), c.ptr(v, 16, "v");
  if (sinks) c.ptr(sinks, 4, "sinks");
  if (weights) c.ptr(weights, 4, "weights");
  if (c.rc) return c.rc;
  SharedArgs a{q, prefix_k, prefix_v, k, v, out, lens, sinks, weights, batch, prefix_len, max_len, n_heads, n_kv_heads,
               head_dim, window, {t[0], t[1]}, {t[2], t[3]}, {t[4], t[5]}, {t[6], t[7], t[8]}, {t[9], t[10], t[11]},
               {t[12], t[13]}, {weights ? strides[14] : 0, weights ? strides[15] : 0}, scale};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == ATTN_BF16)
    shared_rows_kernel<__nv_bfloat16><<<batch * n_kv_heads, 32, 0, s>>>(a);
  else
    shared_rows_kernel<__half><<<batch * n_kv_heads, 32, 0, s>>>(a);
  count_launches(1);
  return c.done(cudaGetLastError());
}
