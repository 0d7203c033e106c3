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
// The sums over disjoint sets of keys join by their (maximum, sum,
// accumulator), so the work is cut three ways:
//   prefix  attn_tc_kernel (tg_attn_tc.cuh): the batch's queries of a key head
//           are the rows of 128-row tiles, so the prefix is read once per tile
//           pair and not once per sequence; pieces of its keys.
//   own     own_kernel: each sequence's keys are read once, in pieces; bound
//           by HBM.  G query heads share a key head, so S^T = K Q^T and
//           O^T += V^T P^T with the heads as the 8 columns of mma.m16n8k16
//           (few rows: the tensor memory path has 128).
//   join    join_kernel: weighted sum of the pieces, the sinks, the outputs;
//           weights from the scores that own_kernel left, once the whole
//           softmax's maximum and sum are known (their order is fixed: results
//           are the same each time).
#include <algorithm>

#include "../../include/tinygiant.h"
#include "tg_attn_tc.cuh"

namespace tg {

constexpr int OWN_KEYS = 128;       // keys per stage: 16 for each consumer warp
constexpr int OWN_BOX = 32;         // rows per TMA box: a sequence's last stage reads at most 31 rows too many
constexpr int OWN_WARPS = 8;
constexpr int OWN_THREADS = (OWN_WARPS + 1) * 32;

struct OwnArgs {
  const void* q;
  const int* lens;
  float* po;          // [(b KH + kh) nso + piece][G][HD]
  float2* pml;        // [(b KH + kh) nso + piece][G]: (c m, l)
  float* scores;      // [b KH + kh][max_len][gp] c s, or null
  long long sq[2];
  int B, KH, G, gp, hd, max_len, window, chunk, nso, ngc;   // ngc: groups of 8 NT heads per key head
  float c;
  DevStatus* st;
};

template <int HD>
struct OwnShape {
  static constexpr int HALF = OWN_KEYS * 128;             // bytes of 64 columns of a stage's K or V
  static constexpr int STAGE = 2 * (HD / 64) * HALF;      // K and V
  static constexpr int STAGES = HD == 128 ? 3 : 6;
  static constexpr int RED = OWN_WARPS * 8 * HD * 4;      // the warps' accumulators of 8 heads
  static constexpr int SMEM = STAGES * STAGE + RED + 1024;
};

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ uint32_t movm(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

struct OwnShared {
  uint64_t full[6], empty[6];
  float2 ml[OWN_WARPS][8];   // each warp's (m, l) of 8 heads
  int abort;
};

// The keys [lo, hi) of piece `pc` of a sequence with len own keys.
__device__ __forceinline__ void own_range(const OwnArgs& a, int len, int pc, int& lo, int& hi) {
  lo = max(pc * a.chunk, a.window > 0 ? max(0, len - a.window) : 0);
  hi = min((pc + 1) * a.chunk, len);
}

// Persistent, one CTA per SM; item = ((b KH + kh) ngc + head group) nso +
// piece.  Warp 8 loads stages ahead, across items; each of warps 0-7 takes 16
// keys of a stage with a running maximum of its own, and the warps' partial
// results join in shared memory at the end of the item.
template <typename T, int HD, int NT>
__global__ void __launch_bounds__(OWN_THREADS, 1) own_kernel(const __grid_constant__ CUtensorMap kmap,
                                                             const __grid_constant__ CUtensorMap vmap, const OwnArgs a) {
  using S = OwnShape<HD>;
  extern __shared__ uint8_t dsm[];
  __shared__ OwnShared sh;
  const int tid = threadIdx.x, wid = tid >> 5, lane = tid & 31;
  uint8_t* stages = dsm + ((1024u - (smem_u32(dsm) & 1023u)) & 1023u);
  float* red = reinterpret_cast<float*>(stages + S::STAGES * S::STAGE);
  volatile int* abort = &sh.abort;
  if (tid == 0) {
    for (int i = 0; i < S::STAGES; i++) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], OWN_WARPS);
    }
    sh.abort = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  auto fail = [&](int site, int u) {
    if (!*abort) set_error(a.st, ERR_WAIT_TIMEOUT, site, blockIdx.x, u);
    *abort = 1;
  };
  const int items = a.B * a.KH * a.ngc * a.nso;
  int n = 0;   // stages so far

  if (wid == OWN_WARPS) {
    bool ok = true;
    for (int it = blockIdx.x; it < items && ok; it += gridDim.x) {
      const int pc = it % a.nso, bk = it / (a.nso * a.ngc), kh = bk % a.KH, b = bk / a.KH;
      int lo, hi;
      own_range(a, min(max(a.lens[b], 0), a.max_len), pc, lo, hi);
      for (int r0 = lo & ~15; r0 < hi; r0 += OWN_KEYS, n++) {
        const int s = n % S::STAGES;
        if (n >= S::STAGES && !at_wait(&sh.empty[s], (n / S::STAGES - 1) & 1, abort)) {
          if (lane == 0) fail(400, it);
          ok = false;
          break;
        }
        const int boxes = min(OWN_KEYS, hi - r0 + OWN_BOX - 1) / OWN_BOX;   // of each column half of K and V
        if (lane == 0) mbar_arrive_expect_tx(&sh.full[s], boxes * 2 * (HD / 64) * OWN_BOX * 128);
        __syncwarp();
        if (lane < boxes * 2 * (HD / 64)) {
          const int bx = lane % boxes, h = lane / boxes;   // h: K halves, then V halves
          tma_load_4d(stages + s * S::STAGE + h * S::HALF + bx * OWN_BOX * 128, h < HD / 64 ? &kmap : &vmap, 64 * (h % (HD / 64)),
                      r0 + bx * OWN_BOX, kh, b, &sh.full[s]);
        }
      }
    }
    if (*abort && lane == 0)   // no copy of this CTA may still be in flight
      for (int i = max(0, n - S::STAGES); i < n; i++) mbar_wait(&sh.full[i % S::STAGES], (i / S::STAGES) & 1);
    return;
  }

  const int g = lane >> 2, cc = lane & 3;
  // this lane's ldmatrix rows within its 16 keys and its 16-byte column
  const int krow = wid * 16 + (lane & 15), kcol = lane >> 4;                                  // K: rows, then k halves
  const int vrow = wid * 16 + (lane & 7) + ((lane >> 4) << 3), vcol = (lane >> 3) & 1;        // V: d halves, then rows
  for (int it = blockIdx.x; it < items; it += gridDim.x) {
    const int pc = it % a.nso, gc = it / a.nso % a.ngc, bk = it / (a.nso * a.ngc), kh = bk % a.KH, b = bk / a.KH;
    int lo, hi;
    own_range(a, min(max(a.lens[b], 0), a.max_len), pc, lo, hi);
    if (lo >= hi) continue;
    // Q^T as B fragments: heads are columns, absent ones and dimensions zero
    uint32_t qf[NT][HD / 16][2];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int hg = (gc * NT + t) * 8 + g;
      const T* q = (const T*)a.q + b * a.sq[0] + (kh * a.G + hg) * a.sq[1];
#pragma unroll
      for (int k = 0; k < HD / 16; k++)
#pragma unroll
        for (int z = 0; z < 2; z++) {
          const int d = k * 16 + z * 8 + cc * 2;
          qf[t][k][z] = hg < a.G && d < a.hd ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
        }
    }
    float o[NT][HD / 16][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      m[t][0] = m[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
#pragma unroll
      for (int k = 0; k < HD / 16; k++) o[t][k][0] = o[t][k][1] = o[t][k][2] = o[t][k][3] = 0.f;
    }
    for (int r0 = lo & ~15; r0 < hi; r0 += OWN_KEYS, n++) {
      const int s = n % S::STAGES;
      if (!at_wait(&sh.full[s], (n / S::STAGES) & 1, abort)) {
        if (lane == 0) fail(401, it);
        break;   // on to the barriers below: every wait from here on fails at once
      }
      const int k0 = r0 + wid * 16;   // this warp's keys k0 .. k0 + 15
      if (k0 < hi) {
        const uint32_t kb = smem_u32(stages + s * S::STAGE), vb = kb + (HD / 64) * S::HALF;
        float x[NT][4];
#pragma unroll
        for (int t = 0; t < NT; t++) x[t][0] = x[t][1] = x[t][2] = x[t][3] = 0.f;
#pragma unroll
        for (int k = 0; k < HD / 16; k++) {
          uint32_t f[4];
          ldsm4(f, kb + (k / 4) * S::HALF + krow * 128 + ((((k % 4) * 2 + kcol) ^ (krow & 7)) << 4));
#pragma unroll
          for (int t = 0; t < NT; t++) mma16816<T>(x[t], f, qf[t][k][0], qf[t][k][1]);
        }
        const bool in0 = k0 + g >= lo && k0 + g < hi, in1 = k0 + g + 8 >= lo && k0 + g + 8 < hi;
        uint32_t p[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
          for (int z = 0; z < 4; z++) x[t][z] = (z < 2 ? in0 : in1) ? x[t][z] * a.c : -INFINITY;
          if (a.scores) {
            float* sc = a.scores + ((size_t)bk * a.max_len + k0 + g) * a.gp + (gc * NT + t) * 8 + cc * 2;
            if ((gc * NT + t) * 8 < a.gp) {
              if (in0) *reinterpret_cast<float2*>(sc) = make_float2(x[t][0], x[t][1]);
              if (in1) *reinterpret_cast<float2*>(sc + 8 * a.gp) = make_float2(x[t][2], x[t][3]);
            }
          }
          float mn[2];
          bool up = false;
#pragma unroll
          for (int z = 0; z < 2; z++) {
            float v = fmaxf(x[t][z], x[t][z + 2]);
#pragma unroll
            for (int sft = 4; sft < 32; sft <<= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, sft));
            mn[z] = fmaxf(m[t][z], v);
            up |= mn[z] > m[t][z];
          }
          if (__any_sync(~0u, up)) {
#pragma unroll
            for (int z = 0; z < 2; z++) {
              const float f = mn[z] > m[t][z] ? at_exp2(m[t][z] - mn[z]) : 1.f;
              m[t][z] = mn[z];
              l[t][z] *= f;
#pragma unroll
              for (int k = 0; k < HD / 16; k++) {
                o[t][k][z] *= f;
                o[t][k][z + 2] *= f;
              }
            }
          }
          float e[4];
#pragma unroll
          for (int z = 0; z < 4; z++) {
            const float mz = m[t][z & 1];
            e[z] = at_exp2(x[t][z] - (mz == -INFINITY ? 0.f : mz));
            l[t][z & 1] += e[z];
          }
          p[t][0] = movm(at_pack<T>(e[0], e[1]));
          p[t][1] = movm(at_pack<T>(e[2], e[3]));
        }
        // V rows outside [lo, hi) may hold anything, infinities and NaN too:
        // their bits are cleared (a register has two keys of one dimension)
        const bool whole = k0 >= lo && k0 + 16 <= hi;
        uint32_t vm[2];
#pragma unroll
        for (int z = 0; z < 2; z++) {
          const int kk = k0 + z * 8 + cc * 2;
          vm[z] = (kk >= lo && kk < hi ? 0x0000ffffu : 0u) | (kk + 1 >= lo && kk + 1 < hi ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int k = 0; k < HD / 16; k++) {
          uint32_t f[4];
          ldsm4t(f, vb + (k / 4) * S::HALF + vrow * 128 + ((((k % 4) * 2 + vcol) ^ (vrow & 7)) << 4));
          if (!whole) f[0] &= vm[0], f[1] &= vm[0], f[2] &= vm[1], f[3] &= vm[1];
#pragma unroll
          for (int t = 0; t < NT; t++) mma16816<T>(o[t][k], f, p[t][0], p[t][1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[s]);
    }
    // join the warps, 8 heads at a time
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
      for (int z = 0; z < 2; z++) {
#pragma unroll
        for (int sft = 4; sft < 32; sft <<= 1) l[t][z] += __shfl_xor_sync(~0u, l[t][z], sft);
        if (g == 0) sh.ml[wid][cc * 2 + z] = make_float2(m[t][z], l[t][z]);
      }
#pragma unroll
      for (int k = 0; k < HD / 16; k++)
#pragma unroll
        for (int z = 0; z < 4; z++) red[(wid * 8 + cc * 2 + (z & 1)) * HD + k * 16 + g + (z >> 1) * 8] = o[t][k][z];
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const int h0 = (gc * NT + t) * 8;
      for (int i = tid; i < 8 * HD; i += OWN_WARPS * 32) {
        const int h = i / HD, d = i % HD;
        float M = -INFINITY, L = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < OWN_WARPS; w++) M = fmaxf(M, sh.ml[w][h].x);
#pragma unroll
        for (int w = 0; w < OWN_WARPS; w++) {
          const float2 ml = sh.ml[w][h];
          if (ml.y == 0.f) continue;   // a warp without keys
          const float f = at_exp2(ml.x - M);
          L = fmaf(ml.y, f, L);
          v = fmaf(red[(w * 8 + h) * HD + d], f, v);
        }
        if (h0 + h < a.G) {
          const size_t at = ((size_t)bk * a.nso + pc) * a.G + h0 + h;
          a.po[at * HD + d] = v;
          if (d == 0) a.pml[at] = make_float2(M, L);
        }
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
    }
  }
}

struct JoinArgs {
  const int* lens;
  const float* sinks;
  float* weights;
  const float *ppo, *opo, *scores;
  const float2 *ppml, *opml;
  void* out;
  long long so[2], sw[2];
  int B, KH, G, gp, hd, tpt, P, nsp, nso, chunk, max_len, window;
};

constexpr int JOIN_THREADS = 256;
constexpr int JOIN_KEYS = 2048;   // own positions whose weights one block adds

// Block (b KH + kh, part): the (maximum, 1 / sum) of each head, then in part 0
// the outputs and in every part the weights of JOIN_KEYS positions.
template <typename T, int HD>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const JoinArgs a) {
  __shared__ float2 fin[128];   // per head: M, 1 / L
  pdl_wait();
  const int bk = blockIdx.x, kh = bk % a.KH, b = bk / a.KH, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int len = min(max(a.lens[b], 0), a.max_len), lo = a.window > 0 ? max(0, len - a.window) : 0;
  const int p0 = lo / a.chunk, p1 = (len + a.chunk - 1) / a.chunk;   // own pieces with keys
  const int j0 = blockIdx.y * JOIN_KEYS;
  if (blockIdx.y > 0 && j0 >= len) return;
  const int ub = b / (2 * a.tpt), r = b % (2 * a.tpt), t = r / a.tpt, tok = r % a.tpt;
  auto pat = [&](int sp, int g) { return ((size_t)(ub * a.nsp + sp) * a.KH + kh) * (2 * AT_ROWS) + t * AT_ROWS + tok * a.G + g; };
  auto oat = [&](int pc, int g) { return ((size_t)bk * a.nso + pc) * a.G + g; };
  for (int g = wid; g < a.G; g += JOIN_THREADS / 32) {
    float M = -INFINITY;
    for (int i = lane; i < a.nsp; i += 32) M = fmaxf(M, a.ppml[pat(i, g)].x);
    for (int i = p0 + lane; i < p1; i += 32) M = fmaxf(M, a.opml[oat(i, g)].x);
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, o));
    const float sk = a.sinks ? a.sinks[kh * a.G + g] * LOG2E : -INFINITY;
    const bool any = M != -INFINITY;
    M = fmaxf(M, sk);
    float L = 0.f;
    for (int i = lane; i < a.nsp; i += 32) {
      const float2 ml = a.ppml[pat(i, g)];
      if (ml.y != 0.f) L = fmaf(ml.y, at_exp2(ml.x - M), L);
    }
    for (int i = p0 + lane; i < p1; i += 32) {
      const float2 ml = a.opml[oat(i, g)];
      if (ml.y != 0.f) L = fmaf(ml.y, at_exp2(ml.x - M), L);
    }
    for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(~0u, L, o);
    const float inv = any && L != 0.f ? 1.f / (L + at_exp2(sk - M)) : L;   // L: 0, or NaN
    if (lane == 0) fin[g] = make_float2(M, inv);
    if (blockIdx.y == 0) {
      constexpr int E = HD / 32;
      float o[E] = {};
      auto add = [&](const float2* pml, const float* po, size_t at) {
        const float2 ml = pml[at];
        if (ml.y == 0.f) return;
        const float f = at_exp2(ml.x - M);
        const float* x = po + at * HD + lane * E;
        if (E == 4) {
          const float4 v = *reinterpret_cast<const float4*>(x);
          o[0] = fmaf(v.x, f, o[0]), o[1] = fmaf(v.y, f, o[1]), o[E - 2] = fmaf(v.z, f, o[E - 2]), o[E - 1] = fmaf(v.w, f, o[E - 1]);
        } else {
          const float2 v = *reinterpret_cast<const float2*>(x);
          o[0] = fmaf(v.x, f, o[0]), o[1] = fmaf(v.y, f, o[1]);
        }
      };
      for (int i = 0; i < a.nsp; i++) add(a.ppml, a.ppo, pat(i, g));
      for (int i = p0; i < p1; i++) add(a.opml, a.opo, oat(i, g));
      T* out = (T*)a.out + b * a.so[0] + (kh * a.G + g) * a.so[1] + lane * E;
      if (lane * E < a.hd)
        for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(out + e) = at_pack<T>(o[e] * inv, o[e + 1] * inv);
    }
  }
  if (!a.weights) return;
  __syncthreads();
  float* w = a.weights + b * a.sw[0] + kh * a.sw[1];
  for (int j = max(j0, lo) + tid; j < min(len, j0 + JOIN_KEYS); j += JOIN_THREADS) {
    const float* sc = a.scores + ((size_t)bk * a.max_len + j) * a.gp;
    float sum = 0.f;
    for (int g = 0; g < a.G; g += 4) {
      const float4 x = *reinterpret_cast<const float4*>(sc + g);
      const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (g + e < a.G) sum = fmaf(at_exp2(xs[e] - fin[g + e].x), fin[g + e].y, sum);
    }
    w[j] += sum;
  }
}

// How the work is cut, and the workspace: prefix and own partial results, scores.
struct SharedSpace {
  int tpt, units, nsp, chunk, nso, gp;
  size_t ppml, ppo, opml, opo, scores, bytes = 0;
  SharedSpace(int B, int P, int max_len, int H, int KH, int hd, bool weights) {
    const int G = H / KH, sms = attn_sms(), HD = hd <= 64 ? 64 : 128;
    tpt = AT_ROWS / G;
    units = (B + 2 * tpt - 1) / (2 * tpt);
    // Prefix: as many pieces as make the longest CTA's work least, counting
    // two blocks' time for a piece's own start and end.
    const int blocks = (P + AT_KEYS - 1) / AT_KEYS;
    nsp = 0;
    long long best = 0;
    for (int n = 1; n <= std::min(blocks, 64); n++) {
      const long long rounds = ((long long)units * KH * n + sms - 1) / sms, cost = rounds * ((blocks + n - 1) / n + 2);
      if (!nsp || cost < best) nsp = n, best = cost;
    }
    // Own keys: pieces of at least two stages, four for each SM if there are
    // that many keys.
    const long long heads = (long long)B * KH, want = (4ll * sms + heads - 1) / heads;
    chunk = std::max(2 * OWN_KEYS, (int)(((max_len + want - 1) / want + OWN_KEYS - 1) / OWN_KEYS * OWN_KEYS));
    nso = (max_len + chunk - 1) / chunk;
    gp = (G + 7) / 8 * 8;
    auto take = [&](size_t n) {
      const size_t o = bytes;
      bytes = (bytes + n + 255) & ~(size_t)255;
      return o;
    };
    const size_t pr = (size_t)units * nsp * KH * 2 * AT_ROWS, orows = (size_t)heads * nso * G;
    ppml = take(8 * pr);
    ppo = take(4 * pr * HD);
    opml = take(8 * orows);
    opo = take(4 * orows * HD);
    scores = take(weights ? 4 * (size_t)heads * max_len * gp : 0);
  }
};

template <typename T, int HD, int NT>
static cudaError_t launch_own(const CUtensorMap& k, const CUtensorMap& v, const OwnArgs& a, int grid, cudaStream_t s) {
  const int smem = OwnShape<HD>::SMEM;
  static std::atomic<unsigned long long> set{0};   // devices whose limit is raised
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !(set.load() >> dev & 1))) {
    e = cudaFuncSetAttribute(own_kernel<T, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess && dev < 64) set |= 1ull << dev;
  }
  if (e != cudaSuccess) return e;
  return launch_pdl(own_kernel<T, HD, NT>, dim3(grid), OWN_THREADS, smem, s, k, v, a);
}

template <typename T, int HD>
static cudaError_t run_shared(const CUtensorMap* m, const AttnTcArgs& ta, int prefix_grid, OwnArgs oa, JoinArgs ja, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  if (prefix_grid > 0) {
    e = launch_attn_tc<T, HD, true>(m[0], m[1], m[2], ta, prefix_grid, s);
    count_launches(1);
  }
  if (e == cudaSuccess && oa.nso > 0) {
    const int nt = oa.G <= 8 ? 1 : 2;
    oa.ngc = (oa.G + 8 * nt - 1) / (8 * nt);
    const int grid = (int)std::min((long long)attn_sms(), (long long)oa.B * oa.KH * oa.ngc * oa.nso);
    e = nt == 1 ? launch_own<T, HD, 1>(m[3], m[4], oa, grid, s) : launch_own<T, HD, 2>(m[3], m[4], oa, grid, s);
    count_launches(1);
  }
  if (e == cudaSuccess) {
    const int parts = ja.weights ? std::max(1, (oa.max_len + JOIN_KEYS - 1) / JOIN_KEYS) : 1;
    e = launch_pdl(join_kernel<T, HD>, dim3(oa.B * oa.KH, parts), JOIN_THREADS, 0, s, ja);
    count_launches(1);
  }
  return e;
}

}  // namespace tg

using namespace tg;

extern "C" size_t tg_attention_shared_workspace(int batch, int prefix_len, int max_len, int n_heads, int n_kv_heads,
                                                int head_dim, int with_weights) {
  if (batch < 0 || prefix_len < 0 || max_len < 0 || n_kv_heads <= 0 || n_heads < n_kv_heads || n_heads / n_kv_heads > AT_ROWS) return 0;
  return SharedSpace(batch, prefix_len, max_len, n_heads, n_kv_heads, head_dim, with_weights != 0).bytes;
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
  c.need(prefix_len < AT_NPOS && cap < AT_NPOS, "too many positions");
  c.need(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && n_heads / n_kv_heads <= 128,
         "n_heads must be a multiple of n_kv_heads, at most 128 times it");
  c.need((long long)batch * n_heads < 1 << 24, "batch x n_heads must be below 2^24");
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
  if (max_len > 0) c.ptr(k, 16, "k"), c.ptr(v, 16, "v");
  if (sinks) c.ptr(sinks, 4, "sinks");
  if (weights) c.ptr(weights, 4, "weights");
  const SharedSpace sp(batch, prefix_len, max_len, n_heads, n_kv_heads, head_dim, weights != nullptr);
  c.need((long long)batch * n_kv_heads * std::max(1, sp.nso) * 16 < 0x7fffffff, "too many positions");
  c.need(workspace_bytes >= sp.bytes, "the workspace is smaller than tg_attention_shared_workspace says");
  if (sp.bytes > 0) c.ptr(workspace, 256, "workspace");
  if (c.rc) return c.rc;

  const int G = n_heads / n_kv_heads;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  AttnTcArgs a{};
  a.out = out;
  a.po = (float*)(ws + sp.ppo);
  a.pml = (float2*)(ws + sp.ppml);
  a.lens = lens;
  a.G = G, a.KH = n_kv_heads, a.hd = head_dim, a.tpt = sp.tpt, a.window = window, a.total_k = prefix_len;
  a.P = prefix_len, a.B = batch, a.nsp = sp.nsp, a.max_len = max_len;
  a.c = scale * LOG2E;
  a.st = attn_status();
  OwnArgs o{q, lens, (float*)(ws + sp.opo), (float2*)(ws + sp.opml), weights ? (float*)(ws + sp.scores) : nullptr, {t[0], t[1]},
            batch, n_kv_heads, G, sp.gp, head_dim, max_len, window, sp.chunk, sp.nso, 1, a.c, a.st};
  JoinArgs j{lens, sinks, weights, a.po, o.po, o.scores, a.pml, o.pml, out, {t[12], t[13]}, {weights ? strides[14] : 0, weights ? strides[15] : 0},
             batch, n_kv_heads, G, sp.gp, head_dim, sp.tpt, prefix_len, sp.nsp, sp.nso, sp.chunk, max_len, window};
  CUtensorMap m[5];
  bool maps = true;
  int grid = 0;
  if (prefix_len > 0) {
    grid = (int)std::min((long long)attn_sms(), (long long)sp.units * sp.nsp * n_kv_heads);
    maps = attn_q_map(&m[0], dtype, q, head_dim, n_heads, batch, t[0], t[1], G, sp.tpt) &&
           attn_kv_map(&m[1], dtype, prefix_k, q, head_dim, n_kv_heads, prefix_len, t[3], t[2]) &&
           attn_kv_map(&m[2], dtype, prefix_v, q, head_dim, n_kv_heads, prefix_len, t[5], t[4]);
  }
  if (max_len > 0)
    maps = maps && attn_cache_map(&m[3], dtype, k, head_dim, cap, n_kv_heads, batch, t[8], t[7], t[6], OWN_BOX) &&
           attn_cache_map(&m[4], dtype, v, head_dim, cap, n_kv_heads, batch, t[11], t[10], t[9], OWN_BOX);
  c.need(maps, "the tensors' shapes and strides do not fit a tensor map");
  if (c.rc) return c.rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = dtype == ATTN_BF16, small = head_dim <= 64;
  return c.done(bf ? (small ? run_shared<__nv_bfloat16, 64>(m, a, grid, o, j, s) : run_shared<__nv_bfloat16, 128>(m, a, grid, o, j, s))
                   : (small ? run_shared<__half, 64>(m, a, grid, o, j, s) : run_shared<__half, 128>(m, a, grid, o, j, s)));
}
