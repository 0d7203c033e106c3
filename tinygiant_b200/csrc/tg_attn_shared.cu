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
//   own     own_kernel: each sequence's keys are read once for every 16 query
//           heads of their key head (its registers hold that many), once in
//           all for up to 16; bound by HBM.  S^T = K Q^T and O^T += V^T P^T
//           with the heads as the 8 columns of mma.m16n8k16 (few rows: the
//           tensor memory path has 128).  All sequences' keys in a row are cut
//           evenly among the CTAs, so lengths may differ at will.
//   join    join_kernel: weighted sum of the pieces, the sinks, the outputs;
//           weights from the scores that own_kernel left, once the whole
//           softmax's maximum and sum are known (their order is fixed: results
//           are the same each time).
// The prefix is bound by the tensor cores and the own keys by HBM, so the two
// kernels run side by side, each on its share of the SMs.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/tinygiant.h"
#include "tg_attn_split.h"
#include "tg_attn_tc.cuh"

namespace tg {

// Rows per TMA box: whole stages come in boxes of 128 rows, a sequence's last
// 64 rows and less in boxes of 32 (a box takes about 85 clocks to issue: with
// 16 boxes of 32 rows in every stage the issuing bound an SM to 46 GB/s).
constexpr int OWN_BOX = 32;
constexpr int OWN_WARPS = 8;        // two groups of four that take stages in turn
constexpr int OWN_THREADS = (OWN_WARPS + 1) * 32;

struct OwnArgs {
  const void* q;
  const int* lens;
  float* po;          // [segment][8 NT][HD], see OwnWalk
  float2* pml;        // [segment][8 NT]: (c m - OFF, l)
  int* starts;        // [batch + 1]: stages of a key head before each sequence
  float* scores;      // [b KH + kh][max_len][gp] c s, or null
  long long sq[2];
  int B, KH, G, gp, hd, max_len, window, ngc;   // ngc: groups of 8 NT heads per key head
  float c, inv_c;     // scale log2(e), and 1 / that
  DevStatus* st;
};

template <int HD>
struct OwnShape {
  static constexpr int HALF = OWN_KEYS * 128;             // bytes of 64 columns of a stage's K or V
  static constexpr int STAGE = 2 * (HD / 64) * HALF;      // K and V
  static constexpr int STAGES = HD == 128 ? 3 : 6, BARS = 2 * STAGES;
  static constexpr int RP = HD + 4;                       // row pitch of the next: lanes with other heads on other banks
  static constexpr int RED = OWN_WARPS * 8 * RP * 4;      // the warps' accumulators of 8 heads
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

// Barriers go by the stage's number modulo twice the ring: then a barrier
// belongs to one group, which sees each of its phases (a wait by parity passes
// if the barrier is a whole phase behind).
struct OwnShared {
  uint64_t full[12], empty[12];
  float2 ml[OWN_WARPS][8];   // each warp's (m, l) of 8 heads
  int sums[OWN_WARPS];
  int b0, before;            // the CTA's first sequence, and the stages of a key head before it
  int abort;
};

// A sequence's own keys [lo, len) and the stages of 128 that they take.
__device__ __forceinline__ int own_len(const int* lens, int b, int max_len) { return min(max(lens[b], 0), max_len); }
__device__ __forceinline__ int own_first(int len, int window) { return window > 0 ? max(0, len - window) & ~15 : 0; }
__device__ __forceinline__ int own_stages(int len, int window) {
  return (len - own_first(len, window) + OWN_KEYS - 1) / OWN_KEYS;
}
// The CTA of n that stage x of `total` falls to: CTA i has the stages
// [i total / n, (i + 1) total / n).
__device__ __forceinline__ int own_cta(long long x, long long total, int n) { return (int)(((x + 1) * n - 1) / total); }

// The stages of a CTA, sequence by sequence, key head by key head (and group
// of heads), as segments: consecutive stages of one (sequence, head).  A
// segment's place among the partial results is its CTA's number plus the
// number of its (sequence, head): two segments differ in one of them at least,
// and neither ever falls.
struct OwnWalk {
  long long x, x1;
  int b, hk, j, len, lo, n, j1;   // sequence, head, first stage; own keys, first key, stages; last stage + 1
  int ahead;                      // the next sequence's own keys, read a sequence early
  __device__ void seq(const OwnArgs& a, int keys) {
    len = keys;
    lo = own_first(len, a.window);
    n = own_stages(len, a.window);
    ahead = b + 1 < a.B ? own_len(a.lens, b + 1, a.max_len) : 0;
  }
  __device__ void start(const OwnArgs& a, int b0, int before, long long x0, long long end) {
    x = x0, x1 = end, b = b0;
    if (x >= x1) return;
    seq(a, own_len(a.lens, b, a.max_len));
    const long long r = x0 - (long long)before * (a.KH * a.ngc);
    hk = (int)(r / n), j = (int)(r % n);
    j1 = (int)min((long long)n, j + x1 - x);
  }
  __device__ bool more() const { return x < x1; }
  __device__ void next(const OwnArgs& a) {
    x += j1 - j;
    if (x >= x1) return;
    j = 0;
    if (++hk == a.KH * a.ngc) {
      hk = 0;
      do {
        b++;
        seq(a, ahead);
      } while (n == 0);   // x < x1: there is another sequence with keys
    }
    j1 = (int)min((long long)n, x1 - x);
  }
};

// Persistent, one CTA per SM of its share.  Warp 8 loads stages ahead, across
// segments.  Warps 0-3 and 4-7 take stages in turn, each warp 32 keys with a
// reference m of its own (moved, as in attn_tc_kernel, only when a score
// exceeds it by LIFT in base 2: one vote in the common case); the warps' partial
// results join in shared memory at the end of a segment.  Bound by HBM: 442 MB
// in 76 us on all SMs (batch 256, 768 keys on average), 0.89 of measured.
template <typename T, int HD, int NT>
__global__ void __launch_bounds__(OWN_THREADS, 1) own_kernel(const __grid_constant__ CUtensorMap kmap,
                                                             const __grid_constant__ CUtensorMap vmap,
                                                             const __grid_constant__ CUtensorMap kend,
                                                             const __grid_constant__ CUtensorMap vend, const OwnArgs a) {
  using S = OwnShape<HD>;
  extern __shared__ uint8_t dsm[];
  __shared__ OwnShared sh;
  const int tid = threadIdx.x, wid = tid >> 5, lane = tid & 31;
  uint8_t* stages = dsm + ((1024u - (smem_u32(dsm) & 1023u)) & 1023u);
  float* red = reinterpret_cast<float*>(stages + S::STAGES * S::STAGE);
  volatile int* abort = &sh.abort;
  if (tid == 0) {
    for (int i = 0; i < S::BARS; i++) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], OWN_WARPS / 2);
    }
    sh.abort = 0;
    fence_mbar_init();
  }
  pdl_wait();
  pdl_trigger();
  // The whole number of stages, then where this CTA's begin.  A thread has
  // one of 256 sequences at a time; up to 256 stay in registers.
  const int HK = a.KH * a.ngc;
  int mine = 0, before = 0, round = 0;   // this thread's sequence: stages, those before it
  auto scan = [&](int b0) {
    const int b = b0 + tid;
    mine = tid < OWN_WARPS * 32 && b < a.B ? own_stages(own_len(a.lens, b, a.max_len), a.window) : 0;
    int y = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const int z = __shfl_up_sync(~0u, y, o);
      if (lane >= o) y += z;
    }
    __syncthreads();
    if (lane == 31 && wid < OWN_WARPS) sh.sums[wid] = y;
    __syncthreads();
    before = round + y - mine;
    for (int i = 0; i < OWN_WARPS; i++) {
      if (i < wid) before += sh.sums[i];
      round += sh.sums[i];
    }
  };
  for (int b0 = 0; b0 < a.B; b0 += OWN_WARPS * 32) scan(b0);
  const long long total = (long long)round * HK;
  const long long ctas = min((long long)gridDim.x, total);   // those that get any: every CTA in between has a segment
  const long long x0 = blockIdx.x < ctas ? total * blockIdx.x / ctas : total;
  const long long x1 = blockIdx.x < ctas ? total * (blockIdx.x + 1) / ctas : total;
  auto note = [&](int b0) {
    const int b = b0 + tid;
    if (tid >= OWN_WARPS * 32 || b >= a.B) return;
    if ((long long)before * HK <= x0 && x0 < (long long)(before + mine) * HK) sh.b0 = b, sh.before = before;
    if (blockIdx.x == 0) {
      a.starts[b] = before;
      if (b == a.B - 1) a.starts[a.B] = before + mine;
    }
  };
  if (a.B <= OWN_WARPS * 32) {
    note(0);
  } else {
    round = 0;
    for (int b0 = 0; b0 < a.B; b0 += OWN_WARPS * 32) {
      scan(b0);
      note(b0);
    }
  }
  __syncthreads();
  auto fail = [&](int site, int u) {
    if (!*abort) set_error(a.st, ERR_WAIT_TIMEOUT, site, blockIdx.x, u);
    *abort = 1;
  };
  OwnWalk wk;
  int n = 0;   // stages so far

  if (wid == OWN_WARPS) {
    bool ok = true;
    for (wk.start(a, sh.b0, sh.before, x0, x1); wk.more() && ok; wk.next(a)) {
      const int kh = wk.hk / a.ngc;
      for (int j = wk.j; j < wk.j1; j++, n++) {
        const int s = n % S::STAGES, r0 = wk.lo + j * OWN_KEYS, old = n - S::STAGES;
        uint64_t* full = &sh.full[n % S::BARS];
        if (old >= 0 && !at_wait(&sh.empty[old % S::BARS], (old / S::BARS) & 1, abort)) {
          if (lane == 0) fail(400, n);
          ok = false;
          break;
        }
        const bool all = wk.len - r0 > OWN_KEYS / 2;
        const int rows = all ? OWN_KEYS : OWN_BOX, boxes = all ? 1 : (wk.len - r0 + OWN_BOX - 1) / OWN_BOX;   // of each column half of K and V
        if (lane == 0) mbar_arrive_expect_tx(full, boxes * 2 * (HD / 64) * rows * 128);
        __syncwarp();
        if (lane < boxes * 2 * (HD / 64)) {
          const int bx = lane % boxes, h = lane / boxes;   // h: K halves, then V halves
          const CUtensorMap* map = h < HD / 64 ? (all ? &kmap : &kend) : (all ? &vmap : &vend);
          tma_load_4d(stages + s * S::STAGE + h * S::HALF + bx * OWN_BOX * 128, map, 64 * (h % (HD / 64)), r0 + bx * OWN_BOX, kh, wk.b, full);
        }
      }
    }
    __syncthreads();   // the other warps are done
    if (*abort && lane == 0)   // some warp gave up: no copy of this CTA may still be in flight at its end
      for (int i = max(0, n - S::STAGES); i < n; i++) mbar_wait(&sh.full[i % S::BARS], (i / S::BARS) & 1);
    return;
  }

  const int g = lane >> 2, cc = lane & 3, wq = wid & 3;
  // this lane's ldmatrix row and 16-byte column of the warp's first 16 keys,
  // for columns 0-15 of each 16: K rows then halves of k, V halves of d then rows
  const int krow = wq * 32 + (lane & 15), vrow = wq * 32 + (lane & 7) + ((lane >> 4) << 3);
  uint32_t ko[4], vo[4];   // byte offsets of the four 16-column groups of a half, swizzled
#pragma unroll
  for (int k = 0; k < 4; k++) {
    ko[k] = krow * 128 + (((k * 2 + (lane >> 4)) ^ (krow & 7)) << 4);
    vo[k] = vrow * 128 + (((k * 2 + ((lane >> 3) & 1)) ^ (vrow & 7)) << 4);
  }
  int turn = 0;                              // the next stage's group
  uint32_t stage = 0, bar = 0, phase = 0;    // and its place, barrier and phase
  for (wk.start(a, sh.b0, sh.before, x0, x1); wk.more(); wk.next(a)) {
    const int b = wk.b, kh = wk.hk / a.ngc, gc = wk.hk % a.ngc, bk = b * a.KH + kh;
    const int lo = a.window > 0 ? max(0, wk.len - a.window) : 0, hi = wk.len;
    const size_t seg = (size_t)blockIdx.x + (size_t)b * HK + wk.hk;
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
    // reference m in base 2, as OFF - m and as the score that exceeds it by LIFT
    float nm[NT][2], lim[NT][2];
#pragma unroll
    for (int t = 0; t < NT; t++) nm[t][0] = nm[t][1] = 0.f, lim[t][0] = lim[t][1] = -INFINITY;
    float* scores = a.scores ? a.scores + (size_t)bk * a.max_len * a.gp + gc * NT * 8 + cc * 2 : nullptr;
    // One step: this warp's keys k0 .. k0 + 31 of a stage.  WHOLE: all of them
    // are the sequence's.
    auto step = [&](auto whole, uint32_t kb, int k0) {
      constexpr bool WHOLE = decltype(whole)::value;
      const uint32_t vb = kb + (HD / 64) * S::HALF;
      float x[2][NT][4];
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int t = 0; t < NT; t++) x[u][t][0] = x[u][t][1] = x[u][t][2] = x[u][t][3] = 0.f;
#pragma unroll
      for (int k = 0; k < HD / 16; k++)
#pragma unroll
        for (int u = 0; u < 2; u++) {
          uint32_t f[4];
          ldsm4(f, kb + ko[k % 4] + (k / 4) * S::HALF + u * 2048);
#pragma unroll
          for (int t = 0; t < NT; t++) mma16816<T>(x[u][t], f, qf[t][k][0], qf[t][k][1]);
        }
      bool up = false;
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const int ka = k0 + 16 * u + g;
        const bool in0 = WHOLE || (ka >= lo && ka < hi), in1 = WHOLE || (ka + 8 >= lo && ka + 8 < hi);
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
          for (int z = 0; z < 4; z++) {
            if (!WHOLE && !(z < 2 ? in0 : in1)) x[u][t][z] = -INFINITY;
            up |= x[u][t][z] > lim[t][z & 1];
          }
          if (a.scores && (gc * NT + t) * 8 < a.gp) {
            float* sc = scores + (size_t)ka * a.gp + t * 8;
            if (in0) *reinterpret_cast<float2*>(sc) = make_float2(x[u][t][0] * a.c, x[u][t][1] * a.c);
            if (in1) *reinterpret_cast<float2*>(sc + 8 * a.gp) = make_float2(x[u][t][2] * a.c, x[u][t][3] * a.c);
          }
        }
      }
      if (__any_sync(~0u, up)) {
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int z = 0; z < 2; z++) {
            float v = fmaxf(fmaxf(x[0][t][z], x[0][t][z + 2]), fmaxf(x[1][t][z], x[1][t][z + 2]));
#pragma unroll
            for (int sft = 4; sft < 32; sft <<= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, sft));
            const float mn = fmaxf(m[t][z], v * a.c), f = mn > m[t][z] ? at_exp2(m[t][z] - mn) : 1.f;
            m[t][z] = mn;
            nm[t][z] = mn == -INFINITY ? 0.f : AttnRange<T>::OFF - mn;
            lim[t][z] = (mn + AttnRange<T>::LIFT) * a.inv_c;
            l[t][z] *= f;
#pragma unroll
            for (int k = 0; k < HD / 16; k++) {
              o[t][k][z] *= f;
              o[t][k][z + 2] *= f;
            }
          }
      }
      uint32_t p[2][NT][2];
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int t = 0; t < NT; t++) {
          float e[4];
#pragma unroll
          for (int z = 0; z < 4; z++) {
            e[z] = at_exp2(fmaf(x[u][t][z], a.c, nm[t][z & 1]));
            l[t][z & 1] += e[z];
          }
          p[u][t][0] = movm(at_pack<T>(e[0], e[1]));
          p[u][t][1] = movm(at_pack<T>(e[2], e[3]));
        }
#pragma unroll
      for (int u = 0; u < 2; u++) {
        // V rows outside [lo, hi) may hold anything, infinities and NaN too:
        // their bits are cleared (a register has two keys of one dimension)
        uint32_t vm[2] = {~0u, ~0u};
        if (!WHOLE)
#pragma unroll
          for (int z = 0; z < 2; z++) {
            const int kk = k0 + 16 * u + z * 8 + cc * 2;
            vm[z] = (kk >= lo && kk < hi ? 0x0000ffffu : 0u) | (kk + 1 >= lo && kk + 1 < hi ? 0xffff0000u : 0u);
          }
#pragma unroll
        for (int k = 0; k < HD / 16; k++) {
          uint32_t f[4];
          ldsm4t(f, vb + vo[k % 4] + (k / 4) * S::HALF + u * 2048);
          if (!WHOLE) f[0] &= vm[0], f[1] &= vm[0], f[2] &= vm[1], f[3] &= vm[1];
#pragma unroll
          for (int t = 0; t < NT; t++) mma16816<T>(o[t][k], f, p[u][t][0], p[u][t][1]);
        }
      }
    };
    for (int j = wk.j; j < wk.j1; j++) {
      if (turn == wid >> 2) {
        if (!at_wait(&sh.full[bar], phase, abort)) {
          if (lane == 0) fail(401, bar);
          break;   // on to the barriers below: every wait from here on fails at once
        }
        const int k0 = wk.lo + j * OWN_KEYS + wq * 32;
        if (k0 < hi) {
          const uint32_t kb = smem_u32(stages) + stage * S::STAGE;
          if (k0 >= lo && k0 + 32 <= hi)
            step(std::true_type{}, kb, k0);
          else
            step(std::false_type{}, kb, k0);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.empty[bar]);
      }
      turn ^= 1;
      if (++stage == S::STAGES) stage = 0;
      if (++bar == S::BARS) bar = 0, phase ^= 1;
    }
    // join the warps, 8 heads at a time
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
      for (int z = 0; z < 2; z++) {
#pragma unroll
        for (int sft = 4; sft < 32; sft <<= 1) l[t][z] += __shfl_xor_sync(~0u, l[t][z], sft);
        if (g == 0) sh.ml[wid][cc * 2 + z] = make_float2(m[t][z] - AttnRange<T>::OFF, l[t][z]);
      }
#pragma unroll
      for (int k = 0; k < HD / 16; k++)
#pragma unroll
        for (int z = 0; z < 4; z++) red[(wid * 8 + cc * 2 + (z & 1)) * S::RP + k * 16 + g + (z >> 1) * 8] = o[t][k][z];
      asm volatile("bar.sync 1, 256;" ::: "memory");
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
          v = fmaf(red[(w * 8 + h) * S::RP + d], f, v);
        }
        const size_t at = seg * (8 * NT) + t * 8 + h;
        a.po[at * HD + d] = v;
        if (d == 0) a.pml[at] = make_float2(M, L);
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
    }
  }
  __syncthreads();   // with the load warp's
}

struct JoinArgs {
  const int *lens, *starts;
  const float* sinks;
  float* weights;
  const float *po, *scores;
  const float2* pml;
  void* out;
  long long so[2], sw[2], own_row;   // own_row: the own segments' first row in pml and po
  int B, KH, G, gp, hd, tpt, nsp, max_len, window, ngc, nt, own_ctas;
};

constexpr int JOIN_THREADS = 256;
constexpr int JOIN_KEYS = 2048;  // own positions whose weights one block adds (512: 26 us instead of 22 at batch 256)

// Block (b KH + kh, part): the weights of JOIN_KEYS own positions, and in part
// 0 the outputs, a warp per head.  Bound by latency: lengths, places, factors,
// then pieces and scores; 22 us at batch 256 with weights (50 MB), 6 us without
// at 33 sequences.
template <typename T, int HD>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const JoinArgs a) {
  __shared__ float2 fin[AT_ROWS];   // per head: M, 1 / the sum
  pdl_wait();
  const int bk = blockIdx.x, kh = bk % a.KH, b = bk / a.KH, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int len = own_len(a.lens, b, a.max_len), lo = a.window > 0 ? max(0, len - a.window) : 0;
  const int j0 = (int)blockIdx.y * JOIN_KEYS;
  if (blockIdx.y > 0 && (j0 >= len || j0 + JOIN_KEYS <= lo)) return;
  const int ub = b / (2 * a.tpt), r = b % (2 * a.tpt), t = r / a.tpt, tok = r % a.tpt;
  const int HK = a.KH * a.ngc, n = a.own_ctas ? own_stages(len, a.window) : 0;
  long long total = 0, first = 0;
  int ctas = 0;
  if (n > 0) {
    total = (long long)a.starts[a.B] * HK;
    first = (long long)a.starts[b] * HK;
    ctas = (int)min((long long)a.own_ctas, total);
  }
  for (int g = wid; g < a.G; g += JOIN_THREADS / 32) {
    // pieces: the prefix's, then the segments of the CTAs c0 .. c1
    const int hk = kh * a.ngc + g / (8 * a.nt), gl = g % (8 * a.nt);
    int c0 = 0, pieces = a.nsp;
    if (n > 0) {
      c0 = own_cta(first + (long long)hk * n, total, ctas);
      pieces += own_cta(first + (long long)(hk + 1) * n - 1, total, ctas) - c0 + 1;
    }
    auto row = [&](int i) -> long long {
      if (i < a.nsp) return ((long long)(ub * a.nsp + i) * a.KH + kh) * (2 * AT_ROWS) + t * AT_ROWS + tok * a.G + g;
      return a.own_row + ((long long)b * HK + hk + c0 + i - a.nsp) * (8 * a.nt) + gl;
    };
    const float2 f = join_scale(pieces, a.pml, a.sinks ? a.sinks[kh * a.G + g] * LOG2E : -INFINITY, row);
    if (lane == 0) fin[g] = f;
    if (blockIdx.y == 0)
      join_row<T, HD>(pieces, a.pml, a.po, f, row, (T*)a.out + b * a.so[0] + (kh * a.G + g) * a.so[1], a.hd);
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

// The workspace of the cut work (tg_attn_split.h): prefix pieces' and own
// segments' partial results, the sequences' first stages, scores.
struct SharedSpace : SharedSplit {
  long long own_row;
  size_t pml, po, starts, scores, bytes = 0;
  SharedSpace(int B, int P, int max_len, int H, int KH, int hd, bool weights) : SharedSplit(B, P, max_len, H, KH, hd, attn_sms()) {
    const int HD = hd <= 64 ? 64 : 128;
    const long long HK = (long long)KH * ngc;
    auto take = [&](size_t n) {
      const size_t o = bytes;
      bytes = (bytes + n + 255) & ~(size_t)255;
      return o;
    };
    own_row = (long long)units * nsp * KH * 2 * AT_ROWS;
    const size_t rows = own_row + (own_ctas ? ((size_t)own_ctas + (size_t)B * HK) * 8 * nt : 0);
    pml = take(8 * rows);
    po = take(4 * rows * HD);
    starts = take(own_ctas ? 4 * ((size_t)B + 1) : 0);
    scores = take(weights ? 4 * (size_t)B * KH * max_len * gp : 0);
  }
};

template <typename T, int HD, int NT>
static cudaError_t launch_own(const CUtensorMap* m, const OwnArgs& a, int grid, cudaStream_t s) {
  const int smem = OwnShape<HD>::SMEM;
  static std::atomic<unsigned long long> set{0};
  const cudaError_t e = attn_smem(own_kernel<T, HD, NT>, smem, set);
  if (e != cudaSuccess) return e;
  return launch_pdl(own_kernel<T, HD, NT>, dim3(grid), OWN_THREADS, smem, s, m[0], m[1], m[2], m[3], a);
}

// The own keys' kernel goes first and lets the prefix start beside it at once;
// the prefix's CTAs, one for each piece, take the SMs that are left, and those
// of the own keys once they are done.  The last of them waits for the own
// keys' kernel, so that the join, which waits for the prefix, follows both.
template <typename T, int HD>
static cudaError_t run_shared(const CUtensorMap* m, AttnTcArgs ta, int pieces, const OwnArgs& oa, const JoinArgs& ja, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  if (ja.own_ctas > 0) {
    e = ja.nt == 1 ? launch_own<T, HD, 1>(m + 3, oa, ja.own_ctas, s) : launch_own<T, HD, 2>(m + 3, oa, ja.own_ctas, s);
    count_launches(1);
  }
  ta.beside = ja.own_ctas > 0;
  if (e == cudaSuccess && pieces > 0) {
    e = launch_attn_tc<T, HD, true>(m[0], m[1], m[2], ta, pieces, s);
    count_launches(1);
  }
  if (e == cudaSuccess) {
    const dim3 grid(ja.B * ja.KH, ja.weights ? std::max(1, (ja.max_len + JOIN_KEYS - 1) / JOIN_KEYS) : 1);
    e = launch_pdl(join_kernel<T, HD>, grid, JOIN_THREADS, 0, s, ja);
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
  c.need((long long)sp.units * sp.nsp * n_kv_heads < 0x7fffffff && max_len / JOIN_KEYS < 65535, "too many positions");
  c.need(workspace_bytes >= sp.bytes, "the workspace is smaller than tg_attention_shared_workspace says");
  if (sp.bytes > 0) c.ptr(workspace, 256, "workspace");
  if (c.rc) return c.rc;

  const int G = n_heads / n_kv_heads;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  AttnTcArgs a{};
  a.out = out;
  a.po = (float*)(ws + sp.po);
  a.pml = (float2*)(ws + sp.pml);
  a.lens = lens;
  a.v = prefix_v, a.sv[0] = t[5], a.sv[1] = t[4];
  a.G = G, a.KH = n_kv_heads, a.hd = head_dim, a.tpt = sp.tpt, a.window = window, a.total_k = prefix_len;
  a.P = prefix_len, a.B = batch, a.nsp = sp.nsp, a.max_len = max_len;
  a.c = scale * LOG2E;
  a.st = attn_status();
  int* starts = (int*)(ws + sp.starts);
  OwnArgs o{q, lens, a.po + sp.own_row * (head_dim <= 64 ? 64 : 128), a.pml + sp.own_row, starts,
            weights ? (float*)(ws + sp.scores) : nullptr, {t[0], t[1]}, batch, n_kv_heads, G, sp.gp, head_dim, max_len, window, sp.ngc,
            a.c, 1.f / a.c, a.st};
  JoinArgs j{lens, starts, sinks, weights, a.po, o.scores, a.pml, out, {t[12], t[13]},
             {weights ? strides[14] : 0, weights ? strides[15] : 0}, sp.own_row, batch, n_kv_heads, G, sp.gp, head_dim, sp.tpt, sp.nsp,
             max_len, window, sp.ngc, sp.nt, sp.own_ctas};
  CUtensorMap m[7];
  bool maps = true;
  int pieces = 0;
  if (prefix_len > 0) {
    pieces = sp.units * sp.nsp * n_kv_heads;
    maps = attn_q_map(&m[0], dtype, q, head_dim, n_heads, batch, t[0], t[1], G, sp.tpt) &&
           attn_kv_map(&m[1], dtype, prefix_k, q, head_dim, n_kv_heads, prefix_len, t[3], t[2]) &&
           attn_kv_map(&m[2], dtype, prefix_v, q, head_dim, n_kv_heads, prefix_len, t[5], t[4]);
  }
  if (max_len > 0)
    for (int i = 0; i < 2; i++) {
      const int rows = i ? OWN_BOX : OWN_KEYS;
      maps = maps && attn_cache_map(&m[3 + 2 * i], dtype, k, head_dim, cap, n_kv_heads, batch, t[8], t[7], t[6], rows) &&
             attn_cache_map(&m[4 + 2 * i], dtype, v, head_dim, cap, n_kv_heads, batch, t[11], t[10], t[9], rows);
    }
  c.need(maps, "the tensors' shapes and strides do not fit a tensor map");
  if (c.rc) return c.rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = dtype == ATTN_BF16, small = head_dim <= 64;
  return c.done(bf ? (small ? run_shared<__nv_bfloat16, 64>(m, a, pieces, o, j, s) : run_shared<__nv_bfloat16, 128>(m, a, pieces, o, j, s))
                   : (small ? run_shared<__half, 64>(m, a, pieces, o, j, s) : run_shared<__half, 128>(m, a, pieces, o, j, s)));
}
