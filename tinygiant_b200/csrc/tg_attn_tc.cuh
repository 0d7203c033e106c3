// tg_attn_tc.cuh — the tensor-core attention kernel of the prompt and shared-
// prefix operators (tcgen05.mma kind::f16, accumulators in tensor memory).
//
// Mathematics.  For a query row and its keys K, with s_j = q . k_j in fp32 and
// c = scale log2(e), one pass over the keys in blocks of 128 keeps a reference
// m, a sum l and an accumulator o:
//   p_j = 2^(c s_j - c m),  l += p_j,  o += p_j v_j;   result o / l.
// m starts as the first block's maximum.  It moves (with l and o scaled by
// 2^(c m_old - c m_new)) only when a block's maximum exceeds it by more than
// 2^8 in the exponent's base: results do not depend on the reference, fp32
// sums and 16-bit p_j hold 2^8 as well as 1, and o is then rarely touched.
// p_j is rounded to the inputs' type for the second product, as tcgen05 wants
// both operands of one type; its error there is that of rounding v once more
// (unit roundoff 2^-8 or 2^-11 of the weighted mean of |v|), the order of the
// output's own rounding.  l sums the unrounded p_j.
//
// Work unit: one key head, two tiles of 128 query rows.  A tile's rows are
// (token, query head of the group) pairs, token-major, so a group of G heads
// fills a tile with 128 / G tokens: K and V tiles are used by the whole group,
// short sequences fill tiles, and the masked corner of the causal diagonal is
// a few tokens wide.  Its keys are the blocks [kb0, kb1).
//
// Warps: 0-3 and 4-7 the softmax of tile 0 and 1 (a thread per row), 8 the TMA
// loads, 9 the MMAs.  Tensor memory: S (128 columns of fp32) and O per tile;
// the 16-bit P overwrites S.  While one tile's softmax runs, the tensor cores
// work on the other tile: P V of its block, then S of its next block.
// Persistent CTAs, one per SM; units come from an atomic counter, longest
// first, so loads and the first S of the next unit overlap the last epilogue.
// Every wait is bounded; a role that gives up records the error and the others
// stop waiting.
#pragma once
#include <cuda.h>

#include <atomic>
#include <type_traits>

#include "tg_attn.h"
#include "tg_ptx.cuh"

namespace tg {

constexpr int AT_ROWS = 128;       // query rows per tile (MMA M)
constexpr int AT_KEYS = 128;       // keys per block (MMA N of S, K of P V)
constexpr int AT_THREADS = 384;   // 12 warps, the last two idle: registers move between whole warpgroups
constexpr int AT_NPOS = 0x3fffffff;

// One piece of work of every key head.
struct __align__(16) AttnEntry {
  int q0, ntok;   // first query row (token) and tokens, at most 2 * (128 / G)
  int p0;         // position of the first token among its sequence's keys
  int k0, nk;     // the sequence's first key row and its keys
  int kb0, kb1;   // key blocks of this piece
  int slot;       // -1: writes the outputs; else the piece's place among the partial results
};

struct AttnHead {
  int n_entries, counter, n_splits, pad[61];
};

// The pieces of a split unit, joined by the combine kernel.
struct __align__(16) AttnSplit {
  int q0, ntok, slot, n;
};

// A sequence's query and key rows; offsets outside the tensors read as their ends.
struct AttnSeq {
  int q0, nq, k0, nk;
};
__device__ __forceinline__ AttnSeq attn_seq(const int* cu_q, const int* cu_k, int s, int total_q, int total_k) {
  AttnSeq r;
  r.q0 = min(max(cu_q[s], 0), total_q);
  r.nq = max(0, min(max(cu_q[s + 1], 0), total_q) - r.q0);
  r.k0 = min(max(cu_k[s], 0), total_k);
  r.nk = max(0, min(max(cu_k[s + 1], 0), total_k) - r.k0);
  return r;
}
// The unit of a sequence's tokens t0 .. t0 + tpu - 1.
__device__ __forceinline__ AttnEntry attn_unit(const AttnSeq& s, int t0, int tpu, int window) {
  AttnEntry e;
  e.q0 = s.q0 + t0;
  e.ntok = min(tpu, s.nq - t0);
  e.p0 = s.nk - s.nq + t0;
  e.k0 = s.k0;
  e.nk = s.nk;
  const int hi = e.p0 + e.ntok, lo = window > 0 ? max(0, e.p0 + 1 - window) : 0;
  e.kb0 = lo / AT_KEYS;
  e.kb1 = hi > 0 ? (hi + AT_KEYS - 1) / AT_KEYS : e.kb0;
  e.slot = -1;
  return e;
}

struct AttnTcArgs {
  AttnHead* head;             // prompt: the plan's
  const AttnEntry* entries;   // prompt: the plan's, or null: at most 32 sequences, nothing split
  const int *cu_q, *cu_k;     // prompt without a plan
  int n_seqs, total_q;
  void* out;
  float* po;                  // partial results [slot * KH + kh][2 * 128][HD]
  float2* pml;                // their (c m, l) [slot * KH + kh][2 * 128]
  const float* sinks;
  const int* lens;            // shared: own keys of each sequence
  long long so[2];
  int G, KH, hd, tpt, window;
  int total_k;                // rows of k and v
  int P, B, nsp, max_len;     // shared: prefix keys, sequences, pieces per unit, bound of lens
  float c;                    // scale log2(e)
  DevStatus* st;
};

// Shared-memory matrix descriptors, 128-byte swizzle.  K-major (Q, K): rows of
// 64 elements (128 bytes), 8-row groups 1024 bytes apart.  MN-major (V): 64
// elements of a key contiguous, 8-key groups 1024 bytes apart, the next 64
// elements AT_KEYS * 128 bytes on.
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t a) {
  return (uint64_t)((a >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t a) {
  return (uint64_t)((a >> 4) & 0x3FFFu) | ((uint64_t)(AT_KEYS * 128u >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) |
         (2ull << 61);
}
// kind::f16: fp32 accumulators, A and B of type T, A K-major, B K- or MN-major.
template <typename T>
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool b_mn) {
  return (1u << 4) | ((std::is_same<T, __nv_bfloat16>::value ? 1u : 0u) << 7) |
         ((std::is_same<T, __nv_bfloat16>::value ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(AT_ROWS >> 4) << 24);
}

__device__ __forceinline__ void at_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void at_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void at_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
               "l"(a), "l"(b), "r"(idesc), "r"(acc)
               : "memory");
}
__device__ __forceinline__ void at_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
               "r"(a), "l"(b), "r"(idesc), "r"(acc)
               : "memory");
}
__device__ __forceinline__ void at_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
#define AT_R4(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3])
#define AT_W4(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3])
__device__ __forceinline__ void at_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : AT_R4(r, 0), AT_R4(r, 4), AT_R4(r, 8), AT_R4(r, 12), AT_R4(r, 16), AT_R4(r, 20), AT_R4(r, 24), AT_R4(r, 28)
      : "r"(taddr));
}
__device__ __forceinline__ void at_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::AT_W4(r, 0),
      AT_W4(r, 4), AT_W4(r, 8), AT_W4(r, 12), AT_W4(r, 16), AT_W4(r, 20), AT_W4(r, 24), AT_W4(r, 28), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void at_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::AT_W4(r, 0),
               AT_W4(r, 4), AT_W4(r, 8), AT_W4(r, 12), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void at_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void at_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One box of a 3-D tensor map into shared memory (no multicast); x is a
// multiple of 64 elements, parts outside the tensor read as zeros.
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                   smem_u32(dst)),
               "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ float at_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t at_pack(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t at_pack<__nv_bfloat16>(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
template <>
__device__ __forceinline__ uint32_t at_pack<__half>(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ float2 at_fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 at_add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tadd.rn.f32x2 rd, ra, rb;\n\t"
      "mov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

template <int HD>
struct AttnTcShape {
  static constexpr int TILE = 128 * HD * 2;               // bytes of a Q tile, a K or a V block
  static constexpr int STAGES = HD == 128 ? 5 : 8;        // K and V blocks in flight
  static constexpr int SMEM = 2 * TILE + STAGES * TILE + 1024;
};

struct AttnTcShared {
  uint64_t q_full, q_empty, kv_full[8], kv_empty[8], s_full[2], p_full[2], o_full[2], unit_full[2], unit_empty[2], aux, drain;
  AttnEntry unit[2];
  int unit_kh[2];             // -1: no more work
  uint32_t tmem;
  int abort;
};

// Waits for phase `parity`; gives up after about a second, or once another
// role has.
__device__ __forceinline__ bool at_wait(uint64_t* bar, uint32_t parity, const volatile int* abort) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity))
    if (*abort || clock64() - t0 > (1ll << 31)) return false;
  return true;
}

template <typename T, int HD, bool SHARED>
__global__ void __launch_bounds__(AT_THREADS, 1) attn_tc_kernel(const __grid_constant__ CUtensorMap qmap,
                                                                const __grid_constant__ CUtensorMap kmap,
                                                                const __grid_constant__ CUtensorMap vmap, const AttnTcArgs a) {
  using S = AttnTcShape<HD>;
  constexpr int NST = S::STAGES, TILE = S::TILE;
  constexpr int TM_O = 2 * AT_KEYS;   // tensor memory: S of tile t at 128 t, O at 256 + HD t
  extern __shared__ uint8_t dsm[];
  __shared__ AttnTcShared sh;
  const int tid = threadIdx.x, wid = tid >> 5, lane = tid & 31;
  uint8_t* qs = dsm + ((1024u - (smem_u32(dsm) & 1023u)) & 1023u);
  uint8_t* kvs = qs + 2 * TILE;
  volatile int* abort = &sh.abort;

  if (wid == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (tid == 288) {
    mbar_init(&sh.q_full, 1);
    mbar_init(&sh.q_empty, 1);
    for (int i = 0; i < NST; i++) {
      mbar_init(&sh.kv_full[i], 1);
      mbar_init(&sh.kv_empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], 4);
      mbar_init(&sh.o_full[i], 1);
      mbar_init(&sh.unit_full[i], 1);
      mbar_init(&sh.unit_empty[i], 9);
    }
    mbar_init(&sh.aux, 1);
    mbar_init(&sh.drain, 1);
    sh.abort = 0;
    fence_mbar_init();
  }
  at_fence_before();
  __syncthreads();
  at_fence_after();
  const uint32_t tmem = sh.tmem;
  pdl_wait();   // the plan comes from the preceding kernel
  pdl_trigger();
  auto fail = [&](int site, int u) {
    if (!*abort) set_error(a.st, ERR_WAIT_TIMEOUT, site, blockIdx.x, u);
    *abort = 1;
  };
  // Without a plan: lane s of the load warp has sequence s, of at most 32, and
  // where its units end among those of all.
  AttnSeq seq{};
  int ends = 0;
  // Entry i of the work (every lane of the load warp calls it).
  auto unit_of = [&](int i) -> AttnEntry {
    if (!SHARED && a.entries) return a.entries[i];
    if (!SHARED) {
      const int s = __ffs(__ballot_sync(~0u, ends > i)) - 1;   // the sequence whose units end past i
      AttnSeq q;
      q.q0 = __shfl_sync(~0u, seq.q0, s), q.nq = __shfl_sync(~0u, seq.nq, s);
      q.k0 = __shfl_sync(~0u, seq.k0, s), q.nk = __shfl_sync(~0u, seq.nk, s);
      const int before = __shfl_sync(~0u, ends, s) - (q.nq + 2 * a.tpt - 1) / (2 * a.tpt);
      return attn_unit(q, (i - before) * 2 * a.tpt, 2 * a.tpt, a.window);
    }
    const int tpu = 2 * a.tpt, nblk = (a.P + AT_KEYS - 1) / AT_KEYS, sp = i % a.nsp;
    AttnEntry e{};
    e.q0 = i / a.nsp * tpu;
    e.ntok = min(tpu, a.B - e.q0);
    e.nk = a.P;
    e.kb0 = (int)((long long)nblk * sp / a.nsp);
    e.kb1 = (int)((long long)nblk * (sp + 1) / a.nsp);
    e.slot = i;
    if (a.window > 0) {   // without the keys that no row of the unit sees
      int lo = a.P;
      for (int r = lane; r < e.ntok; r += 32) lo = min(lo, max(0, a.P + min(max(a.lens[e.q0 + r], 0), a.max_len) - a.window));
      lo = __reduce_min_sync(~0u, lo);
      e.kb0 = lo >= a.P ? e.kb1 : min(e.kb1, max(e.kb0, lo / AT_KEYS));
    }
    return e;
  };
  // The next unit, as the load warp announced it; false at the end.
  int un = 0;
  auto next_unit = [&](AttnEntry& e, int& kh) -> bool {
    const int i = un & 1;
    if (!at_wait(&sh.unit_full[i], (un >> 1) & 1, abort)) {
      fail(300, un);
      return false;
    }
    e = sh.unit[i];
    kh = sh.unit_kh[i];
    return kh >= 0;
  };

  // 168 registers a thread at launch (384 x 168 = 64,512): 216 for the eight
  // softmax warps and 72 for the four others make the same sum.
  if (wid >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  if (wid == 8) {
    // ---- loads
    const int tpu = 2 * a.tpt;
    const bool fixed = SHARED || !a.entries;   // units dealt out in turn
    if (!SHARED && !a.entries) {
      if (lane < a.n_seqs) seq = attn_seq(a.cu_q, a.cu_k, lane, a.total_q, a.total_k);
      ends = max(0, (seq.nq + tpu - 1) / tpu);
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, ends, o);
        if (lane >= o) ends += y;
      }
    }
    const int n_entries = SHARED ? (a.B + tpu - 1) / tpu * a.nsp : a.entries ? a.head->n_entries : __shfl_sync(~0u, ends, 31);
    const int n_work = n_entries * a.KH;
    int issued = 0, qn = 0, auxn = 0;   // blocks, Q loads and corrected blocks so far
    bool ok = true;
    for (int it = 0; ok; it++) {
      int w = (int)blockIdx.x + it * (int)gridDim.x;
      if (!fixed) {
        if (lane == 0) w = atomicAdd(&a.head->counter, 1);
        w = __shfl_sync(~0u, w, 0);
      }
      AttnEntry e{};
      const int kh = w < n_work ? w % a.KH : -1;
      if (kh >= 0) e = unit_of(w / a.KH);
      const int us = it & 1;
      if (it >= 2 && !at_wait(&sh.unit_empty[us], ((it >> 1) - 1) & 1, abort)) {
        if (lane == 0) fail(301, it);
        break;
      }
      if (lane == 0) {
        sh.unit[us] = e;
        sh.unit_kh[us] = kh;
        mbar_arrive(&sh.unit_full[us]);
      }
      if (kh < 0) break;
      if (e.kb0 >= e.kb1) continue;
      const int ntile = e.ntok > a.tpt ? 2 : 1;
      if (qn > 0 && !at_wait(&sh.q_empty, (qn - 1) & 1, abort)) {
        if (lane == 0) fail(302, it);
        break;
      }
      qn++;
      if (lane == 0) {
        mbar_arrive_expect_tx(&sh.q_full, ntile * (HD / 64) * a.G * a.tpt * 128);
        for (int t = 0; t < ntile; t++)
          for (int c = 0; c < HD / 64; c++)
            tma_load_3d(qs + t * TILE + c * 16384, &qmap, 64 * c, kh * a.G, e.q0 + t * a.tpt, &sh.q_full);
      }
      for (int i = 0; i < 2 * (e.kb1 - e.kb0); i++) {
        const int s = issued % NST, row = (e.kb0 + (i >> 1)) * AT_KEYS;
        const bool v = i & 1;
        if (issued >= NST && !at_wait(&sh.kv_empty[s], (issued / NST - 1) & 1, abort)) {
          if (lane == 0) fail(303, it);
          ok = false;
          break;
        }
        uint8_t* dst = kvs + s * TILE;
        // Values behind the sequence's end belong to others: p = 0 does not
        // silence an infinity or NaN there, so those rows are zeroed first.
        // (Keys need nothing: their scores are replaced.)
        const int end = e.nk - row;
        const bool fix = v && end < AT_KEYS && e.k0 + e.nk < a.total_k;
        uint64_t* bar = fix ? &sh.aux : &sh.kv_full[s];
        if (lane == 0) {
          mbar_arrive_expect_tx(bar, TILE);
          for (int c = 0; c < HD / 64; c++)
            tma_load_3d(dst + c * 16384, v ? &vmap : &kmap, 64 * c, e.k0 + row, kh, bar);
        }
        if (fix) {
          if (!at_wait(&sh.aux, auxn & 1, abort)) {
            if (lane == 0) fail(304, it);
            ok = false;
            break;
          }
          auxn++;
          for (int c = 0; c < HD / 64; c++)
            for (int o = max(end, 0) * 8 + lane; o < AT_KEYS * 8; o += 32)
              reinterpret_cast<uint4*>(dst + c * 16384)[o] = make_uint4(0, 0, 0, 0);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.kv_full[s]);
        }
        issued++;
      }
    }
    if (*abort && lane == 0) {   // no copy of this CTA may still be in flight
      for (int i = max(0, issued - NST); i < issued; i++) mbar_wait(&sh.kv_full[i % NST], (i / NST) & 1);
      if (qn > 0) mbar_wait(&sh.q_full, (qn - 1) & 1);
    }
  } else if (wid == 9) {
    // ---- MMAs, issued by one thread
    if (lane == 0) {
      constexpr uint32_t idesc_s = idesc_f16<T>(AT_KEYS, false), idesc_o = idesc_f16<T>(HD, true);
      const uint32_t q0 = smem_u32(qs), kv0 = smem_u32(kvs);
      auto mma_s = [&](int t, int s) {   // S_t = Q_t K^T
#pragma unroll
        for (int k = 0; k < HD / 16; k++) {
          const uint32_t o = (k / 4) * 16384 + (k % 4) * 32;
          at_mma_ss(tmem + t * AT_KEYS, desc_kmajor(q0 + t * TILE + o), desc_kmajor(kv0 + s * TILE + o), idesc_s, k > 0);
        }
        at_commit(&sh.s_full[t]);
      };
      int kvn = 0, qn = 0, pn[2] = {0, 0};
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
        if (ok && !at_wait(bar, parity, abort)) {
          fail(site, un);
          ok = false;
        }
        return ok;
      };
      auto kv_wait = [&](int i, int site) { return wait(&sh.kv_full[i % NST], (i / NST) & 1, site); };
      for (; ok; un++) {
        AttnEntry e;
        int kh;
        if (!next_unit(e, kh)) break;
        mbar_arrive(&sh.unit_empty[un & 1]);
        const int nb = e.kb1 - e.kb0, ntile = e.ntok > a.tpt ? 2 : 1;
        if (nb <= 0) continue;
        if (!wait(&sh.q_full, qn & 1, 310) || !kv_wait(kvn, 311)) break;
        qn++;
        at_fence_after();
        for (int t = 0; t < ntile; t++) mma_s(t, kvn % NST);
        at_commit(&sh.kv_empty[kvn % NST]);
        if (nb == 1) at_commit(&sh.q_empty);
        kvn++;
        for (int j = 0; j < nb && ok; j++) {
          const bool more = j + 1 < nb;
          const int vs = kvn % NST, ks = (kvn + 1) % NST;
          if (!kv_wait(kvn, 312)) break;
          for (int t = 0; t < ntile; t++) {
            if (!wait(&sh.p_full[t], pn[t] & 1, 313)) break;
            pn[t]++;
            at_fence_after();
#pragma unroll
            for (int k = 0; k < AT_KEYS / 16; k++)   // O_t += P_t V
              at_mma_ts(tmem + TM_O + t * HD, tmem + t * AT_KEYS + k * 8, desc_mnmajor(kv0 + vs * TILE + k * 2048), idesc_o,
                        j > 0 || k > 0);
            if (more) {
              if (t == 0 && !kv_wait(kvn + 1, 314)) break;
              mma_s(t, ks);
            } else {
              at_commit(&sh.o_full[t]);
            }
          }
          if (!ok) break;
          at_commit(&sh.kv_empty[vs]);
          if (more) {
            at_commit(&sh.kv_empty[ks]);
            if (j + 2 == nb) at_commit(&sh.q_empty);
          }
          kvn += more ? 2 : 1;
        }
      }
      if (*abort) {   // no MMA of this CTA may still be in flight
        at_commit(&sh.drain);
        mbar_wait(&sh.drain, 0);
      }
    }
    __syncwarp();
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ---- softmax of tile t, a thread per row
    const int t = wid >> 2, row = tid & 127;
    const int tok = row / a.G, g = row - tok * a.G;
    const uint32_t lanes = (uint32_t)(wid & 3) << 21;   // this warp's 32 lanes of tensor memory
    const uint32_t ts = tmem + t * AT_KEYS + lanes, to = tmem + TM_O + t * HD + lanes;
    const float c = a.c;
    int sn = 0, on = 0;
    for (;; un++) {
      AttnEntry e;
      int kh;
      if (!next_unit(e, kh)) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.unit_empty[un & 1]);
      const int tt = t * a.tpt + tok, nb = e.kb1 - e.kb0;
      if (t * a.tpt >= e.ntok) continue;
      const bool valid = tok < a.tpt && tt < e.ntok;
      int hi, lo = 0;   // the row's keys
      if (SHARED) {
        hi = a.P;
        if (a.window > 0 && valid) lo = max(0, a.P + min(max(a.lens[e.q0 + tt], 0), a.max_len) - a.window);
      } else {
        hi = e.p0 + tt + 1;
        if (a.window > 0) lo = max(0, hi - a.window);
      }
      const int wlo = __reduce_max_sync(~0u, valid ? lo : 0), whi = __reduce_min_sync(~0u, valid ? hi : AT_NPOS);
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int j = 0; j < nb; j++) {
        if (!at_wait(&sh.s_full[t], sn & 1, abort)) {
          if (lane == 0) fail(320 + t, un);
          ok = false;
          break;
        }
        sn++;
        at_fence_after();
        uint32_t r[128];
#pragma unroll
        for (int i = 0; i < 4; i++) at_ld32(ts + 32 * i, r + 32 * i);
        at_wait_ld();
        float* s = reinterpret_cast<float*>(r);
        const int base = (e.kb0 + j) * AT_KEYS;
        if (base < wlo || base + AT_KEYS > whi) {
          const int l0 = lo - base, h0 = hi - base;
#pragma unroll
          for (int i = 0; i < 128; i++) s[i] = i >= l0 && i < h0 ? s[i] : -INFINITY;
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int i = 4; i < 128; i++) mx[i & 3] = fmaxf(mx[i & 3], s[i]);
        const float mn = fmaxf(fmaxf(m, fmaxf(mx[0], mx[1])), fmaxf(mx[2], mx[3]));
        if (j == 0) {
          m = mn;
        } else {
          const float d = (mn - m) * c;
          const bool up = d > 8.f;
          if (__any_sync(~0u, up)) {   // P V of the block before is complete: S came behind it
            const float f = up ? at_exp2(-d) : 1.f;
            if (up) m = mn;
            l *= f;
#pragma unroll
            for (int i = 0; i < HD / 32; i++) {
              uint32_t o[32];
              at_ld32(to + 32 * i, o);
              at_wait_ld();
#pragma unroll
              for (int q = 0; q < 32; q++) o[q] = __float_as_uint(__uint_as_float(o[q]) * f);
              at_st32(to + 32 * i, o);
            }
          }
        }
        const float cm = m == -INFINITY ? 0.f : -c * m;
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          uint32_t p[16];
#pragma unroll
          for (int q = 0; q < 16; q++) {
            float2 x = at_fma2(make_float2(s[32 * i + 2 * q], s[32 * i + 2 * q + 1]), make_float2(c, c), make_float2(cm, cm));
            x.x = at_exp2(x.x);
            x.y = at_exp2(x.y);
            sum[q & 1] = at_add2(sum[q & 1], x);
            p[q] = at_pack<T>(x.x, x.y);
          }
          at_st16(ts + 16 * i, p);
        }
        at_wait_st();
        at_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full[t]);
        sum[0] = at_add2(sum[0], sum[1]);
        l += sum[0].x + sum[0].y;
      }
      if (!ok) break;
      if (nb > 0) {
        if (!at_wait(&sh.o_full[t], on & 1, abort)) {
          if (lane == 0) fail(322 + t, un);
          break;
        }
        on++;
        at_fence_after();
      }
      const int h = kh * a.G + g;
      const bool part = SHARED || e.slot >= 0;
      const size_t pr = ((size_t)e.slot * a.KH + kh) * (2 * AT_ROWS) + t * AT_ROWS + row;
      float inv = 1.f;
      if (part) {
        if (valid) a.pml[pr] = make_float2(l == 0.f ? -INFINITY : c * m, l);
      } else {
        if (a.sinks && valid && l != 0.f) l += at_exp2(a.sinks[h] * LOG2E - c * m);
        inv = l == 0.f ? 0.f : 1.f / l;
      }
      T* out = (T*)a.out + (e.q0 + tt) * a.so[0] + h * a.so[1];
      float* po = a.po + pr * HD;
#pragma unroll
      for (int i = 0; i < HD / 32; i++) {
        uint32_t o[32];
        if (nb > 0) {
          at_ld32(to + 32 * i, o);
          at_wait_ld();
        } else {
#pragma unroll
          for (int q = 0; q < 32; q++) o[q] = 0;
        }
        if (!valid) continue;
        if (part) {
          if (nb <= 0) continue;   // l = 0: not read
#pragma unroll
          for (int q = 0; q < 32; q += 4)
            *reinterpret_cast<uint4*>(po + 32 * i + q) = make_uint4(o[q], o[q + 1], o[q + 2], o[q + 3]);
        } else {
#pragma unroll
          for (int q = 0; q < 32; q += 8) {
            uint4 x;
            uint32_t* xs = &x.x;
#pragma unroll
            for (int z = 0; z < 4; z++)
              xs[z] = at_pack<T>(__uint_as_float(o[q + 2 * z]) * inv, __uint_as_float(o[q + 2 * z + 1]) * inv);
            if (32 * i + q < a.hd) *reinterpret_cast<uint4*>(out + 32 * i + q) = x;
          }
        }
      }
      at_fence_before();
    }
  }
  at_fence_before();
  __syncthreads();
  if (wid == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// ---------------------------------------------------------------------
// Host side.

inline CUresult attn_map(CUtensorMap* m, int dtype, const void* p, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                         const cuuint32_t* box) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      fn = nullptr;
    return reinterpret_cast<Encode>(fn);
  }();
  if (!encode) return CUDA_ERROR_NOT_SUPPORTED;
  const cuuint32_t es[4] = {1, 1, 1, 1};
  return encode(m, dtype == ATTN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(p),
                dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// Q as [rows][heads][hd] in boxes of 64 elements x G heads x tpt rows.
inline bool attn_q_map(CUtensorMap* m, int dtype, const void* q, int hd, int H, long long rows, long long s_row, long long s_head,
                       int G, int tpt) {
  const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)H, (cuuint64_t)rows};
  const cuuint64_t st[2] = {(cuuint64_t)s_head * 2, (cuuint64_t)s_row * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)tpt};
  return attn_map(m, dtype, q, 3, dims, st, box) == CUDA_SUCCESS;
}

// K or V as [heads][rows][hd] in boxes of 64 elements x 128 rows.  Without
// rows nothing is loaded; the map then describes any valid address.
inline bool attn_kv_map(CUtensorMap* m, int dtype, const void* p, const void* any, int hd, int KH, long long rows, long long s_row,
                        long long s_head) {
  const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)(rows > 0 ? rows : 1), (cuuint64_t)KH};
  const cuuint64_t st[2] = {(cuuint64_t)s_row * 2, (cuuint64_t)s_head * 2};
  const cuuint32_t box[3] = {64, AT_KEYS, 1};
  return attn_map(m, dtype, rows > 0 ? p : any, 3, dims, st, box) == CUDA_SUCCESS;
}

// A cache [sequences][heads][rows][hd] in boxes of 64 elements x `box_rows` rows.
inline bool attn_cache_map(CUtensorMap* m, int dtype, const void* p, int hd, int rows, int KH, int B, long long s_row, long long s_head,
                           long long s_seq, int box_rows) {
  const cuuint64_t dims[4] = {(cuuint64_t)hd, (cuuint64_t)rows, (cuuint64_t)KH, (cuuint64_t)B};
  const cuuint64_t st[3] = {(cuuint64_t)s_row * 2, (cuuint64_t)s_head * 2, (cuuint64_t)s_seq * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1};
  return attn_map(m, dtype, p, 4, dims, st, box) == CUDA_SUCCESS;
}

// Launch with programmatic stream serialization: the kernel may start while
// its predecessor in the stream runs, and waits for it (pdl_wait) before it
// reads what that wrote.
template <typename K, typename... A>
inline cudaError_t launch_pdl(K kernel, dim3 grid, int block, size_t smem, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

inline int attn_sms() {   // SMs of the current device
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!sms[dev] && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) sms[dev] = 148;
  return sms[dev];
}

template <typename T, int HD, bool SHARED>
inline cudaError_t launch_attn_tc(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const AttnTcArgs& a, int grid,
                                  cudaStream_t s) {
  const int smem = AttnTcShape<HD>::SMEM;
  static std::atomic<unsigned long long> set{0};   // devices whose limit is raised
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !(set.load() >> dev & 1))) {
    e = cudaFuncSetAttribute(attn_tc_kernel<T, HD, SHARED>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess && dev < 64) set |= 1ull << dev;
  }
  if (e != cudaSuccess) return e;
  return launch_pdl(attn_tc_kernel<T, HD, SHARED>, dim3(grid), AT_THREADS, smem, s, q, k, v, a);
}

DevStatus* attn_status();   // the operators' device error record on the current device, or null (tg_attn_prompt.cu)

}  // namespace tg
