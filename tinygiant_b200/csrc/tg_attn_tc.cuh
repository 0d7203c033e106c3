// tg_attn_tc.cuh — the tensor-core attention kernel of the prompt and shared-
// prefix operators (tcgen05.mma kind::f16, accumulators in tensor memory).
//
// Mathematics.  For a query row and its keys K, with s_j = q . k_j in fp32 and
// c = scale log2(e), one pass over the keys in blocks of 128 keeps a reference
// m, a sum l and an accumulator o:
//   p_j = 2^(c s_j - c m),  l += p_j,  o += p_j v_j;   result o / l.
// m starts as the first block's maximum.  It moves (with l and o scaled by
// 2^(c m_old - c m_new)) only when a block's maximum exceeds it by more than
// 2^8 (fp16: 2^5) in the exponent's base: results do not depend on the
// reference, and o is then rarely touched.  p_j is rounded to the inputs' type
// for the second product, as tcgen05 wants both operands of one type; its error
// there is that of rounding v once more (unit roundoff 2^-8 or 2^-11 of the
// weighted mean of |v|), the order of the output's own rounding; fp16's range
// is used whole for that (AttnRange).  l sums the unrounded p_j.
//
// Work unit: one key head, two tiles of 128 query rows.  A tile's rows are
// (token, query head of the group) pairs, token-major, so a group of G heads
// fills a tile with 128 / G tokens: K and V tiles are used by the whole group,
// short sequences fill tiles, and the masked corner of the causal diagonal is
// a few tokens wide.  Its keys are nb blocks from key ks on.
//
// Warps: 0-3 and 4-7 the softmax of tile 0 and 1 (a thread per row), 8 the TMA
// loads, 9 the S products, 10 the P V, 11 the values that not all rows see.
// Tensor memory (512 columns): O of both tiles, the 16-bit P of both, and S, one
// buffer of 128 columns for both tiles at head_dim 128, one for each at 64.  A
// softmax warp takes its S into registers at once and frees the buffer, so the
// next S is computed while it works on its exponentials.  S and P V are issued
// by a thread each: what one has to do between two products would be idle time
// of the tensor cores (8,192 tokens: 549 us with one thread, 461 with two).
// Persistent CTAs, one per SM; units come from an atomic counter, longest
// first.  Every wait is bounded; a role that gives up records the error and the
// others stop waiting.
//
// What bounds it.  A block of 128 keys for both tiles takes the tensor cores
// 2,048 clocks at head_dim 128 and the exponentials 1,792 of the special
// function unit; a softmax warp needs about 3,100 for its block (load 430,
// maximum 350, exponentials and P 1,600, waits).  8,192 tokens, 32 / 4 heads of
// 128, bf16: 427 us, 1.29 PFLOP/s, 0.78 of measured (in a long loop, under the
// power cap, 489 to 501, 0.79 to 0.81 of the sustained rate); fp16 445 (see
// AttnRange); 4,096 at head_dim 64: 116 us.
#pragma once
#include <cuda.h>

#include <atomic>
#include <type_traits>

#include "tg_attn.h"
#include "tg_attn_split.h"
#include "tg_ptx.cuh"

namespace tg {

constexpr int AT_SOFT = 8;         // softmax warps; then one each for loads, S, P V and edges
constexpr int AT_THREADS = 384;
constexpr int AT_NPOS = 0x3fffffff;
constexpr int AT_UNITS = 4;        // units announced ahead
// A unit's noted blocks of values that not all rows see.  A prompt's unit has no
// more (2 tiles of 128 tokens, both ends); a prefix's may, as its sequences'
// windows begin wherever their lengths put them: then all are looked through.
constexpr int AT_EDGES = 8;

// One piece of work of every key head.
struct __align__(16) AttnEntry {
  int q0, ntok;   // first query row (token) and tokens, at most 2 * (128 / G)
  int p0;         // position of the first token among its sequence's keys
  int k0, nk;     // the sequence's first key row and its keys
  int ks, nb;     // this piece's first key and blocks of keys
  int el, eh;     // the keys [el, eh) are those that all rows see
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
  e.ks = lo;
  e.el = window > 0 ? max(0, hi - window) : 0;
  e.eh = e.p0 + 1;
  e.nb = hi > lo ? (hi - lo + AT_KEYS - 1) / AT_KEYS : 0;
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
  float2* pml;                // their (c m - OFF, l) [slot * KH + kh][2 * 128]
  const float* sinks;
  const int* lens;            // shared: own keys of each sequence
  long long so[2];
  const void* v;              // the values, and their strides of rows and heads
  long long sv[2];
  int G, KH, hd, tpt, window;
  int total_k;                // rows of k and v
  int P, B, nsp, max_len;     // shared: prefix keys, sequences, pieces per unit, bound of lens
  int wide;                   // outputs in 32-byte pieces: head_dim a multiple of 16, rows 32-byte aligned
  int beside;                 // shared: launched beside a kernel that it does not wait for
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
__device__ __forceinline__ void at_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : AT_R4(r, 0), AT_R4(r, 4), AT_R4(r, 8), AT_R4(r, 12)
               : "r"(taddr));
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

// 32 aligned bytes in one store: a warp's rows are far apart, and each store
// takes the load/store unit a cycle for every row.
__device__ __forceinline__ void at_store8(void* p, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), AT_W4(r, 0), AT_W4(r, 4) : "memory");
}
__device__ __forceinline__ float at_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Maxima that are NaN if an operand is.
__device__ __forceinline__ float at_max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float at_max2(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
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

// 2^x of a pair on the FMA units, x >= -126 (less, and NaN, counts as that; a
// row with a score of NaN or +inf becomes NaN by its other keys, see cm): x = n + f
// with f in [-1/2, 1/2], 2^f by the degree-4 polynomial of least relative
// error there (2.6e-6, fitted by reweighted least squares), n added to the
// exponent.
__device__ __forceinline__ float2 at_exp2_poly(float2 x) {
  const float2 magic = make_float2(12582912.f, 12582912.f), minus = make_float2(-12582912.f, -12582912.f);   // 1.5 2^23
  auto two = [](float v) { return make_float2(v, v); };
  x.x = fmaxf(x.x, -126.f);
  x.y = fmaxf(x.y, -126.f);
  const float2 t = at_add2(x, magic);
  const float2 n = at_add2(t, minus);
  const float2 f = at_fma2(n, two(-1.f), x);
  float2 p = at_fma2(two(0.009570101276f), f, two(0.05591785908f));
  p = at_fma2(p, f, two(0.2402474433f));
  p = at_fma2(p, f, two(0.6931217909f));
  p = at_fma2(p, f, two(0.9999992847f));
  p.x = __int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23));
  p.y = __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23));
  return p;
}

template <int HD>
struct AttnTcShape {
  static constexpr int TILE = 128 * HD * 2;               // bytes of a Q tile, a K or a V block
  // One pair of exponentials in POLY_OF goes to the FMA units: the special
  // function unit gives 4 values a clock to each quarter of the SM, as long for
  // a block's 128 x 128 as the tensor cores take for both its products (none:
  // 445 us at 8,192 tokens, 1 in 8 431, 1 in 4 440; at head_dim 64, where the
  // products are half as long, 117, 106 and 107 us at 4,096).
  static constexpr int POLY_OF = HD == 128 ? 8 : 4;
  static constexpr int NQ = HD == 128 ? 1 : 2;            // units whose Q is there or on its way
  static constexpr int STAGES = HD == 128 ? 5 : 8;        // K and V blocks in flight, in turn
  // Their barriers: an even number, so that each is K's or V's alone and its
  // waiter sees every phase (a wait by parity passes if the barrier is a whole
  // phase behind).
  static constexpr int BARS = STAGES % 2 ? 2 * STAGES : STAGES;
  static constexpr int SMEM = (2 * NQ + STAGES) * TILE + 1024;
};

struct AttnTcShared {
  uint64_t q_full[2], q_empty[2], kv_full[10], kv_empty[10], s_full[2], s_loaded[2], p_full[2], p_empty[2], unit_full[AT_UNITS],
      unit_empty[AT_UNITS], edge[10], drain[2];
  AttnEntry unit[AT_UNITS];
  int unit_kh[AT_UNITS];      // -1: no more work
  // Edge blocks with values that are not finite: 16 times the unit's number
  // and how many (AT_EDGES + 1: more than are noted); each one's block and its
  // keys, a bit each.
  int bad[AT_UNITS], bad_block[AT_UNITS][AT_EDGES];
  uint32_t bad_keys[AT_UNITS][AT_EDGES][4];
  uint32_t tmem;
  int abort;
  // Copies of the load warp, for the end of a CTA that gave up: blocks and Q
  // loads so far, and of each K / V barrier's last block whether it went
  // through the edge barrier (is) and that barrier's next phase (par).
  int issued, q_issued;
  uint32_t edge_is, edge_par;
};

// Waits for phase `parity`; gives up after about a second, or once another
// role has.  A warp comes here converged, so a poll is one instruction for all
// its lanes and they leave together (a vote on it costs 1 % at 8,192 tokens).
__device__ __forceinline__ bool at_wait(uint64_t* bar, uint32_t parity, const volatile int* abort) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint32_t t0 = clock();   // 32 bits: a second is half of their range
  while (!mbar_try_wait(bar, parity))
    if (*abort || (uint32_t)clock() - t0 > 1u << 31) return false;
  return true;
}

// The same for a warp that has time: it polls a few times in a microsecond, so
// that its quarter of the SM's softmax keeps the issue slots.
__device__ __forceinline__ bool at_wait_idle(uint64_t* bar, uint32_t parity, const volatile int* abort) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint32_t t0 = clock();
  while (!mbar_try_wait(bar, parity)) {
    if (*abort || (uint32_t)clock() - t0 > 1u << 31) return false;
    __nanosleep(200);
  }
  return true;
}

// A place in a ring and its phase, counted on without divisions.
struct AttnRing {
  uint32_t s, ph;
  __device__ __forceinline__ void add(uint32_t k, uint32_t n) {
    s += k;
    if (s >= n) s -= n, ph ^= 1;
  }
};

// Adds to a row's O in tensor memory the values that are not finite of the
// noted keys in [lo, hi) (numbers from the unit's first key on, whose values
// start at v).  All lanes of the warp call it.
template <typename T, int HD>
__device__ __noinline__ void attn_add_odd(uint32_t to, const char* v, long long stride, int hd, int blocks, const int* block,
                                          const uint32_t (*keys)[4], int lo, int hi) {
  for (int i = 0; i < HD / 16; i++) {
    uint32_t o[16];
    at_ld16(to + 16 * i, o);
    at_wait_ld();
    for (int r = 0; r < blocks; r++)
      for (int k = 0; k < AT_KEYS; k++) {
        const int key = block[r] * AT_KEYS + k;
        if (!(keys[r][k / 32] >> (k % 32) & 1) || key < lo || key >= hi) continue;
        const T* x = (const T*)v + key * stride + 16 * i;
#pragma unroll
        for (int q = 0; q < 16; q++) {
          const float y = 16 * i + q < hd ? to_f32(x[q]) : 0.f;
          if (!isfinite(y)) o[q] = __float_as_uint(__uint_as_float(o[q]) + y);
        }
      }
    __syncwarp();
    at_st16(to + 16 * i, o);
    at_wait_st();
  }
}

// Whether a pair of 16-bit values has one that is not finite, a bit for each:
// its exponent bits are all ones, so 1 added to the exponent reaches the sign.
template <typename T>
__device__ __forceinline__ uint32_t at_odd(uint32_t x) {
  constexpr uint32_t EXP = std::is_same<T, __nv_bfloat16>::value ? 0x7f807f80u : 0x7c007c00u;
  constexpr uint32_t ONE = std::is_same<T, __nv_bfloat16>::value ? 0x00800080u : 0x04000400u;
  return ((x & EXP) + ONE) & 0x80008000u;
}
template <typename T>
__device__ __forceinline__ uint32_t at_odd4(uint4 x) {
  return at_odd<T>(x.x) | at_odd<T>(x.y) | at_odd<T>(x.z) | at_odd<T>(x.w);
}

// The same for more blocks than are noted: the unit's first n keys, which not
// all rows see, are read again, a lane per key.
template <typename T, int HD>
__device__ __noinline__ void attn_add_odd_front(uint32_t to, const char* v, long long stride, int hd, int n, int lo, int hi) {
  const int lane = threadIdx.x & 31;
  for (int k0 = 0; k0 < n; k0 += 32) {
    uint32_t odd = 0;
    if (k0 + lane < n) {
      const uint4* x = (const uint4*)((const T*)v + (k0 + lane) * stride);
      for (int i = 0; i < hd / 8; i++) odd |= at_odd4<T>(x[i]);
    }
    for (uint32_t keys = __ballot_sync(~0u, odd != 0); keys; keys &= keys - 1) {
      const int key = k0 + __ffs(keys) - 1;
      const T* x = (const T*)v + key * stride;
      for (int i = 0; i < HD / 16; i++) {
        uint32_t o[16];
        at_ld16(to + 16 * i, o);
        at_wait_ld();
#pragma unroll
        for (int q = 0; q < 16; q++) {
          const float y = key >= lo && key < hi && 16 * i + q < hd ? to_f32(x[16 * i + q]) : 0.f;
          if (!isfinite(y)) o[q] = __float_as_uint(__uint_as_float(o[q]) + y);
        }
        __syncwarp();
        at_st16(to + 16 * i, o);
        at_wait_st();
      }
    }
  }
}

template <typename T, int HD, bool SHARED>
__global__ void __launch_bounds__(AT_THREADS, 1) attn_tc_kernel(const __grid_constant__ CUtensorMap qmap,
                                                                const __grid_constant__ CUtensorMap kmap,
                                                                const __grid_constant__ CUtensorMap vmap, const AttnTcArgs a) {
  using S = AttnTcShape<HD>;
  constexpr int NST = S::STAGES, NBAR = S::BARS, TILE = S::TILE, NQ = S::NQ, W0 = AT_SOFT;
  // tensor memory: S buffers of 128 columns, P of 64 for each tile, O of HD for each
  constexpr int NS = HD == 128 ? 1 : 2, TM_P = NS * AT_KEYS, TM_O = TM_P + AT_KEYS;
  extern __shared__ uint8_t dsm[];
  __shared__ AttnTcShared sh;
  const int tid = threadIdx.x, wid = tid >> 5, lane = tid & 31;
  uint8_t* qs = dsm + ((1024u - (smem_u32(dsm) & 1023u)) & 1023u);
  uint8_t* kvs = qs + 2 * NQ * TILE;
  volatile int* abort = &sh.abort;

  if (wid == W0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (tid == W0 * 32 + 32) {
    for (int i = 0; i < NBAR; i++) {
      mbar_init(&sh.kv_full[i], 1);
      mbar_init(&sh.kv_empty[i], 1);
      mbar_init(&sh.edge[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&sh.q_full[i], 1);
      mbar_init(&sh.q_empty[i], 1);
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.s_loaded[i], W0 / 2);
      mbar_init(&sh.p_full[i], W0 / 2);
      mbar_init(&sh.p_empty[i], 1);
    }
    for (int i = 0; i < AT_UNITS; i++) {
      mbar_init(&sh.unit_full[i], 1);
      mbar_init(&sh.unit_empty[i], W0 + 3);
    }
    for (int i = 0; i < AT_UNITS; i++) sh.bad[i] = -1;
    mbar_init(&sh.drain[0], 1);
    mbar_init(&sh.drain[1], 1);
    sh.abort = 0;
    fence_mbar_init();
  }
  at_fence_before();
  __syncthreads();
  at_fence_after();
  const uint32_t tmem = sh.tmem;
  // The plan comes from the preceding kernel; a prefix beside the own keys'
  // kernel depends on nothing that runs.
  if (!SHARED || !a.beside) {
    pdl_wait();
    pdl_trigger();
  }
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
    const int b0 = (int)((long long)nblk * sp / a.nsp), b1 = (int)((long long)nblk * (sp + 1) / a.nsp);
    e.ks = b0 * AT_KEYS;
    e.nb = b1 - b0;
    e.slot = i;
    e.eh = AT_NPOS;       // behind the prefix there are zeros
    if (a.window > 0) {   // without the keys that no row of the unit sees
      int lo = a.P, most = 0;
      for (int r = lane; r < e.ntok; r += 32) {
        const int first = max(0, a.P + min(max(a.lens[e.q0 + r], 0), a.max_len) - a.window);
        lo = min(lo, first), most = max(most, first);
      }
      lo = __reduce_min_sync(~0u, lo);
      e.el = __reduce_max_sync(~0u, most);
      const int skip = lo >= a.P ? e.nb : min(e.nb, max(0, (lo - e.ks) / AT_KEYS));
      e.ks += skip * AT_KEYS;
      e.nb -= skip;
    }
    return e;
  };
  // The next unit, as the load warp announced it; false at the end.
  int un = 0;
  // Whether some row sees the block from key `row` on only in part, or it
  // reaches behind the sequence's keys into others'.
  auto on_edge = [&](const AttnEntry& e, int row) {
    return row < e.el || row + AT_KEYS > e.eh || (e.nk - row < AT_KEYS && e.k0 + e.nk < a.total_k);
  };
  auto next_unit = [&](AttnEntry& e, int& kh) -> bool {
    const int i = un % AT_UNITS;
    if (!at_wait(&sh.unit_full[i], (un / AT_UNITS) & 1, abort)) {
      fail(300, un);
      return false;
    }
    e = sh.unit[i];
    kh = sh.unit_kh[i];
    return kh >= 0;
  };

  // 168 registers a thread at launch (384 x 168 = 64,512): 216 for the eight
  // softmax warps and 72 for the four others make the same sum.
  if (wid >= W0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  }
  if (wid == W0) {
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
    int issued = 0, qn = 0;   // blocks and Q loads so far
    uint32_t edge_is = 0, edge_par = 0;
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
      const int us = it % AT_UNITS;
      if (it >= AT_UNITS && !at_wait(&sh.unit_empty[us], (it / AT_UNITS - 1) & 1, abort)) {
        if (lane == 0) fail(301, it);
        break;
      }
      if (lane == 0) {
        sh.unit[us] = e;
        sh.unit_kh[us] = kh;
        mbar_arrive(&sh.unit_full[us]);
      }
      if (kh < 0) break;
      if (e.nb <= 0) continue;
      const int ntile = e.ntok > a.tpt ? 2 : 1;
      const int qb = qn % NQ;
      if (qn >= NQ && !at_wait(&sh.q_empty[qb], (qn / NQ - 1) & 1, abort)) {
        if (lane == 0) fail(302, it);
        break;
      }
      qn++;
      if (lane == 0) {
        mbar_arrive_expect_tx(&sh.q_full[qb], ntile * (HD / 64) * a.G * a.tpt * 128);
        for (int t = 0; t < ntile; t++)
          for (int c = 0; c < HD / 64; c++)
            tma_load_3d(qs + (2 * qb + t) * TILE + c * 16384, &qmap, 64 * c, kh * a.G, e.q0 + t * a.tpt, &sh.q_full[qb]);
      }
      for (int i = 0; i < 2 * e.nb; i++) {
        const int s = issued % NST, row = e.ks + (i >> 1) * AT_KEYS;
        const bool v = i & 1;
        const int old = issued - NST;   // the block that was there before
        if (old >= 0 && !at_wait(&sh.kv_empty[old % NBAR], (old / NBAR) & 1, abort)) {
          if (lane == 0) fail(303, it);
          ok = false;
          break;
        }
        uint8_t* dst = kvs + s * TILE;
        // a V block that not all rows see whole goes through the edge warp
        const int b = issued % NBAR;
        const bool edge = v && on_edge(e, row);
        edge_is = edge_is & ~(1u << b) | (uint32_t)edge << b;
        edge_par ^= (uint32_t)edge << b;
        uint64_t* bar = edge ? &sh.edge[b] : &sh.kv_full[b];
        if (lane == 0) {
          mbar_arrive_expect_tx(bar, TILE);
          for (int c = 0; c < HD / 64; c++)
            tma_load_3d(dst + c * 16384, v ? &vmap : &kmap, 64 * c, e.k0 + row, kh, bar);
        }
        issued++;
      }
    }
    if (lane == 0) sh.issued = issued, sh.q_issued = qn, sh.edge_is = edge_is, sh.edge_par = edge_par;
  } else if (wid == W0 + 1 || wid == W0 + 2) {
    // ---- products, each kind issued by a thread of its own: what one has to
    // do between two products does not keep the tensor cores from the other's
    if (lane == 0) {
      bool ok = true, issued = false;
      auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
        if (!at_wait(bar, parity & 1, abort)) {
          fail(site, un);
          ok = false;
        }
        return ok;
      };
      AttnRing unit{0, 0}, qr{0, 0}, kv{wid == W0 + 1 ? 0u : 1u, 0};   // kv: the barrier; K and V take turns
      // Parities of the tiles' S (or P), a bit each (an indexed array would
      // live in local memory).
      uint32_t bits = 0, last = 0;
      for (;; un++) {
        if (!wait(&sh.unit_full[unit.s], unit.ph, 300)) break;
        const int nb = sh.unit[unit.s].nb, ntile = sh.unit[unit.s].ntok > a.tpt ? 2 : 1;
        if (sh.unit_kh[unit.s] < 0) break;
        mbar_arrive(&sh.unit_empty[unit.s]);
        unit.add(1, AT_UNITS);
        if (nb <= 0) continue;
        issued = true;
        if (wid == W0 + 1) {
          constexpr uint32_t idesc = idesc_f16<T>(AT_KEYS, false);
          const uint64_t dq = desc_kmajor(smem_u32(qs) + qr.s * 2 * TILE), dk = desc_kmajor(smem_u32(kvs));
          if (!wait(&sh.q_full[qr.s], qr.ph, 310)) break;
          for (int j = 0; j < nb && ok; j++) {
            if (!wait(&sh.kv_full[kv.s], kv.ph, 311)) break;
            const uint64_t bk = dk + (kv.s < NST ? kv.s : kv.s - NST) * (TILE / 16);
            for (uint32_t t = 0; t < ntile; t++) {
              // The buffer is free once the softmax has loaded what was in it
              // (a barrier's phase before its first counts as complete).
              const uint32_t was = NS == 1 ? last : t;
              if (!wait(&sh.s_loaded[was], (bits >> was) + 1, 312)) break;
              at_fence_after();
              const uint64_t aq = dq + t * (TILE / 16);
#pragma unroll
              for (int k = 0; k < HD / 16; k++) {   // S_t = Q_t K^T
                const uint32_t o = ((k / 4) * 16384 + (k % 4) * 32) / 16;
                at_mma_ss(tmem + (NS == 1 ? 0 : t * AT_KEYS), aq + o, bk + o, idesc, k > 0);
              }
              at_commit(&sh.s_full[t]);
              bits ^= 1u << t;
              last = t;
            }
            at_commit(&sh.kv_empty[kv.s]);
            kv.add(2, NBAR);
          }
          if (!ok) break;
          at_commit(&sh.q_empty[qr.s]);
          qr.add(1, NQ);
        } else {
          constexpr uint32_t idesc = idesc_f16<T>(HD, true);
          const uint64_t dv = desc_mnmajor(smem_u32(kvs));
          for (int j = 0; j < nb && ok; j++) {
            if (!wait(&sh.kv_full[kv.s], kv.ph, 313)) break;
            const uint64_t bv = dv + (kv.s < NST ? kv.s : kv.s - NST) * (TILE / 16);
            for (uint32_t t = 0; t < ntile; t++) {
              const uint32_t d = tmem + TM_O + t * HD, pa = tmem + TM_P + t * (AT_KEYS / 2), par = bits >> t;
              if (!wait(&sh.p_full[t], par, 315)) break;
              at_fence_after();
#pragma unroll
              for (int k = 0; k < AT_KEYS / 16; k++)   // O_t += P_t V
                at_mma_ts(d, pa + k * 8, bv + k * (2048 / 16), idesc, j > 0 || k > 0);
              at_commit(&sh.p_empty[t]);
              bits ^= 1u << t;
            }
            at_commit(&sh.kv_empty[kv.s]);
            kv.add(2, NBAR);
          }
          if (!ok) break;
        }
      }
      if (issued) {   // no product or commit of this CTA may still be in flight at its end
        at_commit(&sh.drain[wid - W0 - 1]);
        mbar_wait(&sh.drain[wid - W0 - 1], 0);
      }
    }
    __syncwarp();
  } else if (wid == W0 + 3) {
    // ---- edges: p = 0 does not silence an infinity or NaN among the values
    // that a row must not see.  Rows behind the sequence's end are zeroed, and
    // such values among the sequence's own rows that not all rows see; those
    // are noted, and the softmax adds them at the end to the rows that do.
    AttnRing kv{1, 0}, unit{0, 0};
    uint32_t bits = 0;   // parities of the edge barriers' next phases
    bool ok = true;
    for (; ok; un++) {
      if (!at_wait_idle(&sh.unit_full[unit.s], unit.ph, abort)) {
        if (lane == 0) fail(330, un);
        break;
      }
      const AttnEntry e = sh.unit[unit.s];
      if (sh.unit_kh[unit.s] < 0) break;
      int nbad = 0;
      for (int j = 0; j < e.nb; j++, kv.add(2, NBAR)) {
        const int row = e.ks + j * AT_KEYS;
        if (!on_edge(e, row)) continue;
        if (!at_wait_idle(&sh.edge[kv.s], bits >> kv.s & 1, abort)) {
          if (lane == 0) fail(331, un);
          ok = false;
          break;
        }
        bits ^= 1u << kv.s;
        uint8_t* dst = kvs + (kv.s < NST ? kv.s : kv.s - NST) * TILE;
        const int end = e.k0 + e.nk < a.total_k ? min(AT_KEYS, max(0, e.nk - row)) : AT_KEYS;
        const int r1 = min(end, max(0, e.el - row)), r2 = min(end, max(r1, e.eh - row));   // not all see [0, r1) and [r2, end)
        uint32_t any = 0;
        for (int c = 0; c < HD / 64; c++) {
          uint4* p = reinterpret_cast<uint4*>(dst + c * 16384);   // 8 words of 16 bytes a row
          for (int o = end * 8 + lane; o < AT_KEYS * 8; o += 32) p[o] = make_uint4(0, 0, 0, 0);
#pragma unroll 4
          for (int o = lane; o < r1 * 8; o += 32) any |= at_odd4<T>(p[o]);
#pragma unroll 4
          for (int o = r2 * 8 + lane; o < end * 8; o += 32) any |= at_odd4<T>(p[o]);
        }
        if (__any_sync(~0u, any != 0)) {
          for (int w = 0; w < 4; w++) {   // a lane per row
            const int r = w * 32 + lane;
            uint32_t x = 0;
            if (r < r1 || (r >= r2 && r < end))
              for (int i = 0; i < HD / 2; i++) {
                uint32_t* p = reinterpret_cast<uint32_t*>(dst + i / 32 * 16384) + r * 32 + i % 32;
                const uint32_t m = at_odd<T>(*p);
                x |= m;
                if (m) *p &= ~((m >> 31) * 0xffff0000u | (m >> 15 & 1) * 0xffffu);
              }
            const uint32_t rows = __ballot_sync(~0u, x != 0);
            if (lane == 0 && nbad < AT_EDGES) sh.bad_keys[unit.s][nbad][w] = rows;
          }
          if (lane == 0) {
            if (nbad < AT_EDGES) sh.bad_block[unit.s][nbad] = j;
            sh.bad[unit.s] = un * 16 + min(nbad, AT_EDGES) + 1;
          }
          nbad++;
        }
        if (end < AT_KEYS || __any_sync(~0u, any != 0)) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // written to
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.kv_full[kv.s]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.unit_empty[unit.s]);
      unit.add(1, AT_UNITS);
    }
  } else if (wid < W0) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ---- softmax of tile t, a thread per row.  What a block does not need is
    // read or computed again at the unit's end: a spilled register costs more,
    // since next to 200 KB of shared memory there is hardly an L1 for it.
    const int t = wid >> 2;
    // tensor memory of this warp's 32 lanes: S, P, O of its tile
    const uint32_t lanes = tmem + ((uint32_t)(wid & 3) << 21);
    const uint32_t ts = lanes + (NS == 1 ? 0 : t * AT_KEYS), tp = lanes + TM_P + t * (AT_KEYS / 2), to = lanes + TM_O + t * HD;
    const float c = a.c;
    const int tok = (tid & 127) / a.G, g = (tid & 127) - tok * a.G;   // the row's token and query head
    uint32_t par = 0;   // blocks so far, modulo 2
    for (;; un++) {
      const volatile AttnEntry* e = &sh.unit[un % AT_UNITS];   // handed back at the unit's end
      {
        AttnEntry first;
        int kh;
        if (!next_unit(first, kh)) break;
      }
      const int nb = e->nb;
      float m = -INFINITY, l = 0.f, sink = -INFINITY;
      int lo = 0, hi = 0;                            // the row's keys
      int lo0 = 0, hi1 = 0, lo1 = 0, hi0 = 0;        // over the warp's rows: keys that some see, keys that all see
      bool valid = false, ok = true;
      const bool mine = t * a.tpt < e->ntok;         // the tile has rows
      if (mine) {
        const int tt = t * a.tpt + tok;
        valid = tok < a.tpt && tt < e->ntok;
        if (SHARED) {
          hi = a.P;
          if (a.window > 0 && valid) lo = max(0, a.P + min(max(a.lens[e->q0 + tt], 0), a.max_len) - a.window);
        } else {
          hi = e->p0 + tt + 1;
          if (a.window > 0) lo = max(0, hi - a.window);
          if (a.sinks && valid && e->slot < 0) sink = a.sinks[sh.unit_kh[un % AT_UNITS] * a.G + g];   // used at the end
        }
        lo0 = __reduce_min_sync(~0u, valid ? lo : AT_NPOS), hi1 = __reduce_max_sync(~0u, valid ? hi : 0);
        lo1 = __reduce_max_sync(~0u, valid ? lo : 0), hi0 = __reduce_min_sync(~0u, valid ? hi : AT_NPOS);
      }
      for (int j = 0; mine && j < nb; j++) {
        if (!at_wait(&sh.s_full[t], par & 1, abort)) {
          fail(320 + t, un);
          ok = false;
          break;
        }
        at_fence_after();
        uint32_t r[AT_KEYS];
#pragma unroll
        for (int i = 0; i < 4; i++) at_ld32(ts + 32 * i, r + 32 * i);
        at_wait_ld();
        at_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.s_loaded[t]);
        float* s = reinterpret_cast<float*>(r);
        // Masked blocks go by chunks of 32 keys: those that no row of the warp
        // sees (dead) need no exponential, and only those at an edge a test
        // for each key.
        const int base = e->ks + j * AT_KEYS;
        unsigned dead = 0;
        const bool clean = base >= lo1 && base + AT_KEYS <= hi0;
        float mx[4] = {m, m, m, m};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int cb = base + 32 * i;
          if (!clean) {
            if (cb >= hi1 || cb + 32 <= lo0) {
              dead |= 1u << i;
              continue;
            }
            if (cb < lo1 || cb + 32 > hi0) {
              const int l0 = lo - cb, h0 = hi - cb;
              unsigned see = h0 >= 32 ? ~0u : h0 <= 0 ? 0u : (1u << h0) - 1;
              see &= l0 <= 0 ? ~0u : l0 >= 32 ? 0u : ~0u << l0;
#pragma unroll
              for (int q = 0; q < 32; q++) s[32 * i + q] = see & (1u << q) ? s[32 * i + q] : -INFINITY;
            }
          }
#pragma unroll
          for (int q = 0; q < 32; q += 8)
#pragma unroll
            for (int z = 0; z < 4; z++) mx[z] = at_max3(mx[z], s[32 * i + q + z], s[32 * i + q + z + 4]);
        }
        const float mn = at_max3(mx[0], mx[1], at_max2(mx[2], mx[3]));
        // P V of the block before: its P may be overwritten, its O scaled (a
        // barrier's phase before its first counts as complete)
        if (!at_wait(&sh.p_empty[t], (par & 1) ^ 1, abort)) {
          fail(324 + t, un);
          ok = false;
          break;
        }
        par ^= 1;
        at_fence_after();
        if (j == 0) {
          m = mn;
        } else {
          const float d = (mn - m) * c;
          const bool up = d > AttnRange<T>::LIFT;
          if (__any_sync(~0u, up)) {
            const float f = up ? at_exp2(-d) : 1.f;
            if (up) m = mn;
            l *= f;
#pragma unroll
            for (int i = 0; i < HD / 16; i++) {
              uint32_t o[16];
              at_ld16(to + 16 * i, o);
              at_wait_ld();
#pragma unroll
              for (int q = 0; q < 16; q++) o[q] = __float_as_uint(__uint_as_float(o[q]) * f);
              at_st16(to + 16 * i, o);
            }
          }
        }
        // Not finite: a score of NaN or +inf makes mn NaN or +inf, then cm and
        // with it every p of the special function unit NaN, as the softmax is.
        // While all scores are -inf, m is too: their p count as 0 (those of the
        // FMA units are 2^-126; a first larger score scales them, and l, by 0).
        const float cm = mn == -INFINITY ? 0.f : fmaf(m, -c, mn - mn + AttnRange<T>::OFF);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        auto scaled = [&](int i) {   // c s - c m + OFF of the pair i
          return at_fma2(make_float2(s[2 * i], s[2 * i + 1]), make_float2(c, c), make_float2(cm, cm));
        };
        if (clean) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            uint32_t p[16];
#pragma unroll
            for (int q = 0; q < 16; q++) {
              float2 x = scaled(16 * i + q);
              if (q % S::POLY_OF == S::POLY_OF - 1) {
                x = at_exp2_poly(x);
              } else {
                x.x = at_exp2(x.x);
                x.y = at_exp2(x.y);
              }
              sum[q & 1] = at_add2(sum[q & 1], x);
              p[q] = at_pack<T>(x.x, x.y);
            }
            at_st16(tp + 16 * i, p);
          }
        } else {   // -inf has to give 0 here
#pragma unroll
          for (int i = 0; i < 4; i++) {
            uint32_t p[16];
            if (dead >> i & 1) {
#pragma unroll
              for (int q = 0; q < 16; q++) p[q] = 0;
            } else {
#pragma unroll
              for (int q = 0; q < 16; q++) {
                float2 x = scaled(16 * i + q);
                x.x = at_exp2(x.x);
                x.y = at_exp2(x.y);
                sum[q & 1] = at_add2(sum[q & 1], x);
                p[q] = at_pack<T>(x.x, x.y);
              }
            }
            at_st16(tp + 16 * i, p);
          }
        }
        at_wait_st();
        at_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full[t]);
        sum[0] = at_add2(sum[0], sum[1]);
        l += sum[0].x + sum[0].y;
      }
      if (!ok) break;
      if (mine) {
        if (m == -INFINITY) l *= 0.f;   // no key, or none above -inf; NaN stays
        const int us = un % AT_UNITS, kh = *(volatile int*)&sh.unit_kh[us], slot = e->slot;
        const bool part = SHARED || slot >= 0;
        float inv = 1.f;
        char* at;   // this thread's outputs, or its part of the partial result
        if (part) {
          const size_t pr = ((size_t)slot * a.KH + kh) * (2 * AT_ROWS) + tid;
          if (valid) a.pml[pr] = make_float2(l == 0.f ? -INFINITY : c * m - AttnRange<T>::OFF, l);
          at = (char*)(a.po + pr * HD);
        } else {
          if (l != 0.f) l += at_exp2(fmaf(sink, LOG2E, AttnRange<T>::OFF - c * m));
          inv = l == 0.f ? 0.f : 1.f / l;
          at = (char*)((T*)a.out + (e->q0 + t * a.tpt + tok) * a.so[0] + (kh * a.G + g) * a.so[1]);
        }
        if (nb > 0) {
          if (!at_wait(&sh.p_empty[t], (par & 1) ^ 1, abort)) {   // the last P V: O is whole
            fail(322 + t, un);
            break;
          }
          at_fence_after();
          const int noted = *(volatile int*)&sh.bad[us], bad = noted >> 4 == un ? noted & 15 : 0;
          if (bad) {
            const char* v = (const char*)((const T*)a.v + (e->k0 + e->ks) * a.sv[0] + kh * a.sv[1]);
            const int from = valid ? lo - e->ks : 1, end = valid ? hi - e->ks : 0;
            if (bad <= AT_EDGES)
              attn_add_odd<T, HD>(to, v, a.sv[0], a.hd, bad, sh.bad_block[us], sh.bad_keys[us], from, end);
            else if (SHARED)
              attn_add_odd_front<T, HD>(to, v, a.sv[0], a.hd, min(min(e->el, e->nk) - e->ks, nb * AT_KEYS), from, end);
          }
        }
#pragma unroll
        for (int i = 0; i < HD / 64; i++) {
          uint32_t o[64];
          if (nb > 0) {
            at_ld32(to + 64 * i, o);
            at_ld32(to + 64 * i + 32, o + 32);
            at_wait_ld();
          } else {
#pragma unroll
            for (int q = 0; q < 64; q++) o[q] = 0;
          }
          if (!valid || (part && nb <= 0)) continue;   // a partial result without keys, l = 0, is not read
          if (part) {
#pragma unroll
            for (int q = 0; q < 64; q += 8) at_store8(at + 256 * i + 4 * q, o + q);
          } else {
            uint32_t y[32];
#pragma unroll
            for (int z = 0; z < 32; z++) y[z] = at_pack<T>(__uint_as_float(o[2 * z]) * inv, __uint_as_float(o[2 * z + 1]) * inv);
            // 32 bytes at a time where they are whole and aligned (window 128: 51.2 us, 53.6 with 16)
            if (a.wide) {
#pragma unroll
              for (int q = 0; q < 4; q++)
                if (64 * i + 16 * q < a.hd) at_store8(at + 128 * i + 32 * q, y + 8 * q);
            } else {
#pragma unroll
              for (int q = 0; q < 8; q++)
                if (64 * i + 8 * q < a.hd) reinterpret_cast<uint4*>(at)[8 * i + q] = make_uint4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]);
            }
          }
        }
        at_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.unit_empty[un % AT_UNITS]);
    }
  }
  at_fence_before();
  __syncthreads();
  if (*abort && tid == W0 * 32) {   // some role gave up: no copy of this CTA may still be in flight at its end
    for (int i = max(0, sh.issued - NST); i < sh.issued; i++) {
      const int b = i % NBAR;
      if (sh.edge_is >> b & 1)
        mbar_wait(&sh.edge[b], (sh.edge_par >> b & 1) ^ 1);
      else
        mbar_wait(&sh.kv_full[b], (i / NBAR) & 1);
    }
    for (int i = max(0, sh.q_issued - NQ); i < sh.q_issued; i++) mbar_wait(&sh.q_full[i % NQ], (i / NQ) & 1);
  }
  __syncwarp();
  if (wid == W0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  if (SHARED && a.beside && blockIdx.x == gridDim.x - 1) pdl_wait();   // this grid ends after the one beside it
}

// ---------------------------------------------------------------------
// Joining partial results.  A row's pieces have (m_i, l_i) in pml, m_i = c m -
// OFF (the factor 2^OFF of their sums taken out), and their accumulators of HD
// values in po; row(i) is the place of piece i of n.
//   M = max(m_i, sink),  f_i = 2^(m_i - M),
//   o = sum f_i o_i / (sum f_i l_i + 2^(sink - M)).
// A warp per row: its lanes weigh 32 pieces at a time, then add them up eight
// at a time with HD / 32 dimensions each.  Pieces without a key (l = 0) have
// no accumulator.  Returns (M, 1 / the whole sum), 0 without keys.
template <typename F>
__device__ __forceinline__ float2 join_scale(int n, const float2* pml, float sink2, F row) {
  const int lane = threadIdx.x & 31;
  float M = -INFINITY, L = 0.f;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const float2 ml = i0 + lane < n ? pml[row(i0 + lane)] : make_float2(-INFINITY, 0.f);
    float m = ml.x;
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    m = fmaxf(M, m);
    float l = ml.y == 0.f ? 0.f : ml.y * at_exp2(ml.x - m);
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
    L = (L == 0.f ? 0.f : L * at_exp2(M - m)) + l;
    M = m;
  }
  if (L == 0.f) return make_float2(0.f, 0.f);
  const float m = fmaxf(M, sink2);
  return make_float2(m, 1.f / (L * at_exp2(M - m) + at_exp2(sink2 - m)));
}
template <typename T, int HD, typename F>
__device__ __forceinline__ void join_row(int n, const float2* pml, const float* po, float2 fin, F row, T* out, int hd) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  float o[E] = {};
  for (int i0 = 0; i0 < n; i0 += 32) {
    const long long r = i0 + lane < n ? (long long)row(i0 + lane) : 0;
    const float2 ml = i0 + lane < n ? pml[r] : make_float2(0.f, 0.f);
    const float f = ml.y == 0.f ? 0.f : at_exp2(ml.x - fin.x) * fin.y;
    unsigned todo = __ballot_sync(~0u, ml.y != 0.f);
    while (todo) {
      float fj[8], x[8][E];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int i = todo ? __ffs(todo) - 1 : -1;
        todo &= todo - 1;
        fj[j] = __shfl_sync(~0u, f, i & 31);
        const long long ri = __shfl_sync(~0u, r, i & 31);
        if (i < 0) fj[j] = 0.f;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float2 v = i < 0 ? make_float2(0.f, 0.f) : *reinterpret_cast<const float2*>(po + ri * HD + lane * E + e);
          x[j][e] = v.x, x[j][e + 1] = v.y;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; j++)
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = fmaf(x[j][e], fj[j], o[e]);
    }
  }
  if (lane * E < hd)
#pragma unroll
    for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(out + lane * E + e) = at_pack<T>(o[e], o[e + 1]);
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

// Raises a kernel's dynamic shared-memory limit on the current device, once, to
// the most that any launch of it asks for: a limit set for each launch could be
// lowered by another thread's before the launch.  set: the devices that have it.
template <typename K>
inline cudaError_t attn_smem(K kernel, int most, std::atomic<unsigned long long>& set) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !(set.load() >> dev & 1))) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e == cudaSuccess && dev < 64) set |= 1ull << dev;
  }
  return e;
}

template <typename T, int HD, bool SHARED>
inline cudaError_t launch_attn_tc(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const AttnTcArgs& a, int grid,
                                  cudaStream_t s) {
  const int smem = AttnTcShape<HD>::SMEM;
  static std::atomic<unsigned long long> set{0};
  const cudaError_t e = attn_smem(attn_tc_kernel<T, HD, SHARED>, smem, set);
  if (e != cudaSuccess) return e;
  return launch_pdl(attn_tc_kernel<T, HD, SHARED>, dim3(grid), AT_THREADS, smem, s, q, k, v, a);
}

DevStatus* attn_status();   // the operators' device error record on the current device, or null (tg_attn_prompt.cu)

}  // namespace tg
