// tg_attn_paged.cu — tg_attention_paged: the newest tokens of each sequence of
// a batch attend to the sequence's pages.
//
// Sequence b has len = lens[b] positions, its n newest the queries; query i is
// at e = len - n + i and attends to the keys j <= e, j > e - window (window 0:
// all).  With x_j = scale q . k_j:
//   o = sum e^(x_j) v_j / (sum e^(x_j) + e^sink).
// In pages of 8 bits k_j and v_j are e4m3 codes times the scales ks, vs of
// their block of 16 keys and key head.
//
// Bound by HBM: each key is read once for the rows (query, head of the group)
// of its key head, up to 16 at a time, so S^T = K Q^T and O^T += V^T P^T run on
// mma.m16n8k16 with keys and dimensions as the 16 and the rows as the 8 columns
// (the tensor-memory path has 128 rows to fill).  Codes are exact in fp16, so
// with them both products are fp16's: q in fp16 as it is, in bf16 times a power
// of two that takes its row's largest value to 2^14 (what falls below fp16's
// least normal value is 2^-28 of that).  Scales never meet the values: ks
// multiplies the scores, and log2(vs) is added to the exponent of the weights
// that meet v.  So there are two running references, one for the sum of the
// weights and one for the accumulators; each warp moves its own only when a
// score exceeds it by LIFT in base 2.
//
// Work: tiles of keys of one (sequence, key head, 16 rows), all in one row cut
// evenly among persistent CTAs; a CTA's tiles go to its eight warps in turn.
// Each warp loads its own tiles ahead with cp.async (pages end anywhere, rows
// that nobody may read come as zeros) and needs no barrier until a unit ends,
// where the warps' results join in shared memory, and those of units that lie in
// several CTAs in a second kernel.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/tinygiant.h"
#include "tg_attn_tc.cuh"
#include "tg_paged.h"

namespace tg {

constexpr int PG_WARPS = 8;
constexpr int PG_THREADS = PG_WARPS * 32;
constexpr int PG_JOIN_THREADS = 256;

struct PagedArgs {
  const void* q;
  const uint8_t *kp, *vp;
  const float *ks, *vs;
  const int *tables, *lens;
  const float* sinks;
  void* out;
  float* po;      // [2 CTA + slot][rows of a unit][HD]
  float4* pml;    // [2 CTA + slot][rows of a unit]: m, l, r
  int4* desc;     // [CTA]: sequence (-1: no unit begins here and ends later), head unit, last CTA
  long long sq[3], so[3];     // sequence, token, head
  long long skp[3], svp[3];   // page, head, row; bytes
  long long sks[3], svs[3];   // page, head, block
  long long st;
  int B, n, rows, rt, KH, G, hd, cols, n_pages, shift, max_len, window;
  int whole;      // units are not cut
  float c;        // scale log2(e)
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at));
  return r;
}
__device__ __forceinline__ uint2 lds8(uint32_t at) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(at));
  return r;
}
__device__ __forceinline__ uint32_t pg_movm(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <typename M>
__device__ __forceinline__ void pg_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (std::is_same<M, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two e4m3 codes, the lower byte first, as fp16.
__device__ __forceinline__ uint32_t pg_codes(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
  return h;
}

// T: type of q and out; CODES: pages of 8 bits; HD: 64 or 128; NT: groups of 8
// rows of a unit.
template <typename T, bool CODES, int HD, int NT>
struct PagedShape {
  using M = typename std::conditional<CODES, __half, T>::type;   // the products' type
  static constexpr int RB = HD * (CODES ? 1 : 2);                // bytes of a row in shared memory
  static constexpr int U = RB <= 128 ? 2 : 1;                    // 16-key parts of a tile
  static constexpr int KEYS = 16 * U;
  static constexpr int CH = RB / 16;                             // 16-byte words of a row
  static constexpr int KC = CH / 4;                              // words of a key row that a lane has
  static constexpr int STEPS = HD / 16;                          // 16-dimension steps of S, 16-dimension parts of O
  static constexpr int HALF = KEYS * RB;                         // K, or V, of a tile
  static constexpr int SLOT = 2 * HALF + 32;                     // and U scales each, and which parts are there
  static constexpr int D = RB == 64 ? 6 : 3;                     // tiles in a warp's ring
  static constexpr int RP = HD + 4;
  static constexpr int RED = PG_WARPS * 8 * RP * 4;
  static constexpr int SMEM = PG_WARPS * D * SLOT + RED;
  // Place of 16-byte word c of row r.  A quarter of a warp reads rows 2 i and
  // 2 i + 1, four words each (K), or words 2 q and 2 q + 1 of rows of one
  // parity (V; half a warp, words of 8 bytes, where rows are 64 bytes): all on
  // different banks.
  static __device__ __forceinline__ int at(int r, int c) {
    if (RB == 64) return (r >> 1) * 128 + ((((r & 1) << 2 | c) ^ ((r >> 1 & 3) << 1)) << 4);
    return r * RB + (c >> 3) * 128 + (((c & 7) ^ (r & 6) ^ ((r & 1) << 2)) << 4);
  }
};

// The tiles of a CTA as segments: consecutive tiles of one unit (sequence, key
// head, 16 rows).  x counts tiles, or units where those are not cut.
struct PagedWalk {
  long long x, x1;
  int b, hu, j, j1, len, lo, n, ahead;
  __device__ __forceinline__ int len_of(const PagedArgs& a, int s) const { return s < a.B ? min(max(a.lens[s], 0), a.max_len) : 0; }
  template <int KEYS>
  __device__ __forceinline__ void seq(const PagedArgs& a, int keys) {
    len = keys;
    lo = paged_first(len, a.n, a.window);
    n = paged_tiles(len, a.n, a.window, KEYS);
    ahead = len_of(a, b + 1);
  }
  // cut: from tile x0 on, `before` tiles of a head unit lie before sequence b0; else from unit x0 on
  template <int KEYS>
  __device__ __forceinline__ void start(const PagedArgs& a, int b0, long long before, long long x0, long long end) {
    const int HU = a.KH * a.rt;
    x = x0, x1 = end, b = b0;
    if (x >= x1) return;
    seq<KEYS>(a, len_of(a, b));
    if (a.whole) {
      hu = (int)(x0 - (long long)b0 * HU) - 1;
      x--;
      j = j1 = 0;
      next<KEYS>(a);
    } else {
      const long long r = x0 - before * HU;
      hu = (int)(r / n), j = (int)(r % n);
      j1 = (int)min((long long)n, j + x1 - x);
    }
  }
  __device__ __forceinline__ bool more() const { return x < x1; }
  template <int KEYS>
  __device__ __forceinline__ void next(const PagedArgs& a) {
    const int HU = a.KH * a.rt;
    if (a.whole) {
      do {   // a unit further, over those without keys
        if (++x >= x1) return;
        if (++hu == HU) hu = 0, b++, seq<KEYS>(a, ahead);
      } while (n == 0);
      j = 0, j1 = n;
      return;
    }
    x += j1 - j;
    if (x >= x1) return;
    j = 0;
    if (++hu == HU) {
      hu = 0;
      do b++, seq<KEYS>(a, ahead);
      while (n == 0);   // x < x1: there is another sequence with keys
    }
    j1 = (int)min((long long)n, x1 - x);
  }
};

// The CTA of n that tile x of `total` falls to: CTA i has [i total / n, (i + 1) total / n).
__device__ __forceinline__ int paged_cta(long long x, long long total, int n) { return (int)(((x + 1) * n - 1) / total); }

struct PagedShared {
  float4 ml[PG_WARPS][8];   // each warp's m, l, r of 8 rows
  long long sums[PG_WARPS], before;
  int b0;
};

template <typename T, bool CODES, int HD, int NT>
__global__ void __launch_bounds__(PG_THREADS, 1) paged_kernel(const PagedArgs a) {
  using S = PagedShape<T, CODES, HD, NT>;
  using M = typename S::M;
  constexpr int KEYS = S::KEYS;
  constexpr float OFF = AttnRange<M>::OFF, LIFT = AttnRange<M>::LIFT;
  extern __shared__ __align__(128) uint8_t dsm[];
  __shared__ PagedShared sh;
  const int tid = threadIdx.x, wid = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int HU = a.KH * a.rt;
  pdl_wait();
  pdl_trigger();
  // Where this CTA's tiles begin.
  long long total, x0, x1;
  int ctas;
  if (a.whole) {
    total = (long long)a.B * HU;
    ctas = (int)min((long long)gridDim.x, total);
    x0 = blockIdx.x < ctas ? total * blockIdx.x / ctas : total;
    x1 = blockIdx.x < ctas ? total * (blockIdx.x + 1) / ctas : total;
    if (tid == 0) sh.b0 = (int)(x0 / HU), sh.before = 0;
  } else {
    int mine = 0;
    long long before = 0, round = 0;   // this thread's sequence: tiles, those before it
    auto scan = [&](int b0) {
      const int b = b0 + tid;
      mine = b < a.B ? paged_tiles(min(max(a.lens[b], 0), a.max_len), a.n, a.window, KEYS) : 0;
      long long y = mine;
      for (int o = 1; o < 32; o <<= 1) {
        const long long z = __shfl_up_sync(~0u, y, o);
        if (lane >= o) y += z;
      }
      __syncthreads();
      if (lane == 31) sh.sums[wid] = y;
      __syncthreads();
      before = round + y - mine;
      for (int i = 0; i < PG_WARPS; i++) {
        if (i < wid) before += sh.sums[i];
        round += sh.sums[i];
      }
    };
    for (int b0 = 0; b0 < a.B; b0 += PG_THREADS) scan(b0);
    total = round * HU;
    // a CTA has a tile for each warp at least
    ctas = (int)max(1ll, min((long long)gridDim.x, total / PG_WARPS));
    x0 = blockIdx.x < ctas ? total * blockIdx.x / ctas : total;
    x1 = blockIdx.x < ctas ? total * (blockIdx.x + 1) / ctas : total;
    auto note = [&](int b0) {
      if (b0 + tid < a.B && before * HU <= x0 && x0 < (before + mine) * HU) sh.b0 = b0 + tid, sh.before = before;
    };
    if (a.B <= PG_THREADS) {
      note(0);
    } else {
      round = 0;
      for (int b0 = 0; b0 < a.B; b0 += PG_THREADS) {
        scan(b0);
        note(b0);
      }
    }
    if (tid == 0) a.desc[blockIdx.x].x = -1;
  }
  __syncthreads();

  uint8_t* ring = dsm + wid * (S::D * S::SLOT);
  float* red = reinterpret_cast<float*>(dsm + PG_WARPS * S::D * S::SLOT);
  const uint32_t ring32 = smem_u32(ring);

  // Loads: a walk of its own, D - 1 of this warp's tiles ahead.
  PagedWalk lw;
  int lj = 0, put = 0, ids[S::U];   // its tile, its place in the ring, its pages
  auto ids_of = [&]() {
#pragma unroll
    for (int u = 0; u < S::U; u++) {
      const int key = (lw.lo & ~15) + lj * KEYS + 16 * u;
      ids[u] = lw.more() && key < lw.len ? paged_page(a.tables + lw.b * a.st, a.cols, key, a.shift, a.n_pages) : -1;
    }
  };
  auto settle = [&]() {   // tiles behind the segment's end are the next one's
    while (lw.more() && lj >= lw.j1) {
      const int over = lj - lw.j1;
      lw.next<KEYS>(a);
      lj = lw.j + over;
    }
  };
  auto load = [&]() {
    if (lw.more()) {
      const int kh = lw.hu / a.rt, k0 = (lw.lo & ~15) + lj * KEYS;
      const uint32_t slot = ring32 + put * S::SLOT;
      constexpr int PER = 32 / S::CH;   // rows of a warp's load
      const int r0 = lane / S::CH, c = lane % S::CH;
      const bool col = c * 16 < a.hd * (CODES ? 1 : 2);
#pragma unroll
      for (int u = 0; u < S::U; u++) {
        const int key = k0 + 16 * u, page = max(ids[u], 0), row = key & ((1 << a.shift) - 1);
        const uint8_t* k = a.kp + page * a.skp[0] + kh * a.skp[1] + (row + r0) * a.skp[2] + c * 16;
        const uint8_t* v = a.vp + page * a.svp[0] + kh * a.svp[1] + (row + r0) * a.svp[2] + c * 16;
#pragma unroll
        for (int i = 0; i < 16; i += PER) {
          const bool in = col && ids[u] >= 0 && key + i + r0 >= lw.lo && key + i + r0 < lw.len;
          const uint32_t to = slot + S::at(16 * u + i + r0, c);
          cp16(to, in ? k + i * a.skp[2] : a.kp, in);
          cp16(to + S::HALF, in ? v + i * a.svp[2] : a.vp, in);
        }
        if (CODES && lane < 2) {
          const int block = row / PAGED_BLOCK;
          const float* s = lane ? a.vs + page * a.svs[0] + kh * a.svs[1] + block * a.svs[2] : a.ks + page * a.sks[0] + kh * a.sks[1] + block * a.sks[2];
          cp4(slot + 2 * S::HALF + (2 * u + lane) * 4, ids[u] >= 0 ? s : a.ks, ids[u] >= 0);
        }
        if (lane == 0) *reinterpret_cast<int*>(ring + put * S::SLOT + 2 * S::HALF + 16 + 4 * u) = ids[u] >= 0;
      }
      lj += PG_WARPS;
      settle();
      ids_of();
    }
    cp_commit();
    if (++put == S::D) put = 0;
  };
  lw.start<KEYS>(a, sh.b0, sh.before, x0, x1);
  lj = lw.more() ? lw.j + wid : 0;
  settle();
  ids_of();
#pragma unroll
  for (int i = 0; i < S::D - 1; i++) load();

  PagedWalk wk;
  wk.start<KEYS>(a, sh.b0, sh.before, x0, x1);
  int tj = wk.more() ? wk.j + wid : 0, get = 0;
  for (; wk.more(); wk.next<KEYS>(a)) {
    const int b = wk.b, kh = wk.hu / a.rt, row0 = wk.hu % a.rt * (8 * NT);
    const int base = wk.len - a.n;   // position of the first query
    // Q^T as B fragments; the rows are columns, absent ones and dimensions zero.
    // A lane's 16-byte words of a key are t4, t4 + 4, ..; their values in turn
    // are the steps' dimensions.
    uint32_t qf[NT][S::STEPS][2];
    float f[NT][2];      // scale log2(e) of this lane's columns' scores, over the power of two in q
    int tok[NT][2];      // and their queries
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int r = row0 + t * 8 + g;
      const T* q = (const T*)a.q + b * a.sq[0] + min(r, a.rows - 1) / a.G * a.sq[1] + (kh * a.G + min(r, a.rows - 1) % a.G) * a.sq[2];
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < S::STEPS; k++)
#pragma unroll
        for (int z = 0; z < 2; z++) {
          constexpr int PW = S::STEPS / S::KC;   // steps of a word
          const int d = (t4 + 4 * (k / PW)) * (4 * PW) + (k % PW) * 4 + z * 2;
          qf[t][k][z] = r < a.rows && d < a.hd ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
          if (CODES && std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const uint32_t m = (h ? qf[t][k][z] >> 16 : qf[t][k][z]) & 0x7fffu;
              if (m < 0x7f80u) top = max(top, m);   // finite ones
            }
          }
        }
      f[t][0] = f[t][1] = a.c;
      if (CODES && std::is_same<T, __nv_bfloat16>::value) {
        top = max(top, __shfl_xor_sync(~0u, top, 1));
        top = max(top, __shfl_xor_sync(~0u, top, 2));
        const int up = min(14 + 127 - (int)(top >> 7), 126);
        const float s = __int_as_float((up + 127) << 23);
#pragma unroll
        for (int k = 0; k < S::STEPS; k++)
#pragma unroll
          for (int z = 0; z < 2; z++) {
            const float lo = __uint_as_float(qf[t][k][z] << 16), hi = __uint_as_float(qf[t][k][z] & 0xffff0000u);
            qf[t][k][z] = at_pack<__half>(lo * s, hi * s);
          }
#pragma unroll
        for (int z = 0; z < 2; z++) f[t][z] = a.c * __int_as_float((127 - __shfl_sync(~0u, up, (t4 * 2 + z) * 4)) << 23);
      }
#pragma unroll
      for (int z = 0; z < 2; z++) tok[t][z] = min(row0 + t * 8 + t4 * 2 + z, a.rows - 1) / a.G;
    }
    float o[NT][S::STEPS][4], m[NT][2], r[NT][2], l[NT][2];   // r: the accumulators' reference (CODES)
    float nm[NT][2], nr[NT][2], limm[NT][2], limr[NT][2];      // OFF - m, and m + LIFT
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
      for (int z = 0; z < 2; z++) {
        m[t][z] = r[t][z] = limm[t][z] = limr[t][z] = -INFINITY;
        nm[t][z] = nr[t][z] = l[t][z] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < S::STEPS; k++) o[t][k][0] = o[t][k][1] = o[t][k][2] = o[t][k][3] = 0.f;
    }
    // the keys that every row sees
    const int all_hi = base + 1, all_lo = a.window > 0 ? max(0, wk.len - a.window) : 0;
    for (; tj < wk.j1; tj += PG_WARPS) {
      load();
      cp_wait<S::D - 1>();
      __syncwarp();
      const uint32_t kb = ring32 + get * S::SLOT, vb = kb + S::HALF;
      const int k0 = (wk.lo & ~15) + tj * KEYS;
      const float* extra = reinterpret_cast<const float*>(ring + get * S::SLOT + 2 * S::HALF);
      float x[S::U][NT][4];
#pragma unroll
      for (int u = 0; u < S::U; u++) {
#pragma unroll
        for (int t = 0; t < NT; t++) x[u][t][0] = x[u][t][1] = x[u][t][2] = x[u][t][3] = 0.f;
#pragma unroll
        for (int w = 0; w < S::KC; w++) {
          const uint4 lo4 = lds16(kb + S::at(16 * u + g, t4 + 4 * w)), hi4 = lds16(kb + S::at(16 * u + g + 8, t4 + 4 * w));
          const uint32_t lo[4] = {lo4.x, lo4.y, lo4.z, lo4.w}, hi[4] = {hi4.x, hi4.y, hi4.z, hi4.w};
          constexpr int PW = S::STEPS / S::KC;
#pragma unroll
          for (int s = 0; s < PW; s++) {
            uint32_t fr[4];
            if (CODES)
              fr[0] = pg_codes(lo[s]), fr[1] = pg_codes(hi[s]), fr[2] = pg_codes(lo[s] >> 16), fr[3] = pg_codes(hi[s] >> 16);
            else
              fr[0] = lo[2 * s & 3], fr[1] = hi[2 * s & 3], fr[2] = lo[2 * s + 1 & 3], fr[3] = hi[2 * s + 1 & 3];
#pragma unroll
            for (int t = 0; t < NT; t++) pg_mma<M>(x[u][t], fr, qf[t][w * PW + s][0], qf[t][w * PW + s][1]);
          }
        }
      }
      // scores in base 2; those that a row does not see: -inf
      bool part = k0 < all_lo || k0 + KEYS > all_hi;
      float lv[S::U];
      bool there[S::U];
#pragma unroll
      for (int u = 0; u < S::U; u++) {
        const float sk = CODES ? extra[2 * u] : 1.f;
        lv[u] = CODES ? __log2f(extra[2 * u + 1]) : 0.f;
        there[u] = reinterpret_cast<const int*>(extra)[4 + u];
        part |= !there[u];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int z = 0; z < 4; z++) x[u][t][z] *= CODES ? f[t][z & 1] * sk : f[t][z & 1];
      }
      if (part) {
#pragma unroll
        for (int u = 0; u < S::U; u++)
#pragma unroll
          for (int t = 0; t < NT; t++)
#pragma unroll
            for (int z = 0; z < 4; z++) {
              const int key = k0 + 16 * u + g + (z >> 1) * 8, at = base + tok[t][z & 1];
              if (!there[u] || key > at || (a.window > 0 && (long long)key <= (long long)at - a.window)) x[u][t][z] = -INFINITY;
            }
      }
      bool up = false;
#pragma unroll
      for (int u = 0; u < S::U; u++)
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int z = 0; z < 4; z++) up |= x[u][t][z] > limm[t][z & 1] || (CODES && x[u][t][z] + lv[u] > limr[t][z & 1]);
      if (__any_sync(~0u, up)) {
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int z = 0; z < 2; z++) {
            float v = -INFINITY, w = -INFINITY;
#pragma unroll
            for (int u = 0; u < S::U; u++) {
              const float y = fmaxf(x[u][t][z], x[u][t][z + 2]);
              v = fmaxf(v, y);
              if (CODES) w = fmaxf(w, y + lv[u]);
            }
#pragma unroll
            for (int sft = 4; sft < 32; sft <<= 1) {
              v = fmaxf(v, __shfl_xor_sync(~0u, v, sft));
              if (CODES) w = fmaxf(w, __shfl_xor_sync(~0u, w, sft));
            }
            if (!CODES) w = v;
            const float mn = fmaxf(m[t][z], v), rn = fmaxf(r[t][z], w);
            const float fm = mn > m[t][z] ? at_exp2(m[t][z] - mn) : 1.f, fr = rn > r[t][z] ? at_exp2(r[t][z] - rn) : 1.f;
            m[t][z] = mn, r[t][z] = rn;
            nm[t][z] = mn == -INFINITY ? 0.f : OFF - mn;
            nr[t][z] = rn == -INFINITY ? 0.f : OFF - rn;
            limm[t][z] = mn + LIFT, limr[t][z] = rn + LIFT;
            l[t][z] *= fm;
#pragma unroll
            for (int k = 0; k < S::STEPS; k++) {
              o[t][k][z] *= fr;
              o[t][k][z + 2] *= fr;
            }
          }
      }
      uint32_t p[S::U][NT][2];
#pragma unroll
      for (int u = 0; u < S::U; u++)
#pragma unroll
        for (int t = 0; t < NT; t++) {
          float e[4];
#pragma unroll
          for (int z = 0; z < 4; z++) {
            const float y = at_exp2(x[u][t][z] + nm[t][z & 1]);
            l[t][z & 1] += y;
            // where the row does not see the key, whatever its scale holds
            e[z] = !CODES ? y : x[u][t][z] == -INFINITY ? 0.f : at_exp2(x[u][t][z] + lv[u] + nr[t][z & 1]);
          }
          p[u][t][0] = pg_movm(at_pack<M>(e[0], e[1]));
          p[u][t][1] = pg_movm(at_pack<M>(e[2], e[3]));
        }
      // O^T += V^T P^T: a lane has the keys 2 t4, 2 t4 + 1 and those 8 on, and
      // HD / 8 dimensions of each; two keys' values of a dimension make a register
#pragma unroll
      for (int u = 0; u < S::U; u++) {
        constexpr int W = HD / 8 * (CODES ? 1 : 2) / 4;   // 32-bit words of a key that a lane has: 2, 4 or 8
        uint32_t v[4][W];
        uint32_t odd = 0;   // values that are not finite
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int row = 16 * u + 2 * t4 + (i & 1) + (i >> 1) * 8;
          if (W == 2) {
            const uint2 y = lds8(vb + S::at(row, g >> 1) + (g & 1) * 8);
            v[i][0] = y.x, v[i][W - 1] = y.y;
          } else {
#pragma unroll
            for (int h = 0; h < W / 4; h++) {
              const uint4 y = lds16(vb + S::at(row, g + 8 * h));
              v[i][4 * h] = y.x, v[i][4 * h + 1] = y.y, v[i][4 * h + 2] = y.z, v[i][4 * h + 3] = y.w;
            }
          }
        }
        if (part && a.n > 1) {   // some rows may see a key and others not: 0 x inf or NaN must not reach those
#pragma unroll
          for (int i = 0; i < 4; i++)
#pragma unroll
            for (int w = 0; w < W; w++) {
              if (CODES) odd |= (v[i][w] & 0x7f7f7f7fu) + 0x01010101u & 0x80808080u;
              else if (std::is_same<T, __half>::value) odd |= (v[i][w] & 0x7c007c00u) + 0x04000400u & 0x80008000u;
              else odd |= (v[i][w] & 0x7f807f80u) + 0x00800080u & 0x80008000u;
            }
          odd = __any_sync(~0u, odd != 0);
        }
#pragma unroll
        for (int k = 0; k < S::STEPS; k++) {
          uint32_t fr[4];
          if (CODES) {   // 16-dimension part k: bytes 2 k and 2 k + 1 of the lane's
            const uint32_t sel = k & 1 ? 0x7362u : 0x5140u;
            const uint32_t y0 = __byte_perm(v[0][k / 2], v[1][k / 2], sel), y1 = __byte_perm(v[2][k / 2], v[3][k / 2], sel);
            fr[0] = pg_codes(y0), fr[1] = pg_codes(y0 >> 16), fr[2] = pg_codes(y1), fr[3] = pg_codes(y1 >> 16);
          } else {
            const int w = k % W;
            fr[0] = __byte_perm(v[0][w], v[1][w], 0x5410), fr[1] = __byte_perm(v[0][w], v[1][w], 0x7632);
            fr[2] = __byte_perm(v[2][w], v[3][w], 0x5410), fr[3] = __byte_perm(v[2][w], v[3][w], 0x7632);
          }
          if (!odd) {
#pragma unroll
            for (int t = 0; t < NT; t++) pg_mma<M>(o[t][k], fr, p[u][t][0], p[u][t][1]);
          } else {   // each query by itself, the keys that it does not see cleared
#pragma unroll
            for (int t = 0; t < NT; t++)
              for (int i = min(row0 + t * 8, a.rows - 1) / a.G; i <= min(row0 + t * 8 + 7, a.rows - 1) / a.G; i++) {
                uint32_t keep[2] = {0u, 0u};
#pragma unroll
                for (int h = 0; h < 4; h++) {
                  const int key = k0 + 16 * u + 2 * t4 + (h & 1) + (h >> 1) * 8, at = base + i;
                  if (key <= at && !(a.window > 0 && (long long)key <= (long long)at - a.window)) keep[h >> 1] |= h & 1 ? 0xffff0000u : 0xffffu;
                }
                const uint32_t mine[4] = {fr[0] & keep[0], fr[1] & keep[0], fr[2] & keep[1], fr[3] & keep[1]};
                float y[4] = {0.f, 0.f, 0.f, 0.f};
                pg_mma<M>(y, mine, p[u][t][0], p[u][t][1]);
#pragma unroll
                for (int z = 0; z < 4; z++)
                  if (tok[t][z & 1] == i) o[t][k][z] += y[z];
              }
          }
        }
      }
      __syncwarp();   // before the next load into this place
      if (++get == S::D) get = 0;
    }
    tj -= wk.j1;
    // Join the warps, 8 rows at a time.
    const bool all = wk.j == 0 && wk.j1 == wk.n;
    const int slot = 2 * blockIdx.x + (wk.j == 0);
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
      for (int z = 0; z < 2; z++) {
#pragma unroll
        for (int sft = 4; sft < 32; sft <<= 1) l[t][z] += __shfl_xor_sync(~0u, l[t][z], sft);
        if (g == 0) sh.ml[wid][t4 * 2 + z] = make_float4(m[t][z] - OFF, l[t][z], r[t][z] - OFF, 0.f);
      }
#pragma unroll
      for (int k = 0; k < S::STEPS; k++)
#pragma unroll
        for (int z = 0; z < 4; z++) {
          // 16-dimension part k: dimensions 2 k and 2 k + 1 of the lane's HD / 8
          constexpr int LW = 4 * S::STEPS / S::KC;   // dimensions of a 16-byte word
          const int e = 2 * k + (z >> 1), d = HD == 64 && CODES ? g * 8 + e : (g + 8 * (e / LW)) * LW + e % LW;
          red[(wid * 8 + t4 * 2 + (z & 1)) * S::RP + d] = o[t][k][z];
        }
      __syncthreads();
      for (int i = tid; i < 8 * HD; i += PG_THREADS) {
        const int h = i / HD, d = i % HD, row = row0 + t * 8 + h;
        float mm = -INFINITY, rr = -INFINITY, L = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < PG_WARPS; w++) mm = fmaxf(mm, sh.ml[w][h].x), rr = fmaxf(rr, sh.ml[w][h].z);
        if (row < a.rows) {
          const float sink = a.sinks && all ? a.sinks[kh * a.G + row % a.G] * LOG2E : -INFINITY;
          mm = fmaxf(mm, sink);
#pragma unroll
          for (int w = 0; w < PG_WARPS; w++) {
            const float4 ml = sh.ml[w][h];
            if (ml.y == 0.f) continue;   // a warp without keys
            L = fmaf(ml.y, at_exp2(ml.x - mm), L);
            if (ml.z != -INFINITY) v = fmaf(red[(w * 8 + h) * S::RP + d], at_exp2(ml.z - rr), v);
          }
          if (all) {
            if (sink != -INFINITY) L += at_exp2(sink - mm);
            if (d < a.hd) {
              const float y = L == 0.f ? 0.f : v == 0.f ? v / L : v / L * at_exp2(rr - mm);
              T* out = (T*)a.out + b * a.so[0] + row / a.G * a.so[1] + (kh * a.G + row % a.G) * a.so[2] + d;
              *reinterpret_cast<uint16_t*>(out) = (uint16_t)at_pack<T>(y, 0.f);
            }
          } else {
            const size_t at = (size_t)slot * (8 * NT) + t * 8 + h;
            a.po[at * HD + d] = v;
            if (d == 0) a.pml[at] = make_float4(mm, L, rr, 0.f);
          }
        }
      }
      __syncthreads();
    }
    if (!all && wk.j == 0 && tid == 0) {
      const int last = paged_cta(wk.x + wk.n - 1, total, ctas);
      a.desc[blockIdx.x] = make_int4(b, wk.hu, last, 0);
    }
  }
  cp_wait<0>();
  // Sequences without a key.
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    if (paged_tiles(min(max(a.lens[b], 0), a.max_len), a.n, a.window, KEYS) > 0) continue;
    const int words = a.hd / 8, H = a.KH * a.G;
    for (int i = tid; i < a.n * H * words; i += PG_THREADS) {
      T* out = (T*)a.out + b * a.so[0] + i / words / H * a.so[1] + i / words % H * a.so[2] + i % words * 8;
      *reinterpret_cast<uint4*>(out) = make_uint4(0, 0, 0, 0);
    }
  }
}

// Block i: the unit that begins in CTA i and ends in a later one, its pieces'
// weighted sum.
template <typename T, int HD, int NT>
__global__ void __launch_bounds__(PG_JOIN_THREADS) paged_join_kernel(const PagedArgs a) {
  pdl_wait();
  const int i = blockIdx.x, lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int4 d = a.desc[i];
  if (d.x < 0) return;
  const int kh = d.y / a.rt, row0 = d.y % a.rt * (8 * NT), pieces = d.z - i + 1;
  auto at = [&](int p, int h) { return (size_t)(p ? 2 * (i + p) : 2 * i + 1) * (8 * NT) + h; };
  for (int h = wid; h < 8 * NT && row0 + h < a.rows; h += PG_JOIN_THREADS / 32) {
    const int row = row0 + h, head = kh * a.G + row % a.G;
    const float sink = a.sinks ? a.sinks[head] * LOG2E : -INFINITY;
    float mm = sink, rr = -INFINITY;
    for (int p = lane; p < pieces; p += 32) {
      const float4 ml = a.pml[at(p, h)];
      mm = fmaxf(mm, ml.x), rr = fmaxf(rr, ml.z);
    }
#pragma unroll
    for (int sft = 16; sft; sft >>= 1) mm = fmaxf(mm, __shfl_xor_sync(~0u, mm, sft)), rr = fmaxf(rr, __shfl_xor_sync(~0u, rr, sft));
    float L = sink != -INFINITY ? at_exp2(sink - mm) : 0.f, v[HD / 32];
#pragma unroll
    for (int e = 0; e < HD / 32; e++) v[e] = 0.f;
#pragma unroll 4
    for (int p = 0; p < pieces; p++) {
      const float4 ml = a.pml[at(p, h)];
      float y[HD / 32];
#pragma unroll
      for (int e = 0; e < HD / 32; e++) y[e] = a.po[at(p, h) * HD + lane + 32 * e];
      if (ml.y == 0.f) continue;
      L = fmaf(ml.y, at_exp2(ml.x - mm), L);
      const float fr = ml.z != -INFINITY ? at_exp2(ml.z - rr) : 0.f;
#pragma unroll
      for (int e = 0; e < HD / 32; e++) v[e] = fmaf(y[e], fr, v[e]);
    }
    T* out = (T*)a.out + d.x * a.so[0] + row / a.G * a.so[1] + head * a.so[2];
#pragma unroll
    for (int e = 0; e < HD / 32; e++) {
      const float y = L == 0.f ? 0.f : v[e] == 0.f ? v[e] / L : v[e] / L * at_exp2(rr - mm);
      if (lane + 32 * e < a.hd) *reinterpret_cast<uint16_t*>(out + lane + 32 * e) = (uint16_t)at_pack<T>(y, 0.f);
    }
  }
}

// What the host settles before the lengths are known.
struct PagedSpace {
  int nt, rt, whole, grid;
  size_t po = 0, pml = 0, desc = 0, bytes = 0;
  PagedSpace(int bits, int batch, int queries, int max_len, int H, int KH, int hd, int sms) {
    const int rows = queries * (H / KH), HD = hd <= 64 ? 64 : 128, keys = HD * bits / 8 <= 128 ? 32 : 16;
    nt = rows <= 8 ? 1 : 2;
    rt = (rows + 8 * nt - 1) / (8 * nt);
    const long long units = (long long)batch * KH * rt, tiles = ((long long)max_len + keys - 1) / keys;
    whole = tiles <= 2 * PG_WARPS;
    const long long most = whole ? units : units * tiles / PG_WARPS;
    grid = (int)std::max(1ll, std::min((long long)sms, most));
    if (whole) return;
    auto take = [&](size_t n) {
      const size_t o = bytes;
      bytes = (bytes + n + 255) & ~(size_t)255;
      return o;
    };
    po = take((size_t)2 * grid * 8 * nt * HD * 4);
    pml = take((size_t)2 * grid * 8 * nt * 16);
    desc = take((size_t)grid * 16);
  }
};

template <typename T, bool CODES, int HD, int NT>
static cudaError_t run_paged(const PagedArgs& a, int grid, cudaStream_t s) {
  const int smem = PagedShape<T, CODES, HD, NT>::SMEM;
  static std::atomic<unsigned long long> set{0};
  cudaError_t e = attn_smem(paged_kernel<T, CODES, HD, NT>, smem, set);
  if (e == cudaSuccess) e = launch_pdl(paged_kernel<T, CODES, HD, NT>, dim3(grid), PG_THREADS, smem, s, a);
  count_launches(1);
  if (e == cudaSuccess && !a.whole && grid > 1) {
    e = launch_pdl(paged_join_kernel<T, HD, NT>, dim3(grid - 1), PG_JOIN_THREADS, 0, s, a);
    count_launches(1);
  }
  return e;
}
template <typename T, bool CODES>
static cudaError_t run_paged(const PagedArgs& a, int nt, int grid, cudaStream_t s) {
  if (a.hd <= 64) return nt == 1 ? run_paged<T, CODES, 64, 1>(a, grid, s) : run_paged<T, CODES, 64, 2>(a, grid, s);
  return nt == 1 ? run_paged<T, CODES, 128, 1>(a, grid, s) : run_paged<T, CODES, 128, 2>(a, grid, s);
}

}  // namespace tg

using namespace tg;

extern "C" size_t tg_attention_paged_workspace(int page_bits, int batch, int n_queries, int max_len, int n_heads,
                                               int n_kv_heads, int head_dim) {
  if (batch <= 0 || n_queries <= 0 || max_len <= 0 || n_kv_heads <= 0 || n_heads < n_kv_heads || n_heads / n_kv_heads > 128 || head_dim <= 0) return 0;
  if ((long long)n_queries * n_heads >= 1 << 24) return 0;
  return PagedSpace(page_bits, batch, n_queries, max_len, n_heads, n_kv_heads, head_dim, attn_sms()).bytes;
}

extern "C" int tg_attention_paged(int dtype, int page_bits, const void* q, const void* k_pages, const void* v_pages,
                                  const float* k_scales, const float* v_scales, void* out, const int* tables,
                                  const int* lens, const float* sinks, int batch, int n_queries, int n_pages, int page,
                                  int table_cols, int max_len, int n_heads, int n_kv_heads, int head_dim,
                                  const int64_t* strides, int window, float scale, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  ArgCheck c("tg_attention_paged");
  c.need(dtype == ATTN_BF16 || dtype == ATTN_FP16, "dtype must be 0 (bf16) or 1 (fp16)");
  c.need(batch >= 0 && n_queries >= 0 && max_len >= 0 && window >= 0, "counts and window must not be negative");
  c.need(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && n_heads / n_kv_heads <= 128,
         "n_heads must be a multiple of n_kv_heads, at most 128 times it");
  c.need((long long)n_queries * n_heads < 1 << 24 && (long long)batch * n_queries * n_heads < 1ll << 31, "too many query rows");
  c.need(head_dim > 0 && head_dim % 8 == 0 && head_dim <= ATTN_MAX_HD, "head_dim must be a multiple of 8, at most 128");
  c.need(std::isfinite(scale) && scale > 0.f, "scale must be finite and positive");
  c.need(strides != nullptr, "strides is null");
  if (c.rc) return c.rc;
  const PoolCheck pool(c, page_bits, n_pages, page, table_cols, batch, n_kv_heads, head_dim, strides + 6);
  const long long n3[3] = {batch, n_queries, n_heads};
  long long t[6];
  for (int i = 0; i < 6; i++) t[i] = c.stride(strides[i], n3[i % 3]);
  c.need(max_len <= (long long)table_cols * page, "max_len must be at most table_cols x page");
  c.need(max_len < AT_NPOS, "too many positions");
  if (c.rc || batch == 0 || n_queries == 0) return c.rc;
  if (n_pages == 0) max_len = 0;
  if (!c.device()) return c.rc;
  c.ptr(q, 16, "q"), c.ptr(out, 16, "out"), c.ptr(lens, 4, "lens");
  if (max_len > 0) {
    c.ptr(k_pages, 16, "k_pages"), c.ptr(v_pages, 16, "v_pages"), c.ptr(tables, 4, "tables");
    if (page_bits == 8) c.ptr(k_scales, 4, "k_scales"), c.ptr(v_scales, 4, "v_scales");
  }
  if (sinks) c.ptr(sinks, 4, "sinks");
  const PagedSpace sp(page_bits, batch, n_queries, max_len, n_heads, n_kv_heads, head_dim, attn_sms());
  c.need(workspace_bytes >= sp.bytes, "the workspace is smaller than tg_attention_paged_workspace says");
  if (sp.bytes > 0) c.ptr(workspace, 256, "workspace");
  if (c.rc) return c.rc;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  PagedArgs a{};
  a.q = q, a.kp = (const uint8_t*)k_pages, a.vp = (const uint8_t*)v_pages, a.ks = k_scales, a.vs = v_scales;
  a.tables = tables, a.lens = lens, a.sinks = sinks, a.out = out;
  a.po = (float*)(ws + sp.po), a.pml = (float4*)(ws + sp.pml), a.desc = (int4*)(ws + sp.desc);
  for (int i = 0; i < 3; i++) {
    a.sq[i] = t[i], a.so[i] = t[3 + i];
    a.skp[i] = pool.kp[i], a.svp[i] = pool.vp[i], a.sks[i] = pool.ks[i], a.svs[i] = pool.vs[i];
  }
  a.st = pool.st, a.B = batch, a.n = n_queries, a.G = n_heads / n_kv_heads, a.KH = n_kv_heads, a.rows = n_queries * a.G, a.rt = sp.rt;
  a.hd = head_dim, a.cols = table_cols, a.n_pages = n_pages, a.shift = pool.shift, a.max_len = max_len, a.window = window;
  a.whole = sp.whole, a.c = scale * LOG2E;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == ATTN_BF16)
    return c.done(page_bits == 8 ? run_paged<__nv_bfloat16, true>(a, sp.nt, sp.grid, s) : run_paged<__nv_bfloat16, false>(a, sp.nt, sp.grid, s));
  return c.done(page_bits == 8 ? run_paged<__half, true>(a, sp.nt, sp.grid, s) : run_paged<__half, false>(a, sp.nt, sp.grid, s));
}
