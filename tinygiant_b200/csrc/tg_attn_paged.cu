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
// mma.m16n8k16 with keys and dimensions as the 16 and the rows as the 8 columns.
// (With 128 keys as the tensor memory's rows one token would be bound by HBM all the
// same; more than 16 rows would read their keys once.)  Codes are exact in fp16, so
// with them both products are fp16's: q in fp16 as it is, in bf16 times a power
// of two that takes its row's largest value to 2^14 or more (fp16 keeps bf16's 8 bits
// down to 2^-31 of that, and nothing below 2^-40).  A weight meets the values in two parts, its
// rounding to 16 bits and what that drops, 22 bits together in fp16 and 16 in bf16:
// of 64 sequences' bf16 outputs one in 1,600 is not the exact value's rounding, with
// one part one in 12 (drafts in fp16: one in 460, and one in 3).  The second product
// costs 3 to 6 % (256 sequences 244 us with one part, 258 with two, 64 35.4 and 36.5,
// drafts under a window 11.9 and 12.5).  Scales never meet the values: ks
// multiplies the scores, and log2(vs) is added to the exponent of the weights
// that meet v.  So there are two running references, one for the sum of the
// weights and one for the accumulators; each warp moves its own only when a
// score exceeds it by LIFT in base 2.
//
// Work: units are a sequence, a key head and up to 16 rows, their tiles 32 keys
// (16 of 256-byte rows).  A group of warps walks the tiles of its units, which
// lie in a row and are cut evenly among the groups, or short ones dealt out whole;
// a group's tiles go to its warps in turn.  Each warp loads its own tiles ahead
// with cp.async (pages end anywhere, and rows that nobody may read come as zeros)
// into places of its own, so no warp waits for another until a unit ends.  There
// the warps' results join in shared memory, and those of units that lie in
// several groups in a second kernel.  Nothing spins, and nothing is summed in an
// order that may change.
//
// What bounds it (32 / 4 heads of 128, codes): 256 sequences of 2,048 to 8,192
// keys, 1.35 GB: 225 us at the full clock, 0.91 of a copy's rate; a tile takes a warp
// about 810 instructions (loads 160, codes to fp16 130, products 48, softmax 140), 0.6
// of the issue slots at that rate.  Call after call the chip's power limit takes the
// clock to 1,560 MHz, and instructions bound it: 259 us.  64 sequences of 1 to 4,096:
// 36 us where the bytes take 20: start and cut 4, units' starts and ends 4, the second
// kernel 5.
//
// Registers: 168 of a thread with 8 rows a unit, up to 255 with 16; with heads of 128
// and codes 24 to 68 bytes are spilled.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "../../include/tinygiant.h"
#include "tg_attn_tc.cuh"
#include "tg_paged.h"

namespace tg {

constexpr int PG_JOIN_THREADS = 256;

struct PagedArgs {
  const void* q;
  const uint8_t *kp, *vp;
  const float *ks, *vs;
  const int *tables, *lens;
  const float* sinks;
  void* out;
  float* po;      // [2 group + slot][rows of a unit][HD]
  float4* pml;    // [2 group + slot][rows of a unit]: m, l, r
  int4* desc;     // [group]: sequence (-1: no unit begins here and ends later), head unit, last group
  long long sq[3], so[3];     // sequence, token, head
  unsigned skp[3], svp[3];    // page, head, row; 16-byte words
  unsigned sks[3], svs[3];    // page, head, block
  long long st;
  int B, n, rows, rt, KH, G, hd, cols, n_pages, shift, max_len, window;
  unsigned by_g;  // 2^32 / G, rounded up (G > 1)
  int whole;      // units are not cut
  int team;       // warps of a group: 4, or 1 or 2 where units are not cut
  int unit;       // what a unit's start and end cost, in tiles of a warp
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
// Two values of a register.
template <typename M>
__device__ __forceinline__ float2 pg_halves(uint32_t two) {
  if (std::is_same<M, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&two));
  return make_float2(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
}
// The query of row r = query G + head of the group: r / G for r < 2^25 (by_g G is
// less than 2^32 + 128).
__device__ __forceinline__ int query_of(const PagedArgs& a, int r) { return a.G == 1 ? r : (int)__umulhi((unsigned)r, a.by_g); }
// What accumulators are multiplied by: 1 over the sum L, whose reference is 2^up of
// theirs; 0 for a row without a key.
__device__ __forceinline__ float paged_factor(float L, float up) {
  return L == 0.f ? 0.f : up == -INFINITY ? 0.f * L : at_exp2(up) / L;
}
// A head's sink in base 2.  +inf, or what leaves fp32 here, is fp32's largest, so that
// it takes all the weight instead of meeting itself as inf - inf.
__device__ __forceinline__ float sink_of(const PagedArgs& a, int head) {
  const float x = a.sinks[head] * LOG2E;
  return x == INFINITY ? FLT_MAX : x;
}
// Four e4m3 codes, the lowest byte first, as two pairs of fp16.
__device__ __forceinline__ void pg_codes(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(four));
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
  static constexpr int WARPS = NT == 1 ? 12 : 8, THREADS = WARPS * 32;
  static constexpr int D = (NT == 1 ? 2 : 3) * (RB == 64 ? 2 : 1);   // tiles in a warp's ring
  static constexpr int RP = HD + 4;                              // pitch of a row of accumulators, in a place of the ring
  // Accumulators in shared and global memory: part k's two dimensions of lane
  // group g at 16 k + 2 g, which all lanes write without bank conflicts; the
  // first of the two:
  static __host__ __device__ __forceinline__ int dim(int k, int g) {
    if (CODES) return HD / 8 * g + 2 * k;
    return k / 4 * 64 + g * 8 + k % 4 * 2;
  }
  static constexpr int SMEM = WARPS * D * SLOT;
  static_assert(8 * RP * 4 <= SLOT && D >= 2, "8 rows of accumulators lie in a place of the ring");
  // Place of 16-byte word c of row r.  A quarter of a warp reads rows 2 i and
  // 2 i + 1, four words each (K), or words 2 q and 2 q + 1 of rows of one
  // parity (V; half a warp, words of 8 bytes, where rows are 64 bytes): all on
  // different banks.
  static __device__ __forceinline__ int at(int r, int c) {
    if (RB == 64) return (r >> 1) * 128 + ((((r & 1) << 2 | c) ^ ((r >> 1 & 3) << 1)) << 4);
    return r * RB + (c >> 3) * 128 + (((c & 7) ^ (r & 6) ^ ((r & 1) << 2)) << 4);
  }
};

// The tiles of a group as segments: consecutive tiles of one unit (sequence,
// key head, 16 rows).  Units lie in a row, `unit` places longer than their tiles
// (none for one without keys), and the places are cut evenly; where units are
// not cut, a place is a unit.
struct PagedWalk {
  long long x, x1;                           // the unit's first place, the end of the group's
  int b, kh, ri, j, j1, len, lo, n, ahead;   // ri: which 16 rows; lo: first key; n: tiles; [j, j1): the segment's
  __device__ __forceinline__ int len_of(const PagedArgs& a, int s) const { return s < a.B ? min(max(a.lens[s], 0), a.max_len) : 0; }
  template <int KEYS>
  __device__ __forceinline__ void seq(const PagedArgs& a, int keys) {
    len = keys;
    lo = paged_first(len, a.n, a.window);
    n = paged_tiles(len, a.n, a.window, KEYS);
    ahead = len_of(a, b + 1);
  }
  __device__ __forceinline__ bool more() const { return x < x1; }
  // On to the next segment with keys.
  template <int KEYS>
  __device__ __forceinline__ void next(const PagedArgs& a) {
    if (!a.whole) x += n + a.unit;
    do {
      if (a.whole) x++;
      if (x >= x1) return;
      if (++ri == a.rt) {
        ri = 0;
        if (++kh == a.KH) {
          kh = 0, b++;
          seq<KEYS>(a, ahead);
        }
      }
    } while (n == 0);   // where units are cut, x < x1: there is another one with keys
    j = 0;
    j1 = a.whole ? n : (int)min((long long)n, x1 - x);
  }
};

// Quotients of numbers that are not negative, in one place: that of 64 bits is long
// in code and time, and seldom needed.
__device__ __noinline__ long long paged_div(long long x, long long y) {
  return (unsigned long long)(x | y) >> 32 ? x / y : (long long)((unsigned)x / (unsigned)y);
}

// The group of n that place x of `total` falls to: group i has [i total / n, (i + 1) total / n).
__device__ __forceinline__ int paged_group(long long x, long long total, int n) { return (int)paged_div((x + 1) * n - 1, total); }

constexpr int PG_MOST = 12;     // warps of a CTA, at most
struct PagedShared {
  float4 ml[PG_MOST][8];        // each warp's m, l, r of 8 rows
  long long sums[PG_MOST], x[PG_MOST], before[PG_MOST];   // each group's first place, the places before its first sequence
  int b0[PG_MOST];                                         // and that
};

// MANY: more than one query of a sequence (the code that keeps apart what some
// see, although it is hardly ever run, takes 100 instructions of each tile's 880).
template <typename T, bool CODES, int HD, int NT, bool MANY>
__global__ void __launch_bounds__((PagedShape<T, CODES, HD, NT>::THREADS), 1) paged_kernel(const PagedArgs a) {
  using S = PagedShape<T, CODES, HD, NT>;
  using M = typename S::M;
  constexpr int KEYS = S::KEYS;
  constexpr float OFF = AttnRange<M>::OFF, LIFT = AttnRange<M>::LIFT;
  extern __shared__ __align__(128) uint8_t dsm[];
  __shared__ PagedShared sh;
  const int tid = threadIdx.x, wid = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int HU = a.KH * a.rt;
  const int mate = wid % a.team, group = (blockIdx.x * S::WARPS + wid) / a.team, groups = gridDim.x * S::WARPS / a.team;
  pdl_wait();
  pdl_trigger();
  // Where this group's tiles begin.
  PagedWalk wk{};
  long long total;
  int parts;   // the groups that have any
  wk.j = wk.j1 = 0;
  if (a.whole) {
    total = (long long)a.B * HU;
    parts = (int)min((long long)groups, total);
    wk.x = group < parts ? paged_div(total * group, parts) : total;
    wk.x1 = group < parts ? paged_div(total * (group + 1), parts) : total;
    if (wk.more()) {
      wk.b = (int)paged_div(wk.x, HU);
      wk.seq<KEYS>(a, wk.len_of(a, wk.b));
      const int hu = (int)(wk.x - (long long)wk.b * HU);
      wk.kh = hu / a.rt, wk.ri = hu % a.rt;
      wk.j1 = wk.n;
      if (wk.n == 0) wk.next<KEYS>(a);
    }
  } else {
    if (mate == 0 && lane == 0) a.desc[group].x = -1;
    // the places of each sequence, those before it: a prefix sum of as many sequences as threads at a time
    long long round = 0, mine, before;
    auto scan = [&](int b) {
      const int n = b < a.B ? paged_tiles(min(max(a.lens[b], 0), a.max_len), a.n, a.window, KEYS) : 0;
      mine = n ? (long long)(n + a.unit) * HU : 0;
      long long y = mine;
      for (int o = 1; o < 32; o <<= 1) {
        const long long z = __shfl_up_sync(~0u, y, o);
        if (lane >= o) y += z;
      }
      __syncthreads();
      if (lane == 31) sh.sums[wid] = y;
      __syncthreads();
      before = round + y - mine;
#pragma unroll
      for (int i = 0; i < S::WARPS; i++) {
        const long long z = sh.sums[i];
        if (i < wid) before += z;
        round += z;
      }
    };
#pragma unroll 1
    for (int first = 0; first < a.B; first += S::THREADS) scan(first + tid);
    total = round;
    // a group has two tiles for each warp at least
    parts = (int)max(1ll, min((long long)groups, paged_div(total, 2 * a.team + a.unit)));
    const bool some = group < parts && total > 0;
    wk.x = some ? paged_div(total * group, parts) : total;
    wk.x1 = some ? paged_div(total * (group + 1), parts) : total;
    if (lane == 0) sh.x[wid] = wk.x;
    if (a.B > S::THREADS) round = 0;
#pragma unroll 1
    for (int first = 0; first < a.B; first += S::THREADS) {
      if (a.B > S::THREADS) scan(first + tid);   // of more sequences than threads: once more, now that the sum is known
      __syncthreads();
#pragma unroll 1
      for (int i = 0; i < S::WARPS; i += a.team) {
        const long long x = sh.x[i];
        if (before <= x && x < before + mine) sh.b0[i] = first + tid, sh.before[i] = before;
      }
    }
    __syncthreads();
    if (some) {
      wk.b = sh.b0[wid - mate];
      wk.seq<KEYS>(a, wk.len_of(a, wk.b));
      const long long r = wk.x - sh.before[wid - mate], hu = paged_div(r, wk.n + a.unit);
      wk.kh = (int)hu / a.rt, wk.ri = (int)hu % a.rt;
      wk.j = (int)(r - hu * (wk.n + a.unit));
      wk.x -= wk.j;
      if (wk.j < wk.n)
        wk.j1 = (int)min((long long)wk.n, wk.x1 - wk.x);
      else   // behind the unit's tiles
        wk.next<KEYS>(a);
    }
  }

  uint8_t* ring = dsm + wid * (S::D * S::SLOT);
  const uint32_t ring32 = smem_u32(ring);

  // Loads: a walk of its own, D - 1 of this warp's tiles ahead.
  PagedWalk lw = wk;
  int lj = wk.j + mate, put = 0, ids[S::U];   // its tile, its place in the ring, its parts' numbers of pages
  constexpr int PER = 32 / S::CH;             // rows of a warp's load
  const int r0 = lane / S::CH, c0 = lane % S::CH;
  const bool col = c0 * 16 < a.hd * (CODES ? 1 : 2);
  const uint32_t to0 = S::at(r0, c0);         // this lane's word of row r0; of row r0 + i: i rows on, and bits 4 to 6 differ by i & 6
  const uint8_t *lk = nullptr, *lv = nullptr;   // this lane's words of the unit's key head
  const float* ls = nullptr;                    // lanes 0 .. 2 U - 1: the scales of K and V of part lane / 2
  const unsigned s_page = lane & 1 ? a.svs[0] : a.sks[0], s_block = lane & 1 ? a.svs[2] : a.sks[2];
  auto head = [&]() {
    if (!lw.more()) return;
    lk = a.kp + 16 * ((uint64_t)lw.kh * a.skp[1] + (uint64_t)r0 * a.skp[2] + c0);
    lv = a.vp + 16 * ((uint64_t)lw.kh * a.svp[1] + (uint64_t)r0 * a.svp[2] + c0);
    if (CODES) ls = lane & 1 ? a.vs + (uint64_t)lw.kh * a.svs[1] : a.ks + (uint64_t)lw.kh * a.sks[1];
    // and its queries, for begin() in a tile or two: a lane has a line
    const int row = lw.ri * (8 * NT) + lane % (8 * NT);
    if (row < a.rows && (HD > 64 || lane < 8 * NT)) {
      const int i = query_of(a, row);
      const T* q = (const T*)a.q + lw.b * a.sq[0] + i * a.sq[1] + (lw.kh * a.G + row - i * a.G) * a.sq[2];
      asm volatile("prefetch.global.L1 [%0];" ::"l"(q + (lane >= 8 * NT && a.hd > 64 ? 64 : 0)));
    }
  };
  auto load = [&]() {
    if (lw.more()) {
      const uint32_t slot = ring32 + put * S::SLOT;
      const int key0 = (lw.lo & ~15) + lj * KEYS;
      int there = 0;
#pragma unroll
      for (int u = 0; u < S::U; u++) {
        const int key = key0 + 16 * u;
        const unsigned row = key & ((1 << a.shift) - 1);
        const bool ok = (unsigned)ids[u] < (unsigned)a.n_pages;
        const unsigned page = ok ? ids[u] : 0;
        const int lo = lw.lo - key - r0, n = ok && col ? lw.len - lw.lo : 0;   // rows [lo, lo + n) from this lane's first on are there
        there |= (int)ok << u;
        const uint8_t* k = lk + 16 * ((uint64_t)page * a.skp[0] + (uint64_t)row * a.skp[2]);
        const uint8_t* v = lv + 16 * ((uint64_t)page * a.svp[0] + (uint64_t)row * a.svp[2]);
#pragma unroll
        for (int i = 0; i < 16; i += PER) {
          const bool in = (unsigned)(i - lo) < (unsigned)n;
          const uint32_t to = slot + (16 * u + i) * S::RB + (to0 ^ (i & 6) << 4);
          cp16(to, k, in);
          cp16(to + S::HALF, v, in);
          k += PER * 16 * (uint64_t)a.skp[2];
          v += PER * 16 * (uint64_t)a.svp[2];
        }
      }
      if (CODES && lane < 2 * S::U) {
        const int u = lane >> 1, id = S::U > 1 && u ? ids[S::U - 1] : ids[0];
        const bool ok = (unsigned)id < (unsigned)a.n_pages;
        const unsigned block = ((key0 + 16 * u) & ((1 << a.shift) - 1)) / PAGED_BLOCK;
        cp4(slot + 2 * S::HALF + 4 * lane, ls + (uint64_t)(ok ? id : 0) * s_page + (uint64_t)block * s_block, ok);
      }
      if (lane == 0) *reinterpret_cast<int*>(ring + put * S::SLOT + 2 * S::HALF + 16) = there;
      if (++put == S::D) put = 0;
      lj += a.team;
    }
    cp_commit();
  };
  // On to the next tile, and its pages, whose numbers have until the next load to come.
  const int* row_of = nullptr;
  auto look = [&](bool again) {
    while (lw.more() && (again || lj >= lw.j1)) {   // tiles behind the segment's end are the next one's
      if (!again) {
        const int over = lj - lw.j1;
        lw.next<KEYS>(a);
        lj = lw.j + over;
      }
      again = false;
      row_of = a.tables + (long long)lw.b * a.st;
      head();
    }
#pragma unroll
    for (int u = 0; u < S::U; u++) {
      const int key = (lw.lo & ~15) + lj * KEYS + 16 * u;
      ids[u] = lw.more() && key < lw.len && (key >> a.shift) < a.cols ? row_of[key >> a.shift] : -1;
    }
  };
  int tj = wk.j + mate, get = 0;
  // this lane's words in the ring: K of key g, words t4 and t4 + 4; V of the keys 2 t4 and 2 t4 + 1
  const uint32_t ko0 = S::at(g, t4), ko1 = S::KC > 1 ? S::at(g, t4 + 4) : 0;
  const uint32_t vo0 = S::RB == 64 ? S::at(2 * t4, g >> 1) + (g & 1) * 8 : S::at(2 * t4, g);
  const uint32_t vo1 = S::RB == 64 ? S::at(2 * t4 + 1, g >> 1) + (g & 1) * 8 : S::at(2 * t4 + 1, g);
  uint32_t qf[NT][S::STEPS][2];
  float f[NT][2];      // scale log2(e) of this lane's columns' scores, over the power of two in q
  int tok[NT][2];      // their queries
  float o[NT][S::STEPS][4], m[NT][2], r[NT][2], l[NT][2];   // r: the accumulators' reference (CODES)
  float nm[NT][2], nr[NT][2], limm[NT][2], limr[NT][2];     // OFF - m, and m + LIFT
  int row0, base;      // the unit's first row, the position of the first query
  // Q^T as B fragments; the rows are columns, absent ones and dimensions zero.
  // A lane's 16-byte words of a key are t4, t4 + 4, ..; their values in turn are
  // the steps' dimensions.
  auto begin = [&]() {
    row0 = wk.ri * (8 * NT), base = wk.len - a.n;
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int row = row0 + t * 8 + g, i = query_of(a, min(row, a.rows - 1));
      const T* q = (const T*)a.q + wk.b * a.sq[0] + i * a.sq[1] + (wk.kh * a.G + min(row, a.rows - 1) - i * a.G) * a.sq[2];
#pragma unroll
      for (int k = 0; k < S::STEPS; k++)
#pragma unroll
        for (int z = 0; z < 2; z++) {
          constexpr int PW = S::STEPS / S::KC;   // steps of a word
          const int d = (t4 + 4 * (k / PW)) * (4 * PW) + (k % PW) * 4 + z * 2;
          qf[t][k][z] = row < a.rows && d < a.hd ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
        }
      f[t][0] = f[t][1] = a.c;
      if (CODES && std::is_same<T, __nv_bfloat16>::value) {
        uint32_t top = 0;   // bits of the largest finite value
#pragma unroll
        for (int k = 0; k < S::STEPS; k++)
#pragma unroll
          for (int z = 0; z < 2; z++) {
            const uint32_t x = qf[t][k][z] & 0x7fffu, y = qf[t][k][z] >> 16 & 0x7fffu;
            top = max(top, max(x < 0x7f80u ? x : 0u, y < 0x7f80u ? y : 0u));
          }
        top = max(top, __shfl_xor_sync(~0u, top, 1));
        top = max(top, __shfl_xor_sync(~0u, top, 2));
        const int up = min(14 + 127 - (int)(top >> 7), 126);
        const float s = __int_as_float((up + 127) << 23);
#pragma unroll
        for (int k = 0; k < S::STEPS; k++)
#pragma unroll
          for (int z = 0; z < 2; z++)
            qf[t][k][z] = at_pack<__half>(__uint_as_float(qf[t][k][z] << 16) * s, __uint_as_float(qf[t][k][z] & 0xffff0000u) * s);
#pragma unroll
        for (int z = 0; z < 2; z++) f[t][z] = a.c * __int_as_float((127 - __shfl_sync(~0u, up, (t4 * 2 + z) * 4)) << 23);
      }
#pragma unroll
      for (int z = 0; z < 2; z++) {
        tok[t][z] = query_of(a, min(row0 + t * 8 + t4 * 2 + z, a.rows - 1));
        m[t][z] = r[t][z] = limm[t][z] = limr[t][z] = -INFINITY;
        nm[t][z] = nr[t][z] = l[t][z] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < S::STEPS; k++) o[t][k][0] = o[t][k][1] = o[t][k][2] = o[t][k][3] = 0.f;
    }
  };
  // This warp's next tile.
  auto tile = [&]() {
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
        const uint32_t from = kb + 16 * u * S::RB + w / 2 * 128 + (w % 2 ? ko1 : ko0);
        const uint4 lo4 = lds16(from), hi4 = lds16(from + 8 * S::RB);
        const uint32_t lo[4] = {lo4.x, lo4.y, lo4.z, lo4.w}, hi[4] = {hi4.x, hi4.y, hi4.z, hi4.w};
        constexpr int PW = S::STEPS / S::KC;
#pragma unroll
        for (int s = 0; s < PW; s++) {
          uint32_t fr[4];
          if (CODES)
            pg_codes(lo[s], fr[0], fr[2]), pg_codes(hi[s], fr[1], fr[3]);
          else
            fr[0] = lo[2 * s & 3], fr[1] = hi[2 * s & 3], fr[2] = lo[2 * s + 1 & 3], fr[3] = hi[2 * s + 1 & 3];
#pragma unroll
          for (int t = 0; t < NT; t++) pg_mma<M>(x[u][t], fr, qf[t][w * PW + s][0], qf[t][w * PW + s][1]);
        }
      }
    }
    // scores in base 2, and (CODES) what they become with the values' scale; those that a row does not see: -inf
    const int there = reinterpret_cast<const int*>(extra)[4];
    const bool part = there != (1 << S::U) - 1 || k0 < (a.window > 0 ? wk.len - a.window : 0) || k0 + KEYS > base + 1;   // not all rows see all keys
    float y[CODES ? S::U : 1][NT][4];
#pragma unroll
    for (int u = 0; u < S::U; u++) {
      const float sk = CODES ? extra[2 * u] : 1.f, lv = CODES ? __log2f(extra[2 * u + 1]) : 0.f;
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const float ft[2] = {CODES ? f[t][0] * sk : f[t][0], CODES ? f[t][1] * sk : f[t][1]};
#pragma unroll
        for (int z = 0; z < 4; z++) {
          x[u][t][z] *= ft[z & 1];
          if (CODES) y[u][t][z] = x[u][t][z] + lv;
        }
      }
    }
    if (part) {
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int z = 0; z < 2; z++) {
          const int hi = base + tok[t][z], lo = a.window > 0 && hi >= a.window ? hi - a.window + 1 : 0;   // the keys that the row sees
#pragma unroll
          for (int u = 0; u < S::U; u++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const int key = k0 + 16 * u + g + h * 8;
              if (!(there >> u & 1) || key > hi || key < lo) {
                x[u][t][z + 2 * h] = -INFINITY;
                if (CODES) y[u][t][z + 2 * h] = -INFINITY;
              }
            }
        }
    }
    float top[NT][2], topy[NT][2];   // of the lane's keys; NaN where no score is a number, which counts as none
    bool up = false;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int z = 0; z < 2; z++) {
        top[t][z] = fmaxf(x[0][t][z], x[0][t][z + 2]);
        if (S::U > 1) top[t][z] = fmaxf(top[t][z], fmaxf(x[S::U - 1][t][z], x[S::U - 1][t][z + 2]));
        up |= top[t][z] > limm[t][z];
        if (CODES) {
          topy[t][z] = fmaxf(y[0][t][z], y[0][t][z + 2]);
          if (S::U > 1) topy[t][z] = fmaxf(topy[t][z], fmaxf(y[S::U - 1][t][z], y[S::U - 1][t][z + 2]));
          up |= topy[t][z] > limr[t][z];
        }
      }
    if (__any_sync(~0u, up)) {
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int z = 0; z < 2; z++) {
          float v = top[t][z], w = CODES ? topy[t][z] : 0.f;
#pragma unroll
          for (int sft = 4; sft < 32; sft <<= 1) {
            v = fmaxf(v, __shfl_xor_sync(~0u, v, sft));
            if (CODES) w = fmaxf(w, __shfl_xor_sync(~0u, w, sft));
          }
          if (!CODES) w = v;
          const bool um = v > limm[t][z], ur = CODES ? w > limr[t][z] : um;   // rows move by their own scores alone
          const float mn = um ? v : m[t][z], rn = ur ? w : r[t][z];
          const float fm = um ? at_exp2(m[t][z] - mn) : 1.f, fr = ur ? at_exp2(r[t][z] - rn) : 1.f;
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
    uint32_t p[S::U][NT][2], pl[S::U][NT][2];   // the weights, and what their rounding drops
#pragma unroll
    for (int u = 0; u < S::U; u++)
#pragma unroll
      for (int t = 0; t < NT; t++) {
        float e[4];
#pragma unroll
        for (int z = 0; z < 4; z++) {
          e[z] = at_exp2(x[u][t][z] + nm[t][z & 1]);
          l[t][z & 1] += e[z];
          if (CODES) e[z] = at_exp2(y[u][t][z] + nr[t][z & 1]);
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const uint32_t w = at_pack<M>(e[2 * h], e[2 * h + 1]);
          const float2 y = pg_halves<M>(w);
          p[u][t][h] = pg_movm(w);
          pl[u][t][h] = pg_movm(at_pack<M>(e[2 * h] - y.x, e[2 * h + 1] - y.y));
        }
      }
    // O^T += V^T P^T: a lane has the keys 2 t4, 2 t4 + 1 and those 8 on, and
    // HD / 8 dimensions of each; two keys' values of a dimension make a register
#pragma unroll
    for (int u = 0; u < S::U; u++) {
      constexpr int W = HD / 8 * (CODES ? 1 : 2) / 4;   // 32-bit words of a key that a lane has: 2, 4 or 8
      uint32_t v[4][W];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t from = vb + (16 * u + 8 * (i >> 1)) * S::RB + (i & 1 ? vo1 : vo0);
        if (W == 2) {
          const uint2 y = lds8(from);
          v[i][0] = y.x, v[i][W - 1] = y.y;
        } else {
#pragma unroll
          for (int h = 0; h < W / 4; h++) {
            const uint4 y = lds16(from + 128 * h);
            v[i][4 * h] = y.x, v[i][4 * h + 1] = y.y, v[i][4 * h + 2] = y.z, v[i][4 * h + 3] = y.w;
          }
        }
      }
      auto part_of = [&](int k, uint32_t (&fr)[4]) {   // dimensions 2 k and 2 k + 1 of the lane's
        if (CODES) {
          const uint32_t sel = k & 1 ? 0x7362u : 0x5140u;
          pg_codes(__byte_perm(v[0][k / 2], v[1][k / 2], sel), fr[0], fr[1]);
          pg_codes(__byte_perm(v[2][k / 2], v[3][k / 2], sel), fr[2], fr[3]);
        } else {
          const int w = k % W;
          fr[0] = __byte_perm(v[0][w], v[1][w], 0x5410), fr[1] = __byte_perm(v[0][w], v[1][w], 0x7632);
          fr[2] = __byte_perm(v[2][w], v[3][w], 0x5410), fr[3] = __byte_perm(v[2][w], v[3][w], 0x7632);
        }
      };
      uint32_t odd = 0;   // values that are not finite, where some rows may see a key and others not: 0 x NaN must not reach those
      if (MANY && part) {
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
      if (!MANY || !odd) {
#pragma unroll
        for (int k = 0; k < S::STEPS; k++) {
          uint32_t fr[4];
          part_of(k, fr);
#pragma unroll
          for (int t = 0; t < NT; t++) {
            pg_mma<M>(o[t][k], fr, p[u][t][0], p[u][t][1]);
            pg_mma<M>(o[t][k], fr, pl[u][t][0], pl[u][t][1]);
          }
        }
      } else {   // each query by itself, the keys that it does not see cleared
#pragma unroll 1
        for (int i = query_of(a, row0); i <= query_of(a, min(row0 + 8 * NT, a.rows) - 1); i++) {
          const int hi = base + i, lo = a.window > 0 && hi >= a.window ? hi - a.window + 1 : 0;
          uint32_t keep[2] = {0u, 0u};
#pragma unroll
          for (int h = 0; h < 4; h++) {
            const int key = k0 + 16 * u + 2 * t4 + (h & 1) + (h >> 1) * 8;
            if (key <= hi && key >= lo) keep[h >> 1] |= h & 1 ? 0xffff0000u : 0xffffu;
          }
#pragma unroll
          for (int k = 0; k < S::STEPS; k++) {
            uint32_t fr[4];
            part_of(k, fr);
            fr[0] &= keep[0], fr[1] &= keep[0], fr[2] &= keep[1], fr[3] &= keep[1];
#pragma unroll
            for (int t = 0; t < NT; t++) {
              float y[4] = {0.f, 0.f, 0.f, 0.f};
              pg_mma<M>(y, fr, p[u][t][0], p[u][t][1]);
              pg_mma<M>(y, fr, pl[u][t][0], pl[u][t][1]);
#pragma unroll
              for (int z = 0; z < 4; z++)
                if (tok[t][z & 1] == i) o[t][k][z] += y[z];
            }
          }
        }
      }
    }
  };
  // The segment's end: the warps' results join, 8 rows at a time; a whole unit
  // becomes outputs, a part of one a piece for the second kernel.
  auto end = [&]() {
    const bool all = wk.j == 0 && wk.j1 == wk.n;
    const size_t slot = 2 * group + (wk.j == 0);
    if (!all && wk.j == 0 && mate == 0 && lane == 0)
      a.desc[group] = make_int4(wk.b, wk.kh * a.rt + wk.ri, paged_group(wk.x + wk.n - 1, total, parts), 0);
    if (a.team == 1) {   // a unit that was not cut, from the registers
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int z = 0; z < 2; z++) {
          float L = l[t][z], mm = m[t][z] - OFF;
#pragma unroll
          for (int sft = 4; sft < 32; sft <<= 1) L += __shfl_xor_sync(~0u, L, sft);
          const int row = row0 + t * 8 + t4 * 2 + z;
          if (row >= a.rows) continue;
          const int head = wk.kh * a.G + row - tok[t][z] * a.G;
          if (a.sinks) {
            const float sink = sink_of(a, head), top = fmaxf(mm, sink);
            if (sink != -INFINITY) L = (L == 0.f ? 0.f : L * at_exp2(mm - top)) + at_exp2(sink - top), mm = top;
          }
          const float f = paged_factor(L, r[t][z] - OFF - mm);
          T* out = (T*)a.out + wk.b * a.so[0] + tok[t][z] * a.so[1] + head * a.so[2];
#pragma unroll
          for (int k = 0; k < S::STEPS; k += 4) {   // eight dimensions in a row
            const int d = S::dim(k, g);
            if (d < a.hd)
              *reinterpret_cast<uint4*>(out + d) = make_uint4(at_pack<T>(o[t][k][z] * f, o[t][k][z + 2] * f), at_pack<T>(o[t][k + 1][z] * f, o[t][k + 1][z + 2] * f),
                                                              at_pack<T>(o[t][k + 2][z] * f, o[t][k + 2][z + 2] * f), at_pack<T>(o[t][k + 3][z] * f, o[t][k + 3][z + 2] * f));
          }
        }
      return;
    }
    auto meet = [&]() {   // the group's warps
      asm volatile("bar.sync %0, %1;" ::"r"(1 + wid / a.team), "r"(32 * a.team) : "memory");
    };
    // each warp's accumulators lie in the place of its ring that is free
    float* red = reinterpret_cast<float*>(ring + put * S::SLOT);
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
      for (int z = 0; z < 2; z++) {
#pragma unroll
        for (int sft = 4; sft < 32; sft <<= 1) l[t][z] += __shfl_xor_sync(~0u, l[t][z], sft);
        if (g == 0) sh.ml[wid][t4 * 2 + z] = make_float4(m[t][z] - OFF, l[t][z], r[t][z] - OFF, __int_as_float(put));
#pragma unroll
        for (int k = 0; k < S::STEPS; k++)
          *reinterpret_cast<float2*>(&red[(t4 * 2 + z) * S::RP + 16 * k + 2 * g]) = make_float2(o[t][k][z], o[t][k][z + 2]);
      }
      meet();
      // Each warp: lane 8 w + h has warp w's share of row h, then the row's factors.
      const int w0 = wid - mate, h8 = row0 + t * 8 + (lane & 7), mine = lane >> 3;
      const float4 ml = mine < a.team ? sh.ml[w0 + mine][lane & 7] : make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
      const bool has = ml.y != 0.f;   // a warp with keys
      float sink = -INFINITY;
      if (a.sinks && all && h8 < a.rows) sink = sink_of(a, wk.kh * a.G + h8 - query_of(a, h8) * a.G);
      float mm = has ? ml.x : -INFINITY, rr = has ? ml.z : -INFINITY;
#pragma unroll
      for (int sft = 8; sft < 32; sft <<= 1) mm = fmaxf(mm, __shfl_xor_sync(~0u, mm, sft)), rr = fmaxf(rr, __shfl_xor_sync(~0u, rr, sft));
      mm = fmaxf(mm, sink);
      const float fr = has && ml.z != -INFINITY ? at_exp2(ml.z - rr) : 0.f;
      float L = has ? ml.y * at_exp2(ml.x - mm) : 0.f;
#pragma unroll
      for (int sft = 8; sft < 32; sft <<= 1) L += __shfl_xor_sync(~0u, L, sft);
      if (sink != -INFINITY) L += at_exp2(sink - mm);
      const float fin = paged_factor(L, rr - mm);
      uint32_t from[4];   // this lane's first pair of each warp
#pragma unroll
      for (int w = 0; w < 4; w++)
        from[w] = smem_u32(dsm) + ((w0 + (w < a.team ? w : 0)) * S::D + __shfl_sync(~0u, __float_as_int(ml.w), w < a.team ? 8 * w : 0)) * S::SLOT + 8 * lane;
#pragma unroll 1
      for (int i = mate * 32; i < 4 * HD; i += 32 * a.team) {
        const int h = i / (HD / 2), at = i % (HD / 2), row = row0 + t * 8 + h;   // pairs from `at` on of row h
        if (row >= a.rows) break;
        float2 v = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; w++) {
          const float f = __shfl_sync(~0u, fr, 8 * w + h);
          const uint2 y = lds8(from[w] + (h * S::RP + 2 * at) * 4);
          if (w < a.team) v.x = fmaf(__uint_as_float(y.x), f, v.x), v.y = fmaf(__uint_as_float(y.y), f, v.y);   // NaN under a weight of 0 too
        }
        if (all) {
          const int query = query_of(a, row), d = S::dim((at + lane) / 8, lane % 8);
          const float f = __shfl_sync(~0u, fin, h);
          if (d < a.hd)
            *reinterpret_cast<uint32_t*>((T*)a.out + wk.b * a.so[0] + query * a.so[1] + (wk.kh * a.G + row - query * a.G) * a.so[2] + d) = at_pack<T>(v.x * f, v.y * f);
        } else {
          *reinterpret_cast<float2*>(a.po + (slot * (8 * NT) + t * 8 + h) * HD + 2 * (at + lane)) = v;
        }
      }
      if (!all && mate == 0 && lane < 8) a.pml[slot * (8 * NT) + t * 8 + lane] = make_float4(mm, L, rr, 0.f);
      meet();
    }
  };

  // D - 1 loads, then for each tile one load more; whoever has no tile left in
  // a segment goes to its end.  Each part stands here once: the code is large
  // (with copies of its parts it was 150 KB, and its fetching took most of the
  // time: 256 sequences 403 us).
  int ahead = 0;
  bool fresh = true;   // a segment that has not begun
  look(true);
#pragma unroll 1
  while (wk.more()) {
    if (++ahead >= S::D) {
#pragma unroll 1
      while (true) {
        if (fresh) begin();
        fresh = tj >= wk.j1;
        if (!fresh) break;
        end();
        tj -= wk.j1;
        wk.next<KEYS>(a);
        if (!wk.more()) break;
      }
      if (fresh) break;   // no more segments
    }
    load();
    look(false);
    if (ahead < S::D) continue;
    cp_wait<S::D - 1>();
    __syncwarp();
    tile();
    __syncwarp();   // before the next load into this place
    if (++get == S::D) get = 0;
    tj += a.team;
  }
  cp_wait<0>();
  // Sequences without a key.
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    if (paged_tiles(min(max(a.lens[b], 0), a.max_len), a.n, a.window, KEYS) > 0) continue;
    const int words = a.hd / 8, H = a.KH * a.G;
    for (int i = tid; i < a.n * H * words; i += S::THREADS) {
      T* out = (T*)a.out + b * a.so[0] + i / words / H * a.so[1] + i / words % H * a.so[2] + i % words * 8;
      *reinterpret_cast<uint4*>(out) = make_uint4(0, 0, 0, 0);
    }
  }
}

// Block (i, y): rows 2 y and 2 y + 1 of the unit that begins in group i and ends
// in a later one, the pieces' weighted sum: four warps have every fourth piece
// each (a long sequence by itself lies in a hundred of them).
template <typename T, bool CODES, int HD, int NT>
__global__ void __launch_bounds__(PG_JOIN_THREADS) paged_join_kernel(const PagedArgs a) {
  __shared__ float2 part[PG_JOIN_THREADS / 32][HD / 2];
  __shared__ float sums[PG_JOIN_THREADS / 32];
  pdl_wait();
  const int i = blockIdx.x, lane = threadIdx.x & 31, wid = threadIdx.x >> 5, w4 = wid & 3, h = 2 * blockIdx.y + (wid >> 2);
  const int4 d = a.desc[i];
  if (d.x < 0) return;
  const int kh = d.y / a.rt, row = d.y % a.rt * (8 * NT) + h, pieces = d.z - i + 1;
  const bool here = row < a.rows;
  const int query = query_of(a, here ? row : 0), head = kh * a.G + (here ? row : 0) - query * a.G;
  auto at = [&](int p) { return (size_t)(p ? 2 * (i + p) : 2 * i + 1) * (8 * NT) + h; };
  const float sink = a.sinks ? sink_of(a, head) : -INFINITY;
  float mm = sink, rr = -INFINITY;
  if (here)
    for (int p = lane; p < pieces; p += 32) {
      const float4 ml = a.pml[at(p)];
      mm = fmaxf(mm, ml.x), rr = fmaxf(rr, ml.z);
    }
#pragma unroll
  for (int sft = 16; sft; sft >>= 1) mm = fmaxf(mm, __shfl_xor_sync(~0u, mm, sft)), rr = fmaxf(rr, __shfl_xor_sync(~0u, rr, sft));
  float L = 0.f;
  float2 v[HD / 64];
#pragma unroll
  for (int e = 0; e < HD / 64; e++) v[e] = make_float2(0.f, 0.f);
  if (here)
#pragma unroll 4
    for (int p = w4; p < pieces; p += 4) {
      const float4 ml = a.pml[at(p)];
      float2 y[HD / 64];
#pragma unroll
      for (int e = 0; e < HD / 64; e++) y[e] = *reinterpret_cast<const float2*>(a.po + at(p) * HD + 2 * lane + 64 * e);
      const float fm = ml.y == 0.f ? 0.f : at_exp2(ml.x - mm), fr = ml.y == 0.f || ml.z == -INFINITY ? 0.f : at_exp2(ml.z - rr);
      L = fmaf(ml.y, fm, L);   // a sum of NaN, which the maxima pass by, stays one
#pragma unroll
      for (int e = 0; e < HD / 64; e++) v[e].x = fmaf(y[e].x, fr, v[e].x), v[e].y = fmaf(y[e].y, fr, v[e].y);
    }
#pragma unroll
  for (int e = 0; e < HD / 64; e++) part[wid][lane + 32 * e] = v[e];
  if (lane == 0) sums[wid] = L;
  __syncthreads();
  if (w4 || !here) return;
#pragma unroll
  for (int w = 1; w < 4; w++) {
    L += sums[wid + w];
#pragma unroll
    for (int e = 0; e < HD / 64; e++) v[e].x += part[wid + w][lane + 32 * e].x, v[e].y += part[wid + w][lane + 32 * e].y;
  }
  if (sink != -INFINITY) L += at_exp2(sink - mm);
  const float fin = paged_factor(L, rr - mm);
#pragma unroll
  for (int e = 0; e < HD / 64; e++) {
    const int pair = lane + 32 * e, to = PagedShape<T, CODES, HD, NT>::dim(pair / 8, pair % 8);
    if (to < a.hd) *reinterpret_cast<uint32_t*>((T*)a.out + d.x * a.so[0] + query * a.so[1] + head * a.so[2] + to) = at_pack<T>(v[e].x * fin, v[e].y * fin);
  }
}

// What the host settles before the lengths are known.
struct PagedSpace {
  int nt, rt, whole, team = 4, unit, grid, groups;
  size_t po = 0, pml = 0, desc = 0, bytes = 0;
  PagedSpace(int bits, int batch, int queries, int max_len, int window, int H, int KH, int hd, int sms) {
    const int rows = queries * (H / KH), HD = hd <= 64 ? 64 : 128, keys = HD * bits / 8 <= 128 ? 32 : 16;
    nt = rows <= 8 ? 1 : 2;
    rt = (rows + 8 * nt - 1) / (8 * nt);
    const int warps = nt == 1 ? 12 : 8;
    const long long units = (long long)batch * KH * rt;
    // keys that a unit's queries read, at most, from a whole block on
    const long long most = window > 0 ? std::min((long long)max_len, (long long)window + queries + 14) : max_len, tiles = (most + keys - 1) / keys;
    whole = tiles <= 16;
    // A group of four shares a unit's tiles and joins at its end, which costs each
    // of them two to three tiles' time; a warp by itself has no one to wait for, but
    // where units are cut it leaves four times the pieces to the second kernel (64
    // sequences 41 us, with groups of two 38, of four 36).
    if (whole)
      while (team > 1 && (long long)sms * warps / team < units) team /= 2;
    unit = 7 * team / 2;
    const long long want = whole ? units : units * tiles / 2;   // groups that can have work
    grid = (int)std::max(1ll, std::min((long long)sms, (want * team + warps - 1) / warps));
    groups = grid * warps / team;
    if (whole) return;
    auto take = [&](size_t n) {
      const size_t o = bytes;
      bytes = (bytes + n + 255) & ~(size_t)255;
      return o;
    };
    po = take((size_t)2 * groups * 8 * nt * HD * 4);
    pml = take((size_t)2 * groups * 8 * nt * 16);
    desc = take((size_t)groups * 16);
  }
};

template <typename T, bool CODES, int HD, int NT, bool MANY>
static cudaError_t run_paged(const PagedArgs& a, const PagedSpace& sp, cudaStream_t s) {
  const int smem = PagedShape<T, CODES, HD, NT>::SMEM;
  static std::atomic<unsigned long long> set{0};
  cudaError_t e = attn_smem(paged_kernel<T, CODES, HD, NT, MANY>, smem, set);
  if (e == cudaSuccess) e = launch_pdl(paged_kernel<T, CODES, HD, NT, MANY>, dim3(sp.grid), PagedShape<T, CODES, HD, NT>::THREADS, smem, s, a);
  count_launches(1);
  if (e == cudaSuccess && !a.whole && sp.groups > 1) {
    e = launch_pdl(paged_join_kernel<T, CODES, HD, NT>, dim3(sp.groups - 1, 4 * NT), PG_JOIN_THREADS, 0, s, a);
    count_launches(1);
  }
  return e;
}
template <typename T, bool CODES>
static cudaError_t run_paged(const PagedArgs& a, const PagedSpace& sp, cudaStream_t s) {
  const bool many = a.n > 1;
  if (a.hd <= 64) {
    if (sp.nt == 1) return many ? run_paged<T, CODES, 64, 1, true>(a, sp, s) : run_paged<T, CODES, 64, 1, false>(a, sp, s);
    return many ? run_paged<T, CODES, 64, 2, true>(a, sp, s) : run_paged<T, CODES, 64, 2, false>(a, sp, s);
  }
  if (sp.nt == 1) return many ? run_paged<T, CODES, 128, 1, true>(a, sp, s) : run_paged<T, CODES, 128, 1, false>(a, sp, s);
  return many ? run_paged<T, CODES, 128, 2, true>(a, sp, s) : run_paged<T, CODES, 128, 2, false>(a, sp, s);
}

}  // namespace tg

using namespace tg;

extern "C" size_t tg_attention_paged_workspace(int page_bits, int batch, int n_queries, int max_len, int window,
                                               int n_heads, int n_kv_heads, int head_dim) {
  if (batch <= 0 || n_queries <= 0 || max_len <= 0 || max_len >= AT_NPOS || window < 0 || n_kv_heads <= 0 || n_heads < n_kv_heads || n_heads / n_kv_heads > 128 || head_dim <= 0) return 0;
  if ((long long)n_queries * n_heads >= 1 << 24) return 0;
  return PagedSpace(page_bits, batch, n_queries, max_len, window, n_heads, n_kv_heads, head_dim, attn_sms()).bytes;
}

int tg::attention_paged(ArgCheck& c, const AttendRecord& r) {
  c.need(r.dtype == ATTN_BF16 || r.dtype == ATTN_FP16, "dtype must be 0 (bf16) or 1 (fp16)");
  c.need(r.max_len < AT_NPOS, "too many positions");
  need_ints(c, &r.batch, 10);
  c.need(r.batch >= 0 && r.n_queries >= 0 && r.max_len >= 0 && r.window >= 0, "counts and window must not be negative");
  c.need(r.n_heads > 0 && r.n_kv_heads > 0 && r.n_heads % r.n_kv_heads == 0 && r.n_heads / r.n_kv_heads <= 128,
         "n_heads must be a multiple of n_kv_heads, at most 128 times it");
  c.need(r.n_queries * r.n_heads < 1 << 24 && r.batch * r.n_queries * r.n_heads < 1ll << 31, "too many query rows");
  c.need(r.head_dim > 0 && r.head_dim % 8 == 0 && r.head_dim <= ATTN_MAX_HD, "head_dim must be a multiple of 8, at most 128");
  c.need(std::isfinite((float)r.scale) && (float)r.scale > 0.f, "scale must be finite and positive");
  if (c.rc) return c.rc;
  const int batch = (int)r.batch, queries = (int)r.n_queries, H = (int)r.n_heads, KH = (int)r.n_kv_heads, hd = (int)r.head_dim;
  const PoolCheck pool(c, (int)r.page_bits, (int)r.n_pages, (int)r.page, (int)r.table_cols, batch, KH, hd, r.strides + 6);
  const long long n3[3] = {batch, queries, H};
  long long t[6];
  for (int i = 0; i < 6; i++) t[i] = c.stride(r.strides[i], n3[i % 3]);
  c.need(r.max_len <= r.table_cols * r.page, "max_len must be at most table_cols x page");
  if (c.rc || batch == 0 || queries == 0) return c.rc;
  const int max_len = r.n_pages == 0 ? 0 : (int)r.max_len;
  if (!c.device()) return c.rc;
  c.ptr(r.q, 16, "q"), c.ptr(r.out, 16, "out"), c.ptr(r.lens, 4, "lens");
  if (max_len > 0) {
    c.ptr(r.k_pages, 16, "k_pages"), c.ptr(r.v_pages, 16, "v_pages"), c.ptr(r.tables, 4, "tables");
    if (r.page_bits == 8) c.ptr(r.k_scales, 4, "k_scales"), c.ptr(r.v_scales, 4, "v_scales");
  }
  if (r.sinks) c.ptr(r.sinks, 4, "sinks");
  const PagedSpace sp((int)r.page_bits, batch, queries, max_len, (int)r.window, H, KH, hd, attn_sms());
  c.need(r.workspace_bytes >= (int64_t)sp.bytes, "the workspace is smaller than tg_attention_paged_workspace says");
  if (sp.bytes > 0) c.ptr(r.workspace, 256, "workspace");
  if (c.rc) return c.rc;
  uint8_t* ws = static_cast<uint8_t*>(r.workspace);
  PagedArgs a{};
  a.q = r.q, a.kp = (const uint8_t*)r.k_pages, a.vp = (const uint8_t*)r.v_pages, a.ks = (const float*)r.k_scales, a.vs = (const float*)r.v_scales;
  a.tables = (const int*)r.tables, a.lens = (const int*)r.lens, a.sinks = (const float*)r.sinks, a.out = r.out;
  a.po = (float*)(ws + sp.po), a.pml = (float4*)(ws + sp.pml), a.desc = (int4*)(ws + sp.desc);
  for (int i = 0; i < 3; i++) {
    a.sq[i] = t[i], a.so[i] = t[3 + i];
    a.skp[i] = (unsigned)(pool.kp[i] / 16), a.svp[i] = (unsigned)(pool.vp[i] / 16);
    a.sks[i] = (unsigned)pool.ks[i], a.svs[i] = (unsigned)pool.vs[i];
  }
  a.st = pool.st, a.B = batch, a.n = queries, a.G = H / KH, a.KH = KH, a.rows = queries * a.G, a.rt = sp.rt;
  a.by_g = (unsigned)(((1ull << 32) + a.G - 1) / a.G);
  a.hd = hd, a.cols = (int)r.table_cols, a.n_pages = (int)r.n_pages, a.shift = pool.shift, a.max_len = max_len, a.window = (int)r.window;
  a.whole = sp.whole, a.team = sp.team, a.unit = sp.unit, a.c = (float)r.scale * LOG2E;
  cudaStream_t s = static_cast<cudaStream_t>(r.stream);
  if (r.dtype == ATTN_BF16)
    return c.done(r.page_bits == 8 ? run_paged<__nv_bfloat16, true>(a, sp, s) : run_paged<__nv_bfloat16, false>(a, sp, s));
  return c.done(r.page_bits == 8 ? run_paged<__half, true>(a, sp, s) : run_paged<__half, false>(a, sp, s));
}

extern "C" int tg_attention_paged(int dtype, int page_bits, const void* q, const void* k_pages, const void* v_pages,
                                  const float* k_scales, const float* v_scales, void* out, const int* tables,
                                  const int* lens, const float* sinks, int batch, int n_queries, int n_pages, int page,
                                  int table_cols, int max_len, int n_heads, int n_kv_heads, int head_dim,
                                  const int64_t* strides, int window, float scale, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  ArgCheck c("tg_attention_paged");
  if (!c.need(strides != nullptr, "strides is null")) return c.rc;
  AttendRecord r{2, dtype, page_bits, q, k_pages, v_pages, k_scales, v_scales, out, tables, lens, sinks, batch, n_queries, n_pages, page,
                 table_cols, max_len, n_heads, n_kv_heads, head_dim, window, {}, scale, workspace, (int64_t)workspace_bytes, stream};
  std::copy(strides, strides + 19, r.strides);
  return attention_paged(c, r);
}
