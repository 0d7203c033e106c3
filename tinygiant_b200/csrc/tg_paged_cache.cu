// tg_paged_cache.cu — what stands around attention over a paged cache:
//   tg_rotary        queries and keys rotated by their positions
//   tg_paged_append  new tokens' keys (rotated) and values written to their pages
//   tg_paged_gather  pages read back as packed rows
//
// Norm:      x <- x / sqrt(mean x^2 + eps) w over a head's dimensions, where
//            weights are given.
// Rotation:  a head's first 2 n dimensions are n pairs, (j, j + n) or
//            (2 j, 2 j + 1); pair j of position p turns by p f_j:
//            a <- s (a cos - b sin), b <- s (b cos + a sin).
// All in fp32 and rounded once.  The angle is taken in turns in 64 bits, its product
// with the position whole, and reduced there to an eighth of a turn: in 32 bits a
// position of 100,000 would leave a sine 7 bits.
//
// Pages of 8 bits (e4m3) have a scale for each key head and block of 16 tokens,
// a power of two: e4m3 keeps 4 bits of every value whatever the factor, so a
// finer scale gains nothing but the exact top of its range, and a block whose
// scale grows when a larger token comes keeps its earlier codes' bits (but for
// those that fall below the format's least normal value).
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "../../include/tinygiant.h"
#include "tg_attn_tc.cuh"
#include "tg_paged.h"

namespace tg {

constexpr int PC_THREADS = 256;
constexpr int PC_WARPS = PC_THREADS / 32;
constexpr int PC_PER_SM = 3;      // CTAs of an SM (with 4, and 64 registers: 8,192 tokens x 36 heads rotated in 31 us instead of 26, 2,048 tokens to 8-bit pages 18 instead of 15; keys and values alone 14 instead of 18)
constexpr int PC_PAIRS = ATTN_MAX_HD / 2;   // pairs of a head, at most
static_assert(PC_THREADS == 4 * PC_PAIRS, "angles of four tokens at a time");
constexpr int PC_CU = 1024;       // sequences whose offsets are kept in shared memory
constexpr int PC_WINDOW = 16;     // packed tokens that a CTA looks through for blocks' first ones, at most
constexpr int PC_TOKENS = 32;     // tokens of a CTA that rotates, at most
constexpr int PC_GATHERS = 5;     // gather CTAs of an SM
constexpr int PC_GATHER = 32;     // tokens of a gather CTA, at most
// A thread has R = 2 or 3 rows of a token; pc_ahead tokens' rows are there or on
// their way.
template <int R>
constexpr int pc_ahead = R == 2 ? 4 : 3;
template <int R>
constexpr int pc_ring_bytes = pc_ahead<R>* R * 16 * PC_THREADS;
static_assert(std::min(pc_ring_bytes<2>, pc_ring_bytes<3>) >= PAGED_BLOCK * ATTN_MAX_HD * 2 * PC_WARPS, "a warp's run of a head");

enum { PC_ROTARY, PC_PAGES16, PC_PAGES8 };

struct CacheArgs {
  const void *q, *k, *v;
  void *qo, *ko;              // rotated q (append: if q is there) and k (tg_rotary)
  uint8_t *kp, *vp;           // pages
  float *ks, *vs;             // scales of 8-bit pages
  const int *tables, *lens, *cu, *positions;
  const double* freqs;
  const float *qw, *kw;       // weights of the norms, or null
  long long sq[2], sk[2], sv[2], sqo[2], sko[2];   // token, head; elements
  long long skp[3], svp[3];   // page, head, row; bytes
  long long sks[3], svs[3];   // page, head, block
  long long st;               // tables' row
  int T, B, per, H, KH, hd, nf, n_pages, cols, shift, token_ctas, window, tokens, parts, each;
  int interleaved;
  double amp, eps64, inv_hd64;   // as they were given; 1 / hd
  float eps, inv_hd;
};

// p f radians in turns, as whole quarters and a rest of an eighth at most.  f / 2 pi is
// a sum of two doubles and the product with p is kept whole, so the rest is off by
// 2^-56 of a turn as long as there are 2^50 of them at most, beyond by 2^-106 of all.
struct Turn {
  int quarters;   // modulo 4
  double rest;
  __device__ __forceinline__ Turn(int p, double f) {
    const double per = 0.15915494309189535, per_low = -9.839338337591243e-18;   // 1 / 2 pi
    const double h = f * per, l = fma(f, per_low, fma(f, per, -h)), t = p * h;
    const double n = rint(4.0 * t), r = fma(-0.25, n, t) + fma((double)p, l, fma((double)p, h, -t));
    const double m = rint(4.0 * r);   // the second double's, where there are so many turns
    rest = fma(-0.25, m, r);
    quarters = (int)fma(-4.0, rint(0.25 * n), n) + (int)fma(-4.0, rint(0.25 * m), m) & 3;
  }
  __device__ __forceinline__ double2 whole(double s, double c) const {   // of the rest's sine and cosine: cosine, sine
    const double cs = quarters & 1 ? -s : c, sn = quarters & 1 ? c : s;
    return quarters & 2 ? make_double2(-cs, -sn) : make_double2(cs, sn);
  }
};
// cos and sin of p f radians, times amp, for fp32: Taylor's series at an eighth of a
// turn at most, the sine off by 2^-29, the cosine by 2^-33.
__device__ __forceinline__ double2 rope_angle(int p, double f, double amp) {
  const Turn t(p, f);
  const double x = 6.2831853071795864769 * t.rest, y = x * x;
  const double s = amp * x * (1 + y * (-1.0 / 6 + y * (1.0 / 120 + y * (-1.0 / 5040 + y * (1.0 / 362880)))));
  const double c = amp * (1 + y * (-1.0 / 2 + y * (1.0 / 24 + y * (-1.0 / 720 + y * (1.0 / 40320 - y * (1.0 / 3628800))))));
  return t.whole(s, c);
}
// The same for fp64.
__device__ __forceinline__ double2 rope_angle64(int p, double f, double amp) {
  const Turn t(p, f);
  double s, c;
  sincospi(2.0 * t.rest, &s, &c);
  return t.whole(amp * s, amp * c);
}

// Eight values of a row are a lane's: the pairs 4 c .. 4 c + 3 of the row's hd / 2.
// Pair j < nf is the dimensions (j, j + nf), or neighbours if interleaved; pairs
// behind those are neighbours and do not turn.  VEC: nf is a multiple of 4, so a
// lane's pairs turn all or none and four values lie together.
struct LanePairs {
  int c, hd, nf;
  bool split;   // (j, j + nf)
  __device__ LanePairs(const CacheArgs& a, int lane_of_row) : c(lane_of_row), hd(a.hd), nf(a.nf), split(!a.interleaved && 4 * lane_of_row < a.nf) {}
  __device__ bool any() const { return 8 * c < hd; }
  __device__ bool turns(int i) const { return 4 * c + i < nf; }
  __device__ int low(int i) const { return split && turns(i) ? 4 * c + i : 8 * c + 2 * i; }
  __device__ int high(int i) const { return split && turns(i) ? 4 * c + i + nf : 8 * c + 2 * i + 1; }
};
// The pairs' first and second values, for the FMA units' two at a time.
struct Pairs {
  float2 a[2], b[2];
};
__device__ __forceinline__ float2 pc_mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
template <typename T>
__device__ __forceinline__ float2 halves(uint32_t w) {
  const uint16_t lo = w & 0xffffu, hi = w >> 16;
  return make_float2(to_f32<T>(*reinterpret_cast<const T*>(&lo)), to_f32<T>(*reinterpret_cast<const T*>(&hi)));
}
// A lane's pairs of a row in shared memory.
template <typename T, bool VEC>
__device__ __forceinline__ void read_pairs(Pairs& x, const LanePairs& m, const uint4* row) {
  const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
  if (VEC && m.split) {
    const uint2 lo = *reinterpret_cast<const uint2*>(p + 4 * m.c), hi = *reinterpret_cast<const uint2*>(p + m.nf + 4 * m.c);
    x.a[0] = halves<T>(lo.x), x.a[1] = halves<T>(lo.y), x.b[0] = halves<T>(hi.x), x.b[1] = halves<T>(hi.y);
  } else {
    uint4 w;
    if (VEC) {
      w = row[m.c];
    } else {
      w.x = (uint32_t)p[m.low(0)] | (uint32_t)p[m.high(0)] << 16, w.y = (uint32_t)p[m.low(1)] | (uint32_t)p[m.high(1)] << 16;
      w.z = (uint32_t)p[m.low(2)] | (uint32_t)p[m.high(2)] << 16, w.w = (uint32_t)p[m.low(3)] | (uint32_t)p[m.high(3)] << 16;
    }
    const float2 y[4] = {halves<T>(w.x), halves<T>(w.y), halves<T>(w.z), halves<T>(w.w)};
    x.a[0] = make_float2(y[0].x, y[1].x), x.b[0] = make_float2(y[0].y, y[1].y);
    x.a[1] = make_float2(y[2].x, y[3].x), x.b[1] = make_float2(y[2].y, y[3].y);
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_pairs(void* row, const LanePairs& m, const Pairs& x) {
  uint16_t* p = static_cast<uint16_t*>(row);
  if (VEC && m.split) {
    *reinterpret_cast<uint2*>(p + 4 * m.c) = make_uint2(at_pack<T>(x.a[0].x, x.a[0].y), at_pack<T>(x.a[1].x, x.a[1].y));
    *reinterpret_cast<uint2*>(p + m.nf + 4 * m.c) = make_uint2(at_pack<T>(x.b[0].x, x.b[0].y), at_pack<T>(x.b[1].x, x.b[1].y));
  } else {
    const uint32_t w[4] = {at_pack<T>(x.a[0].x, x.b[0].x), at_pack<T>(x.a[0].y, x.b[0].y), at_pack<T>(x.a[1].x, x.b[1].x), at_pack<T>(x.a[1].y, x.b[1].y)};
    if (VEC) {
      *reinterpret_cast<uint2*>(p + 8 * m.c) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(p + 8 * m.c + 4) = make_uint2(w[2], w[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        p[m.low(i)] = (uint16_t)w[i];
        p[m.high(i)] = (uint16_t)(w[i] >> 16);
      }
    }
  }
}
// e4m3 codes of a pair, the first in the low byte; NaN stays, infinities must be gone.
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ float2 e4m3_values(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// A lane's codes: of its pairs' first values, and of their second ones.
struct Codes {
  uint32_t a, b;
};
__device__ __forceinline__ Codes codes_of(const Pairs& x) {
  return {e4m3_pair(x.a[0].x, x.a[0].y) | e4m3_pair(x.a[1].x, x.a[1].y) << 16, e4m3_pair(x.b[0].x, x.b[0].y) | e4m3_pair(x.b[1].x, x.b[1].y) << 16};
}
template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t* p, const LanePairs& m, const Codes& y) {
  if (VEC && m.split) {
    *reinterpret_cast<uint32_t*>(p + 4 * m.c) = y.a;
    *reinterpret_cast<uint32_t*>(p + m.nf + 4 * m.c) = y.b;
  } else if (VEC) {
    *reinterpret_cast<uint2*>(p + 8 * m.c) = make_uint2(__byte_perm(y.a, y.b, 0x5140), __byte_perm(y.a, y.b, 0x7362));
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) p[m.low(i)] = (uint8_t)(y.a >> 8 * i), p[m.high(i)] = (uint8_t)(y.b >> 8 * i);
  }
}
template <bool VEC>
__device__ __forceinline__ Codes load_codes(const uint8_t* p, const LanePairs& m) {
  if (VEC && m.split) return {*reinterpret_cast<const uint32_t*>(p + 4 * m.c), *reinterpret_cast<const uint32_t*>(p + m.nf + 4 * m.c)};
  Codes y{0, 0};
#pragma unroll
  for (int i = 0; i < 4; i++) y.a |= (uint32_t)p[m.low(i)] << 8 * i, y.b |= (uint32_t)p[m.high(i)] << 8 * i;
  return y;
}
// All ones in the bytes of four codes that are NaN.
__device__ __forceinline__ uint32_t e4m3_nans(uint32_t four) { return (((four & 0x7f7f7f7fu) + 0x01010101u & 0x80808080u) >> 7) * 0xffu; }

// `instead` in place of what is not finite.
__device__ __forceinline__ void only_finite(Pairs& x, float instead) {
  auto one = [&](float& v) { v = v - v == 0.f ? v : instead; };
#pragma unroll
  for (int e = 0; e < 2; e++) one(x.a[e].x), one(x.a[e].y), one(x.b[e].x), one(x.b[e].y);
}
// The norm over the LPR lanes of N rows (lanes without values have zeros), where
// on[i] is all ones; where it is 0, w[i] (the weights in the lanes' order) has ones.
template <int LPR, int N>
__device__ __forceinline__ void norm_rows(Pairs (&x)[N], const float* const (&w)[N], const uint32_t (&on)[N], const CacheArgs& a) {
  float s[N];
#pragma unroll
  for (int i = 0; i < N; i++) {
    float2 q = pc_mul2(x[i].a[0], x[i].a[0]);
    q = at_fma2(x[i].a[1], x[i].a[1], q);
    q = at_fma2(x[i].b[0], x[i].b[0], q);
    q = at_fma2(x[i].b[1], x[i].b[1], q);
    s[i] = q.x + q.y;
  }
#pragma unroll
  for (int o = LPR / 2; o; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; i++) s[i] += __shfl_xor_sync(~0u, s[i], o);
#pragma unroll
  for (int i = 0; i < N; i++) {
    const float r = __uint_as_float((__float_as_uint(rsqrtf(fmaf(s[i], a.inv_hd, a.eps))) & on[i]) | (0x3f800000u & ~on[i]));
    const float2 rr = make_float2(r, r);
    const float4 u = *reinterpret_cast<const float4*>(w[i]), v = *reinterpret_cast<const float4*>(w[i] + PC_PAIRS);
    x[i].a[0] = pc_mul2(x[i].a[0], pc_mul2(rr, make_float2(u.x, u.y)));
    x[i].a[1] = pc_mul2(x[i].a[1], pc_mul2(rr, make_float2(u.z, u.w)));
    x[i].b[0] = pc_mul2(x[i].b[0], pc_mul2(rr, make_float2(v.x, v.y)));
    x[i].b[1] = pc_mul2(x[i].b[1], pc_mul2(rr, make_float2(v.z, v.w)));
  }
}
// cos and sin of a lane's four pairs.
struct Turns {
  float2 c[2], s[2];
  __device__ __forceinline__ Turns(const float (*turn)[PC_PAIRS], const LanePairs& m) {
    const float4 u = *reinterpret_cast<const float4*>(&turn[0][4 * m.c]), v = *reinterpret_cast<const float4*>(&turn[1][4 * m.c]);
    c[0] = make_float2(u.x, u.y), c[1] = make_float2(u.z, u.w), s[0] = make_float2(v.x, v.y), s[1] = make_float2(v.z, v.w);
  }
};
// Pairs j < nf turned; the others stay as they are, whatever their neighbours hold.
template <bool VEC>
__device__ __forceinline__ void rotate_pairs(Pairs& x, const Turns& t, const LanePairs& m) {
  if (VEC && !m.turns(0)) return;
  const Pairs y = x;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    x.a[i] = at_fma2(y.a[i], t.c[i], pc_mul2(y.b[i], make_float2(-t.s[i].x, -t.s[i].y)));
    x.b[i] = at_fma2(y.b[i], t.c[i], pc_mul2(y.a[i], t.s[i]));
  }
  if (!VEC) {
    if (!m.turns(0)) x.a[0].x = y.a[0].x, x.b[0].x = y.b[0].x;
    if (!m.turns(1)) x.a[0].y = y.a[0].y, x.b[0].y = y.b[0].y;
    if (!m.turns(2)) x.a[1].x = y.a[1].x, x.b[1].x = y.b[1].x;
    if (!m.turns(3)) x.a[1].y = y.a[1].y, x.b[1].y = y.b[1].y;
  }
}
__device__ __forceinline__ Pairs no_pairs() {
  const float2 z = make_float2(0.f, 0.f);
  return Pairs{{z, z}, {z, z}};
}

// Offsets of the sequences, in shared memory where they fit.
__device__ __forceinline__ const int* keep_offsets(const int* cu, int B, int* s_cu) {
  if (!cu || B > PC_CU) return cu;
  for (int i = threadIdx.x; i <= B; i += PC_THREADS) s_cu[i] = cu[i];
  return s_cu;
}

__device__ __forceinline__ void cp16(uint4* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
static_assert(PC_TOKENS >= PC_WINDOW + PAGED_BLOCK - 1, "both kinds of CTAs' tokens");
struct CacheShared {
  int cu[PC_CU + 1];
  alignas(16) float w[3][ATTN_MAX_HD];                              // norms' weights of q and k, in the lanes' order; 1 where there are none, and for v
  alignas(16) float turn[PC_WINDOW + PAGED_BLOCK - 1][2][PC_PAIRS];   // cos, sin of tokens' pairs that turn
  int at[PC_TOKENS];                                                // tokens' positions for the rotation
  int run[PC_WINDOW], len[PC_WINDOW], page[PC_TOKENS], row[PC_TOKENS];   // runs: first token, tokens; runs' or tokens' page and (first) row
  int runs, cover;
};
__device__ __forceinline__ void keep_weights(const CacheArgs& a, CacheShared& sh) {
  for (int i = threadIdx.x; i < a.hd; i += PC_THREADS) {   // pairs' first values, and from PC_PAIRS on their second ones
    const int second = i >= a.hd / 2, j = i - second * (a.hd / 2), at = j + second * PC_PAIRS, d = j >= a.nf || a.interleaved ? 2 * j + second : second ? j + a.nf : j;
    sh.w[0][at] = a.qw ? a.qw[d] : 1.f;
    sh.w[1][at] = a.kw ? a.kw[d] : 1.f;
    sh.w[2][at] = 1.f;
  }
}
__device__ __forceinline__ void keep_turn(float (*turn)[PC_PAIRS], int pair, int pos, double f, double amp) {
  const double2 t = rope_angle(pos, f, amp);
  turn[0][pair] = (float)t.x, turn[1][pair] = (float)t.y;
}

// Rows of nt tokens from t0 on: q, and (tg_rotary, 16-bit pages) k and v.  A row
// is LPR lanes of 8 values; a thread has the same R rows of every token, of
// the `part`-th share of a token's rows, and copies those of the next tokens into
// its own places of a ring in shared memory as it turns this one's.  The angles
// of four tokens are made together, by all threads, while the four before are
// turned.
extern __shared__ uint4 pc_ring[];   // [token % pc_ahead][row][thread]: a row is LPR pieces
template <typename T, int LPR, bool VEC, int MODE, bool NORM, int R>
__device__ __forceinline__ void token_rows(const CacheArgs& a, CacheShared& sh, int t0, int nt, int part) {
  const int tid = threadIdx.x;
  constexpr int ROWS = PC_THREADS / LPR, AHEAD = pc_ahead<R>;
  const LanePairs m(a, tid % LPR);
  const int rows = a.H + (MODE == PC_PAGES8 ? 0 : a.KH) + (MODE == PC_PAGES16 ? a.KH : 0);
  const int first = part * R * ROWS + tid / LPR;   // its rows: first, first + ROWS, ..
  const T* from[R];
  T* to[R];   // q, tg_rotary's k; the head's place in a page
  const float* w[R];
  uint32_t on[R];
  auto fetch = [&](int t) {
    if (t < nt)
#pragma unroll
      for (int i = 0; i < R; i++) {
        const int r = first + i * ROWS;
        if (r < rows && m.any()) cp16(pc_ring + (t % AHEAD * R + i) * PC_THREADS + tid, from[i] + 8 * m.c);
        from[i] += r < a.H ? a.sq[0] : r < a.H + a.KH ? a.sk[0] : a.sv[0];
      }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < R; i++) {
    const int r = first + i * ROWS;
    const long long t = t0;
    const int which = MODE == PC_PAGES8 || r < a.H ? 0 : r < a.H + a.KH ? 1 : 2;
    w[i] = sh.w[which] + (m.any() ? 4 * m.c : 0);
    on[i] = (which == 0 && a.qw) || (which == 1 && a.kw) ? ~0u : 0;
    if (r < a.H) {
      from[i] = (const T*)a.q + t * a.sq[0] + r * a.sq[1];
      to[i] = (T*)a.qo + t * a.sqo[0] + r * a.sqo[1];
    } else if (r < a.H + a.KH) {
      from[i] = (const T*)a.k + t * a.sk[0] + (r - a.H) * a.sk[1];
      to[i] = MODE == PC_ROTARY ? (T*)a.ko + t * a.sko[0] + (r - a.H) * a.sko[1] : (T*)(a.kp + (r - a.H) * a.skp[1]);
    } else {
      from[i] = (const T*)a.v + t * a.sv[0] + (r - a.H - a.KH) * a.sv[1];
      to[i] = (T*)(a.vp + (r - a.H - a.KH) * a.svp[1]);
    }
  }
#pragma unroll
  for (int t = 0; t < AHEAD - 1; t++) fetch(t);
  const int* cu = MODE == PC_ROTARY ? nullptr : keep_offsets(a.cu, a.B, sh.cu);
  if (NORM) keep_weights(a, sh);
  if (MODE != PC_ROTARY) __syncthreads();
  if (tid < nt) {
    int pos = 0, page = -1, row = 0;
    if (MODE == PC_ROTARY) {
      pos = a.positions[t0 + tid];
    } else {
      const PagedToken k = paged_token(cu, a.B, a.per, a.T, t0 + tid);
      page = -2;   // of no sequence
      if (k.seq >= 0) {
        const int p = paged_position(a.lens[k.seq], k.end, t0 + tid);
        pos = a.positions ? a.positions[t0 + tid] : p;
        page = MODE == PC_PAGES16 ? paged_page(a.tables + k.seq * a.st, a.cols, p, a.shift, a.n_pages) : -1;
        row = p & ((1 << a.shift) - 1);
      }
    }
    sh.at[tid] = pos, sh.page[tid] = page, sh.row[tid] = row;
  }
  const int pair = tid % PC_PAIRS, quarter = tid / PC_PAIRS;
  const double f = pair < a.nf ? a.freqs[pair] : 0.0;
  auto angles = [&](int t) {   // of four tokens from t on
    if (t + quarter < nt && pair < a.nf) keep_turn(sh.turn[(t & 4) + quarter], pair, sh.at[t + quarter], f, a.amp);
  };
  __syncthreads();
  angles(0);
#pragma unroll 1
  for (int t = 0; t < nt; t++) {
    if (t % 4 == 0) {
      __syncthreads();
      angles(t + 4);
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 2) : "memory");
    __syncwarp();   // the warp's copies of this token are there, the last one's are read
    fetch(t + AHEAD - 1);
    const Turns turns(sh.turn[t & 7], m);
    const int page = MODE == PC_ROTARY ? -1 : sh.page[t];
    auto read = [&](int i, Pairs& x) {   // lanes of rows that have none take part in the sums
      x = no_pairs();
      if (first + i * ROWS < rows && m.any()) read_pairs<T, VEC>(x, m, pc_ring + (t % AHEAD * R + i) * PC_THREADS + tid - m.c);
    };
    auto write = [&](int i, Pairs& x) {
      const int r = first + i * ROWS;
      const bool is_q = r < a.H, is_v = r >= a.H + a.KH;
      if (r >= rows || !m.any()) return;
      if (MODE != PC_PAGES16 || !is_v) rotate_pairs<VEC>(x, turns, m);
      if (MODE != PC_PAGES16 || is_q) {
        if (page != -2) store_pairs<T, VEC>(to[i], m, x);
        to[i] += is_q ? a.sqo[0] : a.sko[0];
      } else if (page >= 0) {
        const long long at = is_v ? page * a.svp[0] + sh.row[t] * a.svp[2] : page * a.skp[0] + sh.row[t] * a.skp[2];
        store_pairs<T, VEC>((uint8_t*)to[i] + at, m, x);
      }
    };
    if (NORM) {   // the rows' sums side by side: 8,192 tokens x 32 heads 25.4 us, one after another 27; without norms that is slower
      Pairs x[R];
#pragma unroll
      for (int i = 0; i < R; i++) read(i, x[i]);
      norm_rows<LPR, R>(x, w, on, a);
#pragma unroll
      for (int i = 0; i < R; i++) write(i, x[i]);
    } else {
#pragma unroll
      for (int i = 0; i < R; i++) {
        Pairs x;
        read(i, x);
        write(i, x);
      }
    }
  }
}

// Codes are what the formulas' values in 64 bits round to, so that they do not depend
// on how a sum was taken.  In fp32 the sum of squares is 9 roundings deep, half of
// which reach its root, which has 4 2^-24 of its own; with the mean, two products
// and a rotation a value y is off by at most 14.5 2^-24 |(a, b)| <= PC_OFF (|y_a| +
// |y_b|) of its pair.  Where both ends of that interval round to one code, that is
// it; the rows of the others, one value in 7,000, are worked out in 64 bits by the
// whole warp.  The test for doubt takes 2 of 8,192 tokens' 46 us and those rows 6.
// So it is with the scale, where the largest value, off by at most 2 PC_OFF of
// itself, may lie on either side of a border (one block in 100,000).
constexpr float PC_OFF = 0x1p-20f, PC_OFF_MOST = 0x1p-18f;
__device__ __forceinline__ Codes codes_within(const Pairs& x, float off, bool& doubt) {
  Pairs lo, hi;
#pragma unroll
  for (int e = 0; e < 2; e++) {
    float2 d = make_float2(off * (fabsf(x.a[e].x) + fabsf(x.b[e].x)), off * (fabsf(x.a[e].y) + fabsf(x.b[e].y)));
    d.x = fminf(d.x, 1e30f), d.y = fminf(d.y, 1e30f);   // beside a NaN: any doubt
    const float2 one = make_float2(1.f, 1.f), less = make_float2(-1.f, -1.f);
    lo.a[e] = at_fma2(d, less, x.a[e]), lo.b[e] = at_fma2(d, less, x.b[e]);
    hi.a[e] = at_fma2(d, one, x.a[e]), hi.b[e] = at_fma2(d, one, x.b[e]);
  }
  const Codes y = codes_of(lo), z = codes_of(hi);
  doubt = y.a != z.a || y.b != z.b;
  return y;
}
__device__ __forceinline__ float to_odd(double x) {   // rounds to any fewer bits as x does; NaN where fp32 does not hold x
  const float y = __double2float_rz(x);
  return !(fabs(x) <= FLT_MAX) ? NAN : (double)y == x ? y : __uint_as_float(__float_as_uint(y) | 1);
}
// A row's values times inv, to_odd.  row: null for lanes without values; w: the lane's
// weights of a key's norm, null for a row of v.
template <typename T, int LPR, bool VEC, bool NORM>
__device__ __noinline__ Pairs exact_pairs(const CacheArgs& a, const uint4* row, const float* w, int pos, double inv) {
  const LanePairs m(a, threadIdx.x % LPR);
  Pairs x = no_pairs();
  if (row) read_pairs<T, VEC>(x, m, row);
  double r = inv;
  if (NORM) {
    double part[2], sum;
#pragma unroll
    for (int e = 0; e < 2; e++)
      part[e] = ((double)x.a[e].x * x.a[e].x + (double)x.a[e].y * x.a[e].y) + ((double)x.b[e].x * x.b[e].x + (double)x.b[e].y * x.b[e].y);
    sum = part[0] + part[1];
#pragma unroll
    for (int o = LPR / 2; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (w && a.kw) r *= sum > FLT_MAX ? 0.0 : rsqrt(sum * a.inv_hd64 + a.eps64);   // what fp32 does not hold counts as infinite there too
  }
  Pairs y;
  auto pair = [&](int i, float xa, float xb, float& ya, float& yb) {
    double u = xa * r, v = xb * r;
    if (NORM && w) u *= w[i], v *= w[PC_PAIRS + i];
    if (w && m.turns(i)) {
      const double2 t = rope_angle64(pos, a.freqs[4 * m.c + i], a.amp);
      const double z = u * t.x - v * t.y;
      v = v * t.x + u * t.y, u = z;
    }
    ya = to_odd(u), yb = to_odd(v);
  };
  pair(0, x.a[0].x, x.b[0].x, y.a[0].x, y.b[0].x), pair(1, x.a[0].y, x.b[0].y, y.a[0].y, y.b[0].y);
  pair(2, x.a[1].x, x.b[1].x, y.a[1].x, y.b[1].x), pair(3, x.a[1].y, x.b[1].y, y.a[1].y, y.b[1].y);
  return y;
}

// Runs of 8-bit blocks whose first token is one of the `window` packed tokens
// from t0 on: a warp has one run's keys or values of a key head.  Its values are
// worked out twice, for the largest and for the codes: kept in registers they
// leave room for one CTA of an SM instead of three (8,192 tokens with q 171 us
// instead of 47).  Two rows at a time, for their sums' shuffles to overlap.  Keys
// and values of 4 heads, 8,192 tokens, normed: 26 us; 25 MB to read and write take
// 4.  As many CTAs as there are SMs' places take 15: what bounds it is how long one
// takes from its offsets to its scales, and that 512 are one round and a bit.
template <typename T, int LPR, bool VEC, bool NORM>
__device__ __forceinline__ void runs_of_blocks(const CacheArgs& a, CacheShared& sh, int t0) {
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  constexpr int RPP = 32 / LPR;   // rows of a warp at a time
  const int* cu = keep_offsets(a.cu, a.B, sh.cu);
  if (NORM) keep_weights(a, sh);
  __syncthreads();
  if (wid == 0) {
    const int t = t0 + lane;
    int n = 0, p = 0;
    PagedToken k;
    k.seq = -1;
    if (lane < a.window + PAGED_BLOCK - 1 && t < a.T) {
      k = paged_token(cu, a.B, a.per, a.T, t);
      p = k.seq >= 0 ? paged_position(a.lens[k.seq], k.end, t) : 0;
      sh.at[lane] = k.seq >= 0 && a.positions ? a.positions[t] : p;
      n = lane < a.window ? paged_run(k, t, p) : 0;
    }
    const int page = n ? paged_page(a.tables + k.seq * a.st, a.cols, p, a.shift, a.n_pages) : -1;
    const unsigned mine = __ballot_sync(~0u, page >= 0);
    if (page >= 0) {
      const int i = __popc(mine & ((1u << lane) - 1));
      sh.run[i] = lane, sh.len[i] = n, sh.page[i] = page, sh.row[i] = p & ((1 << a.shift) - 1);
    }
    const int cover = __reduce_max_sync(~0u, page >= 0 ? lane + n : 0);
    if (lane == 0) sh.runs = __popc(mine), sh.cover = cover;
  }
  __syncthreads();
  if (!sh.runs) return;
  const LanePairs m(a, lane % LPR);
  const int items = sh.runs * 2 * a.KH;
  const float* const w[2] = {sh.w[1] + (m.any() ? 4 * m.c : 0), sh.w[1] + (m.any() ? 4 * m.c : 0)};
  const uint32_t on[2] = {a.kw ? ~0u : 0, a.kw ? ~0u : 0};
  const bool touched = (NORM && a.kw) || a.nf > 0;
  const float off_by = (NORM && a.kw) || 4 * m.c < a.nf ? PC_OFF : 0.f;   // values that no one touches are exact
  uint4* ring = pc_ring + wid * PAGED_BLOCK * LPR;   // an item's rows
  auto fetch = [&](int item) {
    const int i = item / (2 * a.KH), kh = item % (2 * a.KH) >> 1, is_v = item & 1;
    const long long step = is_v ? a.sv[0] : a.sk[0];
    const T* from = (is_v ? (const T*)a.v + kh * a.sv[1] : (const T*)a.k + kh * a.sk[1]) + (t0 + sh.run[i] + lane / LPR) * step;
    for (int u = 0; u * RPP < sh.len[i]; u++, from += RPP * step)
      if (u * RPP + lane / LPR < sh.len[i] && m.any()) cp16(ring + u * 32 + lane, from + 8 * m.c);
  };
  if (wid < items) fetch(wid);
  if (tid % PC_PAIRS < a.nf) {
    const double f = a.freqs[tid % PC_PAIRS];
    for (int j = tid / PC_PAIRS; j < sh.cover; j += PC_THREADS / PC_PAIRS) keep_turn(sh.turn[j], tid % PC_PAIRS, sh.at[j], f, a.amp);
  }
  __syncthreads();
  for (int item = wid; item < items; item += PC_WARPS) {
    const int i = item / (2 * a.KH), kh = item % (2 * a.KH) >> 1, is_v = item & 1;
    const int j0 = sh.run[i], n = sh.len[i], off = sh.row[i] % PAGED_BLOCK, block = sh.row[i] / PAGED_BLOCK;
    uint8_t* rows = is_v ? a.vp + sh.page[i] * a.svp[0] + kh * a.svp[1] + (long long)block * PAGED_BLOCK * a.svp[2]
                         : a.kp + sh.page[i] * a.skp[0] + kh * a.skp[1] + (long long)block * PAGED_BLOCK * a.skp[2];
    const long long pitch = is_v ? a.svp[2] : a.skp[2];
    float* scale_at = is_v ? a.vs + sh.page[i] * a.svs[0] + kh * a.svs[1] + block * a.svs[2]
                           : a.ks + sh.page[i] * a.sks[0] + kh * a.sks[1] + block * a.sks[2];
    const float before = off ? *scale_at : 0.f;
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    auto values = [&](int u, Pairs (&x)[2]) {   // of the rows u RPP + lane / LPR and RPP on; zeros where there is none
#pragma unroll
      for (int i = 0; i < 2; i++) {
        x[i] = no_pairs();
        if ((u + i) * RPP + lane / LPR < n && m.any()) read_pairs<T, VEC>(x[i], m, ring + ((u + i) * RPP + lane / LPR) * LPR);
      }
      if (is_v) return;
      if (NORM) norm_rows<LPR, 2>(x, w, on, a);
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int j = (u + i) * RPP + lane / LPR;
        if (j < n && m.any()) rotate_pairs<VEC>(x[i], Turns(sh.turn[j0 + j], m), m);
      }
    };
    uint32_t amax;      // bits of the largest finite magnitude
    bool odd = false;   // a value is infinite
    for (;;) {
      float most = 0.f;   // NaN is less than any number here
#pragma unroll 1
      for (int u = 0; u * RPP < n; u += 2) {
        Pairs x[2];
        values(u, x);
#pragma unroll
        for (int i = 0; i < 2; i++) {
          if (odd) only_finite(x[i], 0.f);
#pragma unroll
          for (int e = 0; e < 2; e++)
            most = fmaxf(fmaxf(most, fmaxf(fabsf(x[i].a[e].x), fabsf(x[i].a[e].y))), fmaxf(fabsf(x[i].b[e].x), fabsf(x[i].b[e].y)));
        }
      }
      amax = __reduce_max_sync(~0u, __float_as_uint(most));
      if (odd || amax < 0x7f800000u) break;
      odd = true;
    }
    auto exact = [&](int u, double times) {   // of the rows u RPP + lane / LPR
      const int j = u * RPP + lane / LPR;
      return exact_pairs<T, LPR, VEC, NORM>(a, j < n && m.any() ? ring + j * LPR : nullptr, is_v ? nullptr : w[0], sh.at[j0 + min(j, n - 1)], times);
    };
    const float top = __uint_as_float(amax);
    if (!is_v && touched &&
        paged_scale_exp(__float_as_uint(top - PC_OFF_MOST * top)) != paged_scale_exp(__float_as_uint(top + PC_OFF_MOST * top))) {
      float most = 0.f;
#pragma unroll 1
      for (int u = 0; u * RPP < n; u++) {
        const Pairs x = exact(u, 1.0);
#pragma unroll
        for (int e = 0; e < 2; e++)
          most = fmaxf(fmaxf(most, fmaxf(fabsf(x.a[e].x), fabsf(x.a[e].y))), fmaxf(fabsf(x.b[e].x), fabsf(x.b[e].y)));
      }
      amax = __reduce_max_sync(~0u, __float_as_uint(most));
    }
    const float need = __uint_as_float((uint32_t)(paged_scale_exp(amax) + 127) << 23);
    const float scale = fmaxf(need, before), inv = 1.f / scale;
    const bool fine = __float_as_uint(scale) & 0x7fffffu;   // an earlier scale that is no power of two: two roundings more, v's values too
    const float off_scaled = (is_v ? 0.f : off_by) + (fine ? 0x1p-22f : 0.f);
    if (off && scale > before) {   // the earlier tokens' codes under the larger scale
      const float less = before * inv;   // has 24 bits, a code 4
      auto two = [&](float2 c) {
        auto odd = [&](float x) {
          const float y = __fmul_rz(x, less);
          return fmaf(x, less, -y) == 0.f ? y : __uint_as_float(__float_as_uint(y) | 1);
        };
        return e4m3_pair(odd(c.x), odd(c.y));
      };
      for (int i8 = lane; i8 < off * (a.hd / 8); i8 += 32) {
        uint2* at = reinterpret_cast<uint2*>(rows + i8 / (a.hd / 8) * pitch + i8 % (a.hd / 8) * 8);
        const uint2 w = *at;
        *at = make_uint2(two(e4m3_values(w.x)) | two(e4m3_values(w.x >> 16)) << 16, two(e4m3_values(w.y)) | two(e4m3_values(w.y >> 16)) << 16);
      }
    }
    unsigned again = 0;   // rows with codes in doubt
#pragma unroll 1
    for (int u = 0; u * RPP < n; u += 2) {
      Pairs x[2];
      values(u, x);
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int j = (u + i) * RPP + lane / LPR;
        const bool there = j < n && m.any();
        const float2 f = make_float2(inv, inv);
        if (odd) only_finite(x[i], NAN);
#pragma unroll
        for (int e = 0; e < 2; e++) x[i].a[e] = pc_mul2(x[i].a[e], f), x[i].b[e] = pc_mul2(x[i].b[e], f);
        bool doubt = false;
        const Codes y = is_v && !fine ? codes_of(x[i]) : codes_within(x[i], off_scaled, doubt);
        if (there) store_codes<VEC>(rows + (off + j) * pitch, m, y);
        if (there && doubt) again |= 1u << (u + i);
      }
    }
    for (again = __reduce_or_sync(~0u, again); again; again &= again - 1) {
      const int u = __ffs(again) - 1, j = u * RPP + lane / LPR;
      const Codes y = codes_of(exact(u, 1.0 / scale));
      if (j < n && m.any()) {
        uint8_t* const at = rows + (off + j) * pitch;
        const Codes z = load_codes<VEC>(at, m);   // what fp32 does not hold stays NaN
        const uint32_t na = e4m3_nans(z.a), nb = e4m3_nans(z.b);
        store_codes<VEC>(at, m, Codes{(y.a & ~na) | (z.a & na), (y.b & ~nb) | (z.b & nb)});
      }
    }
    if (lane == 0) *scale_at = scale;
    __syncwarp();   // all have read the rows
    if (item + PC_WARPS < items) fetch(item + PC_WARPS);
  }
}

// Rows of tokens and, beside them in the same launch, runs of 8-bit blocks, so that
// the copies of the one overlap the instructions of the other.  Measured in a
// replayed graph, bf16, heads of 128: 8,192 tokens x 32 heads rotated 22 us (0.94 of
// a copy's rate, part of it from L2: bytes bound it), with norms 26 (instructions);
// the same with 4 key heads to 8-bit pages 46, without norms 37, where 160 MB take
// 24, and to 16-bit pages 37.  A chunk of 2,048 tokens 20; two tokens 5, to 16-bit pages
// 4, of which an empty kernel is 2.
template <typename T, int LPR, bool VEC, int MODE, bool NORM, int R>
__global__ void __launch_bounds__(PC_THREADS, PC_PER_SM) cache_kernel(const __grid_constant__ CacheArgs a) {
  __shared__ CacheShared sh;
  pdl_wait();
  if (MODE == PC_PAGES8 && blockIdx.x >= a.token_ctas) {
    runs_of_blocks<T, LPR, VEC, NORM>(a, sh, (blockIdx.x - a.token_ctas) * a.window);
  } else {
    const int t0 = blockIdx.x / a.parts * a.tokens;
    token_rows<T, LPR, VEC, MODE, NORM, R>(a, sh, t0, min(a.tokens, a.T - t0), blockIdx.x % a.parts);
  }
}

struct GatherArgs {
  const uint8_t *kp, *vp;
  const float *ks, *vs;
  const int *tables, *cu;
  uint8_t *ko, *vo;
  unsigned skp[3], svp[3];    // page, head, row; 16-byte words
  unsigned sks[3], svs[3];    // page, head, block
  unsigned sko[2], svo[2];    // token, head; 16-byte words
  long long st;
  int T, B, KH, hd, n_pages, cols, shift;
  int wide;   // outputs in 32-byte pieces: rows start on 32-byte boundaries
};

// Rows of the packed outputs, 16 bytes of a page's row at a time, three of them
// loaded before the first is stored.  A CTA has `per` tokens; a thread goes
// through their rows (K of all heads, then V, of each token) without divisions,
// and strides are 32-bit numbers of 16-byte words: with 64-bit products the
// kernel was bound by its instructions (185 for 32 x 16 values, 38 us).
template <typename T, bool CODES>
__global__ void __launch_bounds__(PC_THREADS, PC_GATHERS) gather_pages_kernel(const GatherArgs a, int lpr, int per) {
  constexpr int N = 3;
  __shared__ int s_cu[PC_CU + 1], s_page[PC_GATHER], s_row[PC_GATHER];
  pdl_wait();
  const int tid = threadIdx.x, t0 = blockIdx.x * per;
  const int* cu = keep_offsets(a.cu, a.B, s_cu);
  __syncthreads();
  if (tid < per && t0 + tid < a.T) {
    const PagedToken k = paged_token(cu, a.B, 1, a.T, t0 + tid);
    const int p = t0 + tid - k.first;
    s_page[tid] = k.seq < 0 ? -2 : paged_page(a.tables + k.seq * a.st, a.cols, p, a.shift, a.n_pages);   // -2: of no sequence
    s_row[tid] = p & ((1 << a.shift) - 1);
  }
  __syncthreads();
  const int c = tid % lpr, heads = 2 * a.KH, tokens = min(per, a.T - t0), step = PC_THREADS / lpr;
  if (c * (CODES ? 16 : 8) >= a.hd) return;
  const int dj = step / heads, dh = step % heads;
  int j = tid / lpr / heads, h = tid / lpr % heads;   // the thread's row: token and head
  while (j < tokens) {
    uint4 w[N];
    float scale[N];
    uint8_t* to[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
      to[i] = nullptr;
      if (j < tokens && s_page[j] != -2) {
        const int page = s_page[j];
        const bool is_v = h >= a.KH;
        const unsigned kh = is_v ? h - a.KH : h, row = s_row[j];
        to[i] = (is_v ? a.vo : a.ko) + 16 * ((uint64_t)(unsigned)(t0 + j) * (is_v ? a.svo[0] : a.sko[0]) + (uint64_t)kh * (is_v ? a.svo[1] : a.sko[1]) +
                                             c * (CODES ? 2 : 1));
        w[i] = make_uint4(0, 0, 0, 0);
        scale[i] = 0.f;
        if (page >= 0) {
          w[i] = *reinterpret_cast<const uint4*>((is_v ? a.vp : a.kp) + 16 * ((uint64_t)(unsigned)page * (is_v ? a.svp[0] : a.skp[0]) +
                                                                              (uint64_t)row * (is_v ? a.svp[2] : a.skp[2]) + (uint64_t)kh * (is_v ? a.svp[1] : a.skp[1]) + c));
          if (CODES)
            scale[i] = (is_v ? a.vs : a.ks)[(uint64_t)(unsigned)page * (is_v ? a.svs[0] : a.sks[0]) + (uint64_t)(row / PAGED_BLOCK) * (is_v ? a.svs[2] : a.sks[2]) +
                                            (uint64_t)kh * (is_v ? a.svs[1] : a.sks[1])];
        }
      }
      j += dj, h += dh;
      if (h >= heads) h -= heads, j++;
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
      if (!to[i]) continue;
      if (!CODES) {
        *reinterpret_cast<uint4*>(to[i]) = w[i];
      } else {
        const float2 f = make_float2(scale[i], scale[i]);
        auto two = [&](uint32_t code) {
          const float2 v = pc_mul2(e4m3_values(code), f);
          return at_pack<T>(v.x, v.y);
        };
        const uint32_t y[8] = {two(w[i].x), two(w[i].x >> 16), two(w[i].y), two(w[i].y >> 16),
                               two(w[i].z), two(w[i].z >> 16), two(w[i].w), two(w[i].w >> 16)};
        if (a.wide) {
          at_store8(to[i], y);
        } else {
          reinterpret_cast<uint4*>(to[i])[0] = make_uint4(y[0], y[1], y[2], y[3]);
          reinterpret_cast<uint4*>(to[i])[1] = make_uint4(y[4], y[5], y[6], y[7]);
        }
      }
    }
  }
}

template <typename T, int LPR, bool VEC, int MODE, bool NORM, int R>
static cudaError_t launch_cache(const CacheArgs& a, int grid, cudaStream_t s) {
  static std::atomic<unsigned long long> set{0};
  const cudaError_t e = attn_smem(cache_kernel<T, LPR, VEC, MODE, NORM, R>, pc_ring_bytes<R>, set);
  return e == cudaSuccess ? launch_pdl(cache_kernel<T, LPR, VEC, MODE, NORM, R>, dim3(grid), PC_THREADS, pc_ring_bytes<R>, s, a) : e;
}
template <typename T, int MODE, bool NORM, int R>
static cudaError_t launch_cache(const CacheArgs& a, int grid, cudaStream_t s) {
  const bool vec = a.nf % 4 == 0;
  if (a.hd <= 64) return vec ? launch_cache<T, 8, true, MODE, NORM, R>(a, grid, s) : launch_cache<T, 8, false, MODE, NORM, R>(a, grid, s);
  return vec ? launch_cache<T, 16, true, MODE, NORM, R>(a, grid, s) : launch_cache<T, 16, false, MODE, NORM, R>(a, grid, s);
}
template <typename T, int MODE>
static cudaError_t launch_cache(const CacheArgs& a, int grid, cudaStream_t s) {
  count_launches(1);
  if (a.qw || a.kw) return a.each == 2 ? launch_cache<T, MODE, true, 2>(a, grid, s) : launch_cache<T, MODE, true, 3>(a, grid, s);
  return a.each == 2 ? launch_cache<T, MODE, false, 2>(a, grid, s) : launch_cache<T, MODE, false, 3>(a, grid, s);
}

}  // namespace tg

using namespace tg;

namespace tg {

// The CTAs that rotate: rows of a thread (two, where that takes no more rounds over
// a token's rows: 32 heads of 128, 8,192 tokens, normed 27 us instead of 29; 36 in
// two shares of two 33 instead of 28), shares of a token's rows, and tokens of a CTA
// so that the SMs have them all at once, or as few times in a row as PC_TOKENS allow.
static long long token_ctas(CacheArgs& a, long long rows, int per_sm) {
  const int once = PC_THREADS / (a.hd <= 64 ? 8 : 16), most = attn_sms() * per_sm;
  const long long by2 = (rows + 2 * once - 1) / (2 * once), by3 = (rows + 3 * once - 1) / (3 * once);
  a.each = 2 * by2 <= 3 * by3 ? 2 : 3;
  a.parts = (int)(a.each == 2 ? by2 : by3);
  const long long work = (long long)a.T * a.parts, waves = (work + (long long)most * PC_TOKENS - 1) / ((long long)most * PC_TOKENS);
  a.tokens = (int)((work + most * waves - 1) / (most * waves));
  return (long long)((a.T + a.tokens - 1) / a.tokens) * a.parts;
}

static int rotary(ArgCheck& c, const RotaryRecord& r) {
  const int64_t* strides = r.strides;
  c.need(r.dtype == ATTN_BF16 || r.dtype == ATTN_FP16, "dtype must be 0 (bf16) or 1 (fp16)");
  need_ints(c, &r.n_tokens, 6);
  c.need(r.n_tokens >= 0 && r.n_tokens < 1 << 30 && r.n_heads >= 0 && r.n_kv_heads >= 0, "counts must not be negative, and tokens below 2^30");
  c.need(r.n_heads < 1 << 16 && r.n_kv_heads < 1 << 16, "too many heads");
  c.need(r.head_dim > 0 && r.head_dim % 8 == 0 && r.head_dim <= ATTN_MAX_HD, "head_dim must be a multiple of 8, at most 128");
  c.need(r.n_freqs >= 0 && 2 * r.n_freqs <= r.head_dim, "at most head_dim / 2 frequencies");
  c.need(std::isfinite((float)r.amplitude), "amplitude must be finite");
  c.need(std::isfinite((float)r.eps) && r.eps >= 0, "eps must be finite and not negative");
  if (c.rc) return c.rc;
  long long t[8];
  for (int i = 0; i < 8; i++) t[i] = c.stride(strides[i], i % 2 == 0 ? r.n_tokens : i / 2 % 2 == 0 ? r.n_heads : r.n_kv_heads);
  if (c.rc || r.n_tokens == 0 || r.n_heads + r.n_kv_heads == 0) return c.rc;
  if (!c.device()) return c.rc;
  if (r.n_heads) c.ptr(r.q, 16, "q"), c.ptr(r.q_out, 16, "q_out");
  if (r.n_kv_heads) c.ptr(r.k, 16, "k"), c.ptr(r.k_out, 16, "k_out");
  c.ptr(r.positions, 4, "positions");
  if (r.n_freqs) c.ptr(r.freqs, 8, "freqs");
  if (r.q_norm) c.ptr(r.q_norm, 4, "q_norm");
  if (r.k_norm) c.ptr(r.k_norm, 4, "k_norm");
  if (c.rc) return c.rc;
  CacheArgs a{};
  a.q = r.q, a.k = r.k, a.qo = r.q_out, a.ko = r.k_out, a.positions = (const int*)r.positions, a.freqs = (const double*)r.freqs;
  a.qw = (const float*)r.q_norm, a.kw = (const float*)r.k_norm;
  for (int i = 0; i < 2; i++) a.sq[i] = t[i], a.sk[i] = t[2 + i], a.sqo[i] = t[4 + i], a.sko[i] = t[6 + i];
  a.T = (int)r.n_tokens, a.H = (int)r.n_heads, a.KH = (int)r.n_kv_heads, a.hd = (int)r.head_dim, a.nf = (int)r.n_freqs;
  a.interleaved = r.interleaved != 0, a.amp = r.amplitude, a.eps64 = r.eps, a.eps = (float)r.eps, a.inv_hd64 = 1.0 / a.hd, a.inv_hd = 1.f / a.hd;
  cudaStream_t s = static_cast<cudaStream_t>(r.stream);
  const long long grid = token_ctas(a, (long long)a.H + a.KH, PC_PER_SM);
  if (!c.need(grid < 1ll << 31, "too many rows")) return c.rc;
  return c.done(r.dtype == ATTN_BF16 ? launch_cache<__nv_bfloat16, PC_ROTARY>(a, (int)grid, s) : launch_cache<__half, PC_ROTARY>(a, (int)grid, s));
}

static int append(ArgCheck& c, const AppendRecord& r) {
  c.need(r.dtype == ATTN_BF16 || r.dtype == ATTN_FP16, "dtype must be 0 (bf16) or 1 (fp16)");
  need_ints(c, &r.n_tokens, 10);
  c.need(r.n_tokens >= 0 && r.batch >= 0 && r.n_heads >= 0 && r.n_kv_heads > 0, "n_kv_heads must be positive, the other counts not negative");
  c.need(r.n_heads < 1 << 16 && r.n_kv_heads < 1 << 16, "too many heads");
  c.need(r.head_dim > 0 && r.head_dim % 8 == 0 && r.head_dim <= ATTN_MAX_HD, "head_dim must be a multiple of 8, at most 128");
  c.need(r.n_freqs >= 0 && 2 * r.n_freqs <= r.head_dim, "at most head_dim / 2 frequencies");
  c.need(std::isfinite((float)r.amplitude), "amplitude must be finite");
  c.need(std::isfinite((float)r.eps) && r.eps >= 0, "eps must be finite and not negative");
  c.need(r.n_tokens == 0 || r.batch > 0, "tokens without a sequence");
  c.need(r.cu || r.batch == 0 || r.n_tokens % r.batch == 0, "without cu there are as many tokens of each sequence");
  c.need(r.n_tokens < 1 << 30, "too many tokens");
  if (c.rc) return c.rc;
  const PoolCheck pool(c, (int)r.page_bits, (int)r.n_pages, (int)r.page, (int)r.table_cols, (int)r.batch, (int)r.n_kv_heads, (int)r.head_dim,
                       r.strides + 8);
  long long t[8];
  for (int i = 0; i < 8; i++)   // q, k, v, q_out
    t[i] = c.stride(r.strides[i], i % 2 == 0 ? r.n_tokens : i / 2 == 0 || i / 2 == 3 ? r.n_heads : r.n_kv_heads);
  if (c.rc || r.n_tokens == 0) return c.rc;
  if (!c.device()) return c.rc;
  c.ptr(r.k, 16, "k"), c.ptr(r.v, 16, "v"), c.ptr(r.lens, 4, "lens");
  if (r.table_cols) c.ptr(r.tables, 4, "tables");
  if (r.n_pages) c.ptr(r.k_pages, 16, "k_pages"), c.ptr(r.v_pages, 16, "v_pages");
  if (r.n_pages && r.page_bits == 8) c.ptr(r.k_scales, 4, "k_scales"), c.ptr(r.v_scales, 4, "v_scales");
  if (r.n_heads) c.ptr(r.q, 16, "q"), c.ptr(r.q_out, 16, "q_out");
  if (r.cu) c.ptr(r.cu, 4, "cu");
  if (r.positions) c.ptr(r.positions, 4, "positions");
  if (r.n_freqs) c.ptr(r.freqs, 8, "freqs");
  if (r.q_norm) c.ptr(r.q_norm, 4, "q_norm");
  if (r.k_norm) c.ptr(r.k_norm, 4, "k_norm");
  if (c.rc) return c.rc;
  CacheArgs a{};
  a.q = r.q, a.k = r.k, a.v = r.v, a.qo = r.q_out, a.kp = (uint8_t*)r.k_pages, a.vp = (uint8_t*)r.v_pages;
  a.ks = (float*)r.k_scales, a.vs = (float*)r.v_scales, a.tables = (const int*)r.tables, a.lens = (const int*)r.lens, a.cu = (const int*)r.cu;
  a.positions = (const int*)r.positions, a.freqs = (const double*)r.freqs, a.qw = (const float*)r.q_norm, a.kw = (const float*)r.k_norm;
  for (int i = 0; i < 2; i++) a.sq[i] = t[i], a.sk[i] = t[2 + i], a.sv[i] = t[4 + i], a.sqo[i] = t[6 + i];
  for (int i = 0; i < 3; i++) a.skp[i] = pool.kp[i], a.svp[i] = pool.vp[i], a.sks[i] = pool.ks[i], a.svs[i] = pool.vs[i];
  a.st = pool.st;
  a.T = (int)r.n_tokens, a.B = (int)r.batch, a.per = a.T / a.B, a.H = (int)r.n_heads, a.KH = (int)r.n_kv_heads, a.hd = (int)r.head_dim;
  a.nf = (int)r.n_freqs, a.n_pages = (int)r.n_pages, a.cols = (int)r.table_cols, a.shift = pool.shift;
  a.interleaved = r.interleaved != 0, a.amp = r.amplitude, a.eps64 = r.eps, a.eps = (float)r.eps, a.inv_hd64 = 1.0 / a.hd, a.inv_hd = 1.f / a.hd;
  long long ctas = r.page_bits == 16 ? token_ctas(a, (long long)a.H + 2 * a.KH, PC_PER_SM) : a.H ? token_ctas(a, a.H, PC_PER_SM - 1) : 0;
  if (!ctas) a.each = 2;
  if (r.page_bits == 8) {   // the runs' CTAs behind: one of them beside those that rotate, on each SM
    a.token_ctas = (int)ctas;
    a.window = 1;
    while (a.window < PC_WINDOW && (a.T + a.window - 1) / a.window > attn_sms() * PC_PER_SM) a.window *= 2;   // all CTAs there at once
    ctas += (a.T + a.window - 1) / a.window;
  }
  if (!c.need(ctas < 1ll << 31, "too many rows")) return c.rc;
  const int grid = (int)ctas;
  cudaStream_t s = static_cast<cudaStream_t>(r.stream);
  const bool bf = r.dtype == ATTN_BF16;
  if (r.page_bits == 16)
    return c.done(bf ? launch_cache<__nv_bfloat16, PC_PAGES16>(a, grid, s) : launch_cache<__half, PC_PAGES16>(a, grid, s));
  return c.done(bf ? launch_cache<__nv_bfloat16, PC_PAGES8>(a, grid, s) : launch_cache<__half, PC_PAGES8>(a, grid, s));
}

static int gather(ArgCheck& c, const GatherRecord& r) {
  c.need(r.dtype == ATTN_BF16 || r.dtype == ATTN_FP16, "dtype must be 0 (bf16) or 1 (fp16)");
  need_ints(c, &r.total, 7);
  c.need(r.total >= 0 && r.batch >= 0 && r.n_kv_heads > 0, "n_kv_heads must be positive, the other counts not negative");
  c.need(r.n_kv_heads < 1 << 20, "too many heads");
  c.need(r.total < 1 << 30, "total must be below 2^30");
  c.need(r.head_dim > 0 && r.head_dim % 8 == 0 && r.head_dim <= ATTN_MAX_HD, "head_dim must be a multiple of 8, at most 128");
  if (c.rc) return c.rc;
  const PoolCheck pool(c, (int)r.page_bits, (int)r.n_pages, (int)r.page, (int)r.table_cols, (int)r.batch, (int)r.n_kv_heads, (int)r.head_dim,
                       r.strides + 4);
  long long t[4];
  for (int i = 0; i < 4; i++) {
    t[i] = c.stride(r.strides[i], i % 2 == 0 ? r.total : r.n_kv_heads);
    c.need(t[i] < 1ll << 35, "strides of the outputs must be below 2^35 elements");
  }
  if (c.rc || r.total == 0 || r.batch == 0) return c.rc;
  if (!c.device()) return c.rc;
  c.ptr(r.cu, 4, "cu"), c.ptr(r.k_out, 16, "k_out"), c.ptr(r.v_out, 16, "v_out");
  if (r.table_cols) c.ptr(r.tables, 4, "tables");
  if (r.n_pages) c.ptr(r.k_pages, 16, "k_pages"), c.ptr(r.v_pages, 16, "v_pages");
  if (r.n_pages && r.page_bits == 8) c.ptr(r.k_scales, 4, "k_scales"), c.ptr(r.v_scales, 4, "v_scales");
  if (c.rc) return c.rc;
  GatherArgs a{};
  a.kp = (const uint8_t*)r.k_pages, a.vp = (const uint8_t*)r.v_pages, a.ks = (const float*)r.k_scales, a.vs = (const float*)r.v_scales;
  a.tables = (const int*)r.tables, a.cu = (const int*)r.cu, a.ko = (uint8_t*)r.k_out, a.vo = (uint8_t*)r.v_out;
  for (int i = 0; i < 3; i++) {
    a.skp[i] = (unsigned)(pool.kp[i] / 16), a.svp[i] = (unsigned)(pool.vp[i] / 16);
    a.sks[i] = (unsigned)pool.ks[i], a.svs[i] = (unsigned)pool.vs[i];
  }
  for (int i = 0; i < 2; i++) a.sko[i] = (unsigned)(t[i] / 8), a.svo[i] = (unsigned)(t[2 + i] / 8);
  a.st = pool.st, a.T = (int)r.total, a.B = (int)r.batch, a.KH = (int)r.n_kv_heads, a.hd = (int)r.head_dim, a.n_pages = (int)r.n_pages;
  a.cols = (int)r.table_cols, a.shift = pool.shift;
  a.wide = ((uintptr_t)r.k_out | (uintptr_t)r.v_out) % 32 == 0 && (t[0] | t[1] | t[2] | t[3]) % 16 == 0;
  int lpr = 1;
  while (lpr < a.hd / (r.page_bits == 8 ? 16 : 8)) lpr *= 2;
  // tokens of a CTA, at least 4: as many as give every SM the same number of full
  // rounds of CTAs (62,346 rows of 4 key heads, 191 MB: three rounds of 29 tokens 36
  // us, one of 85 38; a copy of as many bytes takes 33)
  const long long most = attn_sms() * PC_GATHERS, waves = (a.T + most * PC_GATHER - 1) / (most * PC_GATHER);
  const int per = (int)std::max(4ll, (a.T + most * waves - 1) / (most * waves));
  const dim3 grid((a.T + per - 1) / per);
  cudaStream_t s = static_cast<cudaStream_t>(r.stream);
  const bool bf = r.dtype == ATTN_BF16;
  count_launches(1);
  if (r.page_bits == 16) return c.done(launch_pdl(gather_pages_kernel<__half, false>, grid, PC_THREADS, 0, s, a, lpr, per));
  return c.done(bf ? launch_pdl(gather_pages_kernel<__nv_bfloat16, true>, grid, PC_THREADS, 0, s, a, lpr, per)
                   : launch_pdl(gather_pages_kernel<__half, true>, grid, PC_THREADS, 0, s, a, lpr, per));
}

}  // namespace tg

extern "C" int tg_rotary(int dtype, const void* q, const void* k, void* q_out, void* k_out, const int* positions,
                         const double* freqs, const float* q_norm, const float* k_norm, int n_tokens, int n_heads,
                         int n_kv_heads, int head_dim, int n_freqs, int interleaved, float amplitude, float eps,
                         const int64_t* strides, void* stream) {
  ArgCheck c("tg_rotary");
  if (!c.need(strides != nullptr, "strides is null")) return c.rc;
  RotaryRecord r{0, dtype, q, k, q_out, k_out, positions, freqs, q_norm, k_norm, n_tokens, n_heads, n_kv_heads, head_dim, n_freqs,
                 interleaved, {}, amplitude, eps, stream};
  std::copy(strides, strides + 8, r.strides);
  return rotary(c, r);
}

extern "C" int tg_paged_append(int dtype, int page_bits, const void* q, const void* k, const void* v, void* q_out,
                               void* k_pages, void* v_pages, float* k_scales, float* v_scales, const int* tables,
                               const int* lens, const int* cu, const int* positions, const double* freqs,
                               const float* q_norm, const float* k_norm, int n_tokens, int batch, int n_pages, int page,
                               int table_cols, int n_heads, int n_kv_heads, int head_dim, int n_freqs, int interleaved,
                               float amplitude, float eps, const int64_t* strides, void* stream) {
  ArgCheck c("tg_paged_append");
  if (!c.need(strides != nullptr, "strides is null")) return c.rc;
  AppendRecord r{1, dtype, page_bits, q, k, v, q_out, k_pages, v_pages, k_scales, v_scales, tables, lens, cu, positions, freqs, q_norm,
                 k_norm, n_tokens, batch, n_pages, page, table_cols, n_heads, n_kv_heads, head_dim, n_freqs, interleaved, {}, amplitude,
                 eps, stream};
  std::copy(strides, strides + 21, r.strides);
  return append(c, r);
}

extern "C" int tg_paged_gather(int dtype, int page_bits, const void* k_pages, const void* v_pages, const float* k_scales,
                               const float* v_scales, const int* tables, const int* cu, void* k_out, void* v_out,
                               int total, int batch, int n_pages, int page, int table_cols, int n_kv_heads, int head_dim,
                               const int64_t* strides, void* stream) {
  ArgCheck c("tg_paged_gather");
  if (!c.need(strides != nullptr, "strides is null")) return c.rc;
  GatherRecord r{3, dtype, page_bits, k_pages, v_pages, k_scales, v_scales, tables, cu, k_out, v_out, total, batch, n_pages, page,
                 table_cols, n_kv_heads, head_dim, {}, stream};
  std::copy(strides, strides + 17, r.strides);
  return gather(c, r);
}

extern "C" int tg_paged_call(const void* record) {
  const int64_t op = record ? *static_cast<const int64_t*>(record) : -1;
  static const char* const names[4] = {"tg_rotary", "tg_paged_append", "tg_attention_paged", "tg_paged_gather"};
  ArgCheck c(op >= 0 && op < 4 ? names[op] : "tg_paged_call", true);
  if (op == 0) return rotary(c, *static_cast<const RotaryRecord*>(record));
  if (op == 1) return append(c, *static_cast<const AppendRecord*>(record));
  if (op == 2) return attention_paged(c, *static_cast<const AttendRecord*>(record));
  if (op == 3) return gather(c, *static_cast<const GatherRecord*>(record));
  c.need(false, "the record's first word must be 0 to 3");
  return c.rc;
}
