// tg_paged.h — where tokens lie in a paged cache: index arithmetic alone, for
// the kernels (tg_paged_cache.cu, tg_attn_paged.cu) and, without CUDA's
// headers, for the host.
//
// Position p of sequence b is row p % page of the page tables[b][p / page].  A
// position below zero or behind the table's columns, and a page outside the
// pool, is no place: nothing is read or written there.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#include "tg_attn.h"
#define TG_HD __host__ __device__ __forceinline__
#else
#define TG_HD inline
#endif

namespace tg {

constexpr int PAGED_BLOCK = 16;      // tokens under one scale
constexpr int PAGED_MIN_EXP = -117;  // smallest scale's exponent: code x scale stays a normal fp32 number (2^-9 2^-117)

// The page of position p, or -1.  shift: log2 of the page's rows.
TG_HD int paged_page(const int* table, int cols, int p, int shift, int n_pages) {
  if (p < 0 || (p >> shift) >= cols) return -1;
  const int page = table[p >> shift];
  return page >= 0 && page < n_pages ? page : -1;
}

// The last b of 0 .. n - 1 with cu[b] <= t, or 0; within bounds whatever cu holds.
TG_HD int paged_search(const int* cu, int n, int t) {
  int lo = 0, hi = n;   // cu[lo] <= t (or lo = 0), cu[hi] > t (or hi = n)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Packed token t: its sequence (-1: of none), the sequence's first packed
// token and the one behind its last.  cu null: `per` tokens of each sequence.
struct PagedToken {
  int seq, first, end;
};
TG_HD PagedToken paged_token(const int* cu, int n_seqs, int per, int total, int t) {
  PagedToken k;
  if (!cu) {
    k.seq = t / per;
    k.first = k.seq * per;
    k.end = k.first + per;
    return k;
  }
  k.seq = paged_search(cu, n_seqs, t);
  k.first = cu[k.seq] > 0 ? cu[k.seq] : 0;
  k.end = cu[k.seq + 1] < total ? cu[k.seq + 1] : total;
  if (t < k.first || t >= k.end) k.seq = -1;
  return k;
}

// The position of packed token t whose sequence has `len` positions with its
// last new token: at most 2^31 - 1, below zero for what is no position.
TG_HD int paged_position(int len, int end, int t) {
  const long long p = (long long)len - ((long long)end - t);
  return p < -0x7fffffffll ? -0x7fffffff : (int)p;
}

// Tokens of one block that a call writes together: their first is the first
// new one of its sequence or the first of its block.  Returns how many there
// are from token t at position p on, 0 if t is not their first or has no place.
TG_HD int paged_run(const PagedToken& k, int t, int p) {
  if (k.seq < 0 || p < 0 || (t != k.first && p % PAGED_BLOCK)) return 0;
  const int room = PAGED_BLOCK - p % PAGED_BLOCK, left = k.end - t;
  return room < left ? room : left;
}

// The exponent of the least power of two under which a value of these fp32
// bits (finite, not negative) fits e4m3's largest, 448 = 1.75 2^8.
TG_HD int paged_scale_exp(uint32_t amax) {
  const int e = (int)(amax >> 23) - 127 - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e > PAGED_MIN_EXP ? e : PAGED_MIN_EXP;
}

// Keys that the queries of a sequence with `len` positions read, [lo, hi), lo
// rounded down to a whole block of 16; its newest `queries` positions ask.
TG_HD int paged_first(int len, int queries, int window) {
  const long long lo = (long long)len - queries + 1 - window;
  return window > 0 && lo > 0 ? (int)lo : 0;
}
TG_HD int paged_tiles(int len, int queries, int window, int keys) {
  const int lo = paged_first(len, queries, window) & ~(PAGED_BLOCK - 1);
  return len > lo ? (int)(((long long)len - lo + keys - 1) / keys) : 0;
}

#ifdef __CUDACC__
// The checks that entries on pages share: the pool, the table, the strides.
struct PoolCheck {
  int shift = 0;
  long long kp[3], vp[3], ks[3] = {}, vs[3] = {}, st = 1;
  // strides: k_pages (page, head, row), v_pages, k_scales (page, head, block), v_scales, tables (row): 13 values
  PoolCheck(ArgCheck& c, int bits, int n_pages, int page, int cols, int batch, int n_kv_heads, int head_dim, const int64_t* t) {
    c.need(bits == 8 || bits == 16, "page_bits must be 8 or 16");
    c.need(n_pages >= 0 && cols >= 0, "n_pages and table_cols must not be negative");
    c.need(page >= 16 && page <= 1 << 20 && (page & (page - 1)) == 0, "page must be a power of two, at least 16");
    c.need(bits == 16 || head_dim % 16 == 0, "head_dim must be a multiple of 16 for pages of 8 bits");
    if (c.rc) return;
    while (1 << shift < page) shift++;
    const long long n[3] = {n_pages, n_kv_heads, page}, nb[3] = {n_pages, n_kv_heads, page / PAGED_BLOCK};
    for (int i = 0; i < 6; i++) {
      long long s = t[i];
      if (n[i % 3] > 1) {
        c.need(s > 0 && s < (1ll << 36) / (bits / 8) && s * bits / 8 % 16 == 0,
               "strides of pages must be positive multiples of 16 bytes, below 2^36 bytes");
      } else {
        s = 0;
      }
      (i < 3 ? kp[i] : vp[i - 3]) = s * bits / 8;
    }
    for (int i = 0; bits == 8 && i < 6; i++) {
      long long s = t[6 + i];
      if (nb[i % 3] > 1)
        c.need(s > 0 && s < 1ll << 31, "strides of scales must be positive and below 2^31");
      else
        s = 0;
      (i < 3 ? ks[i] : vs[i - 3]) = s;
    }
    if (batch > 1) {
      c.need(t[12] > 0, "the stride of tables must be positive");
      st = t[12];
    }
  }
};

// The entries' arguments as one record of 64-bit words, as tg_paged_call takes
// them; the pointers are the caller's word for device memory.
struct RotaryRecord {
  int64_t op, dtype;
  const void *q, *k;
  void *q_out, *k_out;
  const void *positions, *freqs, *q_norm, *k_norm;
  int64_t n_tokens, n_heads, n_kv_heads, head_dim, n_freqs, interleaved, strides[8];
  double amplitude, eps;
  void* stream;
};
struct AppendRecord {
  int64_t op, dtype, page_bits;
  const void *q, *k, *v;
  void *q_out, *k_pages, *v_pages, *k_scales, *v_scales;
  const void *tables, *lens, *cu, *positions, *freqs, *q_norm, *k_norm;
  int64_t n_tokens, batch, n_pages, page, table_cols, n_heads, n_kv_heads, head_dim, n_freqs, interleaved, strides[21];
  double amplitude, eps;
  void* stream;
};
struct AttendRecord {
  int64_t op, dtype, page_bits;
  const void *q, *k_pages, *v_pages, *k_scales, *v_scales;
  void* out;
  const void *tables, *lens, *sinks;
  int64_t batch, n_queries, n_pages, page, table_cols, max_len, n_heads, n_kv_heads, head_dim, window, strides[19];
  double scale;
  void* workspace;
  int64_t workspace_bytes;
  void* stream;
};
struct GatherRecord {
  int64_t op, dtype, page_bits;
  const void *k_pages, *v_pages, *k_scales, *v_scales, *tables, *cu;
  void *k_out, *v_out;
  int64_t total, batch, n_pages, page, table_cols, n_kv_heads, head_dim, strides[17];
  void* stream;
};
// Counts of a record: the n words from `at` on, which have to be 32-bit numbers.
inline void need_ints(ArgCheck& c, const int64_t* at, int n) {
  for (int i = 0; i < n; i++) c.need(at[i] >= INT32_MIN && at[i] <= INT32_MAX, "a count does not fit 32 bits");
}
int attention_paged(ArgCheck& c, const AttendRecord& r);   // tg_attn_paged.cu
#endif

}  // namespace tg
