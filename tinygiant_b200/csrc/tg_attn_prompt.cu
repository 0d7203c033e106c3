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
// Three launches.  plan_kernel (one CTA) reads the lengths on the device and
// lists the units of work, longest first, splitting the keys of those that
// cost more than an SM's share of the whole; the tensor-core kernel
// (tg_attn_tc.cuh) works through the list; combine_kernel joins split units.
// Short sequences need neither plan nor joining.
#include <algorithm>
#include <atomic>

#include "../../include/tinygiant.h"
#include "tg_attn_tc.cuh"

namespace tg {

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_BUCKETS = 512;
constexpr int PLAN_SPLITS = 256;   // split units, at most: each costs over twice an SM's share
// Key blocks of a split unit's piece, at least: 8 tokens on 4,088 keys take
// 24.3 us with 4, 25.2 with 2 and 32.1 with 1 (the join reads more pieces).
constexpr int MIN_PIECE = 4;

static __device__ DevStatus g_attn_status;

// The record's address on each device where an operator with waits was called.
static std::atomic<DevStatus*> g_status_at[ATTN_DEVICES];

DevStatus* attn_status() {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= ATTN_DEVICES) return nullptr;
  DevStatus* at = g_status_at[dev].load();
  if (!at) {
    if (cudaGetSymbolAddress((void**)&at, g_attn_status) != cudaSuccess) {
      cudaGetLastError();
      return nullptr;
    }
    g_status_at[dev] = at;
  }
  return at;
}

// Reports waits that ran out in the operators' kernels, on any device, since
// the last report, and clears the records.  In two steps around the library
// stream's synchronisation, with copies on that stream into pinned memory: no
// other stream is waited for, and where no operator ran nothing is done.
bool attn_status_copy_async(cudaStream_t s, const char* what) {
  for (int i = 0; i < ATTN_DEVICES; i++)
    if (const DevStatus* at = g_status_at[i].load()) {
      const cudaError_t e = cudaMemcpyAsync(attn_status_host() + i, at, sizeof *at, cudaMemcpyDeviceToHost, s);
      if (e != cudaSuccess) {
        set_host_error(100 + (int)e, "%s: reading the attention operators' status failed (%s)", what, cudaGetErrorString(e));
        return false;
      }
    }
  return true;
}
bool attn_finish_copied(cudaStream_t s, const char* what) {
  bool ok = true;
  for (int i = 0; i < ATTN_DEVICES; i++) {
    DevStatus *at = g_status_at[i].load(), *h = attn_status_host() + i;
    if (!at || h->code == 0) continue;
    cudaMemsetAsync(at, 0, sizeof *at, s);
    cudaStreamSynchronize(s);
    set_host_error(200 + h->code, "%s: device error %d at site %d of an attention operator (%d, %d)", what, h->code, h->where, h->a, h->b);
    h->code = 0;
    ok = false;
  }
  return ok;
}

// The operators' waits, by a warp, a warp that has time and a thread, for a
// barrier that nothing arrives at; records how many gave up.
__global__ void __launch_bounds__(96) debug_wait_kernel(DevStatus* st) {
  __shared__ uint64_t bar;
  __shared__ int abort, gave_up;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    abort = gave_up = 0;
    fence_mbar_init();
  }
  __syncthreads();
  const int w = threadIdx.x / 32, lane = threadIdx.x % 32;
  bool ok = true;
  if (w == 0)
    ok = at_wait(&bar, 0, &abort);
  else if (w == 1)
    ok = at_wait_idle(&bar, 0, &abort);
  else if (lane == 0)
    ok = at_wait(&bar, 0, &abort);
  if (!ok && lane == 0) atomicAdd(&gave_up, 1);
  __syncthreads();
  if (threadIdx.x == 0 && gave_up) set_error(st, ERR_WAIT_TIMEOUT, 399, gave_up);
}

struct PlanArgs {
  AttnHead* head;
  AttnEntry* entries;
  AttnSplit* splits;
  const int *cu_q, *cu_k;
  int n_seqs, total_q, total_k, tpu, KH, window, sms;
  int max_entries, max_slots;   // capacities (slots per key head)
};

// One CTA; about 4 us warm, most of it the launch and four barriers.
__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(const PlanArgs a) {
  __shared__ int hist[PLAN_BUCKETS];
  __shared__ AttnSeq seqs[PLAN_THREADS];
  __shared__ int ends[PLAN_THREADS];
  __shared__ int sums[PLAN_THREADS / 32];
  __shared__ AttnEntry split[PLAN_SPLITS];
  __shared__ int split_at[PLAN_SPLITS], split_n[PLAN_SPLITS];
  __shared__ unsigned long long s_total;
  __shared__ int s_max, s_slots, s_splits, s_n;
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  if (tid == 0) s_total = 0, s_max = 0, s_slots = 0, s_splits = 0;
  for (int i = tid; i < PLAN_BUCKETS; i += PLAN_THREADS) hist[i] = 0;
  // PLAN_THREADS sequences from s0 on in shared memory, with where their
  // units end; returns the number of their units
  auto load = [&](int s0) -> int {
    __syncthreads();
    AttnSeq q{};
    if (s0 + tid < a.n_seqs) q = attn_seq(a.cu_q, a.cu_k, s0 + tid, a.total_q, a.total_k);
    int x = (q.nq + a.tpu - 1) / a.tpu;
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(~0u, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sums[w] = x;
    __syncthreads();
    static_assert(PLAN_THREADS == 1024, "a lane for each warp's sum");
    const int s = sums[lane], before = __reduce_add_sync(~0u, lane < w ? s : 0), all = __reduce_add_sync(~0u, s);
    seqs[tid] = q;
    ends[tid] = before + x;
    __syncthreads();
    return all;
  };
  // f(entry, cost) for every unit
  auto each = [&](auto f) {
    for (int s0 = 0; s0 < a.n_seqs; s0 += PLAN_THREADS) {
      const int n = a.n_seqs > PLAN_THREADS ? load(s0) : ends[PLAN_THREADS - 1];
      for (int u = tid; u < n; u += PLAN_THREADS) {
        int lo = 0;   // the first sequence whose units end past u
        for (int step = PLAN_THREADS / 2; step; step >>= 1)
          if (ends[lo + step - 1] <= u) lo += step;
        const AttnSeq q = seqs[lo];
        const AttnEntry e = attn_unit(q, (u - (ends[lo] - (q.nq + a.tpu - 1) / a.tpu)) * a.tpu, a.tpu, a.window);
        f(e, e.nb);
      }
    }
  };
  if (a.n_seqs <= PLAN_THREADS) load(0);
  unsigned long long sum = 0;
  int mx = 0;
  each([&](const AttnEntry& e, int cost) {
    sum += cost;
    mx = max(mx, cost);
  });
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  mx = __reduce_max_sync(~0u, mx);
  if (lane == 0) {
    atomicAdd(&s_total, sum);
    atomicMax(&s_max, mx);
  }
  __syncthreads();
  // Units of more than twice `share` blocks are split into equal pieces of at
  // most `share` (a piece costs a partial result; taken first, a unit of up to
  // twice an SM's share delays the end by less than that: 1,024 tokens take 29
  // us, against 36 with every unit over one share split).  There are at most
  // 2 total / share pieces, which bounds them by the capacity.
  const unsigned long long total = s_total;
  int share = 0x7fffffff;
  if (a.max_slots > 0) {
    const unsigned long long even = (total * a.KH + a.sms - 1) / a.sms, room = (2 * total + a.max_slots - 1) / a.max_slots;
    share = (int)min((unsigned long long)0x7fffffff, max((unsigned long long)MIN_PIECE, max(even, room)));
  }
  auto pieces = [&](int cost) { return cost > 2ll * share ? (cost + share - 1) / share : 1; };
  const int top = max(1, (int)min((long long)s_max, 2ll * share));
  auto bucket = [&](int size) { return top < PLAN_BUCKETS ? top - size : (int)((long long)(top - size) * PLAN_BUCKETS / (top + 1)); };
  each([&](const AttnEntry& e, int cost) {
    const int n = pieces(cost);
    atomicAdd(&hist[bucket((cost + n - 1) / n)], n);
  });
  __syncthreads();
  if (w == 0) {   // exclusive sums: where each bucket starts
    int run = 0;
    for (int b0 = 0; b0 <= min(top, PLAN_BUCKETS - 1); b0 += 32) {
      const int v = hist[b0 + lane];
      int x = v;
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, x, o);
        if (lane >= o) x += y;
      }
      hist[b0 + lane] = run + x - v;
      run += __shfl_sync(~0u, x, 31);
    }
    if (lane == 0) s_n = run;
  }
  __syncthreads();
  each([&](const AttnEntry& e, int cost) {
    const int n = pieces(cost), at = atomicAdd(&hist[bucket((cost + n - 1) / n)], n);
    if (n == 1) {
      if (at < a.max_entries) a.entries[at] = e;
      return;
    }
    AttnEntry x = e;
    x.slot = atomicAdd(&s_slots, n);
    const int i = atomicAdd(&s_splits, 1);
    if (x.slot + n > a.max_slots || i >= PLAN_SPLITS) return;   // not reached: see the bound above
    a.splits[i] = AttnSplit{e.q0, e.ntok, x.slot, n};
    split[i] = x;
    split_at[i] = at;
    split_n[i] = n;
  });
  __syncthreads();
  for (int i = w; i < min(s_splits, PLAN_SPLITS); i += PLAN_THREADS / 32) {   // a warp per split unit, a lane per piece
    const AttnEntry e = split[i];
    const int n = split_n[i];
    for (int p = lane; p < n; p += 32) {
      AttnEntry x = e;
      const int b0 = (int)((long long)e.nb * p / n), b1 = (int)((long long)e.nb * (p + 1) / n);
      x.ks = e.ks + b0 * AT_KEYS;
      x.nb = b1 - b0;
      x.slot = e.slot + p;
      if (split_at[i] + p < a.max_entries) a.entries[split_at[i] + p] = x;
    }
  }
  __syncthreads();
  if (tid == 0) {
    a.head->n_entries = min(s_n, a.max_entries);
    a.head->counter = 0;
    a.head->n_splits = min(min(s_splits, a.max_slots), PLAN_SPLITS);
  }
}

struct CombineArgs {
  const AttnHead* head;
  const AttnSplit* splits;
  const float* po;
  const float2* pml;
  const float* sinks;
  void* out;
  long long so[2];
  int G, KH, hd, tpt;
};

// A warp per (split unit, key head, tile row); bound by the latency of four
// dependent reads: 3 us without splits, 7 us for 32 pieces of 64 rows.
template <typename T, int HD>
__global__ void __launch_bounds__(256) combine_kernel(const CombineArgs a) {
  pdl_wait();
  const int n = a.head->n_splits * a.KH * 2 * AT_ROWS;
  for (int i = blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += gridDim.x * 8) {
    const int row = i % AT_ROWS, t = i / AT_ROWS % 2, kh = i / (2 * AT_ROWS) % a.KH;
    const AttnSplit s = a.splits[i / (2 * AT_ROWS * a.KH)];
    const int tok = row / a.G, g = row - tok * a.G, tt = t * a.tpt + tok, h = kh * a.G + g;
    if (tok >= a.tpt || tt >= s.ntok) continue;
    auto at = [&](int p) { return ((size_t)(s.slot + p) * a.KH + kh) * (2 * AT_ROWS) + t * AT_ROWS + row; };
    const float2 fin = join_scale(s.n, a.pml, a.sinks ? a.sinks[h] * LOG2E : -INFINITY, at);
    join_row<T, HD>(s.n, a.pml, a.po, fin, at, (T*)a.out + (s.q0 + tt) * a.so[0] + h * a.so[1], a.hd);
  }
}

// The workspace: header, entries, splits, then the partial results.
struct PromptSpace {
  int max_entries, max_slots;
  // Without splits (no sequence has more keys than a piece) and with a lane for
  // each sequence the units need no list: three sequences of 14 tokens take 6.8
  // us instead of 14.5 with the plan's launch before.
  bool plan;
  size_t entries, splits, pml, po, bytes;
  PromptSpace(int n_seqs, int total_q, int max_k, int H, int KH, int hd) {
    const long long tpu = 2 * (AT_ROWS / (H / KH)), units = (total_q + tpu - 1) / tpu + n_seqs;
    const long long blocks = (max_k + AT_KEYS - 1) / AT_KEYS;
    // pieces of split units per key head: two per SM, and no more than units of the longest sequence's keys make
    const long long slots = blocks <= MIN_PIECE ? 0 : std::min((long long)(2 * attn_sms() / KH + 1), units * ((blocks + MIN_PIECE - 1) / MIN_PIECE));
    max_slots = (int)slots;
    max_entries = (int)std::min(units + slots, (long long)1 << 30);
    auto take = [&](size_t n) {
      const size_t o = bytes;
      bytes = (bytes + n + 255) & ~(size_t)255;
      return o;
    };
    bytes = 0;
    entries = splits = pml = po = 0;
    plan = max_slots > 0 || n_seqs > 32;
    if (!plan) return;
    take(sizeof(AttnHead));
    entries = take(sizeof(AttnEntry) * max_entries);
    splits = take(sizeof(AttnSplit) * max_slots);
    const size_t rows = (size_t)max_slots * KH * 2 * AT_ROWS;
    pml = take(sizeof(float2) * rows);
    po = take(sizeof(float) * rows * (hd <= 64 ? 64 : 128));
  }
};

template <typename T, int HD>
static cudaError_t run_prompt(const PlanArgs& p, const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, const AttnTcArgs& a,
                              const CombineArgs& c, long long units, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  if (a.entries) {
    e = launch_pdl(plan_kernel, dim3(1), PLAN_THREADS, 0, s, p);
    count_launches(1);
  }
  const long long work = (units + p.max_slots) * p.KH;
  if (e == cudaSuccess) e = launch_attn_tc<T, HD, false>(qm, km, vm, a, (int)std::min((long long)p.sms, work), s);
  count_launches(1);
  if (e == cudaSuccess && p.max_slots > 0) {
    e = launch_pdl(combine_kernel<T, HD>, dim3(8 * p.sms), 256, 0, s, c);
    count_launches(1);
  }
  return e;
}

}  // namespace tg

using namespace tg;

extern "C" int tg_cuda_debug_attn_wait(void) {
  std::lock_guard<std::recursive_mutex> lk(ctx_mutex());
  if (!ensure_init()) return -1;
  DevStatus* st = attn_status();
  if (!st) return -1;
  debug_wait_kernel<<<1, 96, 0, stream()>>>(st);
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return 0;
  set_host_error(100 + (int)e, "tg_cuda_debug_attn_wait: %s", cudaGetErrorString(e));
  return -1;
}

extern "C" size_t tg_attention_prompt_workspace(int n_seqs, int total_q, int max_k, int n_heads, int n_kv_heads,
                                                int head_dim) {
  if (n_seqs < 0 || total_q < 0 || max_k < 0 || n_kv_heads <= 0 || n_heads < n_kv_heads || n_heads / n_kv_heads > AT_ROWS) return 0;
  return PromptSpace(n_seqs, total_q, max_k, n_heads, n_kv_heads, head_dim).bytes;
}

extern "C" int tg_attention_prompt(int dtype, const void* q, const void* k, const void* v, void* out, const int* cu_q,
                                   const int* cu_k, const float* sinks, int n_seqs, int total_q, int total_k,
                                   int max_k, int n_heads, int n_kv_heads, int head_dim, const int64_t* strides,
                                   int window, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  ArgCheck c("tg_attention_prompt");
  c.need(dtype == ATTN_BF16 || dtype == ATTN_FP16, "dtype must be 0 (bf16) or 1 (fp16)");
  c.need(n_seqs >= 0 && total_q >= 0 && total_k >= 0 && max_k >= 0 && window >= 0, "counts and window must not be negative");
  c.need(total_q < AT_NPOS && total_k < AT_NPOS, "too many rows");
  c.need(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && n_heads / n_kv_heads <= 128,
         "n_heads must be a multiple of n_kv_heads, at most 128 times it");
  c.need(head_dim > 0 && head_dim % 8 == 0 && head_dim <= ATTN_MAX_HD, "head_dim must be a multiple of 8, at most 128");
  c.need(std::isfinite(scale) && scale > 0.f, "scale must be finite and positive");
  c.need(strides != nullptr, "strides is null");
  if (c.rc) return c.rc;
  const long long n4[4] = {total_q, n_heads, total_k, n_kv_heads};
  const int dim[8] = {0, 1, 2, 3, 2, 3, 0, 1};
  long long st[8];
  for (int i = 0; i < 8; i++) st[i] = c.stride(strides[i], n4[dim[i]]);
  if (c.rc || total_q == 0) return c.rc;
  c.need(n_seqs > 0, "rows without a sequence");
  window = std::min(window, AT_NPOS);   // beyond any position: position - window stays an int
  if (!c.device()) return c.rc;
  c.ptr(q, 16, "q"), c.ptr(out, 16, "out"), c.ptr(cu_q, 4, "cu_q"), c.ptr(cu_k, 4, "cu_k");
  if (total_k > 0) c.ptr(k, 16, "k"), c.ptr(v, 16, "v");
  if (sinks) c.ptr(sinks, 4, "sinks");
  const PromptSpace sp(n_seqs, total_q, max_k, n_heads, n_kv_heads, head_dim);
  c.need(workspace_bytes >= sp.bytes, "the workspace is smaller than tg_attention_prompt_workspace says");
  if (sp.bytes > 0) c.ptr(workspace, 256, "workspace");
  if (c.rc) return c.rc;

  const int G = n_heads / n_kv_heads, tpt = AT_ROWS / G;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  PlanArgs p{(AttnHead*)ws, (AttnEntry*)(ws + sp.entries), (AttnSplit*)(ws + sp.splits), cu_q, cu_k, n_seqs, total_q, total_k,
             2 * tpt, n_kv_heads, window, attn_sms(), sp.max_entries, sp.max_slots};
  AttnTcArgs a{};
  a.head = p.head;
  a.entries = sp.plan ? p.entries : nullptr;   // null: dealt out in turn
  a.cu_q = cu_q, a.cu_k = cu_k, a.n_seqs = n_seqs, a.total_q = total_q;
  a.out = out;
  a.po = (float*)(ws + sp.po);
  a.pml = (float2*)(ws + sp.pml);
  a.sinks = sinks;
  a.so[0] = st[6], a.so[1] = st[7];
  a.v = v, a.sv[0] = st[4], a.sv[1] = st[5];
  a.G = G, a.KH = n_kv_heads, a.hd = head_dim, a.tpt = tpt, a.window = window, a.total_k = total_k;
  a.wide = head_dim % 16 == 0 && (uintptr_t)out % 32 == 0 && st[6] % 16 == 0 && st[7] % 16 == 0;
  a.c = scale * LOG2E;
  a.st = attn_status();
  CombineArgs cb{p.head, p.splits, a.po, a.pml, sinks, out, {st[6], st[7]}, G, n_kv_heads, head_dim, tpt};
  CUtensorMap qm, km, vm;
  c.need(attn_q_map(&qm, dtype, q, head_dim, n_heads, total_q, st[0], st[1], G, tpt) &&
             attn_kv_map(&km, dtype, k, q, head_dim, n_kv_heads, total_k, st[2], st[3]) &&
             attn_kv_map(&vm, dtype, v, q, head_dim, n_kv_heads, total_k, st[4], st[5]),
         "the tensors' shapes and strides do not fit a tensor map");
  if (c.rc) return c.rc;
  const long long units = (total_q + 2ll * tpt - 1) / (2 * tpt) + n_seqs;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = dtype == ATTN_BF16, small = head_dim <= 64;
  return c.done(bf ? (small ? run_prompt<__nv_bfloat16, 64>(p, qm, km, vm, a, cb, units, s)
                            : run_prompt<__nv_bfloat16, 128>(p, qm, km, vm, a, cb, units, s))
                   : (small ? run_prompt<__half, 64>(p, qm, km, vm, a, cb, units, s)
                            : run_prompt<__half, 128>(p, qm, km, vm, a, cb, units, s)));
}
