// g4_kv.cu -- a paged KV cache and the operations on its pages: growing and
// shrinking sequences, forking them (beams, shared prompts), copying and
// compacting pages.
//
// The bookkeeping lives on the device: a page table [sequence][page], the
// sequences' lengths and a reference count per page.  Every operation reads
// its arguments from device memory and is one or two launches, so that a
// decode step with beam search (select, fork, grow, append, attend) runs
// without a host round trip and can be captured into a graph.  Pages are taken
// lowest number first and in the order of a call's entries, which makes every
// result a function of the state alone.
//
// The planning kernels are one CTA: they scan the reference counts once
// (4 bytes a page; 64 K pages are 256 KB) and their cost is latency, not
// bandwidth.  What is bound by HBM is the copying, one warp per (page, layer,
// K or V, head) strip of consecutive bytes, eight 16-byte loads in flight per
// lane: 1001 pages of 256 KB in 81 us (6.5 TB/s read and written, the measured
// copy rate), 64 shared last pages over 8 layers in 12 us. A fork takes 3 to 4 us,
// planning a resize or a compaction 4 to 6 (thousands of pages).
// The copy is a dependent launch that starts while the plan is made. One launch
// whose other CTAs wait for the planning one was slower: 4 beams forked and
// grown 15.4 against 12.1 us, 64 beams 27.5 against 23.3, the compaction of 1001
// pages 101.5 against 95.3.
#include "g4_common.cuh"
#include "g4_kv.h"

#include <cstring>
#include <new>

namespace g4 {

constexpr int kPlanThreads = 1024;
constexpr int kForkThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 8;

struct KvDev {
  int32_t *table, *lens, *refs;
  unsigned* flags;
  int n_pages, n_seqs, max_pages, max_positions, page_size;
};

static KvDev kv_dev(const g4_kv* kv) {
  return KvDev{kv->table,  kv->lens,      kv->refs,          kv->flags,     kv->n_pages,
               kv->n_seqs, kv->max_pages, kv->max_positions, kv->page_size};
}

// Exclusive prefix sum over the CTA (kPlanThreads threads); total in *sum.
// Callers alternate between two sets of warp_sums, so that one barrier is enough.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* warp_sums, T* sum) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  T x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[w] = x;
  __syncthreads();
  const T mine = warp_sums[lane];
  T s = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  *sum = __shfl_sync(0xffffffffu, s, 31);
  return x - v + __shfl_sync(0xffffffffu, s - mine, w);
}

__device__ __forceinline__ bool page_ok(int p, int n_pages) { return (unsigned)p < (unsigned)n_pages; }

// The pages a thread owns in the scans: kRun consecutive ones per round of the
// CTA, in registers between counting and ranking while one round covers the pool.
constexpr int kRun = 8;
struct PageRun {
  int refs[kRun];
  int first, n_pages;
  __device__ __forceinline__ void load(const int32_t* r, int round, int n) {
    n_pages = n;
    first = (round * kPlanThreads + threadIdx.x) * kRun;
    if (first + kRun <= n) {
      const int4 x = __ldcg(reinterpret_cast<const int4*>(r + first));
      const int4 y = __ldcg(reinterpret_cast<const int4*>(r + first) + 1);
      refs[0] = x.x, refs[1] = x.y, refs[2] = x.z, refs[3] = x.w;
      refs[4] = y.x, refs[5] = y.y, refs[6] = y.z, refs[7] = y.w;
    } else {
#pragma unroll
      for (int j = 0; j < kRun; ++j) refs[j] = first + j < n ? __ldcg(r + first + j) : 0;
    }
  }
  __device__ __forceinline__ bool used(int j) const { return refs[j] > 0; }
  __device__ __forceinline__ bool free(int j) const { return refs[j] <= 0 && first + j < n_pages; }
  __device__ __forceinline__ int count_used() const {
    int c = 0;
#pragma unroll
    for (int j = 0; j < kRun; ++j) c += used(j);
    return c;
  }
  __device__ __forceinline__ int count_free() const {
    int c = 0;
#pragma unroll
    for (int j = 0; j < kRun; ++j) c += free(j);
    return c;
  }
};
__device__ __forceinline__ int page_rounds(int n_pages) { return (n_pages + kPlanThreads * kRun - 1) / (kPlanThreads * kRun); }

// g4_kv_resize, planning: new lengths for the entries' sequences, pages given
// back and taken, and the list of shared last pages to copy.
__global__ void __launch_bounds__(kPlanThreads) kv_resize_kernel(KvDev d, const int32_t* seqs, const int32_t* new_lens,
                                                                 int n, int grow_only, int32_t* free_list, KvMove* moves,
                                                                 int32_t* plan) {
  extern __shared__ int sm[];
  int* owner = sm;              // [n_seqs] first entry naming the sequence
  int* es = owner + d.n_seqs;   // [n] the entry's sequence, -1: not taken part
  int* eo = es + n;             // old length
  int* en = eo + n;             // new length
  int* el = en + n;             // shared-page candidate: the last, partly filled page (-1: none)
  int* ec = el + n;             // 1: that page is copied
  int* ea = ec + n;             // first of the entry's pages in free_list
  __shared__ unsigned long long sums64[2][32];
  __shared__ int sums[2][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, ps = d.page_size;
  grid_dep_launch();
  PageRun run;
  run.load(d.refs, 0, d.n_pages);  // looked at below, again if pages are given back
  for (int i = tid; i < d.n_seqs; i += kPlanThreads) owner[i] = 0x7fffffff;
  __syncthreads();
  unsigned bad = 0;
  int shrinks = 0;
  for (int i = tid; i < n; i += kPlanThreads) {
    int s = seqs[i];
    const int nl = new_lens[i];
    if (s >= d.n_seqs || (s >= 0 && (nl < 0 || nl > d.max_positions))) {
      bad |= KV_BAD_ENTRY;
      s = -1;
    }
    es[i] = s;
    en[i] = nl;
    if (s >= 0) atomicMin(owner + s, i);
  }
  __syncthreads();
  for (int i = tid; i < n; i += kPlanThreads) {
    const int s = es[i];
    el[i] = -1;
    if (s < 0) continue;
    const int old = d.lens[s];
    if (owner[s] != i || old < 0 || old > d.max_positions) {
      bad |= KV_BAD_ENTRY;
      es[i] = -1;
      continue;
    }
    eo[i] = old;
    if (grow_only && en[i] < old) en[i] = old;
    shrinks |= en[i] < old;
    if (en[i] > old && old % ps != 0) {
      const int last = d.table[(size_t)s * d.max_pages + old / ps];
      if (page_ok(last, d.n_pages)) {
        el[i] = last;
      } else {  // the table holds no page where the length says there is one
        bad |= KV_BAD_ENTRY;
        es[i] = -1;
      }
    }
  }
  shrinks = __syncthreads_or(shrinks);
  if (shrinks) {  // sequences that shrink give pages back first
    for (int i = warp; i < n; i += kPlanThreads / 32) {
      if (es[i] < 0 || en[i] >= eo[i]) continue;
      const int32_t* row = d.table + (size_t)es[i] * d.max_pages;
      for (int p = (en[i] + ps - 1) / ps + lane; p < (eo[i] + ps - 1) / ps; p += 32)
        if (page_ok(row[p], d.n_pages)) atomicSub(d.refs + row[p], 1);
    }
    __syncthreads();
  }
  // a shared last page is copied by every sequence that grows into it, except
  // one that is left as its only holder; pages wanted per entry
  // (both sums in one scan: pages in the low 44 bits, since 4096 entries of 2^26
  // pages and a copy each pass 32 bits but not 39, copies, 4096 at most, above)
  constexpr int kCopyShift = 44;
  constexpr unsigned long long kPageMask = (1ull << kCopyShift) - 1;
  unsigned long long base = 0;
  for (int i0 = 0, round = 0; i0 < n; i0 += kPlanThreads, ++round) {
    const int i = i0 + tid;
    int need = 0, copied = 0;
    if (i < n && es[i] >= 0) {
      if (el[i] >= 0) {
        const int held = __ldcg(d.refs + el[i]);
        if (held > 1) {
          int earlier = 0;
          for (int j = 0; j < i; ++j) earlier += el[j] == el[i];
          copied = held - earlier > 1;
        }
      }
      const int more = (en[i] + ps - 1) / ps - (eo[i] + ps - 1) / ps;
      need = max(0, more) + copied;
    }
    unsigned long long sum;
    const unsigned long long at =
        base + block_scan(((unsigned long long)copied << kCopyShift) | (unsigned long long)need, sums64[round & 1], &sum);
    if (i < n) {
      ea[i] = (int)(at & kPageMask);  // (read when all of them have a page: at most n_pages)
      ec[i] = copied;
    }
    if (copied) moves[at >> kCopyShift] = KvMove{el[i], i, eo[i] % ps};  // dst: the entry, its page below
    base += sum;
  }
  const int total = (int)min(base & kPageMask, 0x7fffffffull);  // (there are 2^20 pages at most)
  const int copies = (int)(base >> kCopyShift);
  // the lowest free pages
  int found = 0;
  if (total > 0) {
    for (int round = 0; round < page_rounds(d.n_pages) && found < total; ++round) {
      if (round || shrinks) run.load(d.refs, round, d.n_pages);
      int sum, at = found + block_scan(run.count_free(), sums[round & 1], &sum);
#pragma unroll
      for (int j = 0; j < kRun; ++j)
        if (run.free(j)) {
          if (at < total) free_list[at] = run.first + j;
          ++at;
        }
      found += sum;
    }
  }
  if (bad) atomicOr(d.flags, bad);
  __syncthreads();
  if (found < total) {  // nothing changes: take the given-back pages again
    for (int i = shrinks ? warp : n; i < n; i += kPlanThreads / 32) {
      if (es[i] < 0 || en[i] >= eo[i]) continue;
      const int32_t* row = d.table + (size_t)es[i] * d.max_pages;
      for (int p = (en[i] + ps - 1) / ps + lane; p < (eo[i] + ps - 1) / ps; p += 32)
        if (page_ok(row[p], d.n_pages)) atomicAdd(d.refs + row[p], 1);
    }
    if (tid == 0) {
      atomicOr(d.flags, KV_NO_PAGES);
      plan[0] = 0;
    }
    return;
  }
  for (int k = tid; k < total; k += kPlanThreads) d.refs[free_list[k]] = 1;
  for (int k = tid; k < copies; k += kPlanThreads) {
    const int i = moves[k].dst;
    moves[k].dst = free_list[ea[i]];
    atomicSub(d.refs + moves[k].src, 1);
  }
  for (int i = warp; i < n; i += kPlanThreads / 32) {
    if (es[i] < 0) continue;
    int32_t* row = d.table + (size_t)es[i] * d.max_pages;
    const int have = (eo[i] + ps - 1) / ps, want = (en[i] + ps - 1) / ps, a = ea[i] + ec[i];
    if (lane == 0 && ec[i]) row[have - 1] = free_list[ea[i]];
    for (int p = have + lane; p < want; p += 32) row[p] = free_list[a + p - have];
    for (int p = want + lane; p < have; p += 32) row[p] = -1;
    if (lane == 0) d.lens[es[i]] = en[i];
  }
  if (tid == 0) plan[0] = copies;
}

// g4_kv_fork: dst[i] holds the pages of src[i].  A CTA owns W columns of the
// page table for all entries: it reads every source before it writes, so that
// sequences may be both source and destination (beams that change places).
__global__ void __launch_bounds__(kForkThreads) kv_fork_kernel(KvDev d, const int32_t* src, const int32_t* dst, int n,
                                                               int W) {
  extern __shared__ int sm[];
  int* owner = sm;             // [n_seqs]
  int* es = owner + d.n_seqs;  // [n] source, -1: entry skipped
  int* ed = es + n;            // [n] destination
  int* tile = ed + n;          // [n][W]
  const int tid = threadIdx.x;
  for (int i = tid; i < d.n_seqs; i += kForkThreads) owner[i] = 0x7fffffff;
  __syncthreads();
  unsigned bad = 0;
  for (int i = tid; i < n; i += kForkThreads) {
    int s = src[i], t = dst[i];
    if (s < 0 || t < 0) s = -1;
    else if (s >= d.n_seqs || t >= d.n_seqs) {
      bad |= KV_BAD_ENTRY;
      s = -1;
    } else atomicMin(owner + t, i);
    es[i] = s;
    ed[i] = t;
  }
  __syncthreads();
  for (int i = tid; i < n; i += kForkThreads)
    if (es[i] >= 0 && owner[ed[i]] != i) {
      bad |= KV_BAD_ENTRY;
      es[i] = -1;
    }
  __syncthreads();
  const int c0 = blockIdx.x * W, sub = tid % W, rows = kForkThreads / W, p = c0 + sub;
  int* len = tile + (size_t)n * W;  // [n], CTA 0
  for (int i = tid / W; i < n; i += rows)
    tile[i * W + sub] = es[i] >= 0 && p < d.max_pages ? d.table[(size_t)es[i] * d.max_pages + p] : -1;
  if (blockIdx.x == 0)
    for (int i = tid; i < n; i += kForkThreads) len[i] = es[i] >= 0 ? d.lens[es[i]] : 0;
  __syncthreads();
  for (int i = tid / W; i < n; i += rows) {
    if (es[i] < 0 || p >= d.max_pages || es[i] == ed[i]) continue;
    int32_t* at = d.table + (size_t)ed[i] * d.max_pages + p;
    const int now = tile[i * W + sub], old = *at;
    if (now == old) continue;
    if (page_ok(now, d.n_pages)) atomicAdd(d.refs + now, 1);
    if (page_ok(old, d.n_pages)) atomicSub(d.refs + old, 1);
    *at = now;
  }
  if (blockIdx.x == 0) {
    for (int i = tid; i < n; i += kForkThreads)
      if (es[i] >= 0) d.lens[ed[i]] = len[i];
    if (bad) atomicOr(d.flags, bad);
  }
}

// g4_kv_compact, planning: with L live pages, the k-th live page at or behind
// L moves to the k-th free page before L.
__global__ void __launch_bounds__(kPlanThreads) kv_compact_kernel(KvDev d, int32_t* moved, KvMove* moves,
                                                                  int32_t* plan) {
  __shared__ int sums[2][32];
  grid_dep_launch();
  const int tid = threadIdx.x, rounds = page_rounds(d.n_pages);
  PageRun run;
  int L = 0, which = 0;
  for (int round = 0; round < rounds; ++round) {
    run.load(d.refs, round, d.n_pages);
    int sum;
    block_scan(run.count_used(), sums[which ^= 1], &sum);
    L += sum;
  }
  // free pages before L take the live ones behind it: as many of one as of the other
  int holes = 0, movers = 0;
  for (int round = 0; round < rounds; ++round) {
    if (rounds > 1) run.load(d.refs, round, d.n_pages);
    int gaps = 0, late = 0;
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      gaps += run.free(j) && run.first + j < L;
      late += run.used(j) && run.first + j >= L;
    }
    int sum, hole = holes + block_scan(gaps, sums[which ^= 1], &sum);
    holes += sum;
    int mover = movers + block_scan(late, sums[which ^= 1], &sum);
    movers += sum;
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      if (run.free(j) && run.first + j < L) moves[hole++].dst = run.first + j;
      if (run.used(j) && run.first + j >= L) moves[mover++].src = run.first + j;
    }
  }
  __syncthreads();
  for (int k = tid; k < holes; k += kPlanThreads) {
    const int s = moves[k].src, t = moves[k].dst;
    moves[k].rows = d.page_size;
    moved[s] = t;
    d.refs[t] = __ldcg(d.refs + s);
    d.refs[s] = 0;
  }
  if (tid == 0) {
    plan[0] = holes;
    plan[1] = L;
  }
}

// Copies the first rows positions of pages, all layers, K and V: a warp per
// strip.  moves with *count entries, or (moves == nullptr) n pairs of whole
// pages src -> dst.  table != nullptr: its entries behind the live pages
// (compaction) change to their new numbers.
__global__ void __launch_bounds__(kCopyThreads) kv_copy_kernel(KvDev d, const KvStrip* strips, int n_strips,
                                                               const KvMove* moves, const int32_t* plan,
                                                               const int32_t* src, const int32_t* dst, int n,
                                                               const int32_t* moved, int remap) {
  grid_dep_wait();
  const int lane = threadIdx.x & 31, warps = gridDim.x * (kCopyThreads / 32);
  const int warp = blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5);
  const int count = moves ? plan[0] : n;
  if (remap && count > 0) {
    const int live = plan[1];
    const long long cells = (long long)d.n_seqs * d.max_pages;
    for (long long i = (long long)blockIdx.x * kCopyThreads + threadIdx.x; i < cells;
         i += (long long)gridDim.x * kCopyThreads) {
      const int p = d.table[i];
      if (p >= live && p < d.n_pages) d.table[i] = moved[p];
    }
  }
  const long long units = (long long)count * n_strips;
  for (long long u = warp; u < units; u += warps) {
    const int m = (int)(u / n_strips);
    const KvStrip s = strips[u - (long long)m * n_strips];
    KvMove mv = moves ? moves[m] : KvMove{src[m], dst[m], d.page_size};
    if (mv.src < 0 || mv.dst < 0 || mv.src == mv.dst) continue;
    if (mv.src >= d.n_pages || mv.dst >= d.n_pages) {
      if (lane == 0) atomicOr(d.flags, KV_BAD_ENTRY);
      continue;
    }
    const uint4* from = reinterpret_cast<const uint4*>(s.base + mv.src * s.page_stride);
    uint4* to = reinterpret_cast<uint4*>(s.base + mv.dst * s.page_stride);
    const int chunks = (int)(mv.rows * s.row_bytes / 16);
    for (int c = lane; c < chunks; c += 32 * kCopyUnroll) {
      uint4 x[kCopyUnroll];
#pragma unroll
      for (int j = 0; j < kCopyUnroll; ++j)
        if (c + 32 * j < chunks) x[j] = __ldcs(from + c + 32 * j);
#pragma unroll
      for (int j = 0; j < kCopyUnroll; ++j)
        if (c + 32 * j < chunks) __stcs(to + c + 32 * j, x[j]);
    }
  }
}

// g4_kv_check: the number of free pages, and the record, which starts anew.
__global__ void __launch_bounds__(kPlanThreads) kv_check_kernel(KvDev d) {
  __shared__ int sums[32];
  int mine = 0, sum;
  for (int p = threadIdx.x; p < d.n_pages; p += kPlanThreads) mine += d.refs[p] <= 0;
  block_scan(mine, sums, &sum);
  if (threadIdx.x == 0) {
    d.flags[1] = (unsigned)sum;
    // read and cleared at once: attention on another stream may be recording
    d.flags[2] = atomicExch(d.flags, 0u);
  }
}

static int copy_grid(const g4_kv* kv, long long max_moves) {
  const long long units = max_moves * kv->n_strips, per = kCopyThreads / 32;
  const long long full = (long long)kv->ctx->dev.sms * 8;
  const long long want = (units + per - 1) / per;
  return (int)(want < 1 ? 1 : want < full ? want : full);
}

static size_t resize_smem(const g4_kv* kv, int n) { return ((size_t)kv->n_seqs + 6 * (size_t)n) * 4; }

// Columns of the page table per CTA: whole 128-byte lines while the tile of
// every entry's columns fits 64 KB, 32-byte sectors beyond.
static int fork_width(int n) { return n <= 512 ? 32 : 8; }
static size_t fork_smem(const g4_kv* kv, int n) {
  return ((size_t)kv->n_seqs + 3 * (size_t)n + (size_t)n * fork_width(n)) * 4;
}

static int entries_ok(g4_kv* kv, const char* what, const void* a, const void* b, int n, int most) {
  if (n < 0 || n > most || (n > 0 && (!a || !b))) {
    kv->ctx->set_err("%s: bad arguments (%d entries, at most %d; device arrays)", what, n, most);
    return G4_E_ARG;
  }
  return 0;
}

int kv_resize(g4_kv* kv, const int32_t* seqs, const int32_t* lens, int n, bool grow_only, cudaStream_t st,
              const char* what) {
  g4_ctx* c = kv->ctx;
  if (int r = entries_ok(kv, what, seqs, lens, n, kv->n_seqs)) return r;
  if (n == 0) return 0;
  DeviceScope scope(c);
  if (scope.rc) return scope.rc;
  const KvDev d = kv_dev(kv);
  kv_resize_kernel<<<1, kPlanThreads, resize_smem(kv, n), st>>>(d, seqs, lens, n, grow_only, kv->free_list, kv->moves,
                                                                kv->plan);
  cudaError_t e = cudaGetLastError();
  if (!e)
    e = launch_after(kv_copy_kernel, dim3(copy_grid(kv, n)), dim3(kCopyThreads), 0, st, d, kv->strips, kv->n_strips,
                     kv->moves, kv->plan, nullptr, nullptr, 0, nullptr, 0);
  return e ? c->cuda_fail(e, what) : 0;
}

}  // namespace g4

using namespace g4;

extern "C" {

int g4_kv_create(g4_ctx* c, const g4_kv_config* cfg, g4_kv** out) {
  if (!c) return G4_E_ARG;
  if (!cfg || !out) {
    c->set_err("g4_kv_create: NULL argument");
    return G4_E_ARG;
  }
  *out = nullptr;
  if (cfg->type != G4_TYPE_F32 && cfg->type != G4_TYPE_F16 && cfg->type != G4_TYPE_BF16) {
    c->set_err("g4_kv_create: cache type %d (F32, F16 or BF16)", cfg->type);
    return G4_E_TYPE;
  }
  const int ps = cfg->page_size;
  if (cfg->n_layers < 1 || cfg->n_layers > 1024 || !cfg->n_kv_heads || !cfg->head_size ||
      (ps != 16 && ps != 32 && ps != 64 && ps != 128 && ps != 256) || cfg->n_pages < 1 || cfg->n_pages > kKvMaxPages ||
      cfg->n_seqs < 1 || cfg->n_seqs > kKvMaxSeqs || cfg->max_positions < 1 || cfg->max_positions > (1 << 30)) {
    c->set_err("g4_kv_create: bad configuration (1..1024 layers, pages of 16, 32, 64, 128 or 256 positions, 1..%d "
               "pages, 1..%d sequences, 1..2^30 positions)", kKvMaxPages, kKvMaxSeqs);
    return G4_E_ARG;
  }
  for (int l = 0; l < cfg->n_layers; ++l)
    if (cfg->n_kv_heads[l] < 1 || cfg->n_kv_heads[l] > 256 || cfg->head_size[l] < 8 ||
        cfg->head_size[l] > kKvMaxHeadSize || cfg->head_size[l] % 8) {
      c->set_err("g4_kv_create: layer %d: %d KV heads of size %d (1..256 heads, sizes 8..%d in steps of 8)", l,
                 cfg->n_kv_heads[l], cfg->head_size[l], kKvMaxHeadSize);
      return G4_E_ARG;
    }
  DeviceScope scope(c);
  if (scope.rc) return scope.rc;
  g4_kv* kv = new (std::nothrow) g4_kv();
  if (!kv) return G4_E_NOMEM;
  kv->ctx = c;
  kv->device = c->dev.device;
  std::vector<KvStrip> strips;
  uint64_t bytes = 0;
  try {
    kv->n_layers = cfg->n_layers;
    kv->type = cfg->type;
    kv->elem = cfg->type == G4_TYPE_F32 ? 4 : 2;
    kv->page_size = ps;
    while ((1 << kv->page_shift) < ps) ++kv->page_shift;
    kv->n_pages = cfg->n_pages;
    kv->n_seqs = cfg->n_seqs;
    kv->max_positions = cfg->max_positions;
    kv->max_pages = (cfg->max_positions + ps - 1) / ps;
    kv->n_kv.assign(cfg->n_kv_heads, cfg->n_kv_heads + cfg->n_layers);
    kv->hs.assign(cfg->head_size, cfg->head_size + cfg->n_layers);
    kv->k.resize(cfg->n_layers);
    kv->v.resize(cfg->n_layers);
    kv->k_map.resize(cfg->n_layers);
    kv->v_map.resize(cfg->n_layers);
    for (int l = 0; l < cfg->n_layers; ++l)
      bytes += 2 * (((uint64_t)kv->n_pages * kv->n_kv[l] * ps * kv->hs[l] * kv->elem + 255) / 256 * 256);
    size_t n_strips = 0;
    for (int l = 0; l < cfg->n_layers; ++l) n_strips += 2 * (size_t)kv->n_kv[l];
    strips.reserve(n_strips);
  } catch (...) {
    delete kv;
    c->set_err("g4_kv_create: out of host memory");
    return G4_E_NOMEM;
  }
  if (cudaMalloc(&kv->pool, bytes) != cudaSuccess) {
    cudaGetLastError();
    kv->pool = nullptr;
    g4_kv_free(kv);
    c->set_err("g4_kv_create: cannot allocate %llu bytes of pages", (unsigned long long)bytes);
    return G4_E_NOMEM;
  }
  uint8_t* at = kv->pool;
  for (int l = 0; l < kv->n_layers; ++l) {
    const uint64_t strip = (uint64_t)ps * kv->hs[l] * kv->elem, page = strip * kv->n_kv[l];
    const uint64_t layer = (page * kv->n_pages + 255) / 256 * 256;
    kv->k[l] = at;
    kv->v[l] = at + layer;
    for (int half = 0; half < 2; ++half)
      for (int h = 0; h < kv->n_kv[l]; ++h)
        strips.push_back(KvStrip{at + half * layer + h * strip, page, (uint32_t)(kv->hs[l] * kv->elem), 0});
    at += 2 * layer;
  }
  kv->n_strips = (int)strips.size();
  auto up = [](uint64_t b) { return (b + 255) / 256 * 256; };
  const uint64_t b_table = up((uint64_t)kv->n_seqs * kv->max_pages * 4), b_lens = up((uint64_t)kv->n_seqs * 4),
                 b_refs = up((uint64_t)kv->n_pages * 4), b_strips = up(strips.size() * sizeof(KvStrip)),
                 n_moves = kv->n_pages > kv->n_seqs ? kv->n_pages : kv->n_seqs, b_moves = up(n_moves * sizeof(KvMove));
  const uint64_t meta = b_table + b_lens + 2 * b_refs + b_strips + b_moves + 512;
  if (cudaMalloc(&kv->meta, meta) != cudaSuccess) {
    cudaGetLastError();
    kv->meta = nullptr;
    g4_kv_free(kv);
    c->set_err("g4_kv_create: cannot allocate %llu bytes of page tables", (unsigned long long)meta);
    return G4_E_NOMEM;
  }
  uint8_t* p = kv->meta;
  kv->table = reinterpret_cast<int32_t*>(p);
  p += b_table;
  kv->lens = reinterpret_cast<int32_t*>(p);
  p += b_lens;
  kv->refs = reinterpret_cast<int32_t*>(p);
  p += b_refs;
  kv->free_list = reinterpret_cast<int32_t*>(p);
  p += b_refs;
  kv->strips = reinterpret_cast<KvStrip*>(p);
  p += b_strips;
  kv->moves = reinterpret_cast<KvMove*>(p);
  p += b_moves;
  kv->plan = reinterpret_cast<int32_t*>(p);
  kv->flags = reinterpret_cast<unsigned*>(p + 256);
  cudaError_t e = cudaMemset(kv->pool, 0, bytes);
  if (!e) e = cudaMemset(kv->meta, 0, meta);
  if (!e) e = cudaMemset(kv->table, 0xff, (size_t)kv->n_seqs * kv->max_pages * 4);  // -1: no page
  if (!e) e = cudaMemcpy(kv->strips, strips.data(), strips.size() * sizeof(KvStrip), cudaMemcpyHostToDevice);
  const int optin = (int)c->dev.smem_optin;
  if (!e) e = cudaFuncSetAttribute(kv_resize_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, optin - 1024);
  if (!e) e = cudaFuncSetAttribute(kv_fork_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, optin - 1024);
  cudaFuncAttributes fa;  // loads the kernels, so that a first call may be captured
  if (!e) e = cudaFuncGetAttributes(&fa, kv_compact_kernel);
  if (!e) e = cudaFuncGetAttributes(&fa, kv_copy_kernel);
  if (!e) e = cudaFuncGetAttributes(&fa, kv_check_kernel);
  if (!e) e = (cudaError_t)rope_prepare();
  if (!e) e = (cudaError_t)kv_attend_prepare(kv);
  if (!e) e = cudaDeviceSynchronize();
  if (e) {
    g4_kv_free(kv);
    return c->cuda_fail(e, "g4_kv_create");
  }
  *out = kv;
  return 0;
}

int g4_kv_free(g4_kv* kv) {
  if (!kv) return G4_E_ARG;
  {
    DeviceScope scope(kv->device);
    if (kv->pool) cudaFree(kv->pool);
    if (kv->meta) cudaFree(kv->meta);
  }
  delete kv;
  return 0;
}

void* g4_kv_k(const g4_kv* kv, int layer) {
  return kv && layer >= 0 && layer < kv->n_layers ? kv->k[layer] : nullptr;
}
void* g4_kv_v(const g4_kv* kv, int layer) {
  return kv && layer >= 0 && layer < kv->n_layers ? kv->v[layer] : nullptr;
}
int32_t* g4_kv_table(const g4_kv* kv) { return kv ? kv->table : nullptr; }
int32_t* g4_kv_lens(const g4_kv* kv) { return kv ? kv->lens : nullptr; }
int32_t* g4_kv_refs(const g4_kv* kv) { return kv ? kv->refs : nullptr; }

int g4_kv_resize(g4_kv* kv, const int32_t* seqs, const int32_t* lens, int n, void* stream) {
  return kv ? kv_resize(kv, seqs, lens, n, false, (cudaStream_t)stream, "g4_kv_resize") : G4_E_ARG;
}

int g4_kv_fork(g4_kv* kv, const int32_t* src, const int32_t* dst, int n, void* stream) {
  if (!kv) return G4_E_ARG;
  g4_ctx* c = kv->ctx;
  if (int r = entries_ok(kv, "g4_kv_fork", src, dst, n, kv->n_seqs)) return r;
  if (n == 0) return 0;
  DeviceScope scope(c);
  if (scope.rc) return scope.rc;
  const int W = fork_width(n), grid = (kv->max_pages + W - 1) / W;
  kv_fork_kernel<<<grid, kForkThreads, fork_smem(kv, n), (cudaStream_t)stream>>>(kv_dev(kv), src, dst, n, W);
  cudaError_t e = cudaGetLastError();
  return e ? c->cuda_fail(e, "g4_kv_fork") : 0;
}

int g4_kv_compact(g4_kv* kv, void* stream) {
  if (!kv) return G4_E_ARG;
  g4_ctx* c = kv->ctx;
  DeviceScope scope(c);
  if (scope.rc) return scope.rc;
  cudaStream_t st = (cudaStream_t)stream;
  const KvDev d = kv_dev(kv);
  kv_compact_kernel<<<1, kPlanThreads, 0, st>>>(d, kv->free_list, kv->moves, kv->plan);
  cudaError_t e = cudaGetLastError();
  if (!e)
    e = launch_after(kv_copy_kernel, dim3(copy_grid(kv, kv->n_pages / 2 + 1)), dim3(kCopyThreads), 0, st, d, kv->strips,
                     kv->n_strips, kv->moves, kv->plan, nullptr, nullptr, 0, kv->free_list, 1);
  return e ? c->cuda_fail(e, "g4_kv_compact") : 0;
}

int g4_kv_copy_pages(g4_kv* kv, const int32_t* src, const int32_t* dst, int n, void* stream) {
  if (!kv) return G4_E_ARG;
  g4_ctx* c = kv->ctx;
  if (int r = entries_ok(kv, "g4_kv_copy_pages", src, dst, n, kv->n_pages)) return r;
  if (n == 0) return 0;
  DeviceScope scope(c);
  if (scope.rc) return scope.rc;
  kv_copy_kernel<<<copy_grid(kv, n), kCopyThreads, 0, (cudaStream_t)stream>>>(
      kv_dev(kv), kv->strips, kv->n_strips, nullptr, nullptr, src, dst, n, nullptr, 0);
  cudaError_t e = cudaGetLastError();
  return e ? c->cuda_fail(e, "g4_kv_copy_pages") : 0;
}

int g4_kv_check(g4_kv* kv, int* free_pages, void* stream) {
  if (!kv) return G4_E_ARG;
  g4_ctx* c = kv->ctx;
  DeviceScope scope(c);
  if (scope.rc) return scope.rc;
  cudaStream_t st = (cudaStream_t)stream;
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  cudaError_t e = cudaStreamIsCapturing(st, &cap);
  if (e) return c->cuda_fail(e, "g4_kv_check");
  if (cap != cudaStreamCaptureStatusNone) {
    c->set_err("g4_kv_check: waits for the stream, which is being captured");
    return G4_E_ARG;
  }
  unsigned read[2] = {0, 0};
  kv_check_kernel<<<1, kPlanThreads, 0, st>>>(kv_dev(kv));
  e = cudaGetLastError();
  if (!e) e = cudaMemcpyAsync(read, kv->flags + 1, sizeof read, cudaMemcpyDeviceToHost, st);
  if (!e) e = cudaStreamSynchronize(st);
  if (e) return c->cuda_fail(e, "g4_kv_check");
  const unsigned found = read[1];
  if (free_pages) *free_pages = (int)read[0];
  if (!found) return 0;
  c->set_err("g4_kv_check:%s%s%s%s%s", found & KV_NO_PAGES ? " not enough free pages (the resize changed nothing);" : "",
             found & KV_BAD_ENTRY ? " an entry's sequence, length or page is out of range or named twice;" : "",
             found & KV_NOT_STORED ? " an appended position has no page or lies in a shared one;" : "",
             found & KV_BAD_ROW ? " a row's sequence or position is out of range or sees a position without a page;" : "",
             found & KV_TIMEOUT ? " a bounded wait expired inside a kernel;" : "");
  return found & KV_NO_PAGES ? G4_E_NOMEM : G4_E_DEVICE;
}

}  // extern "C"
