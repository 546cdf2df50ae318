// g4_beam.cu -- beam search's selection: for every group of `beams` rows, the
// `beams` best of all continuations score_b + logit_bt - log sum_t exp(logit_bt).
//
// One pass over the logits, bound by HBM (4 bytes a candidate): a warp takes a
// strip of kStrip consecutive logits of a row and leaves its maximum and its sum
// of exponentials, nothing else; no barrier, no shared memory, no list. A second
// launch, one CTA per group, adds the strips' sums up in 64 bits and finds every
// strip's best score. At most `beams` strips can hold a winner: those first
// in the order (best score, then row and strip). Only they are read again, by a
// warp each, and their `beams` best logits ranked by counting.
//
// Precision: the exponentials (hardware ex2, 2^-22) and a strip's sum are 32-bit:
// the scan is bound by its 4 bytes a candidate and would not be with 64-bit ones.
// A row's logarithm is off by 1e-7 or so, the same for all its tokens; scores are
// then put together and compared in 64 bits. Within a row that is the order of the
// logits; continuations of different rows that lie closer than 1e-7 may change places.
//
// 64 rows of 262144 (16 groups of 4): 21 us, 13.3 for the scan (10.2 at the copy
// rate; 16384 strips are 3.5 waves of the resident warps) and the rest for the pick,
// which is latency: five steps with a barrier each. Selecting in the scan itself
// (sorted maxima and candidates per chunk) took 32 us, a ring of chunks with a
// running bound 33, persistent warps with the next strip in flight 26.
//
// Order: by the score so made, ties to the lower row, then the lower token; equal
// logits of one row have equal scores. Every comparison is on unique pairs, so
// the result does not depend on the order in which warps arrive. A strip that is
// not among the first `beams` holds no winner: each of those has a continuation
// that comes before all of its own.
#include "g4_common.cuh"
#include "g4_kv.h"

#include <cfloat>

namespace g4 {

constexpr int kScanThreads = 128;
constexpr int kStrip = 1024;  // logits per warp: 32 per lane, 4 KB in flight
constexpr int kMaxBeams = 32;
constexpr int kPickThreads = 1024;

// exp(v - m) is taken as 2^((v - m) * kLog2e) with this rounded constant
// throughout, and the logarithm divided by the same one. The maximum is
// subtracted before the factor: a product of a logit of -1e10 is rounded by
// hundreds, one of 2.4e38 is infinite, and such logits are how a vocabulary is
// masked; a difference is exact next to the maximum, and one that overflows is
// -inf, whose term is 0. Every finite strip's sum is then 1 to kStrip.
constexpr float kLog2e = 1.4426950408889634f;

// A strip: its largest logit m (-inf: none) and the sum of 2^((v - m) * kLog2e).
struct StripStat {
  float m, sum;
};

// A number's order as an unsigned word (NaN below everything, the zeros equal).
__device__ __forceinline__ uint32_t order_of(float v) {
  if (!(v == v)) return 0u;
  const uint32_t u = v == 0.f ? 0u : __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ unsigned long long order_of(double v) {
  const unsigned long long u = v == 0.0 ? 0ull : (unsigned long long)__double_as_longlong(v);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

__device__ __forceinline__ float beam_exp2(float x) {  // relative error 2^-22
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A strip's logits, 32 per lane (-inf behind the row's end); returns how lane
// elements map to tokens: first + step * i, in runs of four where the row is
// 16-byte aligned.
struct StripMap {
  int base, quad;
  __device__ __forceinline__ int token(int i) const { return quad ? base + (i >> 2) * 128 + (i & 3) : base + i * 32; }
};
__device__ __forceinline__ StripMap load_strip(const float* row, int vocab, int t0, int lane, float (&v)[32]) {
  const float* x = row + t0;
  StripMap map;
  map.quad = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  map.base = t0 + (map.quad ? 4 * lane : lane);
  if (map.quad && t0 + kStrip <= vocab) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(x) + i * 32 + lane);
      v[4 * i] = f.x;
      v[4 * i + 1] = f.y;
      v[4 * i + 2] = f.z;
      v[4 * i + 3] = f.w;
    }
  } else {
    map.quad = 0;
    map.base = t0 + lane;
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = map.base + 32 * i < vocab ? __ldg(x + lane + 32 * i) : -INFINITY;
  }
  return map;
}

__global__ void __launch_bounds__(kScanThreads) beam_scan_kernel(const float* logits, long long stride, int vocab,
                                                                 const int32_t* finished, int n_rows, int strips,
                                                                 StripStat* stats) {
  const int lane = threadIdx.x & 31;
  const unsigned w = blockIdx.x * (kScanThreads / 32) + (threadIdx.x >> 5);
  grid_dep_launch();
  const unsigned row = w / (unsigned)strips;
  if (row >= (unsigned)n_rows || (finished && finished[row])) return;  // a finished row needs no logits
  float v[32];
  load_strip(logits + (long long)row * stride, vocab, (int)(w - row * strips) * kStrip, lane, v);
  float m0 = -INFINITY, m1 = -INFINITY;  // (a NaN is never the larger one)
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    m0 = fmaxf(m0, v[i]);
    m1 = fmaxf(m1, v[i + 1]);
  }
  const float m = value_of(__reduce_max_sync(0xffffffffu, order_of(fmaxf(m0, m1))));
  const float base = m == -INFINITY ? 0.f : m;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 32; ++i) s[i & 3] += beam_exp2((v[i] - base) * kLog2e);
  float sum = (s[0] + s[1]) + (s[2] + s[3]);
  if (!(sum == sum)) {  // NaNs count as masked
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) sum += v[i] == v[i] ? beam_exp2((v[i] - base) * kLog2e) : 0.f;
  }
  sum = warp_sum(sum);
  if (lane == 0) stats[w] = StripStat{m, sum};
}

// A continuation's or strip's place in the order: larger key first, then lower index.
struct __align__(16) Ranked {
  unsigned long long key;  // 0: none
  long long at;
  __device__ __forceinline__ bool before(const Ranked& o) const {
    return (key > o.key) | ((key == o.key) & (at < o.at));
  }
};

// How many of n entries (shared memory) come before one; a warp together.
__device__ __forceinline__ int warp_rank(const Ranked* all, int n, const Ranked& r, int lane) {
  int rank = 0;
  for (int j = lane; j < n; j += 32) rank += all[j].before(r);
  return (int)__reduce_add_sync(0xffffffffu, (unsigned)rank);
}

// The lanes' entries in order (bitonic).
__device__ __forceinline__ Ranked warp_sort(Ranked r, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) {
      Ranked other;
      other.key = __shfl_xor_sync(0xffffffffu, r.key, o);
      other.at = __shfl_xor_sync(0xffffffffu, (int)r.at, o);
      const bool keep_first = ((lane & o) == 0) == ((lane & size) == 0);
      if (other.before(r) == keep_first) r = other;
    }
  return r;
}

__global__ void __launch_bounds__(kPickThreads) beam_pick_kernel(
    const float* logits, long long stride, int vocab, const StripStat* stats, const float* scores,
    const int32_t* finished, int beams, int strips, int pad_token, float* new_scores, int32_t* parents,
    int32_t* tokens) {
  constexpr int NW = kPickThreads / 32;
  // a row's largest logit and the logarithm of its sum relative to that one. A log
  // probability is (logit - largest) - logarithm: their sum would lose the
  // logarithm beside a largest logit of -1e20, where nothing of a row is live.
  __shared__ double largest[kMaxBeams], log_sum[kMaxBeams], score_of[kMaxBeams];
  __shared__ int done[kMaxBeams];
  __shared__ Ranked lists[NW * kMaxBeams];
  __shared__ Ranked chosen[kMaxBeams];
  __shared__ Ranked cand[kMaxBeams * kMaxBeams];  // at: row and token; until they are scored, key: the logit's order
  __shared__ double cand_score[kMaxBeams * kMaxBeams];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g0 = blockIdx.x * beams;
  if (tid < beams) {
    done[tid] = finished ? finished[g0 + tid] : 0;
    score_of[tid] = (double)scores[g0 + tid];
  }
  __syncthreads();
  grid_dep_wait();
  for (int b = warp; b < beams; b += NW) {
    if (done[b]) continue;
    const StripStat* st = stats + (long long)(g0 + b) * strips;
    float M = -INFINITY;
    double s = 0.0;
    // up to eight strips per lane stay in registers
    constexpr int kHold = 8;
    StripStat x[kHold];
#pragma unroll
    for (int i = 0; i < kHold; ++i) x[i] = lane + 32 * i < strips ? st[lane + 32 * i] : StripStat{-INFINITY, 0.f};
#pragma unroll
    for (int i = 0; i < kHold; ++i) M = fmaxf(M, x[i].m);
    for (int i = lane + 32 * kHold; i < strips; i += 32) M = fmaxf(M, st[i].m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    auto part = [&](const StripStat& t) { return t.m > -INFINITY ? t.sum * beam_exp2((t.m - M) * kLog2e) : 0.f; };
    float near = 0.f;
#pragma unroll
    for (int i = 0; i < kHold; ++i) near += part(x[i]);
    for (int i = lane + 32 * kHold; i < strips; i += 32) s += (double)part(st[i]);
    s += (double)near;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) {
      largest[b] = M == -INFINITY ? 0.0 : (double)M;
      log_sum[b] = M == -INFINITY ? INFINITY : log2(s) / (double)kLog2e;
    }
  }
  __syncthreads();

  // ---- the strips in order of their best score: each warp's first ones, then all
  Ranked kept{0, 0x7fffffff};
  const int total = beams * strips;
  for (int i0 = warp * 32; i0 < total; i0 += kPickThreads) {
    const int i = i0 + lane, b = min(i / strips, beams - 1);
    Ranked r{0, i};
    if (i < total) {
      double sc = -INFINITY;
      if (done[b]) {
        if (i == b * strips) sc = score_of[b];
      } else {
        const float m = stats[(long long)g0 * strips + i].m;
        if (m > -INFINITY) sc = score_of[b] + (((double)m - largest[b]) - log_sum[b]);
      }
      if (sc > -INFINITY) r.key = order_of(sc);
    }
    const unsigned long long least = __shfl_sync(0xffffffffu, kept.key, beams - 1);
    if (!__any_sync(0xffffffffu, r.key > least)) continue;
    r = warp_sort(r, lane);
    if (__all_sync(0xffffffffu, kept.key == 0)) {  // the warp's first
      kept = r;
      continue;
    }
    // both are in order: of entry i and entry 31 - i of the other, the first are the 32 first
    Ranked other;
    other.key = __shfl_sync(0xffffffffu, r.key, 31 - lane);
    other.at = __shfl_sync(0xffffffffu, (int)r.at, 31 - lane);
    if (other.before(kept)) kept = other;
    kept = warp_sort(kept, lane);
  }
  if (lane < beams) lists[warp * beams + lane] = kept;
  if (tid < beams) chosen[tid] = Ranked{0, 0};
  __syncthreads();
  for (int i = warp; i < NW * beams; i += NW) {
    const Ranked r = lists[i];
    if (r.key == 0) continue;
    const int rank = warp_rank(lists, NW * beams, r, lane);
    if (rank < beams && lane == 0) chosen[rank] = r;
  }
  __syncthreads();

  // ---- their best logits: a warp per strip
  for (int r = warp; r < beams; r += NW) {
    const Ranked strip = chosen[r];
    const int b = min((int)strip.at / strips, beams - 1), row = g0 + b;
    float v[32];
    StripMap map{0, 0};
    const bool reads = strip.key != 0 && !done[b];  // the same in every lane
    if (reads) {
      map = load_strip(logits + (long long)row * stride, vocab, ((int)strip.at - b * strips) * kStrip, lane, v);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = v[i] == v[i] ? v[i] : -INFINITY;
    }
    // the lane's largest logit, lowest token first (its elements are in token
    // order); taken, the lane looks for its next one
    float m = -INFINITY;
    int at = 0;
    auto look = [&]() {
      float x[16];
      int i_of[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool second = v[2 * i + 1] > v[2 * i];
        x[i] = second ? v[2 * i + 1] : v[2 * i];
        i_of[i] = 2 * i + second;
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1)
#pragma unroll
        for (int i = 0; i < w; ++i) {
          const bool second = x[2 * i + 1] > x[2 * i];
          x[i] = second ? x[2 * i + 1] : x[2 * i];
          i_of[i] = second ? i_of[2 * i + 1] : i_of[2 * i];
        }
      m = x[0];
      at = i_of[0];
    };
    if (reads) look();
    for (int k = 0; k < beams; ++k) {
      const uint32_t mine = m > -INFINITY ? order_of(m) : 0u;
      const uint32_t top = __reduce_max_sync(0xffffffffu, mine);
      const uint32_t token = (uint32_t)map.token(at);
      const uint32_t first = __reduce_min_sync(0xffffffffu, top && mine == top ? token : 0xffffffffu);
      if (lane == 0) cand[r * beams + k] = Ranked{top, ((long long)row << 32) | first};
      if (top && mine == top && token == first) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i == at) v[i] = -INFINITY;
        look();
      }
      __syncwarp();
    }
    if (lane == 0 && strip.key != 0 && !reads) cand[r * beams] = Ranked{1, ((long long)row << 32) | (uint32_t)pad_token};
  }
  if (tid < beams) {
    new_scores[g0 + tid] = -INFINITY;
    parents[g0 + tid] = -1;
    tokens[g0 + tid] = -1;
  }
  __syncthreads();

  // ---- their scores, and the first of all
  const int n = beams * beams;
  for (int i = tid; i < n; i += kPickThreads) {
    const Ranked c = cand[i];
    if (c.key == 0) continue;
    const int b = (int)(c.at >> 32) - g0;
    const double sc =
        done[b] ? score_of[b] : score_of[b] + (((double)value_of((uint32_t)c.key) - largest[b]) - log_sum[b]);
    cand_score[i] = sc;
    cand[i].key = order_of(sc);
  }
  __syncthreads();
  for (int i = warp; i < n; i += NW) {
    const Ranked c = cand[i];
    if (c.key == 0) continue;
    const int rank = warp_rank(cand, n, c, lane);
    if (rank < beams && lane == 0) {
      new_scores[g0 + rank] = (float)cand_score[i];
      parents[g0 + rank] = (int)(c.at >> 32);
      tokens[g0 + rank] = (int)(uint32_t)c.at;
    }
  }
}

int beam_prepare() {
  cudaFuncAttributes fa;
  cudaError_t e = cudaFuncGetAttributes(&fa, beam_scan_kernel);
  if (!e) e = cudaFuncGetAttributes(&fa, beam_pick_kernel);
  return e;
}

static long long beam_strips(int vocab) { return ((long long)vocab + kStrip - 1) / kStrip; }

}  // namespace g4

using namespace g4;

extern "C" {

size_t g4_beam_select_workspace(int n_rows, int vocab, int beams) {
  if (n_rows < 1 || vocab < 1 || vocab > (1 << 30) || beams < 1 || beams > kMaxBeams) return 0;
  return (size_t)n_rows * beam_strips(vocab) * sizeof(StripStat);
}

int g4_beam_select(g4_ctx* c, const float* logits, int64_t stride, int vocab, const float* scores,
                   const int32_t* finished, int n_rows, int beams, int pad_token, float* new_scores, int32_t* parents,
                   int32_t* tokens, void* work, size_t work_bytes, void* stream) {
  if (!c) return G4_E_ARG;
  const long long strips = vocab > 0 ? beam_strips(vocab) : 0;
  if (n_rows < 0 || vocab < 1 || vocab > (1 << 30) || beams < 1 || beams > kMaxBeams || n_rows % beams ||
      n_rows * strips > (1ll << 30) ||
      (n_rows > 0 && (!logits || !scores || !new_scores || !parents || !tokens || (n_rows > 1 && stride < vocab)))) {
    c->set_err("g4_beam_select: bad arguments (%d rows of %d tokens, %d beams, at most %d; rows a multiple of the "
               "beams)", n_rows, vocab, beams, kMaxBeams);
    return G4_E_ARG;
  }
  if (n_rows == 0) return 0;
  const size_t need = g4_beam_select_workspace(n_rows, vocab, beams);
  if (!work || work_bytes < need || (reinterpret_cast<uintptr_t>(work) & 15)) {
    c->set_err("g4_beam_select: work space of %zu bytes, needs %zu (16-byte aligned)", work ? work_bytes : (size_t)0,
               need);
    return G4_E_ARG;
  }
  DeviceScope scope(c);
  if (scope.rc) return scope.rc;
  cudaStream_t st = (cudaStream_t)stream;
  StripStat* stats = static_cast<StripStat*>(work);
  const unsigned grid = (unsigned)((n_rows * strips + kScanThreads / 32 - 1) / (kScanThreads / 32));
  beam_scan_kernel<<<grid, kScanThreads, 0, st>>>(logits, stride, vocab, finished, n_rows, (int)strips, stats);
  cudaError_t e = cudaGetLastError();
  if (!e)
    e = launch_after(beam_pick_kernel, dim3(n_rows / beams), dim3(kPickThreads), 0, st, logits, stride, vocab, stats,
                     scores, finished, beams, (int)strips, pad_token, new_scores, parents, tokens);
  return e ? c->cuda_fail(e, "g4_beam_select") : 0;
}

}  // extern "C"
