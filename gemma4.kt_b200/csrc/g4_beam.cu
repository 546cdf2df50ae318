// g4_beam.cu -- beam search's selection: for every group of `beams` rows, the
// `beams` best of all continuations score_b + logit_bt - log sum_t exp(logit_bt).
//
// One pass over the logits (bound by HBM: 4 bytes a candidate).  A CTA holds
// kChunk logits of a row in registers and takes from them the chunk's maximum
// and sum of exponentials and its `beams` largest logits: the beams-th largest
// of the threads' own maxima bounds them from below (the warps sort theirs and
// rank them in each other's lists), so only candidates at or above it (beams to
// 32 * beams of kChunk) are ranked, by counting.  A second
// launch joins a group's chunks: the log sums in 64 bits, then the best
// continuations by the same ranking, on 64-bit scores.
//
// Order: within a row by logit, ties to the lower token (the row's constant
// shifts all alike); across rows by the 64-bit score, ties to the lower beam.
// Every comparison is on unique (value, index) pairs, so the result does not
// depend on the order in which candidates arrive.
#include "g4_common.cuh"
#include "g4_kv.h"

namespace g4 {

constexpr int kBeamThreads = 256;
constexpr int kBeamPer = 32;                          // logits per thread
constexpr int kChunk = kBeamThreads * kBeamPer;
constexpr int kMaxBeams = 32;
constexpr int kBeamJoinThreads = 512;

// A float's order as an unsigned word (NaN below everything).
__device__ __forceinline__ uint32_t order_of(float v) {
  if (!(v == v)) return 0u;
  const uint32_t u = __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

struct ChunkStat {
  float m, sum;
};

// The lanes' keys in descending order (bitonic).
__device__ __forceinline__ unsigned long long warp_sort(unsigned long long k, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, o);
      const bool keep_max = ((lane & o) == 0) == ((lane & size) == 0);
      k = (other > k) == keep_max ? other : k;
    }
  return k;
}

__global__ void __launch_bounds__(kBeamThreads, 4)
    beam_chunk_kernel(const float* logits, long long stride, int vocab, const int32_t* finished, int beams, int chunks,
                      unsigned long long* best, ChunkStat* stats) {
  constexpr int NW = kBeamThreads / 32, G = kBeamPer / 4;
  __shared__ unsigned long long top[NW][kMaxBeams];
  __shared__ unsigned long long cand[kMaxBeams * kBeamPer];
  __shared__ unsigned long long bound_s;
  __shared__ float red[NW];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / chunks, c = blockIdx.x - row * chunks;
  grid_dep_launch();
  if (finished && finished[row]) return;  // its one continuation needs no logits
  const float* x = logits + row * stride;
  const int t0 = c * kChunk;
  if (tid == 0) count = 0;
  // group i of a thread: tokens t0 + i * 1024 + 4 tid + {0..3}
  float v[G][4];
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && t0 + kChunk <= vocab;
  if (vec) {
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const float4 f = __ldcs(reinterpret_cast<const float4*>(x + t0 + (i * kBeamThreads + tid) * 4));
      v[i][0] = f.x;
      v[i][1] = f.y;
      v[i][2] = f.z;
      v[i][3] = f.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = t0 + (i * kBeamThreads + tid) * 4 + j;
        v[i][j] = t < vocab ? x[t] : -INFINITY;
      }
  }
  // the thread's largest logit (a NaN is never the larger one) and its group
  float m = -INFINITY;
  int at = 0;
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const float g = fmaxf(fmaxf(v[i][0], v[i][1]), fmaxf(v[i][2], v[i][3]));
    if (g > m) {
      m = g;
      at = i;
    }
  }
  auto key_of = [&](float f, int token) {
    return ((unsigned long long)order_of(f) << 32) | (0xffffffffu - (uint32_t)token);
  };
  // The bound: the beams-th largest of the threads' keys, a key being the
  // largest logit with its group's last token, so at most that of the logit
  // itself: beams candidates reach it, all in threads whose keys do.
  const unsigned long long mine = key_of(m, t0 + (at * kBeamThreads + tid) * 4 + 3);
  const unsigned long long sorted = warp_sort(mine, lane);
  if (lane < beams) top[warp][lane] = sorted;
  const float warp_max = value_of((uint32_t)(__shfl_sync(0xffffffffu, sorted, 0) >> 32));
  if (lane == 0) red[warp] = warp_max;
  __syncthreads();
  float M = red[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) M = fmaxf(M, red[i]);
  if (lane < beams) {
    int rank = lane;
    for (int w = 1; w < NW; ++w) {  // in another warp's list: how many are larger
      const unsigned long long* list = top[(warp + w) % NW];
      int r = 0;
      for (int i = 0; i < beams && list[i] > sorted; ++i) ++r;
      rank += r;
    }
    if (rank == beams - 1) bound_s = sorted;
  }
  const float base = M == -INFINITY ? 0.f : M;
  float s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int i = 0; i < G; ++i) {
    s0 += __expf(v[i][0] - base) + __expf(v[i][1] - base);
    s1 += __expf(v[i][2] - base) + __expf(v[i][3] - base);
  }
  if (!(s0 + s1 == s0 + s1)) {  // NaNs count as masked
    s0 = s1 = 0.f;
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s0 += v[i][j] == v[i][j] ? __expf(v[i][j] - base) : 0.f;
  }
  const float sum = warp_sum(s0 + s1);
  __syncthreads();
  if (lane == 0) red[warp] = sum;
  const unsigned long long bound = bound_s;
  if (mine >= bound) {
    const float bv = value_of((uint32_t)(bound >> 32));
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v[i][j] >= bv) {
          const unsigned long long k = key_of(v[i][j], t0 + (i * kBeamThreads + tid) * 4 + j);
          if (k >= bound) cand[atomicAdd(&count, 1)] = k;
        }
  }
  __syncthreads();
  const int n = count;
  unsigned long long* out = best + ((long long)row * chunks + c) * beams;
  for (int i = tid; i < n; i += kBeamThreads) {
    const unsigned long long k = cand[i];
    int r = 0;
    for (int j = 0; j < n; ++j) r += cand[j] > k;
    if (r < beams) out[r] = k;
  }
  if (tid == 0) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) t += red[i];
    stats[(long long)row * chunks + c] = ChunkStat{M, t};
  }
}

// A 64-bit score's order as an unsigned word.
__device__ __forceinline__ unsigned long long order_of(double v) {
  const long long u = __double_as_longlong(v);
  return u < 0 ? ~(unsigned long long)u : (unsigned long long)u | 0x8000000000000000ull;
}

// One CTA per group: the rows' log sums, their best tokens over the chunks,
// and the group's best continuations.
__global__ void __launch_bounds__(kBeamJoinThreads) beam_join_kernel(
    const unsigned long long* best, const ChunkStat* stats, const float* scores, const int32_t* finished, int beams,
    int chunks, int pad_token, float* new_scores, int32_t* parents, int32_t* tokens) {
  __shared__ double lse[kMaxBeams];
  __shared__ unsigned long long row_key[kMaxBeams][kMaxBeams];  // a row's best logits, in order
  __shared__ unsigned long long cand_key[kMaxBeams * kMaxBeams];
  __shared__ double cand_score[kMaxBeams * kMaxBeams];
  __shared__ int cand_row[kMaxBeams * kMaxBeams], cand_token[kMaxBeams * kMaxBeams];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, NW = kBeamJoinThreads / 32;
  const int g0 = blockIdx.x * beams;
  grid_dep_wait();
  for (int b = warp; b < beams; b += NW) {
    const int row = g0 + b;
    if (finished && finished[row]) continue;
    const ChunkStat* st = stats + (long long)row * chunks;
    const unsigned long long* list = best + (long long)row * chunks * beams;
    // the row's best: sorted blocks of 32 keys, the lists' heads first; a block
    // is looked at only if it can hold one of the best so far
    unsigned long long kept = 0;  // lane i: the i-th largest so far
    const int total = chunks * beams;
    float M = -INFINITY;
    for (int i = lane; i < chunks; i += 32) M = fmaxf(M, st[i].m);
    for (int i0 = 0; i0 < total; i0 += 32) {
      // element i of this order: head i / chunks of chunk i % chunks
      const int i = i0 + lane, head = i / chunks;
      unsigned long long k = i < total ? list[(long long)(i - head * chunks) * beams + head] : 0;
      const unsigned long long least = __shfl_sync(0xffffffffu, kept, beams - 1);
      if (!__any_sync(0xffffffffu, k > least)) continue;
      k = warp_sort(k, lane);
      // both lists descend: the larger of element i and element 31 - i of the other are the 32 largest
      const unsigned long long other = __shfl_sync(0xffffffffu, k, 31 - lane);
      kept = warp_sort(other > kept ? other : kept, lane);
    }
    if (lane < beams) row_key[b][lane] = kept;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    double s = 0.0;
    for (int i = lane; i < chunks; i += 32)
      if (st[i].m > -INFINITY) s += (double)(st[i].sum * expf(st[i].m - M));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) lse[b] = M == -INFINITY ? INFINITY : (double)M + log(s);
  }
  __syncthreads();
  const int n = beams * beams;
  for (int i = tid; i < n; i += kBeamJoinThreads) {
    const int b = i / beams, k = i - b * beams, row = g0 + b;
    double sc = -INFINITY;
    int token = -1;
    if (finished && finished[row]) {
      if (k == 0) {
        sc = (double)scores[row];
        token = pad_token;
      }
    } else {
      const unsigned long long key = row_key[b][k];
      const float v = value_of((uint32_t)(key >> 32));
      if (v > -INFINITY) {
        sc = (double)scores[row] + ((double)v - lse[b]);
        token = (int)(0xffffffffu - (uint32_t)key);
      }
    }
    if (!(sc == sc)) sc = -INFINITY;
    cand_score[i] = sc;
    cand_row[i] = row;
    cand_token[i] = token;
    cand_key[i] = order_of(sc);
  }
  __syncthreads();
  // rank by (score, then beam and token order); i is in beam order, and in
  // token order where a beam's scores tie
  for (int i = tid; i < n; i += kBeamJoinThreads) {
    int r = 0;
    for (int j = 0; j < n; ++j) r += cand_key[j] > cand_key[i] || (cand_key[j] == cand_key[i] && j < i);
    if (r < beams) {
      const bool live = cand_score[i] > -INFINITY;
      new_scores[g0 + r] = live ? (float)cand_score[i] : -INFINITY;
      parents[g0 + r] = live ? cand_row[i] : -1;
      tokens[g0 + r] = live ? cand_token[i] : -1;
    }
  }
}

int beam_prepare() {
  cudaFuncAttributes fa;
  cudaError_t e = cudaFuncGetAttributes(&fa, beam_chunk_kernel);
  if (!e) e = cudaFuncGetAttributes(&fa, beam_join_kernel);
  return e;
}

static long long beam_chunks(int vocab) { return ((long long)vocab + kChunk - 1) / kChunk; }

}  // namespace g4

using namespace g4;

extern "C" {

size_t g4_beam_select_workspace(int n_rows, int vocab, int beams) {
  if (n_rows < 1 || vocab < 1 || vocab > (1 << 30) || beams < 1 || beams > kMaxBeams) return 0;
  return (size_t)n_rows * beam_chunks(vocab) * (beams * 8 + sizeof(ChunkStat));
}

int g4_beam_select(g4_ctx* c, const float* logits, int64_t stride, int vocab, const float* scores,
                   const int32_t* finished, int n_rows, int beams, int pad_token, float* new_scores, int32_t* parents,
                   int32_t* tokens, void* work, size_t work_bytes, void* stream) {
  if (!c) return G4_E_ARG;
  const long long chunks = vocab > 0 ? beam_chunks(vocab) : 0;
  if (n_rows < 0 || vocab < 1 || vocab > (1 << 30) || beams < 1 || beams > kMaxBeams || n_rows % beams || n_rows * chunks > 0x7fffffffll ||
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
  unsigned long long* best = static_cast<unsigned long long*>(work);
  ChunkStat* stats = reinterpret_cast<ChunkStat*>(best + (size_t)n_rows * chunks * beams);
  beam_chunk_kernel<<<(unsigned)(n_rows * chunks), kBeamThreads, 0, st>>>(logits, stride, vocab, finished, beams,
                                                                          (int)chunks, best, stats);
  cudaError_t e = cudaGetLastError();
  if (!e)
    e = launch_after(beam_join_kernel, dim3(n_rows / beams), dim3(kBeamJoinThreads), 0, st, best, stats, scores,
                     finished, beams, (int)chunks, pad_token, new_scores, parents, tokens);
  return e ? c->cuda_fail(e, "g4_beam_select") : 0;
}

}  // extern "C"
