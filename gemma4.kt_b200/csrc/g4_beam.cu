// g4_beam.cu -- beam search's selection: for every group of `beams` rows, the
// `beams` best of all continuations score_b + logit_bt - log sum_t exp(logit_bt).
//
// One pass over the logits (bound by HBM: 4 bytes a candidate).  A CTA holds
// kChunk logits of a row in registers and takes from them the chunk's maximum
// and sum of exponentials and its `beams` largest logits: the beams-th largest
// of the threads' own maxima bounds them from below, so only candidates at or
// above it (beams to 32 * beams of kChunk) are ranked, by counting.  A second
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

__global__ void __launch_bounds__(kBeamThreads) beam_chunk_kernel(const float* logits, long long stride, int vocab,
                                                                  const int32_t* finished, int beams, int chunks,
                                                                  unsigned long long* best, ChunkStat* stats) {
  __shared__ unsigned long long top[kBeamThreads];
  __shared__ unsigned long long cand[kMaxBeams * kBeamPer];
  __shared__ unsigned long long bound_s;
  __shared__ float red[kBeamThreads / 32];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / chunks, c = blockIdx.x - row * chunks;
  grid_dep_launch();
  if (finished && finished[row]) return;  // its one continuation needs no logits
  const float* x = logits + row * stride;
  const int t0 = c * kChunk;
  if (tid == 0) count = 0;
  // element i of a thread: token t0 + (i / 4) * 1024 + 4 tid + i % 4
  float v[kBeamPer];
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
#pragma unroll
  for (int i = 0; i < kBeamPer / 4; ++i) {
    const int t = t0 + (i * kBeamThreads + tid) * 4;
    if (vec && t + 4 <= vocab) {
      const float4 f = __ldcs(reinterpret_cast<const float4*>(x + t));
      v[4 * i] = f.x;
      v[4 * i + 1] = f.y;
      v[4 * i + 2] = f.z;
      v[4 * i + 3] = f.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * i + j] = t + j < vocab ? x[t + j] : -INFINITY;
    }
  }
  float m = -INFINITY;
  int at = 0;
#pragma unroll
  for (int i = 0; i < kBeamPer; ++i) {
    if (!(v[i] == v[i])) v[i] = -INFINITY;  // a NaN is never chosen
    if (v[i] > m) {
      m = v[i];
      at = i;
    }
  }
  auto token_of = [&](int i) { return t0 + ((i >> 2) * kBeamThreads + tid) * 4 + (i & 3); };
  auto key_of = [&](float f, int token) {
    return ((unsigned long long)order_of(f) << 32) | (0xffffffffu - (uint32_t)token);
  };
  const unsigned long long mine = key_of(m, token_of(at));
  top[tid] = mine;
  float M = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (lane == 0) red[warp] = M;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kBeamThreads / 32; ++i) M = fmaxf(M, red[i]);
  // the bound: the beams-th largest of the threads' maxima
  int rank = 0;
  for (int i = 0; i < kBeamThreads; ++i) rank += top[i] > mine;
  if (rank == beams - 1) bound_s = mine;
  const float base = M == -INFINITY ? 0.f : M;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kBeamPer; ++i) s += __expf(v[i] - base);
  s = warp_sum(s);
  __syncthreads();
  if (lane == 0) red[warp] = s;
  const unsigned long long bound = bound_s;
  const float bv = value_of((uint32_t)(bound >> 32));
  if (mine >= bound) {  // only these threads can hold candidates
#pragma unroll
    for (int i = 0; i < kBeamPer; ++i)
      if (v[i] >= bv) {
        const unsigned long long k = key_of(v[i], token_of(i));
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
    for (int i = 0; i < kBeamThreads / 32; ++i) t += red[i];
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
    float M = -INFINITY;
    for (int i = lane; i < chunks; i += 32) M = fmaxf(M, st[i].m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    double s = 0.0;
    for (int i = lane; i < chunks; i += 32)
      if (st[i].m > -INFINITY) s += (double)st[i].sum * exp((double)st[i].m - (double)M);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) lse[b] = M == -INFINITY ? INFINITY : (double)M + log(s);
    // the row's best: repeatedly the largest head of the chunks' ordered lists
    const unsigned long long* list = best + (long long)row * chunks * beams;
    unsigned long long last = ~0ull;
    for (int k = 0; k < beams; ++k) {
      unsigned long long x = 0;
      for (int i = lane; i < chunks * beams; i += 32) {
        const unsigned long long y = list[i];
        if (y < last && y > x) x = y;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long y = __shfl_xor_sync(0xffffffffu, x, o);
        x = y > x ? y : x;
      }
      if (lane == 0) row_key[b][k] = x;
      last = x;
    }
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
