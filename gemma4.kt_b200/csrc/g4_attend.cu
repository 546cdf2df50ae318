// g4_attend.cu -- attention of one new token per row over a paged KV cache:
//   o_h = sum_t p_ht v_t,  p_h = softmax over the visible t of scale * q_h . k_t,
// t visible when t <= pos and (no window, or t > pos - window, or t < sinks).
//
// Bound by HBM: every visible K and V element is read once for all query heads
// of its KV head (4 * heads flops an element).  The products run on the tensor
// cores in the form that wastes least at few heads: positions are the 16 rows
// of the mma's A operand and up to 8 query heads its 8 columns,
//   S^T = K q^T,   O^T += V^T P^T,
// so K rows feed ldmatrix and V rows ldmatrix.trans as they lie in the page,
// S^T and O^T keep a head in the same column of the same thread (its softmax
// statistics and the rescaling of its sums need no exchange), and P^T becomes
// a B operand by one 8 x 8 transpose of registers (movmatrix).
//
// Precision: activations are 32-bit.  q and p are split into parts of the
// cache's type that sum to them (bf16: three parts of 8 bits; f16: two of 11,
// q scaled by a power of two per head so that both parts stay normal); K and V
// enter the mma exactly, sums are fp32.  An fp32 cache is split the same way
// into three bf16 parts as its tile leaves shared memory, the six products
// above 2^-24 are taken.
//
// Work split: the visible positions of all (row, KV head, block of 8 query
// heads) items lie on one line, cut into equal runs of whole units (16
// positions per warp) for a grid that just fills the GPU; each CTA finds its
// run from the device's positions, so ragged batches and one long sequence
// alike keep every SM busy and a captured launch stays right when the
// positions change.  Runs that end inside an item leave (max, sum, O) partials
// in the caller's work space; a second launch joins them in a fixed order.
//
// Warps are independent inside a run: each streams its own 16-position tiles
// through a private ring in shared memory (cp.async, rows of masked positions
// filled with zeros, so what lies there cannot reach the sums), keeps its
// running maximum, sum and O^T in registers, and meets the CTA's other warps
// once per item.
#include "g4_common.cuh"
#include "g4_kv.h"

#include <cuda_bf16.h>

namespace g4 {

constexpr int kHeadBlock = 8;  // query heads per item: the mma's columns
constexpr int kTile = 16;      // positions per warp and step: the mma's rows
constexpr int kJoinThreads = 512;

struct AttendArgs {
  const float* q;
  float* out;
  long long q_stride, out_stride;
  const int32_t *seqs, *pos;
  int n_rows;
  const uint8_t *kp, *vp;
  const int32_t* table;
  unsigned* flags;
  int n_seqs, max_pages, max_positions, page_shift, n_pages;
  int n_kv, group, blocks;  // query heads per KV head, blocks of 8 of them
  int hs;
  float scale_log2;         // scale * log2(e): scores in powers of two
  int window, sinks;
  float* ws;                // [grid][2][kHeadBlock][hs + 2] partials: max, sum, O
};

// Shape of one instantiation: element type, padded head size, warps per CTA
// and stages of a warp's ring (a stage holds 16 rows of K or of V).
template <int TYPE, int HSP>
struct AttendShape {
  static constexpr int kElem = TYPE == F32 ? 4 : 2;
  static constexpr int kStage = kTile * HSP * kElem;
  static constexpr int kWarps = kStage > 16 * 1024 ? 2 : 4;
  // two CTAs per SM where the ring allows it: 64 KB at 2 KB stages, 96 KB otherwise
  static constexpr int kStages = kStage <= 2048 ? 8 : kStage <= 4096 ? 6 : 3;
  static constexpr int kParts = TYPE == F16 ? 2 : 3;
  static constexpr int kCtas = kStage <= 8192 ? 2 : 1;
  static constexpr int kQBytes = kParts * HSP * kHeadBlock * 2;
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kSmem = kRing + kQBytes;
  static constexpr int kUnit = kWarps * kTile;  // positions per unit
  static_assert(kWarps * kHeadBlock * HSP * 4 <= kRing, "the CTA's join reuses the ring");
};

// The units of a row's visible positions: those of the first tokens, then
// those of the window.
struct RowUnits {
  int seq, pos, sink_units, first_unit, units, low;  // low: first position of the window
};

__device__ __forceinline__ RowUnits row_units(const AttendArgs& a, int row, int unit) {
  RowUnits r;
  r.seq = a.seqs[row];
  r.pos = a.pos[row];
  r.units = r.sink_units = r.first_unit = r.low = 0;
  if (r.seq < 0 || r.seq >= a.n_seqs || r.pos < 0 || r.pos >= a.max_positions) return r;
  if (a.window > 0) r.low = max(0, r.pos - a.window + 1);
  r.first_unit = r.low / unit;
  r.sink_units = min((min(a.sinks, r.low) + unit - 1) / unit, r.first_unit);
  r.units = r.sink_units + r.pos / unit - r.first_unit + 1;
  return r;
}

// The grid's cut of the line of units, and where a CTA's run starts.
struct Run {
  long long w0, w1, total;  // units [w0, w1) of total
  int row;                  // row of unit w0
  long long row_start;      // its first unit
};

__device__ __forceinline__ long long run_start(long long total, int grid, int cta) {
  return total * cta / grid;
}

// All threads of the CTA; red holds 32 + 3 long longs.
template <int THREADS>
__device__ Run find_run(const AttendArgs& a, int unit, int items, int cta, int grid, long long* red) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int NW = THREADS / 32;
  long long sum = 0;
  for (int r = tid; r < a.n_rows; r += THREADS) sum += row_units(a, r, unit).units;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if (lane == 0) red[warp] = sum;
  __syncthreads();
  long long total = 0;
  for (int i = 0; i < NW; ++i) total += red[i];
  total *= items;
  // no more CTAs than units: the first ones get one unit each
  const int used = (int)min((long long)grid, total);
  Run run;
  run.total = total;
  run.w0 = cta < used ? run_start(total, used, cta) : total;
  run.w1 = cta < used ? run_start(total, used, cta + 1) : total;
  run.row = 0;
  run.row_start = 0;
  if (run.w0 >= run.w1) return run;
  long long before = 0;
  for (int r0 = 0; r0 < a.n_rows; r0 += THREADS) {
    const int r = r0 + tid;
    long long mine = r < a.n_rows ? (long long)row_units(a, r, unit).units * items : 0, x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) red[warp] = x;
    __syncthreads();
    long long start = before + x - mine, chunk = 0;
    for (int i = 0; i < NW; ++i) {
      if (i < warp) start += red[i];
      chunk += red[i];
    }
    if (mine > 0 && start <= run.w0 && run.w0 < start + mine) {
      red[32] = r;
      red[33] = start;
    }
    before += chunk;
    if (before > run.w0) break;
  }
  __syncthreads();
  run.row = (int)red[32];
  run.row_start = red[33];
  return run;
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <bool HALF>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (HALF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_approx(float x) {  // relative error 2^-22
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 16 bytes global -> shared; zeros where !ok (nothing is read).
__device__ __forceinline__ void cp16_or_zero(uint32_t dst, const void* src, bool ok) {
  const int n = ok ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

// The next part of (x, y) in the mma's type, packed, and what it leaves of them.
template <bool HALF>
__device__ __forceinline__ uint32_t take_part(float& x, float& y) {
  if (HALF) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    x -= f.x;
    y -= f.y;
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  const uint32_t u = *reinterpret_cast<const uint32_t*>(&h);
  x -= __uint_as_float(u << 16);
  y -= __uint_as_float(u & 0xffff0000u);
  return u;
}

// Where 16-byte chunk c of row r lies in a stage: chunks change places within
// a row so that the eight rows of a fragment load hit distinct banks.  fp32
// fragments are pairs of chunks of rows {0..3}, {4..7}, {0,2,4,6} or
// {1,3,5,7}: those sets get distinct even offsets.
template <int TYPE>
__device__ __forceinline__ int chunk_at(int r, int c) {
  return TYPE == F32 ? c ^ (2 * (((r & 7) + ((r >> 2) & 1)) & 3)) : c ^ (r & 7);
}

template <int TYPE, int HSP>
__global__ void __launch_bounds__(AttendShape<TYPE, HSP>::kWarps * 32, AttendShape<TYPE, HSP>::kCtas)
    kv_attend_kernel(const __grid_constant__ AttendArgs a) {
  using S = AttendShape<TYPE, HSP>;
  constexpr bool HALF = TYPE == F16;
  constexpr int NW = S::kWarps, NS = S::kStages, NP = S::kParts, KS = HSP / 16, CPR = HSP * S::kElem / 16;
  extern __shared__ __align__(128) uint8_t smraw[];
  __shared__ long long red[35];
  __shared__ float q_unscale[kHeadBlock];
  __shared__ float stat[NW][kHeadBlock][2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hs = a.hs;
  uint8_t* ring = smraw + (size_t)warp * NS * S::kStage;
  uint2* qf = reinterpret_cast<uint2*>(smraw + S::kRing);  // [part][k step][lane] B fragments
  const uint32_t ring_u = smem_u32(ring);
  const int items = a.n_kv * a.blocks, ks = (hs + 15) / 16, chunks = hs * S::kElem / 16;
  grid_dep_launch();
  const Run run = find_run<NW * 32>(a, S::kUnit, items, blockIdx.x, gridDim.x, red);
  // rows that see nothing: zeros
  for (int r = blockIdx.x; r < a.n_rows; r += gridDim.x) {
    const int seq = a.seqs[r], pos = a.pos[r];
    if (seq < 0) continue;
    if (seq >= a.n_seqs || pos >= a.max_positions) {
      if (tid == 0) atomicOr(a.flags, KV_BAD_ROW);
    } else if (pos < 0) {
      for (int i = tid; i < a.n_kv * a.group * hs; i += NW * 32) a.out[r * a.out_stride + i] = 0.f;
    }
  }
  long long w = run.w0, row_start = run.row_start;
  int row = run.row;
  bool first = true;
  while (w < run.w1) {
    RowUnits ru = row_units(a, row, S::kUnit);
    while (w >= row_start + (long long)ru.units * items) {
      row_start += (long long)ru.units * items;
      ru = row_units(a, ++row, S::kUnit);
    }
    const int item = (int)((w - row_start) / ru.units);
    const int u0 = (int)((w - row_start) - (long long)item * ru.units);
    const int u1 = (int)min((long long)ru.units, u0 + (run.w1 - w));
    const int kvh = item / a.blocks, h0 = (item - kvh * a.blocks) * kHeadBlock, nh = min(kHeadBlock, a.group - h0);
    const float* q = a.q + row * a.q_stride + (long long)(kvh * a.group + h0) * hs;
    const int32_t* pages = a.table + (long long)ru.seq * a.max_pages;
    const int n = u1 - u0;

    // ---- K and V tiles on their way before anything else
    auto tile_pos = [&](int j) {  // first position of this warp's tile of unit u0 + j
      const int u = u0 + j;
      return (u < ru.sink_units ? u : ru.first_unit + u - ru.sink_units) * S::kUnit + warp * kTile;
    };
    auto seen = [&](int t) { return t <= ru.pos && (t >= ru.low || t < a.sinks); };
    auto seen_tile = [&](int t0) { return t0 <= ru.pos && (t0 + kTile > ru.low || t0 < a.sinks); };
    auto tile_page = [&](int j) {  // -1: no position of the tile is visible, or its page is missing
      const int t = tile_pos(j);
      return j < n && seen_tile(t) ? pages[t >> a.page_shift] : -1;
    };
    auto issue = [&](int j, int page, bool is_v, int stage) {
      if (j < n) {
        const int t0 = tile_pos(j);
        const bool have = (unsigned)page < (unsigned)a.n_pages;
        if (!have && seen_tile(t0) && lane == 0) atomicOr(a.flags, KV_BAD_ROW);
        const uint8_t* src = (is_v ? a.vp : a.kp) +
                             (((((long long)(have ? page : 0) * a.n_kv + kvh) << a.page_shift) +
                               (t0 & ((1 << a.page_shift) - 1))) * hs) * S::kElem;
        const uint32_t dst = ring_u + stage * S::kStage;
#pragma unroll
        for (int i = 0; i < kTile * CPR / 32; ++i) {
          const int e = lane + 32 * i, r = e / CPR, c = e % CPR;
          // chunks behind the head's end are zeros up to the next k step
          if (c < ks * S::kElem)
            cp16_or_zero(dst + (uint32_t)(r * CPR + chunk_at<TYPE>(r, c)) * 16u,
                         src + ((long long)r * chunks + (c < chunks ? c : 0)) * 16, have && seen(t0 + r) && c < chunks);
        }
      }
      cp_commit();
    };
    // half tile h is K (even) or V (odd) of tile h / 2; NS - 1 of them in flight
    int next = 0, next_stage = 0;
    int page_a = tile_page(0), page_b = tile_page(1);  // pages of tiles next / 2 and the one behind it
    auto issue_next = [&]() {
      issue(next >> 1, page_a, next & 1, next_stage);
      if (next & 1) {
        page_a = page_b;
        page_b = tile_page((next >> 1) + 2);
      }
      ++next;
      next_stage = next_stage + 1 == NS ? 0 : next_stage + 1;
    };
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) issue_next();

    // ---- q of the block's heads as B fragments: k = dims, n = heads
    if (HALF) {  // a power of two per head brings its largest element to 2^13..2^14
      for (int h = warp; h < kHeadBlock; h += NW) {
        float m = 0.f;
        if (h < nh)
          for (int d = lane; d < hs; d += 32) m = fmaxf(m, fabsf(q[(long long)h * hs + d]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        int e = 0;
        if (m > 0.f && m < INFINITY) frexpf(m, &e);
        if (lane == 0) q_unscale[h] = ldexpf(1.f, max(-100, min(100, e - 14)));
      }
      __syncthreads();
    }
    for (int i = tid; i < ks * 32; i += NW * 32) {
      const int kk = i >> 5, h = (i & 31) >> 2, d = kk * 16 + 2 * (i & 3);
      float x[4] = {0.f, 0.f, 0.f, 0.f};
      if (h < nh) {
        const float f = HALF ? 1.f / q_unscale[h] : 1.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int dd = d + (j & 1) + (j >> 1) * 8;
          x[j] = dd < hs ? q[(long long)h * hs + dd] * f : 0.f;
        }
      }
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        uint2 b;
        b.x = take_part<HALF>(x[0], x[1]);
        b.y = take_part<HALF>(x[2], x[3]);
        qf[(p * KS + kk) * 32 + (i & 31)] = b;
      }
    }
    __syncthreads();
    float sc[2];  // score factors of this thread's two heads
#pragma unroll
    for (int j = 0; j < 2; ++j) sc[j] = a.scale_log2 * (HALF ? q_unscale[2 * (lane & 3) + j] : 1.f);

    // ---- the warp's tiles
    float o[KS][4];
#pragma unroll
    for (int i = 0; i < KS; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    int stage = 0;
    for (int j = 0; j < n; ++j) {
      const int t0 = tile_pos(j);
      // K
      cp_wait<NS - 2>();
      __syncwarp();
      issue_next();
      uint32_t pf[NP][2];
      {
        float s[NP][4];
#pragma unroll
        for (int p = 0; p < NP; ++p) s[p][0] = s[p][1] = s[p][2] = s[p][3] = 0.f;
        const uint32_t kt = ring_u + stage * S::kStage;
        const uint8_t* kg = ring + stage * S::kStage;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
          if (kk < ks) {
            if (TYPE != F32) {
              uint32_t ka[4];
              ldsm4(ka, kt + (uint32_t)((lane & 15) * CPR + chunk_at<TYPE>(lane & 15, 2 * kk + (lane >> 4))) * 16u);
#pragma unroll
              for (int p = 0; p < NP; ++p) {
                const uint2 b = qf[(p * KS + kk) * 32 + lane];
                mma16816<HALF>(s[p], ka, b.x, b.y);
              }
            } else {
              float x[8];
#pragma unroll
              for (int i = 0; i < 4; ++i) {  // (row, row + 8) x (col, col + 8)
                const int r = (lane >> 2) + (i & 1) * 8, c = kk * 4 + (i >> 1) * 2 + ((lane & 3) >> 1);
                const float2 v = *reinterpret_cast<const float2*>(kg + (r * CPR + chunk_at<TYPE>(r, c)) * 16 + (lane & 1) * 8);
                x[2 * i] = v.x;
                x[2 * i + 1] = v.y;
              }
              uint32_t ka[3][4];
#pragma unroll
              for (int p = 0; p < 3; ++p)
#pragma unroll
                for (int i = 0; i < 4; ++i) ka[p][i] = take_part<false>(x[2 * i], x[2 * i + 1]);
#pragma unroll
              for (int p = 0; p < NP; ++p) {  // products of parts i + p <= 2
                const uint2 b = qf[(p * KS + kk) * 32 + lane];
#pragma unroll
                for (int i = 0; i < 3 - p; ++i) mma16816<false>(s[i], ka[i], b.x, b.y);
              }
            }
          }
        }
        // scores: rows t0 + lane / 4 (+ 8), columns heads 2 (lane % 4) (+ 1)
        const bool s0 = seen(t0 + (lane >> 2)), s1 = seen(t0 + (lane >> 2) + 8);
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = s[NP - 1][i];
#pragma unroll
          for (int p = NP - 2; p >= 0; --p) v += s[p][i];
          x[i] = ((i >> 1) ? s1 : s0) ? v * sc[i & 1] : -INFINITY;
        }
        float mn[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mn[h] = fmaxf(x[h], x[h + 2]);
#pragma unroll
          for (int b = 4; b < 32; b <<= 1) mn[h] = fmaxf(mn[h], __shfl_xor_sync(0xffffffffu, mn[h], b));
          mn[h] = fmaxf(mn[h], m[h]);
        }
        if (__any_sync(0xffffffffu, mn[0] != m[0] || mn[1] != m[1])) {
          float f[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            f[h] = mn[h] == -INFINITY ? 1.f : exp2_approx(m[h] - mn[h]);
            l[h] *= f[h];
            m[h] = mn[h];
          }
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            o[i][0] *= f[0];
            o[i][1] *= f[1];
            o[i][2] *= f[0];
            o[i][3] *= f[1];
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // f16 parts: p up to 2^8, so that the second part of a small p stays normal
          const float mm = m[i & 1] == -INFINITY ? 0.f : m[i & 1];
          x[i] = exp2_approx(x[i] - mm + (HALF ? 8.f : 0.f));
          l[i & 1] += x[i];
        }
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          pf[p][0] = transpose8(take_part<HALF>(x[0], x[1]));
          pf[p][1] = transpose8(take_part<HALF>(x[2], x[3]));
        }
      }
      stage = stage + 1 == NS ? 0 : stage + 1;
      // V
      cp_wait<NS - 2>();
      __syncwarp();
      issue_next();
      {
        const uint32_t vt = ring_u + stage * S::kStage;
        const uint8_t* vg = ring + stage * S::kStage;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          if (i < ks) {
            if (TYPE != F32) {
              uint32_t va[4];
              const int r = (lane & 7) + (lane >> 4) * 8;
              ldsm4_t(va, vt + (uint32_t)(r * CPR + chunk_at<TYPE>(r, 2 * i + ((lane >> 3) & 1))) * 16u);
#pragma unroll
              for (int p = 0; p < NP; ++p) mma16816<HALF>(o[i], va, pf[p][0], pf[p][1]);
            } else {
              // V[pos 2 (lane % 4) + {0, 1} (+ 8)][dim lane / 4 (+ 8)]: registers (dim), (dim + 8), then pos + 8
              float x[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const int r = 2 * (lane & 3) + (e & 1) + (e >> 2) * 8, d = i * 16 + (lane >> 2) + ((e >> 1) & 1) * 8;
                x[e] = *reinterpret_cast<const float*>(vg + (r * CPR + chunk_at<TYPE>(r, d >> 2)) * 16 + (d & 3) * 4);
              }
              uint32_t va[3][4];
#pragma unroll
              for (int p = 0; p < 3; ++p)
#pragma unroll
                for (int e = 0; e < 4; ++e) va[p][e] = take_part<false>(x[2 * e], x[2 * e + 1]);
#pragma unroll
              for (int p = NP - 1; p >= 0; --p)
#pragma unroll
                for (int e = 2 - p; e >= 0; --e) mma16816<false>(o[i], va[e], pf[p][0], pf[p][1]);
            }
          }
        }
      }
      stage = stage + 1 == NS ? 0 : stage + 1;
    }
    cp_wait<0>();

    // ---- the CTA's warps meet: common maximum, sums, O
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int b = 4; b < 32; b <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], b);
      if (lane < 4) {
        stat[warp][2 * lane + h][0] = m[h];
        stat[warp][2 * lane + h][1] = l[h];
      }
    }
    __syncthreads();  // also: every warp has left the ring
    float* part = reinterpret_cast<float*>(smraw);  // [NW][kHeadBlock][HSP]
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int head = 2 * (lane & 3) + h;
      float M = -INFINITY;
#pragma unroll
      for (int i = 0; i < NW; ++i) M = fmaxf(M, stat[i][head][0]);
      const float f = m[h] == -INFINITY ? 0.f : exp2_approx(m[h] - M);
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        float* at = part + (warp * kHeadBlock + head) * HSP + i * 16 + (lane >> 2);
        at[0] = o[i][h] * f;
        at[8] = o[i][2 + h] * f;
      }
    }
    __syncthreads();
    const bool whole = u0 == 0 && u1 == ru.units;
    for (int e = tid; e < nh * hs; e += NW * 32) {
      const int h = e / hs, d = e - h * hs;
      float M = -INFINITY, L = 0.f, acc = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) M = fmaxf(M, stat[i][h][0]);
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        L += stat[i][h][0] == -INFINITY ? 0.f : exp2_approx(stat[i][h][0] - M) * stat[i][h][1];
        acc += part[(i * kHeadBlock + h) * HSP + d];
      }
      if (whole) {
        a.out[row * a.out_stride + (long long)(kvh * a.group + h0 + h) * hs + d] = L > 0.f ? acc / L : 0.f;
      } else {
        float* ws = a.ws + ((long long)(blockIdx.x * 2 + (first ? 0 : 1)) * kHeadBlock + h) * (hs + 2);
        if (d == 0) {
          ws[0] = M;
          ws[1] = L;
        }
        ws[2 + d] = acc;
      }
    }
    __syncthreads();  // the ring, the fragments and the statistics are free again
    w += n;
    first = false;
  }
}

// Joins the partials of items that span CTAs: block (c, h) takes head h of the
// item that starts in CTA c and does not end there.
__global__ void __launch_bounds__(kJoinThreads) kv_attend_join_kernel(const __grid_constant__ AttendArgs a, int unit,
                                                                      int grid) {
  __shared__ long long red[35];
  __shared__ float wsum[kJoinThreads / 32];
  __shared__ float acc_s[kJoinThreads / 32][kKvMaxHeadSize];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hs = a.hs, c = blockIdx.x, h = blockIdx.y;
  constexpr int NW = kJoinThreads / 32;
  const int items = a.n_kv * a.blocks;
  const Run run = find_run<kJoinThreads>(a, unit, items, c, grid, red);
  if (run.w0 >= run.w1) return;
  // the item of the run's last unit
  long long row_start = run.row_start;
  int row = run.row;
  RowUnits ru = row_units(a, row, unit);
  while (run.w1 - 1 >= row_start + (long long)ru.units * items) {
    row_start += (long long)ru.units * items;
    ru = row_units(a, ++row, unit);
  }
  const int item = (int)((run.w1 - 1 - row_start) / ru.units);
  const long long i0 = row_start + (long long)item * ru.units, i1 = i0 + ru.units;
  if (i0 < run.w0 || i1 <= run.w1) return;
  const int kvh = item / a.blocks, h0 = (item - kvh * a.blocks) * kHeadBlock;
  if (h >= min(kHeadBlock, a.group - h0)) return;
  const int used = (int)min((long long)grid, run.total);
  int last = c + 1;
  while (run_start(run.total, used, last + 1) < i1) ++last;
  const int own_slot = i0 == run.w0 ? 0 : 1;
  auto partial = [&](int i) {  // of CTA i
    return a.ws + ((long long)(i * 2 + (i == c ? own_slot : 0)) * kHeadBlock + h) * (hs + 2);
  };
  grid_dep_wait();
  float M = -INFINITY;
  for (int i = c + lane; i <= last; i += 32) M = fmaxf(M, __ldcg(partial(i)));
#pragma unroll
  for (int b = 16; b > 0; b >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, b));
  if (M == -INFINITY) M = 0.f;
  // a warp takes every NW-th partial; lanes pairs of dims
  float2 acc[kKvMaxHeadSize / 64];
  float L = 0.f;
#pragma unroll
  for (int u = 0; u < kKvMaxHeadSize / 64; ++u) acc[u] = make_float2(0.f, 0.f);
  for (int i = c + warp; i <= last; i += NW) {
    const float* p = partial(i);
    const float f = exp2_approx(__ldcg(p) - M);
    L = fmaf(f, __ldcg(p + 1), L);
#pragma unroll
    for (int u = 0; u < kKvMaxHeadSize / 64; ++u) {
      const int d = 2 * (lane + 32 * u);
      if (d < hs) {
        const float2 v = __ldcg(reinterpret_cast<const float2*>(p + 2 + d));
        acc[u].x = fmaf(f, v.x, acc[u].x);
        acc[u].y = fmaf(f, v.y, acc[u].y);
      }
    }
  }
  if (lane == 0) wsum[warp] = L;
#pragma unroll
  for (int u = 0; u < kKvMaxHeadSize / 64; ++u) {
    const int d = 2 * (lane + 32 * u);
    if (d < hs) *reinterpret_cast<float2*>(&acc_s[warp][d]) = acc[u];
  }
  __syncthreads();
  for (int d = tid; d < hs; d += kJoinThreads) {
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      s += acc_s[i][d];
      t += wsum[i];
    }
    a.out[row * a.out_stride + (long long)(kvh * a.group + h0 + h) * hs + d] = t > 0.f ? s / t : 0.f;
  }
}

using AttendFn = void (*)(const AttendArgs);
struct AttendPlan {
  AttendFn fn;
  int threads, smem, unit, ctas;
};

template <int TYPE, int HSP>
static AttendPlan attend_plan_s() {
  using S = AttendShape<TYPE, HSP>;
  return AttendPlan{kv_attend_kernel<TYPE, HSP>, S::kWarps * 32, S::kSmem, S::kUnit, S::kCtas};
}
template <int TYPE>
static AttendPlan attend_plan_t(int hs) {
  return hs <= 64    ? attend_plan_s<TYPE, 64>()
         : hs <= 128 ? attend_plan_s<TYPE, 128>()
         : hs <= 256 ? attend_plan_s<TYPE, 256>()
                     : attend_plan_s<TYPE, 512>();
}
static AttendPlan attend_plan(int type, int hs) {
  return type == F32 ? attend_plan_t<F32>(hs) : type == F16 ? attend_plan_t<F16>(hs) : attend_plan_t<BF16>(hs);
}

int kv_attend_prepare(const g4_kv* kv) {
  cudaError_t e = cudaSuccess;
  for (int l = 0; l < kv->n_layers && !e; ++l) {
    const AttendPlan p = attend_plan(kv->type, kv->hs[l]);
    e = cudaFuncSetAttribute(p.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, p.smem);
  }
  cudaFuncAttributes fa;
  if (!e) e = cudaFuncGetAttributes(&fa, kv_attend_join_kernel);
  return e;
}

}  // namespace g4

using namespace g4;

extern "C" {

size_t g4_kv_attend_workspace(const g4_kv* kv, int layer) {
  if (!kv || layer < 0 || layer >= kv->n_layers) return 0;
  const AttendPlan p = attend_plan(kv->type, kv->hs[layer]);
  return (size_t)kv->ctx->dev.sms * p.ctas * 2 * kHeadBlock * (kv->hs[layer] + 2) * sizeof(float);
}

int g4_kv_attend(g4_kv* kv, int layer, const g4_kv_queries* rows, void* work, size_t work_bytes, void* stream) {
  if (!kv) return G4_E_ARG;
  g4_ctx* c = kv->ctx;
  if (!rows || layer < 0 || layer >= kv->n_layers) {
    c->set_err("g4_kv_attend: layer %d of %d, rows %p", layer, kv->n_layers, (const void*)rows);
    return G4_E_ARG;
  }
  const int hs = kv->hs[layer], nkv = kv->n_kv[layer], n = rows->n_rows;
  const long long width = (long long)rows->n_heads * hs;
  if (n < 0 || n > (1 << 20) || rows->n_heads < 1 || rows->n_heads > 4096 || rows->n_heads % nkv || rows->window < 0 ||
      rows->sinks < 0 || !(rows->scale > -1e30f && rows->scale < 1e30f) ||
      (n > 0 && (!rows->q || !rows->out || !rows->seqs || !rows->pos ||
                 (n > 1 && (rows->q_stride < width || rows->out_stride < width))))) {
    c->set_err("g4_kv_attend: bad arguments (%d rows, %d query heads over %d KV heads of %d, window %d, sinks %d, scale "
               "%g; rows at least heads x head size apart)", n, rows->n_heads, nkv, hs, rows->window, rows->sinks,
               (double)rows->scale);
    return G4_E_ARG;
  }
  if (n == 0) return 0;
  const size_t need = g4_kv_attend_workspace(kv, layer);
  if (!work || work_bytes < need || (reinterpret_cast<uintptr_t>(work) & 15)) {
    c->set_err("g4_kv_attend: work space of %zu bytes, needs %zu (16-byte aligned)", work ? work_bytes : (size_t)0, need);
    return G4_E_ARG;
  }
  DeviceScope scope(c);
  if (scope.rc) return scope.rc;
  AttendArgs a{};
  a.q = rows->q;
  a.out = rows->out;
  a.q_stride = rows->q_stride;
  a.out_stride = rows->out_stride;
  a.seqs = rows->seqs;
  a.pos = rows->pos;
  a.n_rows = n;
  a.kp = kv->k[layer];
  a.vp = kv->v[layer];
  a.table = kv->table;
  a.flags = kv->flags;
  a.n_seqs = kv->n_seqs;
  a.max_pages = kv->max_pages;
  a.max_positions = kv->max_positions;
  a.page_shift = kv->page_shift;
  a.n_pages = kv->n_pages;
  a.n_kv = nkv;
  a.group = rows->n_heads / nkv;
  a.blocks = (a.group + kHeadBlock - 1) / kHeadBlock;
  a.hs = hs;
  a.scale_log2 = rows->scale * 1.4426950408889634f;
  a.window = rows->window;
  a.sinks = rows->window > 0 ? rows->sinks : 0;
  a.ws = static_cast<float*>(work);
  const AttendPlan p = attend_plan(kv->type, hs);
  const int grid = c->dev.sms * p.ctas;
  cudaStream_t st = (cudaStream_t)stream;
  p.fn<<<grid, p.threads, p.smem, st>>>(a);
  cudaError_t e = cudaGetLastError();
  if (!e)
    e = launch_after(kv_attend_join_kernel, dim3(grid, a.group < kHeadBlock ? a.group : kHeadBlock), dim3(kJoinThreads),
                     0, st, a, p.unit, grid);
  return e ? c->cuda_fail(e, "g4_kv_attend") : 0;
}

}  // extern "C"
