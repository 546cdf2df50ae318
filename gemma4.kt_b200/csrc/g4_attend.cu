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
// enter the mma exactly.  The tensor core cuts its sums off: they are taken
// fresh every few steps and added in fp32 (without: 1e-6 to 3e-6 of the result
// off, growing with the context; with: 2e-7 to 6e-7, less than fp32 matrix
// products). Weights are 32-bit powers of two by the hardware's ex2 (2^-22), their
// sums 32-bit, where the contiguous batch takes exponentials in 64 bits: one per
// position and head, which the products would wait for, and an error below what
// the products leave.  An fp32 cache is multiplied in fp32, two products an instruction:
// K and V split into parts as well would need six mma steps for one (64
// sequences to 4000, 8 heads over one of 256: 106 us against 83).
//
// Work split: the visible positions of all (row, KV head, block of 8 query
// heads) items lie on one line, cut into equal runs of whole units (16
// positions per warp) for a grid that just fills the GPU; each CTA finds its
// run from the device's positions, so ragged batches and one long sequence
// alike keep every SM busy and a captured launch stays right when the
// positions change.  Runs that end inside an item leave (max, sum, O) partials
// in the caller's work space; a second launch joins them in a fixed order.
//
// Bound where (time of the GPU alone): 96 ragged sequences to 12001 (64 heads over
// 8 of 128, bf16) run at the measured copy rate (360 us for 2.37 GB), one of 131071
// (f16) at 91% of it (90 us); 64 sequences with a window of 512 (16 heads over 8 of
// 256, bf16) at 73% (51 us): what is left is the start of a run (position, page,
// first bytes: 4 us) and the join (3 us). A call of a few positions takes 9 to 14.
//
// Inside a run one warp brings units in (TMA boxes of 16 positions x 128 bytes
// of a head, swizzled so that fragment loads hit distinct banks; K and V of a
// unit are two stages of one ring) and runs ahead over the ends of items, so
// HBM stays busy while the others finish one. The other warps own 16 or 32
// positions of every unit each, keep their running maximum, sum and O^T in
// registers, and meet once per item. Positions that a row does not see are
// left out of the scores by selection and their V rows are zeroed in shared
// memory, so what lies there cannot reach the sums; boxes without a visible
// position are not loaded.
#include "g4_common.cuh"
#include "g4_kv.h"

#include <cudaTypedefs.h>
#include <cuda_bf16.h>

namespace g4 {

constexpr int kHeadBlock = 8;  // query heads per item: the mma's columns
constexpr int kTile = 16;      // positions per warp and step: the mma's rows
constexpr int kJoinThreads = 256;
// What an item counts beside its units in the work split (0 / 1 / 2: 64 windowed
// sequences 63 / 51 / 52 us, 128 of 10 to 300 positions 38 / 31 / 30).
constexpr int kItemUnits = 1;
constexpr int kMaxGrid = 512;  // CTAs (a B200 takes 296)
static_assert(kKvMaxHeadSize <= 2 * kJoinThreads, "two dims per thread of the join");

struct AttendArgs {
  const float* q;
  float* out;
  long long q_stride, out_stride;
  const int32_t *seqs, *pos;
  int n_rows;
  const int32_t* table;
  unsigned* flags;
  int n_seqs, max_pages, max_positions, page_shift, n_pages;
  int n_kv, group, blocks;  // query heads per KV head, blocks of 8 of them
  int hs;
  float scale_log2;         // scale * log2(e): scores in powers of two
  int window, sinks;
  float* ws;                // [grid][2][kHeadBlock][hs + 2] partials: max, sum, O
  int4* joins;              // [grid] the item that a CTA goes on with: row (-1: none), item, first CTA and its slot, last CTA
};

// Shape of one instantiation: element type, padded head size, groups of warps
// that own positions, 16-position tiles per group, stages of the ring (a stage
// holds a unit's K or V). Two CTAs per SM share 192 KB of ring where a stage is
// 32 KB or less; a wider head takes the SM's memory for one, and for an fp32
// cache several warps split its dims, so that eight warps compute.
template <int TYPE, int HSP, int MT>
struct AttendShape {
  static constexpr int kElem = TYPE == F32 ? 4 : 2;
  static constexpr int kRow = HSP * kElem;  // bytes of a position, padded
  static constexpr int kWarps = kRow > 1024 ? 2 : 4;  // groups
  static constexpr int kTiles = MT;
  static constexpr int kSplit = TYPE != F32 ? 1 : kRow > 1024 ? 4 : kRow > 512 ? 2 : 1;  // warps of a group: each its part of the dims
  static constexpr int kAll = kWarps * kSplit;
  static constexpr int kUnit = kWarps * kTiles * kTile;  // positions per unit
  static constexpr int kStage = kUnit * kRow;
  static constexpr int kStages = kStage <= 16384 ? 6 : 3;
  static constexpr int kCtas = kStage <= 32768 ? 2 : 1;
  static constexpr int kParts = TYPE == F16 ? 2 : 3;
  static constexpr int kBlocks = kRow / 128;              // 128-byte blocks of a row
  static constexpr int kBlockBytes = kUnit * 128;         // one block of every position
  static constexpr int kRing = kStages * kStage;
  // q: the parts' fragments, or (F32) rows of heads 16 bytes apart in the banks
  static constexpr int kQPitch = HSP + 4;
  static constexpr int kQBytes = TYPE == F32 ? kHeadBlock * kQPitch * 4 : kParts * HSP * kHeadBlock * 2;
  static constexpr int kPBytes = TYPE == F32 ? kAll * MT * 512 : 0;  // F32: a tile's weights
  static constexpr int kMeet = kAll * kWarps * 512;       // where the warps meet; shares the fragments' memory
  static constexpr int kSwap = kSplit > 1 ? 2 * kAll * MT * 512 : 0;  // a group's partial scores, two units in turn
  static constexpr int kSmem = kRing + (kQBytes + kPBytes > kMeet ? kQBytes + kPBytes : kMeet) + kSwap;
  static constexpr int kThreads = (kAll + 1) * 32;
};

// The units of a row's visible positions: those of the first tokens, then
// those of the window.
struct RowUnits {
  int seq, pos, sink_units, first_unit, units, low;  // low: first position of the window
};

__device__ __forceinline__ RowUnits row_units(const AttendArgs& a, int seq, int pos, int unit) {
  RowUnits r;
  r.seq = seq;
  r.pos = pos;
  r.units = r.sink_units = r.first_unit = r.low = 0;
  if (r.seq < 0 || r.seq >= a.n_seqs || r.pos < 0 || r.pos >= a.max_positions) return r;
  if (a.window > 0) r.low = max(0, r.pos - a.window + 1);
  r.first_unit = r.low / unit;
  r.sink_units = min((min(a.sinks, r.low) + unit - 1) / unit, r.first_unit);
  r.units = r.sink_units + r.pos / unit - r.first_unit + 1;
  return r;
}

// An item's length on the line: its units, and a fixed part that stands for
// what every item costs beside them (fragments of q, the warps' meeting).
__device__ __forceinline__ int line_units(const RowUnits& r) { return r.units ? r.units + kItemUnits : 0; }

// Quotient of a long dividend that is usually short: a 64-bit division costs
// several hundred cycles, which every CTA would wait for.
__device__ __forceinline__ long long quotient(long long x, long long d) {
  return ((x | d) >> 32) == 0 ? (long long)((uint32_t)x / (uint32_t)d) : x / d;
}

// The line's cut into runs: the first `extra` CTAs have base + 1 of it, the
// others base (no more CTAs than length: the first ones get one each).
struct Cut {
  long long total, base;
  int used, extra;
  __device__ __forceinline__ void make(long long length, int grid) {
    total = length;
    used = (int)min((long long)grid, length);
    base = used ? quotient(length, used) : 0;
    extra = (int)(length - base * used);
  }
  __device__ __forceinline__ long long start(int cta) const { return cta * base + min(cta, extra); }
  __device__ __forceinline__ int cta_of(long long x) const {
    const long long wide = extra * (base + 1);
    return x < wide ? (int)quotient(x, base + 1) : extra + (int)quotient(x - wide, base);
  }
};

// A CTA's run and where it starts.
struct Run {
  long long w0, w1;     // [w0, w1) of the line
  int row, seq, pos;    // row of w0
  long long row_start;  // where it begins
  Cut cut;
};

// All threads of the CTA. Up to a row per thread one scan gives both the
// total and the place of w0; more rows are walked a second time.
template <int THREADS>
__device__ Run find_run(const AttendArgs& a, int unit, int items, int cta, int grid, long long* red) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int NW = THREADS / 32;
  Run run;
  long long mine = 0, x = 0, before = 0, chunk = 0;
  int seq = -1, pos = -1;
  auto scan = [&](int r) {  // mine: units of row r; x: of the rows up to r in this chunk; chunk: of the chunk
    seq = r < a.n_rows ? a.seqs[r] : -1;
    pos = r < a.n_rows ? a.pos[r] : -1;
    mine = (long long)line_units(row_units(a, seq, pos, unit)) * items;
    x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) red[warp] = x;
    __syncthreads();
    chunk = 0;
    for (int i = 0; i < NW; ++i) {
      if (i < warp) x += red[i];
      chunk += red[i];
    }
  };
  long long total = 0;
  for (int r0 = 0; r0 < a.n_rows; r0 += THREADS) {
    scan(r0 + tid);
    total += chunk;
  }
  run.cut.make(total, grid);
  run.w0 = run.w1 = total;
  run.row = run.seq = run.pos = 0;
  run.row_start = 0;
  if (cta >= run.cut.used) return run;
  run.w0 = run.cut.start(cta);
  run.w1 = run.cut.start(cta + 1);
  for (int r0 = 0; r0 < a.n_rows; r0 += THREADS) {
    if (a.n_rows > THREADS) scan(r0 + tid);
    const long long start = before + x - mine;
    if (mine > 0 && start <= run.w0 && run.w0 < start + mine) {
      red[NW] = r0 + tid;
      red[NW + 1] = start;
      red[NW + 2] = ((long long)seq << 32) | pos;
    }
    before += chunk;
    if (before > run.w0) break;
  }
  __syncthreads();
  run.row = (int)red[NW];
  run.row_start = red[NW + 1];
  run.seq = (int)(red[NW + 2] >> 32);
  run.pos = (int)red[NW + 2];
  return run;
}

// The same for up to 4 rows per lane: every warp finds the run by itself.
__device__ __forceinline__ Run find_run_small(const AttendArgs& a, int unit, int items, int cta, int grid) {
  const int lane = threadIdx.x & 31, per = (a.n_rows + 31) / 32;
  int seq[4], pos[4];
  long long len[4], mine = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = lane * per + i;
    const bool have = i < per && r < a.n_rows;
    seq[i] = have ? a.seqs[r] : -1;
    pos[i] = have ? a.pos[r] : -1;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    len[i] = (long long)line_units(row_units(a, seq[i], pos[i], unit)) * items;
    mine += len[i];
  }
  long long x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  Run run;
  run.cut.make(__shfl_sync(0xffffffffu, x, 31), grid);
  run.w0 = run.w1 = run.cut.total;
  run.row = run.seq = run.pos = 0;
  run.row_start = 0;
  if (cta >= run.cut.used) return run;
  run.w0 = run.cut.start(cta);
  run.w1 = run.cut.start(cta + 1);
  long long start = x - mine;
  bool found = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (!found && len[i] > 0 && start <= run.w0 && run.w0 < start + len[i]) {
      found = true;
      run.row = lane * per + i;
      run.seq = seq[i];
      run.pos = pos[i];
    }
    if (!found) start += len[i];
  }
  const int who = __ffs(__ballot_sync(0xffffffffu, found)) - 1;
  run.row = __shfl_sync(0xffffffffu, run.row, who);
  run.seq = __shfl_sync(0xffffffffu, run.seq, who);
  run.pos = __shfl_sync(0xffffffffu, run.pos, who);
  run.row_start = __shfl_sync(0xffffffffu, start, who);
  return run;
}

// A walk over a run: the part of one item after the other.
struct Walk {
  long long w, row_start;
  int row, item, u0, n;  // units [u0, u0 + n) of the row's item
  int next_seq, next_pos;
  RowUnits ru;
  __device__ __forceinline__ void load_row(const AttendArgs& a) {  // of the row behind this one
    next_seq = row + 1 < a.n_rows ? a.seqs[row + 1] : -1;
    next_pos = row + 1 < a.n_rows ? a.pos[row + 1] : -1;
  }
  __device__ __forceinline__ void start(const AttendArgs& a, const Run& r, int unit) {
    w = r.w0;
    row = r.row;
    row_start = r.row_start;
    if (w >= r.w1) return;
    ru = row_units(a, r.seq, r.pos, unit);
    load_row(a);
  }
  __device__ __forceinline__ bool next(const AttendArgs& a, const Run& r, int unit, int items) {
    while (w < r.w1) {
      const int len = line_units(ru);
      if (w >= row_start + (long long)len * items) {
        row_start += (long long)len * items;
        ru = row_units(a, next_seq, next_pos, unit);
        ++row;
        load_row(a);
        continue;
      }
      item = (int)quotient(w - row_start, len);
      const int at = (int)(w - row_start - (long long)item * len), to = (int)min((long long)len, at + (r.w1 - w));
      u0 = max(0, at - kItemUnits);
      n = max(0, to - kItemUnits) - u0;
      w += to - at;
      if (n > 0) return true;
    }
    return false;
  }
  __device__ __forceinline__ long long item_end() const { return row_start + (long long)(item + 1) * line_units(ru); }
  __device__ __forceinline__ int position(int j, int unit) const {  // first of unit u0 + j
    const int u = u0 + j;
    return (u < ru.sink_units ? u : ru.first_unit + u - ru.sink_units) * unit;
  }
  __device__ __forceinline__ bool seen(int t, int sinks) const { return t <= ru.pos && (t >= ru.low || t < sinks); }
  __device__ __forceinline__ bool seen_tile(int t0, int sinks) const {
    return t0 <= ru.pos && (t0 + kTile > ru.low || t0 < sinks);
  }
  // every position of the tile
  __device__ __forceinline__ bool whole_tile(int t0, int sinks) const {
    return t0 + kTile - 1 <= ru.pos && (t0 >= ru.low || t0 + kTile <= sinks);
  }
};

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
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_approx(float x) {  // relative error 2^-22
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A box of 16 positions x 128 bytes of one head of a page.
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int slot, int head, int page,
                                        uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(slot), "r"(head), "r"(page), "r"(smem_u32(bar))
      : "memory");
}
template <int THREADS>
__device__ __forceinline__ void bar_compute() {  // the computing warps
  asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
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

// Two fp32 multiply-adds at once.
__device__ __forceinline__ void fma2(unsigned long long& c, unsigned long long a, unsigned long long b) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(a), "l"(b));
}
__device__ __forceinline__ float2 halves(unsigned long long x) {
  return make_float2(__uint_as_float((uint32_t)x), __uint_as_float((uint32_t)(x >> 32)));
}

// Byte offset of 16-byte chunk c of position r in a stage: 128-byte blocks of
// all positions one after the other, chunks swizzled within a row's block.
template <int BLOCK>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return (uint32_t)((c >> 3) * BLOCK + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

template <int TYPE, int HSP, int MT>
__global__ void __launch_bounds__(AttendShape<TYPE, HSP, MT>::kThreads, AttendShape<TYPE, HSP, MT>::kCtas)
    kv_attend_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ CUtensorMap k_map,
                     const __grid_constant__ CUtensorMap v_map) {
  using S = AttendShape<TYPE, HSP, MT>;
  constexpr bool HALF = TYPE == F16;
  constexpr int NW = S::kWarps, NS = S::kStages, NP = S::kParts, KS = HSP / 16, BLK = S::kBlockBytes;
  constexpr int DS = S::kSplit, NA = S::kAll, KSW = KS / DS;  // a warp's mma steps: [split * KSW, split * KSW + KSW)
  constexpr int KG = 4;  // mma steps whose operands are read together: a 128-byte block of a 16-bit head
  extern __shared__ __align__(1024) uint8_t smraw[];
  __shared__ long long red[NA + 4];
  __shared__ float q_unscale[kHeadBlock], q_max[NA][kHeadBlock];
  __shared__ float stat[NW][kHeadBlock][2];
  __shared__ __align__(8) uint64_t full[NS], empty[NS];
  __shared__ unsigned boxes[NS];  // the 16-position boxes of a stage that were loaded
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hs = a.hs;
  const int group = warp / DS, split = warp % DS;
  // F32: a lane multiplies four positions with four heads for a quarter of the
  // dims (bits 0 and 2), and weighs four dims of 64 for the same four heads
  // (bit 1): twice the products per load of an mma's layout, into which two
  // exchanges bring the scores.
  const int bit0 = lane & 1, bit2 = (lane >> 2) & 1, heads4 = (lane & 2) * 2;
  const int dim4 = (lane >> 3) * 4 + bit2 * 2 + bit0;
  auto four_heads = [&](const float (&f)[2], float (&all)[4]) {  // of this lane's two, in an mma's layout
    const float x = __shfl_xor_sync(0xffffffffu, f[0], 1), y = __shfl_xor_sync(0xffffffffu, f[1], 1);
    all[0] = bit0 ? x : f[0];
    all[1] = bit0 ? y : f[1];
    all[2] = bit0 ? f[0] : x;
    all[3] = bit0 ? f[1] : y;
  };
  const uint32_t ring = smem_u32(smraw);
  uint2* qf = reinterpret_cast<uint2*>(smraw + S::kRing);     // [part][k step][lane] B fragments of q
  float* qs = reinterpret_cast<float*>(smraw + S::kRing);     // (F32) q [head][kQPitch]
  float* weights = reinterpret_cast<float*>(smraw + S::kRing + S::kQBytes) + warp * MT * 128;  // (F32) [position][head]
  float4* meet = reinterpret_cast<float4*>(smraw + S::kRing);  // [split][step][group][lane], between items
  float4* swap = reinterpret_cast<float4*>(smraw + S::kSmem - S::kSwap);  // [2][group][split][tile][lane]
  int swap_at = 0;
  const int items = a.n_kv * a.blocks, ks = (hs + 15) / 16;
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, NA);
    }
    fence_barrier_init();
  }
  grid_dep_launch();
  const Run run = a.n_rows <= 128 ? find_run_small(a, S::kUnit, items, blockIdx.x, gridDim.x)
                                  : find_run<S::kThreads>(a, S::kUnit, items, blockIdx.x, gridDim.x, red);
  __syncthreads();  // the barriers are set up (find_run may return before its last one)
  Walk k;
  k.start(a, run, S::kUnit);
  int stage = 0;
  uint32_t phase = 0;
  auto step = [&]() {
    if (++stage == NS) {
      stage = 0;
      phase ^= 1u;
    }
  };

  if (warp == NA) {
    // ---- the loading warp: lane b brings box b of every unit
    const int nblk = (hs * S::kElem + 127) / 128;
    int issued = 0;
    bool ok = true;
    while (ok && k.next(a, run, S::kUnit, items)) {
      const int32_t* pages = a.table + (long long)k.ru.seq * a.max_pages;
      const int kvh = k.item / a.blocks;
      auto page_of = [&](int j, bool& seen) {
        const int t = k.position(j, S::kUnit) + lane * kTile;
        seen = lane < NW * MT && j < k.n && k.seen_tile(t, a.sinks);
        return seen ? pages[t >> a.page_shift] : -1;
      };
      // (kept beside the page: looked at when its turn comes, the load stays in flight; a
      // mark in the page's number itself cost 387 against 373 us for 96 rows to 12001)
      bool seen, seen_after;
      int page = page_of(0, seen);
      for (int j = 0; j < k.n && ok; ++j) {
        const int after = page_of(j + 1, seen_after);
        const bool have = page >= 0 && page < a.n_pages;
        if (seen && !have) atomicOr(a.flags, KV_BAD_ROW);
        const unsigned mask = __ballot_sync(0xffffffffu, have);
        const int slot = (k.position(j, S::kUnit) + lane * kTile) & ((1 << a.page_shift) - 1);
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          if (issued >= NS && !mbar_wait_bounded(empty + stage, phase ^ 1u)) {
            ok = false;
            break;
          }
          if (lane == 0) {
            boxes[stage] = mask;
            mbar_arrive_expect_tx(full + stage, (uint32_t)(__popc(mask) * nblk) * 2048u);
          }
          __syncwarp();
          if (have) {
            const uint32_t dst = ring + stage * S::kStage + lane * 2048;
            for (int b = 0; b < nblk; ++b)
              tma_box(dst + b * BLK, half ? &v_map : &k_map, b * (128 / S::kElem), slot, kvh, page, full + stage);
          }
          ++issued;
          step();
        }
        page = after;
        seen = seen_after;
      }
    }
    if (!ok) {  // the copies still in flight land before the CTA may leave
      if (lane == 0) atomicOr(a.flags, KV_TIMEOUT);
      for (int i = 0; i < NS && i < issued; ++i) {
        if (--stage < 0) {
          stage = NS - 1;
          phase ^= 1u;
        }
        mbar_wait_bounded(full + stage, phase);
      }
    }
    return;
  }

  // ---- the computing warps
  bool dead = false;  // a wait expired: no more waits, the results are void
  auto arrived = [&]() {
    if (!dead && !mbar_wait_bounded(full + stage, phase)) {
      dead = true;
      if (lane == 0) atomicOr(a.flags, KV_TIMEOUT);
    }
  };
  auto release = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + stage);
    step();
  };
  // q of an item's heads, as the B fragments hold it (k = dims, n = heads): the
  // values of this thread's fragment registers, read before the item begins
  constexpr int QL = (KS + NA - 1) / NA;
  float qv[QL][4];
  auto load_q = [&]() {
    const int kvh = k.item / a.blocks, h0 = (k.item - kvh * a.blocks) * kHeadBlock, nh = min(kHeadBlock, a.group - h0);
    const float* q = a.q + k.row * a.q_stride + (long long)(kvh * a.group + h0) * hs;
    const bool vec = ((reinterpret_cast<uintptr_t>(a.q) & 7) | (a.q_stride & 1)) == 0;
#pragma unroll
    for (int i = 0; i < QL; ++i) {
      const int kk = warp + NA * i, h = lane >> 2, d = kk * 16 + 2 * (lane & 3);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float* at = q + (long long)h * hs + d + 8 * j;
        float2 v = make_float2(0.f, 0.f);
        if (h < nh && d + 8 * j < hs) {
          if (vec) v = *reinterpret_cast<const float2*>(at);
          else v = make_float2(at[0], at[1]);
        }
        qv[i][2 * j] = v.x;
        qv[i][2 * j + 1] = v.y;
      }
    }
  };
  bool first = true, more = k.next(a, run, S::kUnit, items);
  if (tid == 0 && (!more || k.u0 == 0)) a.joins[blockIdx.x].x = -1;
  constexpr bool kAhead = QL <= 8;  // room in registers to read q during the meeting before
  if (kAhead && more) load_q();
  while (more) {
    const int row = k.row, item = k.item, n = k.n;
    const int kvh = item / a.blocks, h0 = (item - kvh * a.blocks) * kHeadBlock, nh = min(kHeadBlock, a.group - h0);
    if (!kAhead) load_q();
    if (HALF) {  // a power of two per head brings its largest element to 2^13..2^14
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < QL; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) m = fmaxf(m, fabsf(qv[i][j]));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      if ((lane & 3) == 0) q_max[warp][lane >> 2] = m;
      bar_compute<NA * 32>();
      m = q_max[0][lane >> 2];
#pragma unroll
      for (int i = 1; i < NA; ++i) m = fmaxf(m, q_max[i][lane >> 2]);
      int e = 0;
      if (m > 0.f && m < INFINITY) frexpf(m, &e);
      e = max(-126, e - 14);  // (a float's exponent is 128 at most: the factor 2^-e is a normal number at both ends)
      if (warp == 0 && (lane & 3) == 0) q_unscale[lane >> 2] = ldexpf(1.f, e);
      const float f = ldexpf(1.f, -e);
#pragma unroll
      for (int i = 0; i < QL; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) qv[i][j] *= f;
    }
#pragma unroll
    for (int i = 0; i < QL; ++i) {
      const int kk = warp + NA * i;
      if constexpr (TYPE == F32) {
        if (kk < KS) {
          float* at = qs + (lane >> 2) * S::kQPitch + kk * 16 + 2 * (lane & 3);
          *reinterpret_cast<float2*>(at) = make_float2(qv[i][0], qv[i][1]);
          *reinterpret_cast<float2*>(at + 8) = make_float2(qv[i][2], qv[i][3]);
        }
      } else if (kk < KS)
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          uint2 b;
          b.x = take_part<HALF>(qv[i][0], qv[i][1]);
          b.y = take_part<HALF>(qv[i][2], qv[i][3]);
          qf[(p * KS + kk) * 32 + lane] = b;
        }
    }
    bar_compute<NA * 32>();
    float sc[2];  // score factors of this thread's two heads
#pragma unroll
    for (int j = 0; j < 2; ++j) sc[j] = a.scale_log2 * (HALF ? q_unscale[2 * (lane & 3) + j] : 1.f);

    // ---- the warp's tiles of every unit
    float o[KSW][4];
#pragma unroll
    for (int i = 0; i < KSW; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    for (int j = 0; j < n; ++j) {
      const int t0 = k.position(j, S::kUnit) + group * MT * kTile;  // the group's first position
      arrived();
      const unsigned mine = (boxes[stage] >> (group * MT)) & ((1u << MT) - 1u);
      if (mine == 0) {  // nothing visible here
        release();
        arrived();
        release();
        continue;
      }
      uint32_t pf[MT][NP][2];
      bool partial = false;
      {
        float score[MT][4];
#pragma unroll
        for (int t = 0; t < MT; ++t) score[t][0] = score[t][1] = score[t][2] = score[t][3] = 0.f;
        if constexpr (TYPE == F32) {
          // each product sum in two halves, even and odd dims
          const uint8_t* kg = smraw + stage * S::kStage;
          unsigned long long acc[MT][4][4];
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[t][j >> 2][j & 3] = 0ull;
          // (chunks behind the head's end are zeros up to the block's)
#pragma unroll 4
          for (int c0 = split * KSW * 4; c0 < min(ks, (split + 1) * KSW) * 4; c0 += 4) {
            const int c = c0 + bit2 * 2 + bit0;
            ulonglong2 qh[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) qh[h] = *reinterpret_cast<const ulonglong2*>(qs + (heads4 + h) * S::kQPitch + 4 * c);
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int r = (group * MT + t) * kTile + (lane >> 3) * 2 + (j & 1) + (j >> 1) * 8;
                const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(kg + chunk_at<BLK>(r, c));
#pragma unroll
                for (int h = 0; h < 4; ++h) fma2(acc[t][j][h], x.x, qh[h].x);
#pragma unroll
                for (int h = 0; h < 4; ++h) fma2(acc[t][j][h], x.y, qh[h].y);
              }
          }
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            float u[4][2];  // positions j, the lane's own two heads
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float v[4];
#pragma unroll
              for (int h = 0; h < 4; ++h) {
                const float2 x = halves(acc[t][j][h]);
                v[h] = x.x + x.y;
              }
#pragma unroll
              for (int e = 0; e < 2; ++e)
                u[j][e] = (bit0 ? v[2 + e] : v[e]) + __shfl_xor_sync(0xffffffffu, bit0 ? v[e] : v[2 + e], 1);
            }
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                score[t][2 * r + e] = (bit2 ? u[2 * r + 1][e] : u[2 * r][e]) +
                                     __shfl_xor_sync(0xffffffffu, bit2 ? u[2 * r][e] : u[2 * r + 1][e], 4);
          }
        } else {
          // The tensor core cuts its sums off instead of rounding them, so the first
          // parts' products, which carry the score, go into fresh sums every few steps
          // and are added in fp32; the others' (2^-8 and less) stay in one chain each.
          float s[MT][NP][4];
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int p = 0; p < NP; ++p) s[t][p][0] = s[t][p][1] = s[t][p][2] = s[t][p][3] = 0.f;
          const uint32_t kt = ring + stage * S::kStage;
          // steps behind the head's end multiply what the map filled with zeros
#pragma unroll 2
          for (int k0 = split * KSW; k0 < min(ks, (split + 1) * KSW); k0 += KG) {
            uint2 b[KG][NP];
            uint32_t ka[KG][MT][4];
#pragma unroll
            for (int g = 0; g < KG; ++g) {
#pragma unroll
              for (int p = 0; p < NP; ++p) b[g][p] = qf[(p * KS + k0 + g) * 32 + lane];
#pragma unroll
              for (int t = 0; t < MT; ++t)
                ldsm4(ka[g][t], kt + chunk_at<BLK>((group * MT + t) * kTile + (lane & 15), 2 * (k0 + g) + (lane >> 4)));
            }
            float fresh[2][MT][4];
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
              for (int i = 0; i < 4; ++i) fresh[0][t][i] = fresh[1][t][i] = 0.f;
#pragma unroll
            for (int g = 0; g < KG; ++g) {
#pragma unroll
              for (int t = 0; t < MT; ++t) mma16816<HALF>(fresh[g & 1][t], ka[g][t], b[g][0].x, b[g][0].y);
#pragma unroll
              for (int p = 1; p < NP; ++p)
#pragma unroll
                for (int t = 0; t < MT; ++t) mma16816<HALF>(s[t][p], ka[g][t], b[g][p].x, b[g][p].y);
            }
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
              for (int i = 0; i < 4; ++i) score[t][i] += fresh[0][t][i] + fresh[1][t][i];
          }
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float v = s[t][NP - 1][i];
#pragma unroll
              for (int p = NP - 2; p >= 0; --p) v += s[t][p][i];
              score[t][i] += v;
            }
        }
        release();
        // the sum over the group's warps
        if (DS > 1) {
          float4* at = swap + ((swap_at * NW + group) * DS) * MT * 32 + lane;
          swap_at ^= 1;
#pragma unroll
          for (int t = 0; t < MT; ++t)
            at[(split * MT + t) * 32] = make_float4(score[t][0], score[t][1], score[t][2], score[t][3]);
          asm volatile("bar.sync %0, %1;" ::"r"(2 + group), "n"(DS * 32) : "memory");
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            score[t][0] = score[t][1] = score[t][2] = score[t][3] = 0.f;
#pragma unroll
            for (int d = 0; d < DS; ++d) {  // the same order in every warp
              const float4 x = at[(d * MT + t) * 32];
              score[t][0] += x.x;
              score[t][1] += x.y;
              score[t][2] += x.z;
              score[t][3] += x.w;
            }
          }
        }
        // scores: rows t0 + lane / 4 (+ 8), columns heads 2 (lane % 4) (+ 1)
        float x[MT][4], mn[2] = {m[0], m[1]};
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const int tt = t0 + t * kTile;
          const bool have = (mine >> t) & 1u, whole = have && k.whole_tile(tt, a.sinks);
          partial |= !whole;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool vis = whole || (have && k.seen(tt + (lane >> 2) + (i >> 1) * 8, a.sinks));
            x[t][i] = vis ? score[t][i] * sc[i & 1] : -INFINITY;
          }
          mn[0] = fmaxf(mn[0], fmaxf(x[t][0], x[t][2]));
          mn[1] = fmaxf(mn[1], fmaxf(x[t][1], x[t][3]));
        }
#pragma unroll
        for (int b = 4; b < 32; b <<= 1) {
          mn[0] = fmaxf(mn[0], __shfl_xor_sync(0xffffffffu, mn[0], b));
          mn[1] = fmaxf(mn[1], __shfl_xor_sync(0xffffffffu, mn[1], b));
        }
        if (__any_sync(0xffffffffu, mn[0] != m[0] || mn[1] != m[1])) {
          float f[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            f[h] = mn[h] == -INFINITY ? 1.f : exp2_approx(m[h] - mn[h]);
            l[h] *= f[h];
            m[h] = mn[h];
          }
          float fs[4];
          if constexpr (TYPE == F32) four_heads(f, fs);
#pragma unroll
          for (int i = 0; i < KSW; ++i) {
            if constexpr (TYPE == F32) {  // a dim's four heads
              o[i][0] *= fs[0];
              o[i][1] *= fs[1];
              o[i][2] *= fs[2];
              o[i][3] *= fs[3];
            } else {  // two dims' two heads
              o[i][0] *= f[0];
              o[i][1] *= f[1];
              o[i][2] *= f[0];
              o[i][3] *= f[1];
            }
          }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // f16 parts: p up to 2^8, so that the second part of a small p stays normal
            const float mm = m[i & 1] == -INFINITY ? 0.f : m[i & 1];
            x[t][i] = exp2_approx(x[t][i] - mm + (HALF ? 8.f : 0.f));
            l[i & 1] += x[t][i];
          }
          if constexpr (TYPE == F32) {
            float2* at = reinterpret_cast<float2*>(weights + (t * kTile + (lane >> 2)) * 8) + (lane & 3);
            at[0] = make_float2(x[t][0], x[t][1]);
            at[8 * 4] = make_float2(x[t][2], x[t][3]);
          } else {
#pragma unroll
            for (int p = 0; p < NP; ++p) {
              pf[t][p][0] = transpose8(take_part<HALF>(x[t][0], x[t][1]));
              pf[t][p][1] = transpose8(take_part<HALF>(x[t][2], x[t][3]));
            }
          }
        }
      }
      arrived();
      if (TYPE == F32) __syncwarp();  // the weights are there
      {
        const uint32_t vt = ring + stage * S::kStage;
        const uint8_t* vg = smraw + stage * S::kStage;
        if (partial) {  // V rows that are not seen become zeros (the warp's dims of them)
          for (int e = lane; e < MT * kTile * 8; e += 32) {
            const int r = e >> 3, t = t0 + r;
            if (!((mine >> (r / kTile)) & 1u) || !k.seen(t, a.sinks))
              for (int b = split * (KSW * S::kElem / 8); b < min((ks * S::kElem + 7) / 8, (split + 1) * (KSW * S::kElem / 8)); ++b)
                *reinterpret_cast<uint4*>(smraw + stage * S::kStage + b * BLK + (group * MT * kTile + r) * 128 + (e & 7) * 16) =
                    make_uint4(0, 0, 0, 0);
          }
          // ordered before the stage's next load, which another proxy writes
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        // (a tile's sums are fresh, too, and added to O in fp32)
        if (TYPE != F32) {
#pragma unroll
          for (int i = 0; i < KSW; i += KG) {
            if (split * KSW + i < ks) {
              float fresh[KG][4];
#pragma unroll
              for (int g = 0; g < KG; ++g) fresh[g][0] = fresh[g][1] = fresh[g][2] = fresh[g][3] = 0.f;
#pragma unroll
              for (int t = 0; t < MT; ++t) {
                uint32_t va[KG][4];
                const int r = (group * MT + t) * kTile + (lane & 7) + (lane >> 4) * 8;
#pragma unroll
                for (int g = 0; g < KG; ++g)
                  ldsm4_t(va[g], vt + chunk_at<BLK>(r, 2 * (split * KSW + i + g) + ((lane >> 3) & 1)));
#pragma unroll
                for (int p = NP - 1; p >= 0; --p)
#pragma unroll
                  for (int g = 0; g < KG; ++g) mma16816<HALF>(fresh[g], va[g], pf[t][p][0], pf[t][p][1]);
              }
#pragma unroll
              for (int g = 0; g < KG; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i + g][e] += fresh[g][e];
            }
          }
        } else {
          // o[4 g + d] are the lane's four heads of its dim d of the g-th 64
          unsigned long long acc[KSW][2];
#pragma unroll
          for (int i = 0; i < KSW; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              acc[i][e] = (unsigned long long)__float_as_uint(o[i][2 * e]) |
                          (unsigned long long)__float_as_uint(o[i][2 * e + 1]) << 32;
#pragma unroll 8
          for (int p = 0; p < MT * kTile; ++p) {
            const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(weights + p * 8 + heads4);
            const int r = group * MT * kTile + p;
#pragma unroll
            for (int g = 0; g < KSW / 4; ++g) {
              if (split * KSW * 16 + g * 64 < hs) {
                const uint4 x = *reinterpret_cast<const uint4*>(vg + chunk_at<BLK>(r, split * KSW * 4 + g * 16 + dim4));
                const uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                  const unsigned long long vv = (unsigned long long)v[d] | (unsigned long long)v[d] << 32;
                  fma2(acc[4 * g + d][0], vv, w.x);
                  fma2(acc[4 * g + d][1], vv, w.y);
                }
              }
            }
          }
#pragma unroll
          for (int i = 0; i < KSW; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float2 y = halves(acc[i][e]);
              o[i][2 * e] = y.x;
              o[i][2 * e + 1] = y.y;
            }
        }
      }
      release();
    }

    const bool whole = k.u0 == 0 && n == k.ru.units;
    if (k.u0 > 0 && tid == 0) {  // begun by another CTA: where its parts are, for the join
      const long long end = k.item_end(), begin = end - line_units(k.ru);
      const int from = run.cut.cta_of(begin + kItemUnits);
      const int slot = run.cut.start(from) < begin;  // the first of its CTA's parts, or its last
      a.joins[blockIdx.x] = make_int4(row, item, from * 2 + slot, run.cut.cta_of(end - 1));
    }
    // ---- the warps meet: common maximum, sums, O
    more = k.next(a, run, S::kUnit, items);
    if (kAhead && more) load_q();  // on its way meanwhile
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int b = 4; b < 32; b <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], b);
      if (split == 0 && lane < 4) {  // (a group's warps have the same)
        stat[group][2 * lane + h][0] = m[h];
        stat[group][2 * lane + h][1] = l[h];
      }
    }
    bar_compute<NA * 32>();  // also: every warp has read its last q fragment
    float f[2], inv[2];
    float* ws = a.ws + (long long)(blockIdx.x * 2 + (first ? 0 : 1)) * kHeadBlock * (hs + 2);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int head = 2 * (lane & 3) + h;
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) M = fmaxf(M, stat[i][head][0]);
#pragma unroll
      for (int i = 0; i < NW; ++i) L += stat[i][head][0] == -INFINITY ? 0.f : exp2_approx(stat[i][head][0] - M) * stat[i][head][1];
      f[h] = m[h] == -INFINITY ? 0.f : exp2_approx(m[h] - M);
      inv[h] = !whole ? 1.f : L > 0.f ? 1.f / L : 0.f;
      if (!whole && warp == 0 && lane < 4 && head < nh) {
        ws[(long long)head * (hs + 2)] = M;
        ws[(long long)head * (hs + 2) + 1] = L;
      }
    }
    // The same lane of every group's warp for a part of the dims holds the same
    // dims and heads: they lay NW steps of 16 dims side by side, each adds up and
    // stores one of them.
    float fs[4], invs[4];
    if constexpr (TYPE == F32) {
      four_heads(f, fs);
      four_heads(inv, invs);
    }
    float4* mine_at = meet + split * (NW * NW * 32);
    float* out = whole ? a.out + row * a.out_stride + (long long)(kvh * a.group + h0) * hs : ws + 2;
    const int out_pitch = whole ? hs : hs + 2;
#pragma unroll
    for (int i0 = 0; i0 < KSW; i0 += NW) {
      if (i0 < ks) {  // (the same for all warps)
        if (i0) bar_compute<NA * 32>();  // the steps before have been added up
#pragma unroll
        for (int i = 0; i < NW; ++i)
          mine_at[(i * NW + group) * 32 + lane] =
              TYPE == F32 ? make_float4(o[i0 + i][0] * fs[0], o[i0 + i][1] * fs[1], o[i0 + i][2] * fs[2], o[i0 + i][3] * fs[3])
                          : make_float4(o[i0 + i][0] * f[0], o[i0 + i][1] * f[1], o[i0 + i][2] * f[0], o[i0 + i][3] * f[1]);
        bar_compute<NA * 32>();
        float4 acc = mine_at[group * NW * 32 + lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) {
          const float4 x = mine_at[(group * NW + w) * 32 + lane];
          acc.x += x.x;
          acc.y += x.y;
          acc.z += x.z;
          acc.w += x.w;
        }
        if constexpr (TYPE == F32) {
          const int i = i0 + group, d = split * KSW * 16 + (i >> 2) * 64 + dim4 * 4 + (i & 3);
          float* at = out + heads4 * out_pitch + d;
          if (d < hs) {
            if (heads4 < nh) at[0] = acc.x * invs[0];
            if (heads4 + 1 < nh) at[out_pitch] = acc.y * invs[1];
            if (heads4 + 2 < nh) at[2 * out_pitch] = acc.z * invs[2];
            if (heads4 + 3 < nh) at[3 * out_pitch] = acc.w * invs[3];
          }
          continue;
        }
        const int d = (split * KSW + i0 + group) * 16 + (lane >> 2), head = 2 * (lane & 3);
        float* at = out + head * out_pitch + d;
        if (head < nh && d < hs) at[0] = acc.x * inv[0];
        if (head + 1 < nh && d < hs) at[out_pitch] = acc.y * inv[1];
        if (head < nh && d + 8 < hs) at[8] = acc.z * inv[0];
        if (head + 1 < nh && d + 8 < hs) at[out_pitch + 8] = acc.w * inv[1];
      }
    }
    bar_compute<NA * 32>();  // the meeting place and the statistics are free again
    first = false;
  }
  // rows that see nothing: zeros
  for (int r = blockIdx.x; r < a.n_rows; r += gridDim.x) {
    const int seq = a.seqs[r], pos = a.pos[r];
    if (seq < 0) continue;
    if (seq >= a.n_seqs || pos >= a.max_positions) {
      if (tid == 0) atomicOr(a.flags, KV_BAD_ROW);
    } else if (pos < 0) {
      for (int i = tid; i < a.n_kv * a.group * hs; i += NA * 32) a.out[r * a.out_stride + i] = 0.f;
    }
  }
}

// Joins the partials of items that span CTAs. A block belongs to the item that
// the CTA of its number goes on with. Few parts: one block, its warps shared out
// over the heads.
// Many: the item's blocks share its heads and dims, one range of dims of one
// head each, the longer the item the narrower.
__global__ void __launch_bounds__(kJoinThreads) kv_attend_join_kernel(const __grid_constant__ AttendArgs a) {
  __shared__ float red[kJoinThreads / 32];
  __shared__ float weight[kMaxGrid], sum[kMaxGrid];
  __shared__ __align__(8) float acc_s[2 * kJoinThreads];  // [group][dims]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hs = a.hs;
  constexpr int NW = kJoinThreads / 32;
  static_assert(NW == kHeadBlock, "a warp per head");
  grid_dep_wait();
  const int4 j = __ldcg(a.joins + blockIdx.x);
  if (j.x < 0) return;
  const int kvh = j.y / a.blocks, h0 = (j.y - kvh * a.blocks) * kHeadBlock, c = j.z >> 1, slot = j.z & 1;
  const int nh = min(kHeadBlock, a.group - h0), n = j.w - c + 1;  // partials, in CTAs c..c + n - 1
  const int task = (int)blockIdx.x - c - 1;
  float* out = a.out + j.x * a.out_stride + (long long)(kvh * a.group + h0) * hs;
  if (n <= kHeadBlock) {
    const int heads = nh <= 1 ? 1 : nh <= 2 ? 2 : nh <= 4 ? 4 : 8, head = warp & (heads - 1);
    if (task > 0 || head >= nh) return;
    auto part = [&](int i) {
      return a.ws + ((long long)((c + i) * 2 + (i == 0 ? slot : 0)) * kHeadBlock + head) * (hs + 2);
    };
    const float2 ml = lane < n ? __ldcg(reinterpret_cast<const float2*>(part(lane))) : make_float2(-INFINITY, 0.f);
    float M = ml.x;
#pragma unroll
    for (int b = 4; b > 0; b >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, b));
    M = __shfl_sync(0xffffffffu, M, 0);
    if (M == -INFINITY) M = 0.f;
    const float w = exp2_approx(ml.x - M), L = warp_sum(w * ml.y), inv = L > 0.f ? 1.f / L : 0.f;
    for (int d0 = warp / heads * 64; d0 < hs; d0 += NW / heads * 64) {  // (the same for every lane)
      const int d = d0 + 2 * lane;
      float2 v[kHeadBlock], acc = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kHeadBlock; ++i)
        v[i] = i < n && d < hs ? __ldcg(reinterpret_cast<const float2*>(part(i) + 2 + d)) : make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kHeadBlock; ++i) {
        const float wi = __shfl_sync(0xffffffffu, w, i);  // 0 behind the last
        acc.x = fmaf(wi, v[i].x, acc.x);
        acc.y = fmaf(wi, v[i].y, acc.y);
      }
      if (d < hs) {
        out[head * hs + d] = acc.x * inv;
        out[head * hs + d + 1] = acc.y * inv;
      }
    }
    return;
  }
  // n - 1 blocks, at least as many as heads: ranges per head (of 16 dims at least)
  const int ranges = min((n - 1) / nh, max(1, hs / 16)), h = task / ranges, share = (hs / 2 + ranges - 1) / ranges;
  if (h >= nh) return;
  const int d0 = 2 * share * (task - h * ranges), per = min(share, (hs - d0) / 2);  // pairs of dims
  if (per <= 0) return;
  auto partial = [&](int i) {  // of CTA i
    return a.ws + ((long long)(i * 2 + (i == c ? slot : 0)) * kHeadBlock + h) * (hs + 2);
  };
  // every partial's weight: 2^(its maximum - the common one)
  float M = -INFINITY;
  for (int i = tid; i < n; i += kJoinThreads) {
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(partial(c + i)));
    weight[i] = ml.x;
    sum[i] = ml.y;
    M = fmaxf(M, ml.x);
  }
#pragma unroll
  for (int b = 16; b > 0; b >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, b));
  if (lane == 0) red[warp] = M;
  __syncthreads();
  M = red[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) M = fmaxf(M, red[i]);
  if (M == -INFINITY) M = 0.f;
  for (int i = tid; i < n; i += kJoinThreads) {  // (the thread's own entries)
    weight[i] = exp2_approx(weight[i] - M);
    sum[i] *= weight[i];
  }
  __syncthreads();
  // threads own two dims each; groups of them take every groups-th partial
  const int groups = kJoinThreads / per, g = tid / per, d = 2 * (tid - g * per);
  if (g < groups) {
    float2 acc = make_float2(0.f, 0.f);
#pragma unroll 8
    for (int i = g; i < n; i += groups) {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(partial(c + i) + 2 + d0 + d));
      acc.x = fmaf(weight[i], v.x, acc.x);
      acc.y = fmaf(weight[i], v.y, acc.y);
    }
    *reinterpret_cast<float2*>(acc_s + g * 2 * per + d) = acc;
  }
  float L = 0.f;
  for (int i = lane; i < n; i += 32) L += sum[i];
  L = warp_sum(L);
  __syncthreads();
  for (int e = tid; e < 2 * per; e += kJoinThreads) {
    float s = 0.f;
    for (int i = 0; i < min(groups, n); ++i) s += acc_s[i * 2 * per + e];
    out[h * hs + d0 + e] = L > 0.f ? s / L : 0.f;
  }
}

using AttendFn = void (*)(const AttendArgs, const CUtensorMap, const CUtensorMap);
struct AttendPlan {
  AttendFn fn;
  int threads, smem, ctas;
};

template <int TYPE, int HSP, int MT>
static AttendPlan attend_plan_s() {
  using S = AttendShape<TYPE, HSP, MT>;
  return AttendPlan{kv_attend_kernel<TYPE, HSP, MT>, S::kThreads, S::kSmem, S::kCtas};
}
// Two tiles per warp share the fragments of q and the softmax's exchange; one
// leaves finer stages in the ring. For short rows the work decides: under the
// power cap of a long run 96 sequences to 12001 (bf16, heads of 128) take 352 us
// with two and 404 with one, although a short burst takes 354 and 360.
template <int TYPE>
static AttendPlan attend_plan_t(int hs) {
  return hs <= 64    ? attend_plan_s<TYPE, 64, 2>()
         : hs <= 128 ? attend_plan_s<TYPE, 128, TYPE == F32 ? 1 : 2>()
         : hs <= 256 ? attend_plan_s<TYPE, 256, 1>()
                     : attend_plan_s<TYPE, 512, 1>();
}
static AttendPlan attend_plan(int type, int hs) {
  return type == F32 ? attend_plan_t<F32>(hs) : type == F16 ? attend_plan_t<F16>(hs) : attend_plan_t<BF16>(hs);
}

// 16 positions x 128 bytes of one head of a page, zeros beyond the head's end.
static bool make_map(PFN_cuTensorMapEncodeTiled_v12000 encode, CUtensorMap* map, const g4_kv* kv, int layer, void* base) {
  const cuuint64_t hs = kv->hs[layer], ps = kv->page_size, nkv = kv->n_kv[layer], e = kv->elem;
  const cuuint64_t dims[4] = {hs, ps, nkv, (cuuint64_t)kv->n_pages};
  const cuuint64_t strides[3] = {hs * e, ps * hs * e, nkv * ps * hs * e};
  const cuuint32_t box[4] = {(cuuint32_t)(128 / e), kTile, 1, 1}, step[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type = kv->type == G4_TYPE_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : kv->type == G4_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                             : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return encode(map, type, 4, base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int attend_grid(const g4_ctx* c, const AttendPlan& p) {
  const int full = c->dev.sms * p.ctas;
  return full < kMaxGrid ? full : kMaxGrid;
}

int kv_attend_prepare(g4_kv* kv) {
  void* entry = nullptr;
  cudaDriverEntryPointQueryResult q{};
  cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &entry, cudaEnableDefault, &q);
  if (!e && (q != cudaDriverEntryPointSuccess || !entry)) e = cudaErrorNotSupported;
  for (int l = 0; l < kv->n_layers && !e; ++l) {
    auto encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(entry);
    if (!make_map(encode, &kv->k_map[l], kv, l, kv->k[l]) || !make_map(encode, &kv->v_map[l], kv, l, kv->v[l]))
      e = cudaErrorInvalidValue;
  }
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
  const size_t grid = attend_grid(kv->ctx, p);
  return grid * (sizeof(int4) + 2 * kHeadBlock * (kv->hs[layer] + 2) * sizeof(float));
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
  const AttendPlan p = attend_plan(kv->type, hs);
  const int grid = attend_grid(c, p);
  a.joins = static_cast<int4*>(work);
  a.ws = reinterpret_cast<float*>(a.joins + grid);
  cudaStream_t st = (cudaStream_t)stream;
  p.fn<<<grid, p.threads, p.smem, st>>>(a, kv->k_map[layer], kv->v_map[layer]);
  cudaError_t e = cudaGetLastError();
  if (!e)
    e = launch_after(kv_attend_join_kernel, dim3(grid), dim3(kJoinThreads), 0, st, a);
  return e ? c->cuda_fail(e, "g4_kv_attend") : 0;
}

}  // extern "C"
