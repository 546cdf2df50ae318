// g4_rope.cu -- rotary positions and the write path of the paged cache: per
// row the query/key norms, the rotation of queries and keys, and the new K and
// V rows stored into their page, in one pass over q, k and v.
//
// Mathematics: pair m of a head turns by the angle pos * f_m,
//   (a, b) -> g * (a cos - b sin, a sin + b cos),
// with pairs (m, m + rot/2) or (2m, 2m + 1).  The plan holds f_m / 2 pi in 64
// bits: pos * f_m reaches 1e6 radians, where a 32-bit product is off by 0.1.
// The turns are reduced to [-1/2, 1/2] in 64 bits and only then rounded, so the
// angle is right to 1e-7 at every position.
//
// Bound by HBM: every input and output element moves once.  A warp owns a head
// vector: its elements stay in registers as groups of four (two pairs), the
// squares are summed by shuffles. The cosines and sines of a row are computed
// once per CTA (64-bit products and conversions cost as much as the row's
// memory traffic when every warp repeats them: 8004 rows of 48 heads of 128 took
// 104 us so, 85 with one computation per CTA) while the heads' elements are on
// their way. The row's place is a chain of three loads (position, page, holders),
// longer than the row's own traffic, so many small CTAs beat few with much in
// flight: two heads a warp in flight and seven CTAs per SM 61 us (5.9 TB/s in a
// burst, 5.5 under the power cap), six heads and four CTAs 75. One row takes 3 us.
#include "g4_common.cuh"
#include "g4_kv.h"

#include <cuda_bf16.h>

#include <cmath>
#include <new>

struct g4_rope {
  g4_ctx* ctx = nullptr;
  int device = 0;
  int head_size = 0, rot = 0, interleaved = 0;
  float factor = 1.f;
  double* turns = nullptr;  // [rot / 2] turns per position
};

namespace g4 {

constexpr int kAppendThreads = 256;

struct AppendArgs {
  const float *q, *k, *v;
  float* q_out;
  long long q_stride, k_stride, v_stride, out_stride;  // floats between rows
  const int32_t *seqs, *pos;
  int n_rows, n_q, n_kv, hs;
  const double* turns;  // nullptr: no rotation
  int rot, interleaved;
  float factor;
  const float *q_norm, *k_norm;
  int norm_v;
  float eps;
  // the cache's layer (k == nullptr: queries alone)
  uint8_t *kp, *vp;
  const int32_t *table, *refs;
  unsigned* flags;
  int n_seqs, max_pages, max_positions, page_shift, n_pages;
  int heads_per_cta, ctas_per_row;
};

template <int TYPE>
__device__ __forceinline__ void store2(uint8_t* base, long long at, float x, float y) {
  if (TYPE == F32) {
    reinterpret_cast<float2*>(base)[at / 2] = make_float2(x, y);
  } else if (TYPE == F16) {
    reinterpret_cast<__half2*>(base)[at / 2] = __floats2half2_rn(x, y);
  } else {
    reinterpret_cast<__nv_bfloat162*>(base)[at / 2] = __floats2bfloat162_rn(x, y);
  }
}
template <int TYPE>
__device__ __forceinline__ void store4(uint8_t* base, long long at, float4 v) {
  if (TYPE == F32) {
    reinterpret_cast<float4*>(base)[at / 4] = v;
  } else {
    uint2 u;
    if (TYPE == F16) {
      const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
      u = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
      const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
      u = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
    reinterpret_cast<uint2*>(base)[at / 4] = u;
  }
}

// NQ groups of four elements per lane (head sizes up to 128 * NQ), HB heads of
// a warp in flight together. A CTA takes heads_per_cta heads of one row; its
// warps share the row's cosines and sines.
template <int TYPE, int NQ, int HB>
__global__ void __launch_bounds__(kAppendThreads, NQ == 1 ? 7 : NQ == 2 ? 6 : 4)
    kv_append_kernel(const __grid_constant__ AppendArgs a) {
  __shared__ float4 turn[kKvMaxHeadSize / 4];  // cosine and sine of a group's two pairs
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int NW = kAppendThreads / 32;
  const long long row = blockIdx.x / a.ctas_per_row;
  const int heads = a.n_q + 2 * a.n_kv, quads = a.hs / 4, rq = a.rot / 4, half = a.rot / 2;
  const int c0 = (int)(blockIdx.x - row * a.ctas_per_row) * a.heads_per_cta;
  const int h0 = c0 + warp, h1 = min(c0 + a.heads_per_cta, heads);  // every NW-th head
  // a group is two pairs: elements (2m, 2m + 1) with (2m, 2m + 1) + rot / 2, or four consecutive ones
  bool split[NQ];
  int lo[NQ];
#pragma unroll
  for (int u = 0; u < NQ; ++u) {
    const int m = lane + 32 * u;
    split[u] = m < rq && !a.interleaved;
    lo[u] = split[u] ? 2 * m : 4 * m;
  }
  auto source = [&](int h) {
    return h < a.n_q             ? a.q + row * a.q_stride + (long long)h * a.hs
           : h < a.n_q + a.n_kv  ? a.k + row * a.k_stride + (long long)(h - a.n_q) * a.hs
                                 : a.v + row * a.v_stride + (long long)(h - a.n_q - a.n_kv) * a.hs;
  };
  auto load = [&](int h, float4 (&x)[NQ]) {
    const float* p = source(h);
#pragma unroll
    for (int u = 0; u < NQ; ++u) {
      x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (lane + 32 * u >= quads) continue;
      if (split[u]) {
        const float2 f = __ldg(reinterpret_cast<const float2*>(p + lo[u]));
        const float2 g = __ldg(reinterpret_cast<const float2*>(p + lo[u] + half));
        x[u] = make_float4(f.x, f.y, g.x, g.y);
      } else {
        x[u] = __ldg(reinterpret_cast<const float4*>(p + lo[u]));
      }
    }
  };
  // the first heads' elements are on their way before the row's position is known
  float4 x[HB][NQ];
#pragma unroll
  for (int i = 0; i < HB; ++i)
    if (h0 + i * NW < h1) load(h0 + i * NW, x[i]);
  const int seq = a.seqs ? a.seqs[row] : 0, pos = a.pos[row];
  if (seq < 0) return;  // a padding row
  if (pos < 0 || (a.k && (seq >= a.n_seqs || pos >= a.max_positions))) {
    if (threadIdx.x == 0 && a.flags) atomicOr(a.flags, KV_BAD_ROW);
    return;
  }
  // the row's page: a position without one, or in a page that sequences share, is not stored
  const bool stores = a.k && h1 > a.n_q;
  const int page = stores ? a.table[(long long)seq * a.max_pages + (pos >> a.page_shift)] : -1;
  for (int m = threadIdx.x; m < 2 * rq; m += kAppendThreads) {
    const double t = (double)pos * a.turns[m];
    float s, c;
    sincospif(2.f * (float)(t - rint(t)), &s, &c);
    reinterpret_cast<float2*>(turn)[m] = make_float2(c * a.factor, s * a.factor);
  }
  const bool known = (unsigned)page < (unsigned)a.n_pages;
  const int refs = known ? a.refs[page] : 2;
  __syncthreads();
  long long slot = -1;
  if (refs <= 1) slot = (((long long)page * a.n_kv) << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
  else if (stores && threadIdx.x == 0) atomicOr(a.flags, KV_NOT_STORED);
  float4 cs[NQ];
#pragma unroll
  for (int u = 0; u < NQ; ++u) cs[u] = lane + 32 * u < rq ? turn[lane + 32 * u] : make_float4(1.f, 0.f, 1.f, 0.f);
  for (int hb = h0; hb < h1; hb += HB * NW) {
    if (hb > h0) {
#pragma unroll
      for (int i = 0; i < HB; ++i)
        if (hb + i * NW < h1) load(hb + i * NW, x[i]);
    }
#pragma unroll
    for (int i = 0; i < HB; ++i) {
      const int h = hb + i * NW;
      const bool is_q = h < a.n_q, is_k = !is_q && h < a.n_q + a.n_kv;
      if (h >= h1 || (!is_q && slot < 0)) break;
      const int hh = is_q ? h : is_k ? h - a.n_q : h - a.n_q - a.n_kv;
      const float* nw = is_q ? a.q_norm : is_k ? a.k_norm : nullptr;
      if (nw || (!is_q && !is_k && a.norm_v)) {
        float ss = 0.f;
#pragma unroll
        for (int u = 0; u < NQ; ++u)
          ss += x[i][u].x * x[i][u].x + x[i][u].y * x[i][u].y + x[i][u].z * x[i][u].z + x[i][u].w * x[i][u].w;
        // The factor in 32 bits, to 2^-22, next to products that round to 2^-24. Root and
        // quotient in 64 bits, as the contiguous batch takes them, cost 95.9 against 81.5
        // us for 8004 rows of 32 + 8 + 8 heads of 128, 54.2 against 50.7 for 4096 of 16 + 8
        // + 8 of 256; the outputs' error (7e-8 relative L2 of fp32 ones) is the plain form's.
        const float s = rsqrtf(warp_sum(ss) / a.hs + a.eps);
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
          if (lane + 32 * u >= quads) continue;
          float2 f = make_float2(1.f, 1.f), g = f;
          if (nw) {
            f = __ldg(reinterpret_cast<const float2*>(nw + lo[u]));
            g = __ldg(reinterpret_cast<const float2*>(nw + lo[u] + (split[u] ? half : 2)));
          }
          x[i][u].x *= f.x * s;
          x[i][u].y *= f.y * s;
          x[i][u].z *= g.x * s;
          x[i][u].w *= g.y * s;
        }
      }
#pragma unroll
      for (int u = 0; u < NQ; ++u) {
        if (lane + 32 * u >= quads) continue;
        float4 v = x[i][u];
        if ((is_q || is_k) && lane + 32 * u < rq) {  // (times 1 and 0 would spread an infinity to its neighbour)
          // pairs (x, z), (y, w) of a split group, (x, y), (z, w) otherwise
          const float b0 = split[u] ? v.z : v.y, a1 = split[u] ? v.y : v.z;
          const float y0 = v.x * cs[u].x - b0 * cs[u].y, z0 = v.x * cs[u].y + b0 * cs[u].x;
          const float y1 = a1 * cs[u].z - v.w * cs[u].w, z1 = a1 * cs[u].w + v.w * cs[u].z;
          v = split[u] ? make_float4(y0, y1, z0, z1) : make_float4(y0, z0, y1, z1);
        }
        if (is_q) {
          float* o = a.q_out + row * a.out_stride + (long long)hh * a.hs;
          if (split[u]) {
            *reinterpret_cast<float2*>(o + lo[u]) = make_float2(v.x, v.y);
            *reinterpret_cast<float2*>(o + lo[u] + half) = make_float2(v.z, v.w);
          } else {
            *reinterpret_cast<float4*>(o + lo[u]) = v;
          }
        } else {
          const long long at = (slot + ((long long)hh << a.page_shift)) * a.hs + lo[u];
          uint8_t* pool = is_k ? a.kp : a.vp;
          if (split[u]) {
            store2<TYPE>(pool, at, v.x, v.y);
            store2<TYPE>(pool, at + half, v.z, v.w);
          } else {
            store4<TYPE>(pool, at, v);
          }
        }
      }
    }
  }
}

using AppendFn = void (*)(const AppendArgs);
template <int TYPE>
static AppendFn append_fn_t(int hs, bool many) {
  if (many) return hs <= 128 ? kv_append_kernel<TYPE, 1, 2> : hs <= 256 ? kv_append_kernel<TYPE, 2, 1> : kv_append_kernel<TYPE, 4, 1>;
  return hs <= 128 ? kv_append_kernel<TYPE, 1, 1> : hs <= 256 ? kv_append_kernel<TYPE, 2, 1> : kv_append_kernel<TYPE, 4, 1>;
}
static AppendFn append_fn(int type, int hs, bool many) {
  return type == F32   ? append_fn_t<F32>(hs, many)
         : type == F16 ? append_fn_t<F16>(hs, many)
                       : append_fn_t<BF16>(hs, many);
}

static cudaError_t launch_append(const DeviceInfo& dev, int type, AppendArgs a, cudaStream_t st) {
  const int heads = a.n_q + (a.k ? 2 * a.n_kv : 0);
  if (!a.k) a.n_kv = 0;
  // Heads per warp: one while the rows do not fill the GPU (a decode step is
  // latency: every head vector its own warp, 64 rows of 32 heads 4.0 us); a whole
  // row per CTA, which computes its turns once, when that leaves every SM 32 warps
  // (8004 rows: 62 us; with a head per warp 85).
  constexpr int kWarps = kAppendThreads / 32;
  const bool many = (long long)a.n_rows * kWarps >= (long long)dev.sms * 32;
  a.heads_per_cta = many ? heads : kWarps;
  a.ctas_per_row = (heads + a.heads_per_cta - 1) / a.heads_per_cta;
  const long long grid = (long long)a.n_rows * a.ctas_per_row;
  if (grid > 0x7fffffffll) return cudaErrorInvalidValue;
  append_fn(type, a.hs, many && heads > kWarps)<<<(unsigned)grid, kAppendThreads, 0, st>>>(a);
  return cudaGetLastError();
}

int rope_prepare() {
  cudaFuncAttributes fa;
  cudaError_t e = cudaSuccess;
  for (int type : {F32, F16, BF16})
    for (int hs : {128, 256, 512})
      for (bool many : {false, true})
        if (!e) e = cudaFuncGetAttributes(&fa, append_fn(type, hs, many));
  return e;
}

// (one row has no distance to the next)
static bool rows_ok(const void* p, long long stride, int heads, int hs, int n) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 &&
         (n <= 1 || (stride % 4 == 0 && stride >= (long long)heads * hs));
}

}  // namespace g4

using namespace g4;

extern "C" {

int g4_rope_create(g4_ctx* c, const g4_rope_config* cfg, g4_rope** out) {
  if (!c) return G4_E_ARG;
  if (!cfg || !out) {
    c->set_err("g4_rope_create: NULL argument");
    return G4_E_ARG;
  }
  *out = nullptr;
  const int rot = cfg->rot_dim;
  if (cfg->head_size < 8 || cfg->head_size > kKvMaxHeadSize || cfg->head_size % 8 || rot < 4 || rot > cfg->head_size ||
      rot % 4 || !(cfg->theta > 1.0) || std::isinf(cfg->theta) ||
      (cfg->layout != G4_ROPE_HALF && cfg->layout != G4_ROPE_INTERLEAVED)) {
    c->set_err("g4_rope_create: head size %d (8..%d in steps of 8), %d rotated (4..head size in steps of 4), base %g "
               "(above 1), layout %d", cfg->head_size, kKvMaxHeadSize, rot, cfg->theta, cfg->layout);
    return G4_E_ARG;
  }
  const bool yarn = cfg->scaling == G4_ROPE_YARN;
  if ((cfg->scaling != G4_ROPE_UNSCALED && cfg->scaling != G4_ROPE_LINEAR && !yarn) ||
      (cfg->scaling != G4_ROPE_UNSCALED && (!(cfg->factor > 0.0) || std::isinf(cfg->factor))) ||
      (yarn && (cfg->original_ctx < 1 || !(cfg->beta_fast > 0.0) || !(cfg->beta_slow > 0.0) || std::isinf(cfg->beta_fast) ||
                std::isinf(cfg->beta_slow))) ||
      !(std::fabs(cfg->attn_factor) < 1e30)) {
    c->set_err("g4_rope_create: scaling %d with factor %g, original context %d, betas %g / %g", cfg->scaling,
               cfg->factor, cfg->original_ctx, cfg->beta_fast, cfg->beta_slow);
    return G4_E_ARG;
  }
  const double kPi = 3.14159265358979323846;
  double turns[kKvMaxHeadSize / 2];
  double low = 0, high = 0;
  if (yarn) {
    // the pair that makes r turns over the original context
    auto pair_of = [&](double r) {
      return rot * std::log(cfg->original_ctx / (r * 2.0 * kPi)) / (2.0 * std::log(cfg->theta));
    };
    low = std::fmax(std::floor(pair_of(cfg->beta_fast)), 0.0);
    high = std::fmin(std::ceil(pair_of(cfg->beta_slow)), rot - 1.0);
  }
  for (int m = 0; m < rot / 2; ++m) {
    double f = std::pow(cfg->theta, -2.0 * m / rot);
    if (cfg->freq_factors) {
      if (!(std::fabs(cfg->freq_factors[m]) > 0.f)) {
        c->set_err("g4_rope_create: frequency factor %d is %g", m, cfg->freq_factors[m]);
        return G4_E_ARG;
      }
      f /= cfg->freq_factors[m];
    }
    if (cfg->scaling == G4_ROPE_LINEAR) f /= cfg->factor;
    if (yarn) {
      const double part = std::fmin(1.0, std::fmax(0.0, (m - low) / std::fmax(high - low, 1e-3)));
      f = f / cfg->factor * part + f * (1.0 - part);
    }
    turns[m] = f / (2.0 * kPi);
  }
  DeviceScope scope(c);
  if (scope.rc) return scope.rc;
  g4_rope* r = new (std::nothrow) g4_rope();
  if (!r) return G4_E_NOMEM;
  r->ctx = c;
  r->device = c->dev.device;
  r->head_size = cfg->head_size;
  r->rot = rot;
  r->interleaved = cfg->layout == G4_ROPE_INTERLEAVED;
  r->factor = cfg->attn_factor != 0.0 ? (float)cfg->attn_factor
              : yarn                  ? (float)(0.1 * std::log(std::fmax(cfg->factor, 1.0)) + 1.0)
                                      : 1.f;
  cudaError_t e = cudaMalloc(&r->turns, sizeof(double) * (rot / 2));
  if (e) {
    cudaGetLastError();
    r->turns = nullptr;
    g4_rope_free(r);
    c->set_err("g4_rope_create: cannot allocate the frequency table");
    return G4_E_NOMEM;
  }
  e = cudaMemcpy(r->turns, turns, sizeof(double) * (rot / 2), cudaMemcpyHostToDevice);
  if (!e) e = (cudaError_t)rope_prepare();
  if (e) {
    g4_rope_free(r);
    return c->cuda_fail(e, "g4_rope_create");
  }
  *out = r;
  return 0;
}

int g4_rope_free(g4_rope* r) {
  if (!r) return G4_E_ARG;
  {
    DeviceScope scope(r->device);
    if (r->turns) cudaFree(r->turns);
  }
  delete r;
  return 0;
}

int g4_rope_apply(const g4_rope* r, const float* x, int64_t x_stride, float* out, int64_t out_stride, int n_heads,
                  const int32_t* pos, int n_rows, void* stream) {
  if (!r) return G4_E_ARG;
  g4_ctx* c = r->ctx;
  if (n_rows < 0 || n_heads < 1 || n_heads > 4096 ||
      (n_rows > 0 && (!x || !out || !pos || !rows_ok(x, x_stride, n_heads, r->head_size, n_rows) ||
                      !rows_ok(out, out_stride, n_heads, r->head_size, n_rows)))) {
    c->set_err("g4_rope_apply: bad arguments (%d rows of %d heads; rows 16-byte aligned and at least heads x head "
               "size apart)", n_rows, n_heads);
    return G4_E_ARG;
  }
  if (n_rows == 0) return 0;
  DeviceScope scope(c);
  if (scope.rc) return scope.rc;
  AppendArgs a{};
  a.q = x;
  a.q_stride = x_stride;
  a.q_out = out;
  a.out_stride = out_stride;
  a.pos = pos;
  a.n_rows = n_rows;
  a.n_q = n_heads;
  a.hs = r->head_size;
  a.turns = r->turns;
  a.rot = r->rot;
  a.interleaved = r->interleaved;
  a.factor = r->factor;
  const cudaError_t e = launch_append(c->dev, F32, a, (cudaStream_t)stream);
  return e ? c->cuda_fail(e, "g4_rope_apply") : 0;
}

int g4_kv_append(g4_kv* kv, int layer, const g4_kv_rows* rows, const g4_rope* rope, void* stream) {
  if (!kv) return G4_E_ARG;
  g4_ctx* c = kv->ctx;
  if (!rows || layer < 0 || layer >= kv->n_layers) {
    c->set_err("g4_kv_append: layer %d of %d, rows %p", layer, kv->n_layers, (const void*)rows);
    return G4_E_ARG;
  }
  const int hs = kv->hs[layer], nkv = kv->n_kv[layer], n = rows->n_rows;
  const int nq = rows->q ? rows->n_heads : 0;
  const bool stores = rows->k || rows->v;
  if (n < 0 || nq < 0 || nq > 4096 || (rows->q && nq < 1) ||
      (n > 0 && (!rows->seqs || !rows->pos || (!stores && !nq) ||
                 (stores && (!rows->k || !rows->v || !rows_ok(rows->k, rows->k_stride, nkv, hs, n) ||
                             !rows_ok(rows->v, rows->v_stride, nkv, hs, n))) ||
                 (nq && (!rows->q_out || !rows_ok(rows->q, rows->q_stride, nq, hs, n) ||
                         !rows_ok(rows->q_out, rows->q_out_stride, nq, hs, n)))))) {
    c->set_err("g4_kv_append: bad arguments (%d rows, %d query heads, head size %d; K and V together or neither; rows "
               "16-byte aligned and at least heads x head size apart)", n, nq, hs);
    return G4_E_ARG;
  }
  if (rope && (rope->head_size != hs || rope->device != c->dev.device)) {
    c->set_err("g4_kv_append: the rotary plan is for head size %d on device %d, the layer has %d on %d",
               rope->head_size, rope->device, hs, c->dev.device);
    return G4_E_ARG;
  }
  if ((reinterpret_cast<uintptr_t>(rows->q_norm) | reinterpret_cast<uintptr_t>(rows->k_norm)) & 7) {
    c->set_err("g4_kv_append: norm weights must be 8-byte aligned");
    return G4_E_ARG;
  }
  if (n == 0) return 0;
  DeviceScope scope(c);
  if (scope.rc) return scope.rc;
  AppendArgs a{};
  a.q = rows->q;
  a.k = rows->k;
  a.v = rows->v;
  a.q_out = rows->q_out;
  a.q_stride = rows->q_stride;
  a.k_stride = rows->k_stride;
  a.v_stride = rows->v_stride;
  a.out_stride = rows->q_out_stride;
  a.seqs = rows->seqs;
  a.pos = rows->pos;
  a.n_rows = n;
  a.n_q = nq;
  a.n_kv = nkv;
  a.hs = hs;
  if (rope) {
    a.turns = rope->turns;
    a.rot = rope->rot;
    a.interleaved = rope->interleaved;
    a.factor = rope->factor;
  }
  a.q_norm = rows->q_norm;
  a.k_norm = rows->k_norm;
  a.norm_v = rows->norm_v;
  a.eps = rows->eps;
  a.kp = kv->k[layer];
  a.vp = kv->v[layer];
  a.table = kv->table;
  a.refs = kv->refs;
  a.flags = kv->flags;
  a.n_seqs = kv->n_seqs;
  a.max_pages = kv->max_pages;
  a.max_positions = kv->max_positions;
  a.page_shift = kv->page_shift;
  a.n_pages = kv->n_pages;
  const cudaError_t e = launch_append(c->dev, kv->type, a, (cudaStream_t)stream);
  return e ? c->cuda_fail(e, "g4_kv_append") : 0;
}

}  // extern "C"
