// g4_kv.h -- the paged KV cache behind g4_kv_* (include/g4.h) and what its
// translation units share.
#pragma once
#include "g4.h"
#include "g4_ctx.h"

#include <cuda.h>

#include <vector>

constexpr int kKvMaxSeqs = 4096;
constexpr int kKvMaxPages = 1 << 20;
constexpr int kKvMaxHeadSize = 512;

// Bits of a cache's device status word (g4_kv_check).
enum KvFlag : unsigned {
  KV_NO_PAGES = 1u,  // g4_kv_resize: fewer free pages than the call needs
  KV_BAD_ENTRY = 2u, // a sequence, length or page out of range, or a sequence twice in one call
  KV_NOT_STORED = 4u,// g4_kv_append: position without a page, or in a page that sequences share
  KV_TIMEOUT = 16u,  // a bounded wait inside a kernel expired
  KV_BAD_ROW = 8u,   // g4_kv_attend / g4_kv_append: sequence or position out of range, or a visible position without a page
};

// One (layer, K or V, KV head): a page's positions are row_bytes apart from
// base + page * page_stride.
struct KvStrip {
  uint8_t* base;
  uint64_t page_stride;
  uint32_t row_bytes;
  uint32_t pad;
};

struct KvMove {
  int src, dst, rows;
};

struct g4_kv {
  g4_ctx* ctx = nullptr;
  int device = 0;
  int n_layers = 0, type = 0, elem = 0, page_size = 0, page_shift = 0, n_pages = 0, n_seqs = 0, max_positions = 0;
  int max_pages = 0;  // pages of one sequence (the table's width)
  int n_strips = 0;
  std::vector<int> n_kv, hs;
  std::vector<uint8_t*> k, v;  // per layer [n_pages][n_kv][page_size][hs]
  std::vector<CUtensorMap> k_map, v_map;  // per layer: 16 positions x 128 bytes of a head in a page, 128-byte swizzle
  uint8_t* pool = nullptr;
  uint8_t* meta = nullptr;     // everything below, one allocation
  int32_t *table = nullptr, *lens = nullptr, *refs = nullptr;
  unsigned* flags = nullptr;   // [0] status bits; g4_kv_check leaves free pages in [1] and the bits it took in [2]
  KvStrip* strips = nullptr;   // [n_strips]
  // work space of the calls that change the cache (ordered by the caller)
  int32_t* free_list = nullptr;  // [n_pages] free pages a call takes / the new id of every moved page
  KvMove* moves = nullptr;       // [max(n_pages, n_seqs)]
  int32_t* plan = nullptr;       // [0] number of moves, [1] live pages
};

namespace g4 {

// The context's device for the length of a call; the caller's comes back.
struct DeviceScope {
  int prev = -1, rc = 0;
  explicit DeviceScope(g4_ctx* c) {
    if (const cudaError_t e = enter(c->dev.device)) rc = c->cuda_fail(e, "cudaSetDevice");
  }
  // For handles that are freed after their context.
  explicit DeviceScope(int device) { rc = enter(device); }
  cudaError_t enter(int device) {
    cudaError_t e = cudaGetDevice(&prev);
    if (e == cudaSuccess && prev != device) e = cudaSetDevice(device);
    else prev = -1;
    return e;
  }
  ~DeviceScope() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

// Programmatic dependent launch: the kernel may start while the one before it
// on the stream runs, and waits for it with grid_dep_wait().
template <typename... KArgs, typename... Args>
cudaError_t launch_after(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

// Set-up of the kernels of one translation unit on the current device (loads
// them, so that a first call may be captured); cudaError_t as int.
int kv_attend_prepare(g4_kv* kv);
// g4_kv_resize; grow_only: a sequence that is longer than its entry asks for keeps its length.
int kv_resize(g4_kv* kv, const int32_t* seqs, const int32_t* lens, int n, bool grow_only, cudaStream_t st,
              const char* what);
int rope_prepare();
int beam_prepare();

}  // namespace g4
