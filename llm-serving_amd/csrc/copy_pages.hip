// Pages of a paged cache copied to other pages of it, in every layer's K and V pool, in one
// launch: pool[dst[i]] = pool[src[i]].
//
// A byte copy, bound by memory. The page ids and the pools' addresses travel by value in the kernel
// arguments: no device buffer to fill and keep alive, no host wait, and a captured launch keeps its ids.
// A workgroup moves kGroupBytes of one page of one pool, 16 bytes per thread and load with all loads
// before the first store; both sides are touched once, so both carry the nontemporal hint.
#include "common.h"

namespace miattn {
namespace {

constexpr int kMaxPools = 64;   // 512 bytes of kernel arguments
constexpr int kMaxMoves = 192;  // 1536 bytes
constexpr int kPerThread = 4;
constexpr int kGroupBytes = 256 * 16 * kPerThread;

struct CopyArgs {
  uint8_t* pool[kMaxPools];
  int32_t src[kMaxMoves], dst[kMaxMoves];
  int64_t page_bytes;
};

__global__ __launch_bounds__(256) void copy_pages_vec(CopyArgs a) {
  uint8_t* pool = a.pool[blockIdx.z];
  const uint8_t* from = pool + int64_t(a.src[blockIdx.y]) * a.page_bytes;
  uint8_t* to = pool + int64_t(a.dst[blockIdx.y]) * a.page_bytes;
  const int64_t at = int64_t(blockIdx.x) * kGroupBytes + threadIdx.x * 16;
  uint4 v[kPerThread];
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int64_t o = at + i * (256 * 16);
    if (o < a.page_bytes) v[i] = load16_nt(from + o);
  }
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int64_t o = at + i * (256 * 16);
    if (o < a.page_bytes) store16_nt(to + o, v[i]);
  }
}

// Pages or pools that are not a multiple of 16 bytes.
__global__ __launch_bounds__(256) void copy_pages_bytes(CopyArgs a) {
  uint8_t* pool = a.pool[blockIdx.z];
  const uint8_t* from = pool + int64_t(a.src[blockIdx.y]) * a.page_bytes;
  uint8_t* to = pool + int64_t(a.dst[blockIdx.y]) * a.page_bytes;
  for (int i = 0; i < kGroupBytes / 256; ++i) {
    const int64_t o = int64_t(blockIdx.x) * kGroupBytes + i * 256 + threadIdx.x;
    if (o < a.page_bytes) to[o] = from[o];
  }
}

}  // namespace
}  // namespace miattn

extern "C" int mi_copy_pages(void* const* host_pools, int n_pools, int64_t page_bytes, int64_t n_blocks,
                             const int32_t* host_src, const int32_t* host_dst, int n_moves, void* stream) {
  using namespace miattn;
  if (n_pools < 0 || n_moves < 0 || page_bytes < 1 || n_blocks < 0) {
    return fail(MI_ERR_INVALID, "mi_copy_pages: bad sizes n_pools=%d n_moves=%d page_bytes=%lld n_blocks=%lld", n_pools,
                n_moves, (long long)page_bytes, (long long)n_blocks);
  }
  if (n_pools == 0 || n_moves == 0) return MI_OK;
  if (host_pools == nullptr || host_src == nullptr || host_dst == nullptr) {
    return fail(MI_ERR_INVALID, "mi_copy_pages: NULL argument");
  }
  bool vec = page_bytes % 16 == 0;
  for (int i = 0; i < n_pools; ++i) {
    if (host_pools[i] == nullptr) return fail(MI_ERR_INVALID, "mi_copy_pages: pool %d is NULL", i);
    vec = vec && reinterpret_cast<uintptr_t>(host_pools[i]) % 16 == 0;
  }
  for (int i = 0; i < n_moves; ++i) {
    if (host_src[i] < 0 || host_src[i] >= n_blocks || host_dst[i] < 0 || host_dst[i] >= n_blocks) {
      return fail(MI_ERR_INVALID, "mi_copy_pages: move %d (%d -> %d) is outside the pool's %lld blocks", i, host_src[i],
                  host_dst[i], (long long)n_blocks);
    }
  }
  const int64_t groups = (page_bytes + kGroupBytes - 1) / kGroupBytes;
  if (groups > 0x7fffffff) return fail(MI_ERR_UNSUPPORTED, "mi_copy_pages: a page of %lld bytes", (long long)page_bytes);
  for (int p0 = 0; p0 < n_pools; p0 += kMaxPools) {
    const int np = n_pools - p0 < kMaxPools ? n_pools - p0 : kMaxPools;
    for (int m0 = 0; m0 < n_moves; m0 += kMaxMoves) {
      const int nm = n_moves - m0 < kMaxMoves ? n_moves - m0 : kMaxMoves;
      CopyArgs a{};
      a.page_bytes = page_bytes;
      for (int i = 0; i < np; ++i) a.pool[i] = static_cast<uint8_t*>(host_pools[p0 + i]);
      for (int i = 0; i < nm; ++i) {
        a.src[i] = host_src[m0 + i];
        a.dst[i] = host_dst[m0 + i];
      }
      const dim3 grid(unsigned(groups), nm, np);
      if (vec) {
        hipLaunchKernelGGL(copy_pages_vec, grid, dim3(256), 0, static_cast<hipStream_t>(stream), a);
      } else {
        hipLaunchKernelGGL(copy_pages_bytes, grid, dim3(256), 0, static_cast<hipStream_t>(stream), a);
      }
      const int rc = launch_status("mi_copy_pages");
      if (rc != MI_OK) return rc;
    }
  }
  return MI_OK;
}
