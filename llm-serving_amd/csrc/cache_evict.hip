// Rows of a paged cache cut to a budget by the weight that attention gave their tokens, per layer, row and KV head.
//
// Of a row of n > budget tokens, the first `sinks`, the last `recent` and the budget - sinks - recent heaviest of the others
// stay (NaN above every number; of equal weights the lower index), in their order: kept[p] is the p-th of them, and
//   K[p], V[p], weights[p] = K[kept[p]], V[kept[p]], weights[kept[p]]  for p < budget,  weights[budget .. n) = 0,  seqlen = budget.
// Every KV head keeps tokens of its own: a pool row (token, KV head) is what moves.
//
// Two launches. The first finds kept: the weights as integers that order like them, in registers, and the budget's
// threshold 8 bits at a time by counting in LDS (bit by bit with ballots and a barrier each: 11.4 us against 6.2 for
// 224 rows of 1088 tokens, 26.8 against 15.4 for 1024 of up to 4096); then one ordered pass of ballots gives each
// kept token its place. The second moves the rows, bound by memory: 2 * D * element size read and written per kept
// (token, KV head), 50 us for 235 MB and 116 us for 510 MB with places drawn at random, 4.4 to 4.7 TB/s of the 5.1 that
// a large copy reaches. K and V have workgroups of their own; where the rows go to other blocks, so have stretches
// of a row. In place, one workgroup goes up a row: p <= kept[p], so a stretch's sources are never below the
// places already written, and a barrier between its loads and its stores is all the order that it needs; it is as large
// as one may be, for fewer of them (a row of 1088 tokens cut to 1024 in 28 layers 88 us with the host's share, 32 of them
// 1567, 4.8 TB/s; with 256 threads 110 and 1610).
#include <algorithm>

#include "common.h"

namespace miattn {
namespace {

constexpr int kMaxLayers = 64;  // 1 KiB of kernel arguments

struct EvictArgs {
  uint8_t* k[kMaxLayers];
  uint8_t* v[kMaxLayers];
  const int32_t* table;
  const int32_t* to;
  int64_t bts0, tos0, ws0, ws1, ws2;
  int32_t* seqlen;
  float* weights;
  int32_t* kept;   // [layers][B][H_kv][budget]: token of the row
  int32_t* slots;  // the same: its slot in the pool, -1 outside
  int32_t* rows;   // [B]: lengths before
  int32_t* err;
  int B, H_kv, block_size, max_blocks, n_blocks, budget, recent, sinks, in_place, last;
};

// Integers that order like the weights: 0 is below all of them.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.0f);  // -0 and 0 are equal
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int row_length(int len, const EvictArgs& a) {
  const int capacity = a.max_blocks * a.block_size;
  return max(0, min(len, capacity));
}

// The slot of a row's token i (page id read from its table), -1 where the table names no block of the pool.
__device__ __forceinline__ int slot_of(const int32_t* table, int i, const EvictArgs& a) {
  const int page = table[i / a.block_size];
  return uint32_t(page) < uint32_t(a.n_blocks) ? page * a.block_size + i % a.block_size : -1;
}

// Items: weights per thread, held in registers; 0 for rows of any length, which read them again in each of up to 5 passes
// (256 rows of 20000 tokens 57 us so, 29.5 held; 128 of 60000 154 and 72). With 16, 32 and 64 of them 18, 116 and 358
// scalars (the ballots of every round, kept for both loops over them) spill to lanes of vector registers, none to memory.
template <int NT, int Items>
__global__ __launch_bounds__(NT) void evict_select_kernel(EvictArgs a) {
  constexpr int W = NT / 64, E = Items * W;  // a count per wave and round
  constexpr bool kLong = Items == 0;
  static_assert(kLong || E % 64 == 0, "whole counts per lane");
  __shared__ int sm[2][W], sm_eq[2][W];
  __shared__ __align__(16) uint32_t counts[kLong ? 4 : E];
  __shared__ __align__(16) int hist[256];
  const int h = blockIdx.x, b = blockIdx.y, l = blockIdx.z;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int n = row_length(a.seqlen[b], a);
  if (h == 0 && l == 0 && tid == 0) a.rows[b] = n;
  if (n <= a.budget) return;  // uniform
  const float* w = a.weights + l * a.ws0 + b * a.ws1 + h * a.ws2 + a.sinks;
  const int32_t* table = a.table + b * a.bts0;
  const int64_t at = ((int64_t(l) * a.B + b) * a.H_kv + h) * a.budget;
  int32_t* kept = a.kept + at;
  int32_t* slots = a.slots + at;
  const int count = n - a.sinks - a.recent;           // candidates
  const int need = a.budget - a.sinks - a.recent;     // of them to keep: 0 <= need < count
  for (int i = tid; i < a.sinks; i += NT) kept[i] = i;
  for (int i = tid; i < a.recent; i += NT) kept[a.budget - a.recent + i] = n - a.recent + i;
  // The places in the pool, all at once at the end: looked up where a token is kept, each round of the pass below waited for
  // its table entries (25 us of the 1024 rows' pass, 22 so).
  auto look_up = [&] {
    __syncthreads();  // the list is written
    for (int p = tid; p < a.budget; p += NT) slots[p] = slot_of(table, kept[p], a);
  };
  if (need == 0) {
    look_up();
    return;
  }
  const int rounds = (count + NT - 1) / NT;
  uint32_t held[kLong ? 1 : Items];
  auto load = [&](int j) {
    const int i = j * NT + tid;
    return i < count ? order_of(w[i]) : 0u;
  };
  if constexpr (!kLong) {
#pragma unroll
    for (int j = 0; j < Items; ++j) held[j] = load(j);
  }
  // The threshold T, the need-th largest weight, 8 bits at a time from the top: the weights whose upper bits are T's are
  // counted by their next 8, and the digit is the one whose bin the need-th falls into. Ends when that bin is taken whole.
  uint32_t T = 0;
  int left = need;  // to be taken from the weights that share T's bits so far
  bool whole = false;
  for (int shift = 24; shift >= 0 && !whole; shift -= 8) {
    for (int i = tid; i < 256; i += NT) hist[i] = 0;
    __syncthreads();
    const uint32_t above_mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    auto tally = [&](uint32_t x) {
      // (0 is no weight)
      if (x != 0 && ((x ^ T) & above_mask) == 0) atomicAdd(&hist[(x >> shift) & 255], 1);
    };
    if constexpr (kLong) {
      for (int j = 0; j < rounds; ++j) tally(load(j));
    } else {
#pragma unroll
      for (int j = 0; j < Items; ++j) {
        if (j < rounds) tally(held[j]);
      }
    }
    __syncthreads();
    // every wave finds the digit by itself: lane l holds the bins 255 - 4 l .. 252 - 4 l, from the heaviest down
    int4 bins = *reinterpret_cast<const int4*>(&hist[252 - 4 * lane]);
    const int mine = bins.x + bins.y + bins.z + bins.w;
    const int upto = wave_inclusive_scan(mine), before = upto - mine;
    const uint64_t owner = __ballot(before < left && left <= upto);
    const int o = __ffsll(static_cast<unsigned long long>(owner)) - 1;
    const int b3 = __builtin_amdgcn_readlane(bins.w, o), b2 = __builtin_amdgcn_readlane(bins.z, o);
    const int b1 = __builtin_amdgcn_readlane(bins.y, o), b0 = __builtin_amdgcn_readlane(bins.x, o);
    int taken = __builtin_amdgcn_readlane(before, o), digit = 255 - 4 * o, in_bin = b3;
    if (taken + in_bin < left) taken += in_bin, --digit, in_bin = b2;
    if (taken + in_bin < left) taken += in_bin, --digit, in_bin = b1;
    if (taken + in_bin < left) taken += in_bin, --digit, in_bin = b0;
    left -= taken;
    T |= uint32_t(digit) << shift;
    whole = left == in_bin;
    __syncthreads();  // the bins are read before they are cleared
  }
  // T's lower bits are 0 where its last bin is taken whole: everything from T on stays. Else those above T stay and
  // the first `equal` at T.
  const int equal = whole ? 0 : left;
  if (whole) --T;  // (a bin of weights is not at 0, so T is not)
  const uint64_t below = (uint64_t(1) << lane) - 1;
  // a kept weight's place: the heavier ones before it and those at the threshold that stay
  auto put = [&](int j, uint32_t x, int gt, int eq) {
    if (x > T || (x == T && eq < equal)) kept[a.sinks + gt + min(eq, equal)] = a.sinks + j * NT + tid;
  };
  if constexpr (kLong) {
    int turn = 0, gt_run = 0, eq_run = 0;
    for (int j = 0; j < rounds; ++j) {
      const uint32_t x = load(j);
      const uint64_t bg = __ballot(x > T), be = __ballot(x == T);
      turn ^= 1;
      if (lane == 0) {
        sm[turn][wave] = __popcll(bg);
        sm_eq[turn][wave] = __popcll(be);
      }
      __syncthreads();
      int g = gt_run, q = eq_run;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        g += i < wave ? sm[turn][i] : 0;
        q += i < wave ? sm_eq[turn][i] : 0;
        gt_run += sm[turn][i];
        eq_run += sm_eq[turn][i];
      }
      put(j, x, g + __popcll(bg & below), q + __popcll(be & below));
    }
  } else {
    // the counts of every round and wave, above the threshold in the lower half, at it in the upper (65536 of either would not
    // fit, but no start has so many before it); one scan gives each
    // round its start (a barrier per round and 1024 threads: 22 us, 15.4 so, the 1024 rows)
    constexpr int P = E / 64;
#pragma unroll
    for (int j = 0; j < Items; ++j) {
      const uint64_t bg = __ballot(held[j] > T), be = __ballot(held[j] == T);
      if (lane == 0) counts[j * W + wave] = uint32_t(__popcll(bg)) | uint32_t(__popcll(be)) << 16;
    }
    __syncthreads();
    uint32_t before = 0, mine = 0;  // of this lane's P counts: those before the one of this wave's, all of them
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const uint32_t c = counts[lane * P + i];
      if (i < wave % P) before += c;
      mine += c;
    }
    before += uint32_t(wave_inclusive_scan(int(mine))) - mine;
#pragma unroll
    for (int j = 0; j < Items; ++j) {
      if (j < rounds) {
        const uint32_t start = __builtin_amdgcn_readlane(before, (j * W + wave) / P);
        const uint64_t bg = __ballot(held[j] > T), be = __ballot(held[j] == T);
        put(j, held[j], int(start & 0xffff) + __popcll(bg & below), int(start >> 16) + __popcll(be & below));
      }
    }
  }
  look_up();
}

constexpr int kPerThread = 8;  // 16-byte loads of a thread before its first store

// LPR lanes of 16 bytes per (token, KV head) row.
template <int LPR, int NT>
__global__ __launch_bounds__(NT) void evict_move_kernel(EvictArgs a) {
  constexpr int kRows = NT / LPR, kStretch = kRows * kPerThread, kRowBytes = LPR * 16;
  const int tid = threadIdx.x;
  const int l = blockIdx.x / (a.B * a.H_kv), bh = blockIdx.x - l * (a.B * a.H_kv);
  const int b = bh / a.H_kv, h = bh - b * a.H_kv;
  const int n = a.rows[b], keep = min(n, a.budget);
  const bool cut = n > a.budget;
  const int64_t at = ((int64_t(l) * a.B + b) * a.H_kv + h) * a.budget;
  const int32_t* kept = a.kept + at;
  if (blockIdx.y == 2) {  // the weights, and (once) the row's length: in place, one workgroup
    if (!cut || blockIdx.z != 0) return;
    float* w = a.weights + l * a.ws0 + b * a.ws1 + h * a.ws2;
    for (int p0 = 0; p0 < keep; p0 += NT * kPerThread) {
      float x[kPerThread];
#pragma unroll
      for (int j = 0; j < kPerThread; ++j) {
        const int p = p0 + j * NT + tid;
        x[j] = p < keep ? w[kept[p]] : 0.0f;
      }
#pragma unroll
      for (int j = 0; j < kPerThread; ++j) asm volatile("" : "+v"(x[j]));  // landed
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kPerThread; ++j) {
        const int p = p0 + j * NT + tid;
        if (p < keep) w[p] = x[j];
      }
    }
    for (int i = keep + tid; i < n; i += NT) w[i] = 0.0f;
    if (a.last && l == 0 && h == 0 && tid == 0) a.seqlen[b] = keep;
    return;
  }
  if (!cut && a.in_place) return;
  uint8_t* pool = blockIdx.y == 0 ? a.k[l] : a.v[l];
  const int32_t* slots = a.slots + at;
  const int32_t* table = a.table + b * a.bts0;
  const int32_t* to = a.to + b * a.tos0;
  const int row = tid / LPR, c = tid - row * LPR;
  const int64_t slot_bytes = int64_t(a.H_kv) * kRowBytes;
  pool += int64_t(h) * kRowBytes + c * 16;
  for (int p0 = blockIdx.z * kStretch; p0 < keep; p0 += gridDim.z * kStretch) {
    int src[kPerThread], dst[kPerThread];
    uint4 x[kPerThread];
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
      const int p = p0 + j * kRows + row;
      src[j] = dst[j] = -1;
      if (p < keep) {
        src[j] = cut ? slots[p] : slot_of(table, p, a);
        dst[j] = slot_of(to, p, a);
        if ((src[j] < 0 || dst[j] < 0) && a.err != nullptr) atomicCAS(a.err, 0, b + 1);
      }
    }
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
      x[j] = make_uint4(0u, 0u, 0u, 0u);
      if (src[j] >= 0 && dst[j] >= 0 && src[j] != dst[j]) x[j] = load16_nt(pool + src[j] * slot_bytes);
    }
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) asm volatile("" : "+v"(x[j].x), "+v"(x[j].y), "+v"(x[j].z), "+v"(x[j].w));
    if (a.in_place) __syncthreads();  // every source of the stretch has been read before any place of it is written
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
      if (src[j] >= 0 && dst[j] >= 0 && src[j] != dst[j]) store16_nt(pool + dst[j] * slot_bytes, x[j]);
    }
  }
}

template <int LPR>
int launch_move(const EvictArgs& a, int layers, hipStream_t s) {
  if (a.in_place) {
    hipLaunchKernelGGL((evict_move_kernel<LPR, 1024>), dim3(layers * a.B * a.H_kv, 3), dim3(1024), 0, s, a);
  } else {
    constexpr int stretch = 256 / LPR * kPerThread;
    const int nz = std::min((a.budget + stretch - 1) / stretch, 256);
    hipLaunchKernelGGL((evict_move_kernel<LPR, 256>), dim3(layers * a.B * a.H_kv, 3, nz), dim3(256), 0, s, a);
  }
  return launch_status("mi_cache_evict (move)");
}

size_t list_bytes(int layers, int B, int H_kv, int budget) {
  return (size_t(layers) * B * H_kv * budget * sizeof(int32_t) + 15) / 16 * 16;
}

}  // namespace
}  // namespace miattn

extern "C" size_t mi_cache_evict_workspace_size(int n_layers, int B, int H_kv, int budget) {
  if (n_layers < 1 || B < 1 || H_kv < 1 || budget < 1) return 0;
  return 2 * miattn::list_bytes(std::min(n_layers, miattn::kMaxLayers), B, H_kv, budget) + size_t(B) * sizeof(int32_t);
}

extern "C" int mi_cache_evict(void* const* host_k_pools, void* const* host_v_pools, int n_layers, int64_t n_blocks,
                              int block_size, int H_kv, int row_bytes, const int32_t* block_table, int64_t bt_stride,
                              int max_blocks, const int32_t* to_table, int64_t to_stride, int to_blocks,
                              int32_t* seqlen, float* weights, const int64_t* weight_strides, int B, int budget,
                              int recent, int sinks, void* workspace, size_t workspace_bytes, int32_t* error_word,
                              void* stream) {
  using namespace miattn;
  if (n_layers < 0 || B < 0 || H_kv < 1 || n_blocks < 1 || block_size < 1 || max_blocks < 1 || to_blocks < 1) {
    return fail(MI_ERR_INVALID, "mi_cache_evict: bad sizes (layers %d, rows %d, H_kv %d, blocks %lld of %d, tables of %d and %d)",
                n_layers, B, H_kv, (long long)n_blocks, block_size, max_blocks, to_blocks);
  }
  if (budget < 1 || recent < 0 || sinks < 0 || int64_t(recent) + sinks > budget) {
    return fail(MI_ERR_INVALID, "mi_cache_evict: budget %d must be positive and hold recent %d + sinks %d", budget, recent, sinks);
  }
  if (row_bytes < 16 || row_bytes > 1024 || (row_bytes & (row_bytes - 1)) != 0) {
    return fail(MI_ERR_UNSUPPORTED, "mi_cache_evict: rows of 16 to 1024 bytes, a power of two, got %d", row_bytes);
  }
  const int64_t capacity = int64_t(max_blocks) * block_size;
  if (n_blocks * block_size > INT32_MAX || capacity > INT32_MAX || int64_t(to_blocks) * block_size > INT32_MAX) {
    return fail(MI_ERR_UNSUPPORTED, "mi_cache_evict: pools and tables must stay below 2^31 tokens");
  }
  if (int64_t(to_blocks) * block_size < std::min<int64_t>(budget, capacity)) {
    return fail(MI_ERR_INVALID, "mi_cache_evict: %d destination blocks of %d do not hold %d tokens", to_blocks, block_size, budget);
  }
  if (B == 0 || n_layers == 0) return MI_OK;
  if (B > 65535 || int64_t(std::min(n_layers, kMaxLayers)) * B * H_kv >= (1 << 22)  /* 2^32 threads */) {
    return fail(MI_ERR_UNSUPPORTED, "mi_cache_evict: grid too large (B=%d, H_kv=%d)", B, H_kv);
  }
  if (host_k_pools == nullptr || host_v_pools == nullptr || block_table == nullptr || to_table == nullptr ||
      seqlen == nullptr || weights == nullptr || weight_strides == nullptr) {
    return fail(MI_ERR_INVALID, "mi_cache_evict: a required pointer is NULL");
  }
  // a budget past what a table holds never cuts a row: no list is written or read
  if (budget > capacity) budget = int(capacity);
  if (recent + sinks > budget) {  // nothing is cut, so which tokens would stay does not matter
    recent = std::min(recent, budget);
    sinks = std::min(sinks, budget - recent);
  }
  const size_t need = mi_cache_evict_workspace_size(n_layers, B, H_kv, budget);
  if (workspace == nullptr || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16 != 0) {
    return fail(MI_ERR_WORKSPACE, "mi_cache_evict: a 16-byte aligned workspace of %zu bytes is needed, got %zu", need,
                workspace_bytes);
  }
  for (int l = 0; l < n_layers; ++l) {
    if (host_k_pools[l] == nullptr || host_v_pools[l] == nullptr ||
        (reinterpret_cast<uintptr_t>(host_k_pools[l]) | reinterpret_cast<uintptr_t>(host_v_pools[l])) % 16 != 0) {
      return fail(MI_ERR_INVALID, "mi_cache_evict: layer %d's pools must be 16-byte aligned", l);
    }
  }
  EvictArgs a{};
  a.table = block_table;
  a.to = to_table;
  a.bts0 = bt_stride;
  a.tos0 = to_stride;
  a.ws0 = weight_strides[0];
  a.ws1 = weight_strides[1];
  a.ws2 = weight_strides[2];
  a.seqlen = seqlen;
  const size_t list = list_bytes(std::min(n_layers, kMaxLayers), B, H_kv, budget);
  a.kept = static_cast<int32_t*>(workspace);
  a.slots = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + list);
  a.rows = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + 2 * list);
  a.err = error_word;
  a.B = B;
  a.H_kv = H_kv;
  a.block_size = block_size;
  a.max_blocks = max_blocks;
  a.n_blocks = int(n_blocks);
  a.budget = budget;
  a.recent = recent;
  a.sinks = sinks;
  a.in_place = to_table == block_table && (to_stride == bt_stride || B == 1);
  hipStream_t s = static_cast<hipStream_t>(stream);
  for (int l0 = 0; l0 < n_layers; l0 += kMaxLayers) {
    const int layers = std::min(n_layers - l0, kMaxLayers);
    for (int i = 0; i < layers; ++i) {
      a.k[i] = static_cast<uint8_t*>(host_k_pools[l0 + i]);
      a.v[i] = static_cast<uint8_t*>(host_v_pools[l0 + i]);
    }
    a.weights = weights + l0 * a.ws0;
    a.last = l0 + layers == n_layers;
    const dim3 grid(H_kv, B, layers);
    if (capacity <= 512 * 8) {
      hipLaunchKernelGGL((evict_select_kernel<512, 8>), grid, dim3(512), 0, s, a);
    } else if (capacity <= 1024 * 16) {
      hipLaunchKernelGGL((evict_select_kernel<1024, 16>), grid, dim3(1024), 0, s, a);
    } else if (capacity <= 1024 * 32) {
      hipLaunchKernelGGL((evict_select_kernel<1024, 32>), grid, dim3(1024), 0, s, a);
    } else if (capacity <= 1024 * 64) {
      hipLaunchKernelGGL((evict_select_kernel<1024, 64>), grid, dim3(1024), 0, s, a);
    } else {
      hipLaunchKernelGGL((evict_select_kernel<1024, 0>), grid, dim3(1024), 0, s, a);
    }
    int rc = launch_status("mi_cache_evict (select)");
    if (rc != MI_OK) return rc;
    switch (row_bytes / 16) {
      case 1: rc = launch_move<1>(a, layers, s); break;
      case 2: rc = launch_move<2>(a, layers, s); break;
      case 4: rc = launch_move<4>(a, layers, s); break;
      case 8: rc = launch_move<8>(a, layers, s); break;
      case 16: rc = launch_move<16>(a, layers, s); break;
      case 32: rc = launch_move<32>(a, layers, s); break;
      default: rc = launch_move<64>(a, layers, s); break;
    }
    if (rc != MI_OK) return rc;
  }
  return MI_OK;
}
