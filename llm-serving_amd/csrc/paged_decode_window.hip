// The paged decode under a sliding window with sinks (kernels: paged_decode.h): row b sees its first `sinks`
// tokens and its last `window` ones. Same bytes per visible token as the plain form and nothing for the others; the splits
// are planned over the visible tokens, so a batch of rows far longer than the window is cut evenly. Bound by the reads:
// 32 rows of 128 to 16384 tokens under 2048 + 4, H 16 / H_kv 8 / D 128 bf16, 254 MB a layer: 41 us of splits + 4.7 of merges,
// 5.5 TB/s; 16 rows of up to 40000 under 4096 + 64, H 8 / H_kv 2 / D 256 fp16, 132 MB: 27 + 4.6; one row of 6000 under
// 1024 + 4 7.0 + 3.8, its round trips (a call is 10 us on the host, 8.6 of them the two launches).
// As the plain form over as many tokens, in a graph: 32 rows of 2052 seen 47.9 us (plain 47.2 to 48.9), 16 of 4160 at head_dim 256
// 31.4 (33 to 36), one of 1028 10.2 (9.7), 8 of 260 9.1 (8.9).
#include "paged_decode.h"

namespace miattn {
namespace {

int windowed(Windowed& w, int window, int sinks) {
  if (window < 1 || sinks < 0) {
    return fail(MI_ERR_INVALID, "mi_paged_decode_window: window must be >= 1 and sinks >= 0, got %d and %d", window, sinks);
  }
  w.most = int(std::min<int64_t>(int64_t(window) + sinks, INT32_MAX));
  w.sinks = sinks;
  return MI_OK;
}

// Tables that no row outgrows the window in: the plain form's result, which has the one-launch kernel for short
// rows (1 row of 8 tokens 10.8 -> 7.2 us a call on the host).
bool hides_nothing(const Windowed& w, int block_size, int max_blocks) {
  return int64_t(max_blocks) * block_size <= w.most;
}

}  // namespace
}  // namespace miattn

extern "C" int mi_paged_decode_window(const void* q, const void* k_cache, const void* v_cache,
                                      const int32_t* block_table, const int32_t* seqlen, void* out, int B, int H,
                                      int H_kv, int D, int block_size, int max_blocks, const int64_t* strides,
                                      float scale, int dtype, int window, int sinks, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  using namespace miattn;
  Windowed w{};
  const int rc = windowed(w, window, sinks);
  if (rc != MI_OK) return rc;
  if (hides_nothing(w, block_size, max_blocks)) {
    return mi_paged_decode(q, k_cache, v_cache, block_table, seqlen, out, B, H, H_kv, D, block_size, max_blocks, strides,
                           scale, dtype, workspace, workspace_bytes, stream);
  }
  return paged_decode_entry(q, k_cache, v_cache, block_table, seqlen, out, B, H, H_kv, D, block_size, max_blocks,
                            strides, scale, dtype, workspace, workspace_bytes, stream, w);
}

extern "C" int mi_paged_decode_fused_window(const void* qkv, int64_t row_stride, int qkv_parts, const void* q_norm_w,
                                            const void* k_norm_w, const void* cos_tab, const void* sin_tab,
                                            int64_t n_pos, int rotary_dim, const int64_t* pos, const void* slot_ids,
                                            int slot_bits, void* k_cache, void* v_cache, const int32_t* block_table,
                                            const int32_t* seqlen, void* out, int B, int H, int H_kv, int D,
                                            int block_size, int max_blocks, int64_t n_slots, const int64_t* strides,
                                            float scale, float eps, int norm_mode, int dtype, int window, int sinks,
                                            void* workspace, size_t workspace_bytes, int32_t* error_word,
                                            void* stream) {
  using namespace miattn;
  Windowed w{};
  int rc = windowed(w, window, sinks);
  if (rc != MI_OK) return rc;
  FusedArgs fa{};
  rc = fused_args(fa, qkv, row_stride, qkv_parts, q_norm_w, k_norm_w, cos_tab, sin_tab, n_pos, rotary_dim, pos,
                  slot_ids, slot_bits, B, H, H_kv, D, n_slots, eps, norm_mode, dtype, error_word);
  if (rc != MI_OK) return rc;
  return paged_decode_entry(nullptr, k_cache, v_cache, block_table, seqlen, out, B, H, H_kv, D, block_size, max_blocks,
                            strides, scale, dtype, workspace, workspace_bytes, stream, w, &fa);
}
