// Decode through a window: one token's attention over the last `window` cached tokens of its request and the
// first `sinks` ones, in an uncompressed paged cache.
//
// out_h = sum_s p_s v_s / sum_s p_s, p_s = 2^(scale log2(e) q_h . k_s - m), over the places s of a request of L
// tokens with s >= L - window or s < sinks. attend_kernel<.., AT_WINDOW, ..> (paged_attend.hpp) takes the pages that
// hold such places (window_pages.hpp) and no others: blocks between are not read, nor their table entries. Its arithmetic
// and rounding are those of the other decodes over 16-bit caches.
//
// Memory bounds a batch: 512 bytes a token seen and KV head. 32 requests over 32 KV heads with a window of 1024 and 16 first
// tokens (533 MB) 98 us, 5.4 TB/s. One request of 65536 tokens, window 4096, over 8 KV heads (17 MB, 3.4 us of memory) takes
// 12.5 us, 8.8 in the workgroups (table entry, page, product, one after the other) and 4.1 in the merge's launch.
// Requests see about as much as each other whatever their lengths are, so the split is one for all (window_splits), where the
// 8-bit decode, which has no bound on a batch's spread of lengths without a window, cuts ranges.
#include <algorithm>

#include "common.hpp"
#include "paged_attend.hpp"

namespace starkv {

namespace {

template <int DT>
__global__ __launch_bounds__(64) void window_merge_kernel(const AttendParams p) {
    attend_merge_head<DT>(p, blockIdx.y, blockIdx.x);
}

// A call's requests see about the same number of pages: one round of the device, as the decode over selected blocks.
int window_splits(int n, int num_kv_heads, int span, int window, int sinks) {
    return attend_splits((int64_t)n * num_kv_heads, seen_pages_most(span, window, sinks), 2, 8);
}

}  // namespace

}  // namespace starkv

using namespace starkv;

extern "C" {

size_t starkv_window_decode_workspace_bytes(int n, int num_heads, int num_kv_heads, int max_seq_len, int window, int sinks) {
    if (n < 1 || num_kv_heads < 1 || num_heads < num_kv_heads || max_seq_len < 1 || window < 1 || sinks < 0) return 256;
    const int splits = window_splits(n, num_kv_heads, max_seq_len, window, sinks);
    return splits == 1 ? 256 : (size_t)n * num_heads * splits * AT_PART * 4;
}

int starkv_window_decode(void* stream, const void* query, int64_t q_s0, int64_t q_s1, const void* k_cache,
                         const void* v_cache, int64_t c_s0, int64_t c_s1, int64_t c_s2, int dtype, int block_size,
                         int64_t num_blocks, const int32_t* block_table, int64_t bt_s0, int64_t bt_s1, int bt_width,
                         const int32_t* seq_lens, int n, int num_heads, int num_kv_heads, int max_seq_len, int window,
                         int sinks, float scale, void* out, int64_t o_s0, int64_t o_s1, void* workspace,
                         size_t workspace_bytes) {
    clear_error();
    SKV_CHECK(n >= 0 && n <= 65535 && max_seq_len >= 1, "window_decode: n=%d (up to 65535) max_seq_len=%d", n, max_seq_len);
    SKV_CHECK(window >= 1 && sinks >= 0, "window_decode: window=%d sinks=%d", window, sinks);
    if (n == 0) return STARKV_OK;
    AttendParams p = {};
    const int rc = attend_setup(p, "window_decode", query, q_s0, q_s1, k_cache, v_cache, c_s0, c_s1, c_s2, dtype,
                                block_size, num_blocks, block_table, bt_s0, bt_s1, bt_width, seq_lens, n, num_heads,
                                num_kv_heads, scale, out, o_s0, o_s1, workspace);
    if (rc != STARKV_OK) return rc;
    const size_t need = starkv_window_decode_workspace_bytes(n, num_heads, num_kv_heads, max_seq_len, window, sinks);
    SKV_CHECK(workspace_bytes >= need, "window_decode: workspace %zu bytes < %zu", workspace_bytes, need);
    p.span = std::min(p.span, max_seq_len);
    p.window = window; p.sinks = sinks;
    p.splits = window_splits(n, num_kv_heads, max_seq_len, window, sinks);
    p.part = (float*)workspace;
    const int err = attend_launch<AT_WINDOW>(stream, dtype, p);
    if (err != STARKV_OK || p.splits == 1) return err;
    if (dtype == STARKV_BF16)
        hipLaunchKernelGGL(window_merge_kernel<STARKV_BF16>, dim3(num_heads, n), dim3(64), 0, (hipStream_t)stream, p);
    else
        hipLaunchKernelGGL(window_merge_kernel<STARKV_F16>, dim3(num_heads, n), dim3(64), 0, (hipStream_t)stream, p);
    SKV_HIP(hipGetLastError());
    return STARKV_OK;
}

}  // extern "C"
