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
// 11.3 us, 8.8 in the workgroups (table entry, page, product, one after the other), the rest in the merge's launch.
// Requests longer than the window see about as much as each other, so the split is one for all (window_splits), where the
// 8-bit decode, which has no bound on a batch's spread of lengths without a window, cuts ranges. Below the window the longest
// sets the time: 24 requests of 100 to 8191 tokens over 8 KV heads, window 8192, 97 us, of their mean length each 85.
#include <algorithm>

#include "common.hpp"
#include "paged_attend.hpp"

namespace starkv {

namespace {

template <int DT>
__global__ __launch_bounds__(64) void window_merge_kernel(const AttendParams p) {
    attend_merge_head<DT>(p, blockIdx.y, blockIdx.x);
}

// The same by WAVES waves, a run of splits each, whose loads all go out at once.
constexpr int WAVES = 8;

// Requests of so many splits are joined by WAVES waves: a request of 8000 tokens over 8 KV heads through a window of 1024 (9
// splits) 8.4 -> 8.2 us, of 4096 (33) 12.9 -> 11.5, of 8000 (63) 15.9 -> 13.2; 500 tokens (4) 7.9 by one wave and 8.1 by 8.
constexpr int JOIN = 8;

template <int DT>
__global__ __launch_bounds__(64 * WAVES) void window_join_kernel(const AttendParams p) {
    static_assert(AT_MAX_SPLITS <= 16 * WAVES, "16 splits a wave");
    __shared__ float2 s_ref[WAVES], s_sum[WAVES][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), b = blockIdx.y, hq = blockIdx.x;
    const int run = (p.splits + WAVES - 1) / WAVES, first = wave * run, count = min(run, p.splits - first);
    const float* pp = p.part + (((int64_t)b * p.Hkv * p.G + hq) * p.splits + first) * AT_PART;
    float m = -INFINITY, f = 0.f;
    if (lane < count) {
        m = pp[lane * AT_PART];
        f = pp[lane * AT_PART + 1];
    }
    float2 a = make_float2(0.f, 0.f), v[16];
#pragma unroll
    for (int u = 0; u < 16; ++u)
        if (u < count) v[u] = *(const float2*)(pp + u * AT_PART + 4 + 2 * lane);
    const float M1 = wave_max(m), e = m == -INFINITY ? 1.f : exp2f(m - M1), l1 = wave_sum(f * e);
#pragma unroll
    for (int u = 0; u < 16; ++u) {
        if (u < count) {
            const float fs = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(e), u));
            a.x = fmaf(v[u].x, fs, a.x);
            a.y = fmaf(v[u].y, fs, a.y);
        }
    }
    if (lane == 0) s_ref[wave] = make_float2(M1, l1);
    s_sum[wave][lane] = a;
    __syncthreads();
    if (wave > 0) return;
    float M = -INFINITY, lt = 0.f;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) M = fmaxf(M, s_ref[k].x);
    a = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < WAVES; ++k) {
        const float fs = s_ref[k].x == -INFINITY ? 1.f : exp2f(s_ref[k].x - M);
        const float2 x = s_sum[k][lane];
        lt = fmaf(s_ref[k].y, fs, lt);
        a.x = fmaf(x.x, fs, a.x);
        a.y = fmaf(x.y, fs, a.y);
    }
    const int64_t o = b * p.o_s0 + hq * p.o_s1 + 2 * lane;
    store_f(p.out, o, DT, M == -INFINITY ? 0.f : a.x / lt);
    store_f(p.out, o + 1, DT, M == -INFINITY ? 0.f : a.y / lt);
}

// A call's requests are taken to see about the same number of pages: one round of the device, as the decode over selected blocks.
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
    const bool join = p.splits >= JOIN, bf = dtype == STARKV_BF16;
    const void* fn = join ? bf ? (const void*)&window_join_kernel<STARKV_BF16> : (const void*)&window_join_kernel<STARKV_F16>
                          : bf ? (const void*)&window_merge_kernel<STARKV_BF16> : (const void*)&window_merge_kernel<STARKV_F16>;
    void* args[] = {(void*)&p};
    SKV_HIP(hipLaunchKernel(fn, dim3(num_heads, n), dim3(join ? 64 * WAVES : 64), args, 0, (hipStream_t)stream));
    return STARKV_OK;
}

}  // extern "C"
