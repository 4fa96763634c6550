// Decode over a part of a long uncompressed cache: a cheap score picks the blocks a token attends to.
//
// key_bounds_kernel keeps, per cache block and KV head, the least and the largest key elementwise:
// lo[d] = min_t k_t[d], hi[d] = max_t k_t[d] over the block's tokens. Then for every token t of the
// block q . k_t <= sum_d max(q_d lo_d, q_d hi_d), and summed over the G query heads of a KV head, which
// share the blocks they read,
//     score = sum_g sum_d max(q_gd lo_d, q_gd hi_d) = sum_d (sum_g max(q_gd, 0)) hi_d + (sum_g min(q_gd, 0)) lo_d:
// one product of 256 terms a block, whatever G. score_kernel forms it, select_kernel keeps the blocks of
// the largest scores (topk_select.hpp) between the first `sink` and the last `recent` ones, and
// attend_kernel<.., AT_SPARSE, ..> (paged_attend.hpp) attends to their tokens.
//
// Scores are summed in 64 bits and rounded once to fp32: a choice must not change with the order of a
// sum (a block that one order puts first and another second changes the output by its whole weight).
// The vector unit has the rate: the same kernel in 32 bits takes the same time, which is memory's and its
// ramp (32 requests of up to 2048 blocks over 8 KV heads, 160 MB: 36 us).
#include <algorithm>

#include "common.hpp"
#include "paged_attend.hpp"
#include "topk_select.hpp"

namespace starkv {

namespace {

template <int DT>
__device__ __forceinline__ void values8(const uint4& w, float* o) {
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (DT == STARKV_BF16) {
            o[2 * k] = __uint_as_float(ws[k] << 16);
            o[2 * k + 1] = __uint_as_float(ws[k] & 0xffff0000u);
        } else {
            o[2 * k] = (float)__builtin_bit_cast(_Float16, (uint16_t)(ws[k] & 0xffffu));
            o[2 * k + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(ws[k] >> 16));
        }
    }
}

// ---------------------------------------------------------------------------
// Bounds of the blocks that hold a request's last max_new tokens
// ---------------------------------------------------------------------------
struct BoundsParams {
    const uint16_t* kc; int64_t c_s0, c_s1, c_s2;  // elements
    uint16_t* bounds; int64_t b_s0, b_s1, b_s2;    // [num_blocks][Hkv][2][128]
    int64_t num_blocks;
    const int32_t* bt; int64_t bt_s0, bt_s1;
    const int32_t* seq_lens; int span;
    int Hkv, block_size, max_new, per;             // per: blocks a request at most
};

// A lane takes 8 dimensions of one head over the block's tokens: 16 lanes a head, the heads of a token
// side by side. Nothing crosses lanes; keys are read once, a token's heads as one run of memory: two
// prompts of 16384 tokens over 32 heads (285 MB) 55 us, 5.1 TB/s; one block of 64 requests 4, three
// dependent reads' latency.
template <int DT>
__global__ __launch_bounds__(256) void key_bounds_kernel(const BoundsParams p) {
    const int b = blockIdx.y, width = 16 * p.Hkv;
    const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int L = min(max(p.seq_lens[b], 0), p.span);
    const int j = (int)(item / width) + max(L - p.max_new, 0) / p.block_size;  // the block of the request
    const int at = (int)(item % width), h = at >> 4, d = 8 * (at & 15);
    const int64_t t0 = (int64_t)j * p.block_size;
    if (item / width >= p.per || t0 >= L) return;
    const int blk = p.bt[b * p.bt_s0 + j * p.bt_s1];
    if (blk < 0 || blk >= p.num_blocks) return;
    const int tokens = min(p.block_size, (int)(L - t0));
    const uint16_t* k = p.kc + blk * p.c_s0 + h * p.c_s2 + d;
    float lo[8], hi[8];
    values8<DT>(*(const uint4*)k, lo);
#pragma unroll
    for (int e = 0; e < 8; ++e) hi[e] = lo[e];
#pragma unroll 4
    for (int t = 1; t < tokens; ++t) {
        float f[8];
        values8<DT>(*(const uint4*)(k + t * p.c_s1), f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {  // NaN stays: its block's score is NaN, which counts as the largest
            lo[e] = __builtin_elementwise_minimum(lo[e], f[e]);
            hi[e] = __builtin_elementwise_maximum(hi[e], f[e]);
        }
    }
    uint32_t w[2][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float x, y;  // values of DT already
        w[0][e] = attend_pack<DT>(lo[2 * e], lo[2 * e + 1], x, y);
        w[1][e] = attend_pack<DT>(hi[2 * e], hi[2 * e + 1], x, y);
    }
    uint16_t* o = p.bounds + blk * p.b_s0 + h * p.b_s1 + d;
    *(uint4*)o = make_uint4(w[0][0], w[0][1], w[0][2], w[0][3]);
    *(uint4*)(o + p.b_s2) = make_uint4(w[1][0], w[1][1], w[1][2], w[1][3]);
}

// ---------------------------------------------------------------------------
// Scores and choice
// ---------------------------------------------------------------------------
struct SelectParams {
    const uint16_t* q; int64_t q_s0, q_s1;
    const uint16_t* bounds; int64_t b_s0, b_s1, b_s2; int64_t num_blocks;
    const int32_t* bt; int64_t bt_s0, bt_s1;
    const int32_t* seq_lens; int span;
    int Hkv, G, bs_shift, keep, sink, recent;  // block_size = 16 << bs_shift
    int cap;                                   // blocks a request at most
    float* score;                              // [n][Hkv][cap]
    int32_t* sel;                              // [n][Hkv][keep]
};

__device__ __forceinline__ int select_blocks_of(const SelectParams& p, int b) {
    const int L = min(max(p.seq_lens[b], 0), p.span);
    return (int)(((int64_t)L + (16 << p.bs_shift) - 1) >> (p.bs_shift + 4));
}

constexpr int SC_U = 4;  // blocks a 16-lane row has in flight

template <int CTL>
__device__ __forceinline__ double add_dpp(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTL, 0xF, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTL, 0xF, 0xF, true);
    return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// 16 lanes a (block, head), 8 dimensions of both bounds each. A workgroup of 16 rows takes a request's
// blocks for `heads` KV heads at once (a power of two up to 16), as they lie in memory: 4 heads of a
// block are 2 KB that a wave reads as one run (one head a workgroup read 512 bytes here and there). A row
// takes SC_U consecutive blocks at a time, with its head's query part in registers.
template <int DT>
__global__ __launch_bounds__(256) void score_kernel(const SelectParams p, int heads) {
    const int b = blockIdx.z, row = threadIdx.x >> 4, d = 8 * (threadIdx.x & 15);
    const int nb = select_blocks_of(p, b), last = nb - p.recent;  // blocks behind `last` are read unscored
    const int h = blockIdx.y * heads + (row & (heads - 1)), step = 16 / heads * SC_U;
    int j0 = blockIdx.x * step + row / heads * SC_U;
    if (nb <= p.keep || h >= p.Hkv) return;
    double up[8], down[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) up[e] = down[e] = 0.0;
    for (int g0 = 0; g0 < p.G; g0 += 4) {  // four rows on their way at a time
        uint4 w[4];
#pragma unroll
        for (int g = 0; g < 4; ++g)
            w[g] = *(const uint4*)(p.q + b * p.q_s0 + (int64_t)(h * p.G + min(g0 + g, p.G - 1)) * p.q_s1 + d);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            if (g0 + g >= p.G) continue;
            float f[8];
            values8<DT>(w[g], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                up[e] += (double)__builtin_elementwise_maximum(f[e], 0.f);
                down[e] += (double)__builtin_elementwise_minimum(f[e], 0.f);
            }
        }
    }
    float* score = p.score + ((int64_t)b * p.Hkv + h) * p.cap;
    for (; j0 < last; j0 += step * gridDim.x) {
        uint4 lo[SC_U], hi[SC_U];
        int blk[SC_U];
#pragma unroll
        for (int u = 0; u < SC_U; ++u) {
            blk[u] = p.bt[b * p.bt_s0 + min(j0 + u, nb - 1) * p.bt_s1];
            if (blk[u] < 0 || blk[u] >= p.num_blocks) blk[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < SC_U; ++u) {
            const uint16_t* x = p.bounds + max(blk[u], 0) * p.b_s0 + h * p.b_s1 + d;
            lo[u] = *(const uint4*)x;
            hi[u] = *(const uint4*)(x + p.b_s2);
        }
#pragma unroll
        for (int u = 0; u < SC_U; ++u) {
            float a[8], c[8];
            values8<DT>(lo[u], a);
            values8<DT>(hi[u], c);
            double s = 0.0;
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fma(up[e], (double)c[e], fma(down[e], (double)a[e], s));
            s = add_dpp<0xB1>(s);
            s = add_dpp<0x4E>(s);
            s = add_dpp<0x141>(s);
            s = add_dpp<0x140>(s);
            if (d == 0 && j0 + u < last) score[j0 + u] = blk[u] < 0 ? -INFINITY : (float)s;
        }
    }
}

template <int RUN>
__global__ __launch_bounds__(TK_THR) void select_kernel(const SelectParams p) {
    __shared__ TopkShared sh;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const int nb = select_blocks_of(p, b);
    int32_t* sel = p.sel + ((int64_t)b * p.Hkv + h) * p.keep;
    if (nb <= p.keep) {
        for (int i = tid; i < p.keep; i += TK_THR) sel[i] = i < nb ? i : -1;
        return;
    }
    const int middle = nb - p.sink - p.recent, k = p.keep - p.sink - p.recent;
    for (int i = tid; i < p.sink + p.recent; i += TK_THR)
        sel[i < p.sink ? i : k + i] = i < p.sink ? i : middle + i;
    if (k == 0) return;
    const float* score = p.score + ((int64_t)b * p.Hkv + h) * p.cap + p.sink;
    topk_ascending<RUN>(sh, middle, k, [&](int i) { return score[i]; },
                        [&](int pos, int i, float) { sel[p.sink + pos] = p.sink + i; });
}

template <int DT>
__global__ __launch_bounds__(64) void attend_merge_kernel(const AttendParams p) {
    attend_merge_head<DT>(p, blockIdx.y, blockIdx.x);
}

}  // namespace

}  // namespace starkv

using namespace starkv;

extern "C" {

int starkv_key_bounds(void* stream, const void* k_cache, int64_t c_s0, int64_t c_s1, int64_t c_s2, int dtype,
                      int block_size, int64_t num_blocks, void* bounds, int64_t b_s0, int64_t b_s1, int64_t b_s2,
                      const int32_t* block_table, int64_t bt_s0, int64_t bt_s1, int bt_width, const int32_t* seq_lens,
                      int n, int num_kv_heads, int max_new) {
    clear_error();
    SKV_CHECK(n >= 0 && n <= 65535 && num_kv_heads >= 1 && max_new >= 0, "key_bounds: n=%d (up to 65535) num_kv_heads=%d max_new=%d",
              n, num_kv_heads, max_new);
    if (n == 0 || max_new == 0) return STARKV_OK;
    SKV_CHECK(k_cache && bounds && block_table && seq_lens, "key_bounds: null pointer");
    SKV_CHECK(dtype == STARKV_BF16 || dtype == STARKV_F16, "key_bounds: bf16 or fp16");
    SKV_CHECK(block_shift(block_size) >= 0, "key_bounds: block_size must be 16 times a power of two");
    SKV_CHECK(num_blocks >= 1 && num_blocks <= 0x7fffffff && bt_width >= 1, "key_bounds: empty cache or block table");
    SKV_CHECK(((uintptr_t)k_cache | (uintptr_t)bounds) % 16 == 0 && (c_s0 | c_s1 | c_s2 | b_s0 | b_s1 | b_s2) % 8 == 0,
              "key_bounds: rows must be 16-byte aligned");
    BoundsParams p = {};
    p.kc = (const uint16_t*)k_cache; p.c_s0 = c_s0; p.c_s1 = c_s1; p.c_s2 = c_s2;
    p.bounds = (uint16_t*)bounds; p.b_s0 = b_s0; p.b_s1 = b_s1; p.b_s2 = b_s2;
    p.num_blocks = num_blocks;
    p.bt = block_table; p.bt_s0 = bt_s0; p.bt_s1 = bt_s1;
    p.seq_lens = seq_lens; p.span = (int)std::min<int64_t>((int64_t)bt_width * block_size, 0x7ffffff0);
    p.Hkv = num_kv_heads; p.block_size = block_size;
    p.max_new = std::min(max_new, p.span);
    p.per = std::min((p.max_new - 1) / block_size + 2, bt_width);  // the first of them may begin before the new tokens
    if (p.max_new == 1) p.per = 1;
    const dim3 grid((unsigned)(((int64_t)p.per * num_kv_heads * 16 + 255) / 256), n);
    if (dtype == STARKV_BF16)
        hipLaunchKernelGGL(key_bounds_kernel<STARKV_BF16>, grid, dim3(256), 0, (hipStream_t)stream, p);
    else
        hipLaunchKernelGGL(key_bounds_kernel<STARKV_F16>, grid, dim3(256), 0, (hipStream_t)stream, p);
    SKV_HIP(hipGetLastError());
    return STARKV_OK;
}

static int select_cap(int bt_width, int block_size, int max_seq_len) {
    return (int)std::min<int64_t>(bt_width, ((int64_t)max_seq_len + block_size - 1) / block_size);
}

size_t starkv_select_blocks_workspace_bytes(int n, int num_kv_heads, int bt_width, int block_size, int max_seq_len) {
    if (n < 1 || num_kv_heads < 1 || bt_width < 1 || block_size < 1 || max_seq_len < 1) return 256;
    return std::max<size_t>(256, (size_t)n * num_kv_heads * select_cap(bt_width, block_size, max_seq_len) * 4);
}

int starkv_select_blocks(void* stream, const void* query, int64_t q_s0, int64_t q_s1, const void* bounds, int64_t b_s0,
                         int64_t b_s1, int64_t b_s2, int dtype, int block_size, int64_t num_blocks,
                         const int32_t* block_table, int64_t bt_s0, int64_t bt_s1, int bt_width,
                         const int32_t* seq_lens, int n, int num_heads, int num_kv_heads, int max_seq_len, int keep,
                         int sink, int recent, int32_t* selected, void* workspace, size_t workspace_bytes) {
    clear_error();
    SKV_CHECK(n >= 0 && n <= 65535 && max_seq_len >= 1, "select_blocks: n=%d (up to 65535) max_seq_len=%d", n, max_seq_len);
    SKV_CHECK(sink >= 0 && recent >= 0 && keep >= 1 && sink <= keep && recent <= keep - sink,
              "select_blocks: keep %d blocks, %d first and %d last ones among them", keep, sink, recent);
    if (n == 0) return STARKV_OK;
    SKV_CHECK(query && bounds && block_table && seq_lens && selected && workspace, "select_blocks: null pointer");
    SKV_CHECK(num_kv_heads >= 1 && num_kv_heads <= 65535 && num_heads >= num_kv_heads && num_heads % num_kv_heads == 0,
              "select_blocks: %d query heads over %d KV heads", num_heads, num_kv_heads);
    SKV_CHECK(dtype == STARKV_BF16 || dtype == STARKV_F16, "select_blocks: bf16 or fp16");
    SKV_CHECK(block_shift(block_size) >= 0, "select_blocks: block_size must be 16 times a power of two");
    SKV_CHECK(num_blocks >= 1 && num_blocks <= 0x7fffffff && bt_width >= 1, "select_blocks: empty cache or block table");
    SKV_CHECK(((uintptr_t)query | (uintptr_t)bounds) % 16 == 0 && (q_s0 | q_s1 | b_s0 | b_s1 | b_s2) % 8 == 0,
              "select_blocks: rows must be 16-byte aligned");
    const size_t need = starkv_select_blocks_workspace_bytes(n, num_kv_heads, bt_width, block_size, max_seq_len);
    SKV_CHECK(workspace_bytes >= need, "select_blocks: workspace %zu bytes < %zu", workspace_bytes, need);
    SelectParams p = {};
    p.q = (const uint16_t*)query; p.q_s0 = q_s0; p.q_s1 = q_s1;
    p.bounds = (const uint16_t*)bounds; p.b_s0 = b_s0; p.b_s1 = b_s1; p.b_s2 = b_s2; p.num_blocks = num_blocks;
    p.bt = block_table; p.bt_s0 = bt_s0; p.bt_s1 = bt_s1;
    p.cap = select_cap(bt_width, block_size, max_seq_len);
    p.seq_lens = seq_lens; p.span = (int)std::min<int64_t>(max_seq_len, (int64_t)bt_width * block_size);
    p.Hkv = num_kv_heads; p.G = num_heads / num_kv_heads; p.bs_shift = block_shift(block_size);
    p.keep = keep; p.sink = sink; p.recent = recent;
    p.score = (float*)workspace; p.sel = selected;
    if (p.cap > keep && keep > sink + recent) {
        int heads = 1;
        while (heads < num_kv_heads && heads < 16) heads *= 2;
        const int64_t groups = (num_kv_heads + heads - 1) / heads, step = 16 / heads * SC_U, most = (p.cap + step - 1) / step;
        const int64_t want = 4096 / (groups * n);
        const dim3 grid((unsigned)std::min<int64_t>(most, std::max<int64_t>(1, want)), (unsigned)groups, n);
        if (dtype == STARKV_BF16)
            hipLaunchKernelGGL(score_kernel<STARKV_BF16>, grid, dim3(256), 0, (hipStream_t)stream, p, heads);
        else
            hipLaunchKernelGGL(score_kernel<STARKV_F16>, grid, dim3(256), 0, (hipStream_t)stream, p, heads);
        SKV_HIP(hipGetLastError());
    }
    const int run = topk_run(p.cap);
    const void* fn = run == TK_FEW ? (const void*)&select_kernel<TK_FEW>
                     : run == TK_MANY ? (const void*)&select_kernel<TK_MANY>
                     : run         ? (const void*)&select_kernel<TK_MOST>
                                   : (const void*)&select_kernel<0>;
    void* args[] = {(void*)&p};
    SKV_HIP(hipLaunchKernel(fn, dim3(num_kv_heads, n), dim3(TK_THR), args, 0, (hipStream_t)stream));
    return STARKV_OK;
}

// Requests of one call have about the same work, so one round of the device is even: 64 requests of 4096 selected
// tokens over 8 KV heads 189 us with workgroups for 2 a CU, 194 for 4, 205 for 8.
static int sparse_splits(int n, int num_kv_heads, int pages) {
    return attend_splits((int64_t)n * num_kv_heads, pages, 2, 8);
}

size_t starkv_sparse_decode_workspace_bytes(int n, int num_heads, int num_kv_heads, int block_size, int keep) {
    if (n < 1 || num_kv_heads < 1 || num_heads < num_kv_heads || block_size < 16 || keep < 1) return 256;
    const int64_t pages = (int64_t)keep * (block_size / 16);
    const int splits = sparse_splits(n, num_kv_heads, (int)std::min<int64_t>(pages, 1 << 27));
    return splits == 1 ? 256 : (size_t)n * num_heads * splits * AT_PART * 4;
}

int starkv_sparse_decode(void* stream, const void* query, int64_t q_s0, int64_t q_s1, const void* k_cache,
                         const void* v_cache, int64_t c_s0, int64_t c_s1, int64_t c_s2, int dtype, int block_size,
                         int64_t num_blocks, const int32_t* block_table, int64_t bt_s0, int64_t bt_s1, int bt_width,
                         const int32_t* seq_lens, int n, int num_heads, int num_kv_heads, const int32_t* selected,
                         int64_t sel_s0, int64_t sel_s1, int keep, float scale, void* out, int64_t o_s0, int64_t o_s1,
                         void* workspace, size_t workspace_bytes) {
    clear_error();
    SKV_CHECK(n >= 0 && n <= 65535 && keep >= 1, "sparse_decode: n=%d (up to 65535) keep=%d", n, keep);
    if (n == 0) return STARKV_OK;
    AttendParams p = {};
    const int rc = attend_setup(p, "sparse_decode", query, q_s0, q_s1, k_cache, v_cache, c_s0, c_s1, c_s2, dtype,
                                block_size, num_blocks, block_table, bt_s0, bt_s1, bt_width, seq_lens, n, num_heads,
                                num_kv_heads, scale, out, o_s0, o_s1, workspace);
    if (rc != STARKV_OK) return rc;
    SKV_CHECK(selected, "sparse_decode: null pointer");
    SKV_CHECK((int64_t)keep * (block_size / 16) <= 1 << 27, "sparse_decode: keep %d blocks of %d", keep, block_size);
    const size_t need = starkv_sparse_decode_workspace_bytes(n, num_heads, num_kv_heads, block_size, keep);
    SKV_CHECK(workspace_bytes >= need, "sparse_decode: workspace %zu bytes < %zu", workspace_bytes, need);
    const int pages = keep << p.bs_shift;
    p.sel = selected; p.sel_s0 = sel_s0; p.sel_s1 = sel_s1; p.keep = keep;
    p.splits = sparse_splits(n, num_kv_heads, pages);
    p.pps = (pages + p.splits - 1) / p.splits;
    p.part = (float*)workspace;
    const int err = attend_launch<AT_SPARSE>(stream, dtype, p);
    if (err != STARKV_OK || p.splits == 1) return err;
    if (dtype == STARKV_BF16)
        hipLaunchKernelGGL(attend_merge_kernel<STARKV_BF16>, dim3(num_heads, n), dim3(64), 0, (hipStream_t)stream, p);
    else
        hipLaunchKernelGGL(attend_merge_kernel<STARKV_F16>, dim3(num_heads, n), dim3(64), 0, (hipStream_t)stream, p);
    SKV_HIP(hipGetLastError());
    return STARKV_OK;
}

}  // extern "C"
