// Eviction by accumulated attention weight, for uncompressed caches.
//
// starkv_weighted_decode is a paged decode over a request's whole cache that also sums up what each
// cached token weighs: weights[b, h, t] += sum_g softmax_g(t) over the G query heads of KV head h (the
// newest token's entry starts there: it is set). attend_kernel<.., AT_SCORES, ..> (paged_attend.hpp) leaves every
// score behind (4 bytes a query head and token beside 512 bytes of keys and values), weigh_kernel turns
// them into weights once the splits' references and sums are known, and joins the splits' outputs. A
// token's entry belongs to one thread, which sums the heads in order: no atomics, the same bits every run.
//
// starkv_evict cuts each request and KV head to `keep` tokens: the first `sink`, the last `recent` and
// those of the largest weights between (topk_select.hpp). The order of tokens stays, so `recent` means the
// same at the next eviction, and kept[j] >= j ascends: compact_kernel moves row kept[j] to row j in place,
// reading rows of a chunk before any of them is written; a later chunk's sources lie behind every
// earlier chunk's targets (a handful of heads moves all rows at once instead, through the workspace:
// stage_kernel). Columns are independent of each other, so K and V, and for few requests their
// halves of 128 bytes, go to workgroups of their own. 16 requests of 8 KV heads cut from 4097 to 8192 tokens
// to 2048: the choice 11 us (one CU a head), the move 55 (268 MB, 4.9 TB/s; a large copy's rate is 5.0).
#include <algorithm>

#include "common.hpp"
#include "paged_attend.hpp"
#include "topk_select.hpp"

namespace starkv {

namespace {

struct WeighParams {
    AttendParams a;
    float* w; int64_t w_s0, w_s1;  // weights [n][Hkv][>= span], last dimension contiguous
    int chunks;                    // workgroups of WG_TOKENS tokens a (request, KV head)
};

constexpr int WG_TOKENS = 1024;

// blockIdx.x < chunks: weights of WG_TOKENS tokens of a (request, KV head); behind them, where there are
// splits, four query heads' outputs a workgroup.
template <int DT>
__global__ __launch_bounds__(256) void weigh_kernel(const WeighParams wp) {
    const AttendParams& p = wp.a;
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, H = p.Hkv * p.G;
    if ((int)blockIdx.x >= wp.chunks) {
        const int g = 4 * (blockIdx.x - wp.chunks) + (tid >> 6);
        if (g < p.G) attend_merge_head<DT>(p, b, h * p.G + g);
        return;
    }
    const int L = attend_length(p, b), t0 = blockIdx.x * WG_TOKENS;
    if (t0 >= L) return;
    // The tokens' sums so far and the first heads' scores are on their way while the heads' sums are formed.
    constexpr int U = WG_TOKENS / 256, AHEAD = 4;
    const float* lg = p.lg + ((int64_t)b * p.Hkv + h) * p.lg_row;
    float* w = wp.w + b * wp.w_s0 + h * wp.w_s1;
    const float* at[U];
    float old[U], sum[U], ahead[AHEAD][U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int t = min(t0 + 256 * u + tid, L - 1);
        at[u] = lg + (int64_t)(t >> 4) * p.G * 16 + (t & 15);
        old[u] = w[t];
        sum[u] = 0.f;
    }
#pragma unroll
    for (int g = 0; g < AHEAD; ++g)
#pragma unroll
        for (int u = 0; u < U; ++u) ahead[g][u] = at[u][16 * min(g, p.G - 1)];
    // Each head's largest reference and the inverse of its sum of weights above it, 16 lanes a head.
    __shared__ float s_ref[AT_MAX_GROUP], s_inv[AT_MAX_GROUP];
    const int g16 = tid >> 4;
    if (g16 < p.G) {
        const float* pp = p.part + ((int64_t)b * H + h * p.G + g16) * p.splits * AT_PART;
        float m[AT_MAX_SPLITS / 16], l[AT_MAX_SPLITS / 16], M = -INFINITY, all = 0.f;
#pragma unroll
        for (int x = 0; x < AT_MAX_SPLITS / 16; ++x) {
            const int s = (tid & 15) + 16 * x;
            m[x] = s < p.splits ? pp[s * AT_PART] : -INFINITY;
            l[x] = s < p.splits ? pp[s * AT_PART + 1] : 0.f;
            M = fmaxf(M, m[x]);
        }
        M = row16_max(M);
#pragma unroll
        for (int x = 0; x < AT_MAX_SPLITS / 16; ++x) all = fmaf(l[x], m[x] == -INFINITY ? 1.f : exp2f(m[x] - M), all);
        all = row16_sum(all);
        if ((tid & 15) == 0) {
            s_ref[g16] = M == -INFINITY ? 0.f : M;  // no block of the cache: weights of 0
            s_inv[g16] = M == -INFINITY ? 0.f : AT_DOWN<DT> / all;
        }
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < AHEAD; ++g)
        if (g < p.G) {
#pragma unroll
            for (int u = 0; u < U; ++u) sum[u] = fmaf(exp2f(ahead[g][u] - s_ref[g]), s_inv[g], sum[u]);
        }
    for (int g = AHEAD; g < p.G; ++g) {
        float s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) s[u] = at[u][16 * g];
#pragma unroll
        for (int u = 0; u < U; ++u) sum[u] = fmaf(exp2f(s[u] - s_ref[g]), s_inv[g], sum[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int t = t0 + 256 * u + tid;
        if (t < L) w[t] = t == L - 1 ? sum[u] : old[u] + sum[u];
    }
}

struct EvictParams {
    uint16_t* kc; uint16_t* vc; int64_t c_s0, c_s1, c_s2; int block_shift; int64_t num_blocks;
    const int32_t* bt; int64_t bt_s0, bt_s1;
    const int32_t* seq_lens; int span;
    const float* w; int64_t w_s0, w_s1;
    int Hkv, cap, keep, sink, recent;
    int32_t* new_lens; float* new_w;  // [n], [n][Hkv][cap]
    int32_t* kept;                    // [n][Hkv][keep]: the kept tokens, ascending
    uint16_t* aside;                  // stage_kernel: [n][Hkv][keep][2][128]
};

__device__ __forceinline__ int evict_length(const EvictParams& p, int b) { return min(max(p.seq_lens[b], 0), p.span); }

template <int RUN>
__global__ __launch_bounds__(TK_THR) void evict_select_kernel(const EvictParams p) {
    __shared__ TopkShared sh;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const int L = evict_length(p, b), left = min(L, p.keep);
    const float* w = p.w + b * p.w_s0 + h * p.w_s1;
    float* nw = p.new_w + ((int64_t)b * p.Hkv + h) * p.cap;
    if (h == 0 && tid == 0) p.new_lens[b] = left;
    for (int i = left + tid; i < p.cap; i += TK_THR) nw[i] = 0.f;
    if (L <= p.keep) {
        for (int i = tid; i < L; i += TK_THR) nw[i] = w[i];
        return;
    }
    int32_t* kept = p.kept + ((int64_t)b * p.Hkv + h) * p.keep;
    const int middle = L - p.sink - p.recent, k = p.keep - p.sink - p.recent;
    for (int i = tid; i < p.sink + p.recent; i += TK_THR) {
        const int from = i < p.sink ? i : middle + i, to = i < p.sink ? i : k + i;
        kept[to] = from;
        nw[to] = w[from];
    }
    if (k == 0) return;
    w += p.sink;
    topk_ascending<RUN>(sh, middle, k, [&](int i) { return w[i]; },
                         [&](int pos, int i, float x) {
                             kept[p.sink + pos] = p.sink + i;
                             nw[p.sink + pos] = x;
                         });
}

constexpr int CP_THR = 1024, CP_U = 4;

// A round: CP_U rows' slices of a lane, on their way or read.
struct Round {
    uint4 v[CP_U];
    int64_t to[CP_U];  // element offset of the target, -1: stays
};

// 2^lanes lanes a row's slice of 16 << lanes bytes, CP_U slices a lane and chunk. Two chunks are on their way
// at a time: a chunk is written behind a barrier that waits for its own rows only. A chunk's tokens and their
// blocks are read two and one chunk ahead and before the rows that are on their way: reads arrive in their
// order, and one that is waited for behind rows waits for the rows.
__global__ __launch_bounds__(CP_THR) void compact_kernel(const EvictParams p, int lanes) {
    const int h = blockIdx.y, b = blockIdx.z;
    if (evict_length(p, b) <= p.keep) return;
    const int slice = threadIdx.x & ((1 << lanes) - 1), row = threadIdx.x >> lanes, step = CP_THR >> lanes;
    uint16_t* c = (blockIdx.x & 1 ? p.vc : p.kc) + h * p.c_s2 + ((blockIdx.x >> 1) << lanes) * 8 + 8 * slice;
    const int mask = (1 << p.block_shift) - 1, chunk = CP_U * step;
    const int32_t* kept = p.kept + ((int64_t)b * p.Hkv + h) * p.keep;
    const int32_t* bt = p.bt + b * p.bt_s0;
    int t1[CP_U], t2[CP_U], sb[CP_U], db[CP_U];  // tokens of the next chunk and the one after, blocks of the next
    const auto tokens = [&](int j0, int (&t)[CP_U]) {
#pragma unroll
        for (int u = 0; u < CP_U; ++u) t[u] = kept[min(j0 + u * step + row, p.keep - 1)];
    };
    const auto blocks = [&](int j0, const int (&t)[CP_U]) {
#pragma unroll
        for (int u = 0; u < CP_U; ++u) {
            sb[u] = bt[(t[u] >> p.block_shift) * p.bt_s1];
            db[u] = bt[(min(j0 + u * step + row, p.keep - 1) >> p.block_shift) * p.bt_s1];
        }
    };
    // The chunk at j0 sets out; behind it wait the tokens of the third and the blocks of the second after it.
    const auto read = [&](int j0, Round& r) {
        int64_t from[CP_U];
#pragma unroll
        for (int u = 0; u < CP_U; ++u) {
            const int j = j0 + u * step + row;
            const bool moves = j < p.keep && t1[u] != j && sb[u] >= 0 && sb[u] < p.num_blocks && db[u] >= 0 && db[u] < p.num_blocks;
            from[u] = moves ? sb[u] * p.c_s0 + (t1[u] & mask) * p.c_s1 : -1;
            r.to[u] = moves ? db[u] * p.c_s0 + (j & mask) * p.c_s1 : -1;
            t1[u] = t2[u];
        }
        tokens(j0 + 2 * chunk, t2);
        blocks(j0 + chunk, t1);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int u = 0; u < CP_U; ++u) {
            r.v[u] = make_uint4(0, 0, 0, 0);
            if (from[u] >= 0) r.v[u] = *(const uint4*)(c + from[u]);
        }
    };
    const auto write = [&](Round& r) {
#pragma unroll
        for (int u = 0; u < CP_U; ++u) asm volatile("" : "+v"(r.v[u].x), "+v"(r.v[u].y), "+v"(r.v[u].z), "+v"(r.v[u].w));
        lds_barrier();  // every lane has its rows of this chunk
#pragma unroll
        for (int u = 0; u < CP_U; ++u)
            if (r.to[u] >= 0) *(uint4*)(c + r.to[u]) = r.v[u];
    };
    Round x, y;
    tokens(0, t1);
    tokens(chunk, t2);
    blocks(0, t1);
    read(0, x);
    for (int j0 = 0; j0 < p.keep; j0 += 2 * chunk) {
        read(j0 + chunk, y);
        write(x);
        read(j0 + 2 * chunk, x);
        write(y);
    }
}

constexpr int ST_ROWS = 64;  // rows a workgroup, four a lane

// A few long rows of caches: one workgroup a column slice moves a chunk after the other, and a handful of them
// leave the device idle. Here every row moves at once, in two launches: the sources that are targets too (token
// kept[j] < keep) are copied aside, then all rows are written, from there or from behind the kept part.
// 16 lanes a row.
template <bool BACK>
__global__ __launch_bounds__(256) void stage_kernel(const EvictParams p) {
    const int h = blockIdx.y, b = blockIdx.z;
    if (evict_length(p, b) <= p.keep) return;
    const int d = 8 * (threadIdx.x & 15), j0 = blockIdx.x * ST_ROWS + (threadIdx.x >> 4), mask = (1 << p.block_shift) - 1;
    const int64_t unit = (int64_t)b * p.Hkv + h;
    const int32_t* kept = p.kept + unit * p.keep;
    const int32_t* bt = p.bt + b * p.bt_s0;
    uint16_t* aside = p.aside + unit * p.keep * 256 + d;  // [keep][K, V][128]
    uint4 vk[4], vv[4];
    int64_t to[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int j = min(j0 + 16 * u, p.keep - 1), t = kept[j];
        const int sb = bt[(t >> p.block_shift) * p.bt_s1], db = bt[(j >> p.block_shift) * p.bt_s1];
        const bool saved = t < p.keep;
        const bool moves = j0 + 16 * u < p.keep && t != j && sb >= 0 && sb < p.num_blocks && db >= 0 &&
                           db < p.num_blocks && (BACK || saved);
        const int64_t from = sb * p.c_s0 + (t & mask) * p.c_s1 + h * p.c_s2 + d;
        const uint16_t* k = BACK && saved ? aside + (int64_t)j * 256 : p.kc + from;
        const uint16_t* v = BACK && saved ? aside + (int64_t)j * 256 + 128 : p.vc + from;
        to[u] = moves ? BACK ? db * p.c_s0 + (j & mask) * p.c_s1 + h * p.c_s2 + d : (int64_t)j * 256 : -1;
        vk[u] = vv[u] = make_uint4(0, 0, 0, 0);
        if (moves) {
            vk[u] = *(const uint4*)k;
            vv[u] = *(const uint4*)v;
        }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (to[u] >= 0) {
            *(uint4*)((BACK ? p.kc : aside) + to[u]) = vk[u];
            *(uint4*)((BACK ? p.vc : aside + 128) + to[u]) = vv[u];
        }
}

}  // namespace

}  // namespace starkv

using namespace starkv;

extern "C" {

static size_t weighted_logits_bytes(int n, int num_heads, int max_seq_len) {
    return (size_t)n * num_heads * (((size_t)max_seq_len + 15) / 16 * 16) * 4;
}

// Requests of one call differ in length: many workgroups, of which the short requests' end at once. 24 requests of
// 1000 to 8191 tokens over 8 KV heads 141 us with workgroups for 2 a CU, 120 for 4, 110 for 8, 108 for 16.
static int weighted_splits(int n, int num_kv_heads, int max_seq_len) {
    return attend_splits((int64_t)n * num_kv_heads, (int)(((int64_t)max_seq_len + 15) / 16), 16, 16);
}

size_t starkv_weighted_decode_workspace_bytes(int n, int num_heads, int num_kv_heads, int max_seq_len) {
    if (n < 1 || num_kv_heads < 1 || num_heads < num_kv_heads || max_seq_len < 1) return 256;
    return weighted_logits_bytes(n, num_heads, max_seq_len) +
           (size_t)n * num_heads * weighted_splits(n, num_kv_heads, max_seq_len) * AT_PART * 4;
}

int starkv_weighted_decode(void* stream, const void* query, int64_t q_s0, int64_t q_s1, const void* k_cache,
                           const void* v_cache, int64_t c_s0, int64_t c_s1, int64_t c_s2, int dtype, int block_size,
                           int64_t num_blocks, const int32_t* block_table, int64_t bt_s0, int64_t bt_s1, int bt_width,
                           const int32_t* seq_lens, int n, int num_heads, int num_kv_heads, int max_seq_len,
                           float scale, float* weights, int64_t w_s0, int64_t w_s1, int weights_len, void* out,
                           int64_t o_s0, int64_t o_s1, void* workspace, size_t workspace_bytes) {
    clear_error();
    SKV_CHECK(n >= 0 && n <= 65535 && max_seq_len >= 1 && max_seq_len <= 1 << 30,
              "weighted_decode: n=%d (up to 65535) max_seq_len=%d", n, max_seq_len);
    if (n == 0) return STARKV_OK;
    WeighParams wp = {};
    AttendParams& p = wp.a;
    const int rc = attend_setup(p, "weighted_decode", query, q_s0, q_s1, k_cache, v_cache, c_s0, c_s1, c_s2, dtype,
                                block_size, num_blocks, block_table, bt_s0, bt_s1, bt_width, seq_lens, n, num_heads,
                                num_kv_heads, scale, out, o_s0, o_s1, workspace);
    if (rc != STARKV_OK) return rc;
    SKV_CHECK(num_kv_heads <= 65535, "weighted_decode: %d KV heads", num_kv_heads);
    SKV_CHECK(weights && weights_len >= max_seq_len, "weighted_decode: weights of %d tokens for max_seq_len=%d",
              weights_len, max_seq_len);
    const size_t need = starkv_weighted_decode_workspace_bytes(n, num_heads, num_kv_heads, max_seq_len);
    SKV_CHECK(workspace_bytes >= need, "weighted_decode: workspace %zu bytes < %zu", workspace_bytes, need);
    p.span = std::min(p.span, max_seq_len);
    const int pages = (p.span + 15) / 16;
    p.splits = weighted_splits(n, num_kv_heads, max_seq_len);
    p.pps = (pages + p.splits - 1) / p.splits;
    p.lg = (float*)workspace;
    p.lg_row = ((int64_t)max_seq_len + 15) / 16 * 16 * p.G;
    p.part = (float*)((char*)workspace + weighted_logits_bytes(n, num_heads, max_seq_len));
    wp.w = weights; wp.w_s0 = w_s0; wp.w_s1 = w_s1;
    wp.chunks = (p.span + WG_TOKENS - 1) / WG_TOKENS;
    const int err = attend_launch<AT_SCORES>(stream, dtype, p);
    if (err != STARKV_OK) return err;
    const dim3 grid(wp.chunks + (p.splits > 1 ? (p.G + 3) / 4 : 0), num_kv_heads, n);
    if (dtype == STARKV_BF16)
        hipLaunchKernelGGL(weigh_kernel<STARKV_BF16>, grid, dim3(256), 0, (hipStream_t)stream, wp);
    else
        hipLaunchKernelGGL(weigh_kernel<STARKV_F16>, grid, dim3(256), 0, (hipStream_t)stream, wp);
    SKV_HIP(hipGetLastError());
    return STARKV_OK;
}

// Up to 8 heads in a call their rows move through the workspace, all at once (up to twice the bytes). In order / at
// once, us a call, choice included: 1 head 65536 -> 57000 tokens 360 / 72, 8 heads 32768 -> 28000 292 / 105, 8192 -> 7000
// 46 / 32, 2176 -> 2048 20 / 20, 16 heads 8192 -> 7000 46 / 46, 2176 -> 2048 22 / 25. Not past 1 GiB of workspace.
static bool evict_staged(int n, int num_kv_heads, int keep) {
    const int64_t units = (int64_t)n * num_kv_heads;
    return units <= 8 && units * keep <= 1 << 21;
}

static size_t evict_kept_bytes(int n, int num_kv_heads, int weights_len, int keep) {
    return ((size_t)n * num_kv_heads * std::min(keep, weights_len) * 4 + 255) / 256 * 256;
}

size_t starkv_evict_workspace_bytes(int n, int num_kv_heads, int weights_len, int keep) {
    if (n < 1 || num_kv_heads < 1 || weights_len < 1 || keep < 1) return 256;
    const size_t rows = keep < weights_len && evict_staged(n, num_kv_heads, keep) ? (size_t)n * num_kv_heads * keep : 0;
    return evict_kept_bytes(n, num_kv_heads, weights_len, keep) + rows * 512;
}

int starkv_evict(void* stream, void* k_cache, void* v_cache, int64_t c_s0, int64_t c_s1, int64_t c_s2, int dtype,
                 int block_size, int64_t num_blocks, const int32_t* block_table, int64_t bt_s0, int64_t bt_s1,
                 int bt_width, const int32_t* seq_lens, int n, int num_kv_heads, const float* weights, int64_t w_s0,
                 int64_t w_s1, int weights_len, int keep, int sink, int recent, int32_t* new_lens, float* new_weights,
                 void* workspace, size_t workspace_bytes) {
    clear_error();
    SKV_CHECK(n >= 0 && n <= 65535 && num_kv_heads >= 1 && num_kv_heads <= 65535,
              "evict: n=%d (up to 65535) num_kv_heads=%d", n, num_kv_heads);
    SKV_CHECK(sink >= 0 && recent >= 0 && keep >= 1 && sink <= keep && recent <= keep - sink,
              "evict: keep %d tokens, %d first and %d last ones among them", keep, sink, recent);
    if (n == 0) return STARKV_OK;
    SKV_CHECK(k_cache && v_cache && block_table && seq_lens && weights && new_lens && new_weights && workspace,
              "evict: null pointer");
    SKV_CHECK(dtype == STARKV_BF16 || dtype == STARKV_F16, "evict: bf16 or fp16");
    SKV_CHECK(block_shift(block_size) >= 0, "evict: block_size must be 16 times a power of two");
    SKV_CHECK(num_blocks >= 1 && num_blocks <= 0x7fffffff && bt_width >= 1 && weights_len >= 1,
              "evict: empty cache, block table or weights");
    SKV_CHECK(((uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0 && (c_s0 | c_s1 | c_s2) % 8 == 0,
              "evict: cache rows must be 16-byte aligned");
    const size_t need = starkv_evict_workspace_bytes(n, num_kv_heads, weights_len, keep);
    SKV_CHECK(workspace_bytes >= need && (uintptr_t)workspace % 16 == 0, "evict: workspace %zu bytes < %zu, or unaligned",
              workspace_bytes, need);
    EvictParams p = {};
    p.kc = (uint16_t*)k_cache; p.vc = (uint16_t*)v_cache; p.c_s0 = c_s0; p.c_s1 = c_s1; p.c_s2 = c_s2;
    p.block_shift = block_shift(block_size) + 4; p.num_blocks = num_blocks;
    p.bt = block_table; p.bt_s0 = bt_s0; p.bt_s1 = bt_s1;
    p.seq_lens = seq_lens; p.span = (int)std::min<int64_t>((int64_t)bt_width * block_size, weights_len);
    p.w = weights; p.w_s0 = w_s0; p.w_s1 = w_s1;
    p.Hkv = num_kv_heads; p.cap = weights_len; p.keep = keep; p.sink = sink; p.recent = recent;
    p.new_lens = new_lens; p.new_w = new_weights; p.kept = (int32_t*)workspace;
    const int run = topk_run(p.span);
    const void* fn = run == TK_FEW ? (const void*)&evict_select_kernel<TK_FEW>
                     : run == TK_MANY ? (const void*)&evict_select_kernel<TK_MANY>
                     : run         ? (const void*)&evict_select_kernel<TK_MOST>
                                   : (const void*)&evict_select_kernel<0>;
    void* args[] = {(void*)&p};
    SKV_HIP(hipLaunchKernel(fn, dim3(num_kv_heads, n), dim3(TK_THR), args, 0, (hipStream_t)stream));
    if (p.span > keep && evict_staged(n, num_kv_heads, keep)) {
        p.aside = (uint16_t*)((char*)workspace + evict_kept_bytes(n, num_kv_heads, weights_len, keep));
        const dim3 grid((keep + ST_ROWS - 1) / ST_ROWS, num_kv_heads, n);
        hipLaunchKernelGGL(stage_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream, p);
        SKV_HIP(hipGetLastError());
        hipLaunchKernelGGL(stage_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream, p);
        SKV_HIP(hipGetLastError());
    } else if (p.span > keep) {
        // Whole rows a workgroup where those fill 256 CUs, else their halves: 4097 to 8192 -> 2048 tokens of 16 requests
        // of 8 KV heads 72 us whole, 77 in halves; 4096 -> 2048 of 64 requests 239, 251; 8192 -> 7000 of 8 requests
        // 127, 117; one of 32 heads 2176 -> 2048 29, 22 (in quarters 27).
        const int lanes = (int64_t)n * num_kv_heads >= 128 ? 4 : 3;
        hipLaunchKernelGGL(compact_kernel, dim3(32 >> lanes, num_kv_heads, n), dim3(CP_THR), 0, (hipStream_t)stream, p,
                           lanes);
        SKV_HIP(hipGetLastError());
    }
    return STARKV_OK;
}

}  // extern "C"
