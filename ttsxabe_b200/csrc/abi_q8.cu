// The C ABI of the 8-bit KV cache: host-side refusals and the launches. As in
// abi.cu every range is checked here, before anything is launched.
#include "kv_q8.cuh"

#include <math.h>
#include <stdlib.h>
#include <string.h>

#include <algorithm>
#include <new>
#include <utility>
#include <vector>

namespace {

constexpr float kLog2e = 1.4426950408889634f;

bool fits_i32(size_t x) { return x <= 0x7fffffffu; }

size_t cache_bytes(size_t kv_heads, size_t hd, size_t cap)
{
    return (size_t)q8_layout((int)kv_heads, (int)hd, (int)(cap / kQ8Block)).bytes;
}

// The shapes every entry takes.
llmtie_status check_geometry(llmtie_gpu *g, size_t batch, size_t kv_heads, size_t hd)
{
    if (!g) return llmtie_fail(LLMTIE_ERR_INVALID, "null device handle");
    cudaSetDevice(g->ordinal);
    if ((hd != 64 && hd != 128) || kv_heads == 0) return llmtie_unsupported(hd, kv_heads, kv_heads);
    if (kv_heads > 4096) return llmtie_fail(LLMTIE_ERR_INVALID, "an 8-bit cache of %zu KV heads", kv_heads);
    if (batch > 65536) return llmtie_fail(LLMTIE_ERR_INVALID, "a batch of %zu", batch);
    return LLMTIE_OK;
}

// One cache of a table, holding (or about to hold) `live` tokens.
llmtie_status check_cache(const void *base, int32_t cap, long long live)
{
    if (!base) return llmtie_fail(LLMTIE_ERR_INVALID, "null 8-bit cache");
    if (((uintptr_t)base & 15u) != 0) return llmtie_misaligned("an 8-bit cache", base, 16);
    if (cap <= 0 || cap % kQ8Block != 0) {
        return llmtie_fail(LLMTIE_ERR_RAGGED_BLOCK, "an 8-bit cache with a capacity of %d, which is not a multiple of %d",
                           cap, kQ8Block);
    }
    if (live < 0 || live > cap) {
        return llmtie_fail(LLMTIE_ERR_CACHE_OVERRUN, "appending at %lld to a cache with room for %d", live, cap);
    }
    return LLMTIE_OK;
}

// Caches that one call writes must not share memory, nor one that it writes with one
// that it reads: they would race. (Those that it only reads may be the same.)
typedef std::vector<std::pair<uintptr_t, size_t>> Spans;
llmtie_status check_apart(Spans &writes, const Spans &reads = Spans())
{
    std::sort(writes.begin(), writes.end());
    bool meet = false;
    for (size_t i = 1; i < writes.size(); i++) meet = meet || writes[i].first < writes[i - 1].first + writes[i - 1].second;
    for (const auto &r : reads) {
        // the first that starts at or behind it, and the one before
        const auto w = std::lower_bound(writes.begin(), writes.end(), std::make_pair(r.first, (size_t)0));
        meet = meet || (w != writes.end() && w->first < r.first + r.second);
        meet = meet || (w != writes.begin() && r.first < (w - 1)->first + (w - 1)->second);
    }
    if (meet) return llmtie_fail(LLMTIE_ERR_INVALID, "two caches of one call share memory");
    return LLMTIE_OK;
}

bool meet(const void *a, size_t a_bytes, const void *b, size_t b_bytes)
{
    return (uintptr_t)a < (uintptr_t)b + b_bytes && (uintptr_t)b < (uintptr_t)a + a_bytes;
}

// A buffer that the call writes, or reads while it writes the cache, in a cache's memory.
llmtie_status check_clear(const char *what, const void *p, size_t bytes, const void *cache, size_t cache_size)
{
    if (p && bytes && meet(p, bytes, cache, cache_size)) {
        return llmtie_fail(LLMTIE_ERR_INVALID, "%s: memory of an 8-bit cache of the same call", what);
    }
    return LLMTIE_OK;
}

llmtie_status overrun(size_t need, size_t have)
{
    return llmtie_fail(LLMTIE_ERR_SLICE_OVERRUN, "reading to %zu in a buffer of %zu", need, have);
}

// cu_seqlens ascending from >= 0; *total is its last entry.
llmtie_status check_rows(const int32_t *cu, size_t batch, size_t *total)
{
    if (cu[0] < 0) return llmtie_fail(LLMTIE_ERR_INVALID, "cu_seqlens starts at %d", cu[0]);
    for (size_t b = 0; b < batch; b++) {
        if (cu[b + 1] < cu[b]) return llmtie_fail(LLMTIE_ERR_INVALID, "cu_seqlens is not ascending");
    }
    *total = (size_t)cu[batch];
    return LLMTIE_OK;
}

// (the tables an entry makes may find no memory: an error, not an exception)
#define NO_MEMORY_IS_AN_ERROR                                                              \
    catch (const std::bad_alloc &)                                                         \
    {                                                                                      \
        return llmtie_fail(LLMTIE_ERR_DRIVER, "no host memory for the tables of the call"); \
    }

#define TRY(x)                              \
    do {                                    \
        const llmtie_status try_s = (x);    \
        if (try_s != LLMTIE_OK) return try_s; \
    } while (0)

// How the decode kernel would go over jobs [b0, b0 + LLMTIE_Q8_MAX_SEQ).
llmtie_status plan_jobs(llmtie_gpu *g, const std::vector<DecodeQ8Seq> &jobs, size_t b0, size_t kv_heads, size_t head_dim,
                        DecodeQ8Plan &plan)
{
    int per[LLMTIE_Q8_MAX_SEQ], clusters[2];
    const int n = (int)std::min<size_t>(LLMTIE_Q8_MAX_SEQ, jobs.size() - b0);
    for (int b = 0; b < n; b++) per[b] = (jobs[b0 + b].live + kQ8Block - 1) / kQ8Block;
    const cudaError_t e = decode_q8_clusters((int)head_dim, clusters);
    if (e != cudaSuccess) return llmtie_driver_fail("decode_q8", e);
    plan_decode_q8(plan, per, n, (int)kv_heads, (int)head_dim, g->sm_count, clusters);
    return LLMTIE_OK;
}

// The decode kernel over any number of jobs, LLMTIE_Q8_MAX_SEQ a launch.
llmtie_status run_jobs(llmtie_gpu *g, const std::vector<DecodeQ8Seq> &jobs, const float *q, void *out, int32_t out_f16,
                       size_t heads, size_t kv_heads, size_t head_dim, float scale, int32_t causal, int32_t weigh,
                       llmtie_decode_scratch *scratch)
{
    for (size_t b0 = 0; b0 < jobs.size(); b0 += LLMTIE_Q8_MAX_SEQ) {
        DecodeQ8Params p;
        memset(&p, 0, sizeof(p));
        p.nseq = (int)std::min<size_t>(LLMTIE_Q8_MAX_SEQ, jobs.size() - b0);
        long long units = 0, blocks = 0;
        bool empty = false;
        for (int b = 0; b < p.nseq; b++) {
            p.seq[b] = jobs[b0 + b];
            const int t = p.seq[b].live;
            empty = empty || t == 0;
            p.unit0[b] = (int)units;
            p.stat0[b] = blocks;
            units += (long long)((t + kQ8Block - 1) / kQ8Block) * (long long)kv_heads;
            blocks += (long long)p.seq[b].full * (long long)kv_heads;
        }
        p.causal = causal ? 1 : 0;
        p.q = q;
        p.out = out;
        if (units > 0x3fffffffll) return llmtie_fail(LLMTIE_ERR_INVALID, "a launch over %lld blocks of the caches", units);
        p.unit0[p.nseq] = (int)units;
        p.heads = (int)heads;
        p.kv_heads = (int)kv_heads;
        p.out_f16 = out_f16 ? 1 : 0;
        p.sl2 = scale * kLog2e;
        p.status = g->timeout_site;
        p.wait_cycles = g->wait_cycles;
        DecodeQ8Plan plan;
        TRY(plan_jobs(g, jobs, b0, kv_heads, head_dim, plan));
        cudaError_t err;
        const int grid = plan.grid;
        p.cluster = plan.cluster;
        p.parts = plan.parts;
        p.over = plan.over;
        const long long shares = units + (long long)p.over * p.nseq * (long long)kv_heads;
        p.each = grid ? (int)(shares / grid) : 0;
        p.more = grid ? (int)(shares % grid) : 0;
        const size_t pairs = (size_t)p.nseq * kv_heads;
        const size_t slots = (size_t)(p.cluster ? std::max(grid / p.cluster, 1) : std::max(2 * grid, 1)) * 8;
        p.part_o = (float *)workspace_reserve(scratch->q8_part, slots * (head_dim + 2) * sizeof(float), g->stream, &err);
        if (!p.part_o) return llmtie_driver_fail("allocating", err);
        p.part_ml = (float2 *)(p.part_o + slots * head_dim);
        const size_t had = scratch->q8_ctr.bytes;
        p.ctr = (unsigned *)workspace_reserve(scratch->q8_ctr, pairs * 8 * sizeof(unsigned), g->stream, &err);
        if (!p.ctr) return llmtie_driver_fail("allocating", err);
        if (scratch->q8_ctr.bytes != had) {
            err = cudaMemsetAsync(p.ctr, 0, scratch->q8_ctr.bytes, g->stream);
            if (err != cudaSuccess) return llmtie_driver_fail("zeroing", err);
        }
        if (weigh && blocks > 0) {
            p.stats = (float2 *)workspace_reserve(scratch->q8_stats, ((size_t)blocks + pairs) * 8 * sizeof(float2), g->stream, &err);
            if (!p.stats) return llmtie_driver_fail("allocating", err);
            p.fin = p.stats + blocks * 8;
        }
        LaunchScope ls(g, head_dim == 128 ? "decode_q8_128" : "decode_q8_64");
        err = launch_decode_q8(g->stream, p, (int)head_dim, grid);
        if (err != cudaSuccess) return llmtie_driver_fail("decode_q8", err);
        if (p.stats) g->launches++;            // two kernels in that launcher then
        if (empty && grid > 0) g->launches++;  // and another that writes the zeros
        TRY(ls.done());
    }
    return LLMTIE_OK;
}

}  // namespace

extern "C" size_t llmtie_kv_q8_bytes(size_t kv_heads, size_t head_dim, size_t cap)
{
    if ((head_dim != 64 && head_dim != 128) || kv_heads == 0 || kv_heads > 4096 || cap % kQ8Block != 0 || !fits_i32(cap)) return 0;
    return cache_bytes(kv_heads, head_dim, cap);
}

extern "C" llmtie_status llmtie_kv_alloc_q8(llmtie_gpu *g, size_t kv_heads, size_t head_dim, size_t cap, void **cache)
{
    TRY(check_geometry(g, 0, kv_heads, head_dim));
    if (!cache) return llmtie_fail(LLMTIE_ERR_INVALID, "null output pointer");
    if (cap == 0 || cap % kQ8Block != 0 || !fits_i32(cap)) {
        return llmtie_fail(LLMTIE_ERR_RAGGED_BLOCK, "an 8-bit cache with a capacity of %zu, which is not a multiple of %d",
                           cap, kQ8Block);
    }
    return llmtie_zeros(g, cache_bytes(kv_heads, head_dim, cap), cache);
}

extern "C" llmtie_status llmtie_rope_inv_freq(llmtie_gpu *g, const float *freq_div, size_t head_dim, float theta,
                                              float *out, size_t out_len)
{
    if (!g) return llmtie_fail(LLMTIE_ERR_INVALID, "null device handle");
    cudaSetDevice(g->ordinal);
    if (head_dim == 0 || head_dim % 2 != 0) {
        return llmtie_fail(LLMTIE_ERR_ODD_HEAD_DIM, "rotating heads of %zu, which is not even", head_dim);
    }
    if (!out) return llmtie_fail(LLMTIE_ERR_INVALID, "null output pointer");
    if (out_len < head_dim / 2) return overrun(head_dim / 2, out_len);
    if (!fits_i32(head_dim)) return llmtie_fail(LLMTIE_ERR_INVALID, "a head of %zu", head_dim);
    LaunchScope ls(g, "rope_inv_freq");
    launch_rope_inv_freq(g->stream, out, freq_div, (int)head_dim, theta);
    return ls.done();
}

extern "C" llmtie_status llmtie_rope_append_q8(llmtie_gpu *g, const float *q, size_t q_len, float *q_out, size_t q_out_len,
                                               const float *k, size_t k_len, const float *v, size_t v_len,
                                               const int32_t *cu_seqlens, size_t batch, void *const *caches,
                                               const int32_t *past, const int32_t *pos, const int32_t *cap,
                                               const float *inv_freq, size_t inv_len, size_t heads, size_t kv_heads,
                                               size_t head_dim)
try {
    TRY(check_geometry(g, batch, kv_heads, head_dim));
    if (!cu_seqlens || !caches || !past || !pos || !cap) return llmtie_fail(LLMTIE_ERR_INVALID, "null sequence table");
    if (batch == 0) return LLMTIE_OK;
    size_t total;
    TRY(check_rows(cu_seqlens, batch, &total));
    const bool turn_q = q != nullptr && inv_freq != nullptr;
    if (turn_q && (heads == 0 || heads > 65536)) return llmtie_unsupported(head_dim, heads, kv_heads);
    if (k_len < total * kv_heads * head_dim || v_len < total * kv_heads * head_dim) {
        return overrun(total * kv_heads * head_dim, std::min(k_len, v_len));
    }
    if (total > (size_t)cu_seqlens[0] && (!k || !v)) return llmtie_fail(LLMTIE_ERR_INVALID, "null key or value rows");
    if (((uintptr_t)k & 15u) != 0) return llmtie_misaligned("the key rows", k, 16);
    if (((uintptr_t)v & 15u) != 0) return llmtie_misaligned("the value rows", v, 16);
    if (inv_freq && inv_len < head_dim / 2) return overrun(head_dim / 2, inv_len);
    if (turn_q) {
        const size_t need = total * heads * head_dim;
        if (!q_out) return llmtie_fail(LLMTIE_ERR_INVALID, "null output pointer");
        if (q_len < need || q_out_len < need) return overrun(need, std::min(q_len, q_out_len));
        if (((uintptr_t)q & 15u) != 0) return llmtie_misaligned("the query", q, 16);
        if (((uintptr_t)q_out & 15u) != 0) return llmtie_misaligned("the rotated query", q_out, 16);
        // in place, or clear of everything the call reads
        const size_t kv_bytes = total * kv_heads * head_dim * 4;
        if ((q_out != q && meet(q_out, need * 4, q, need * 4)) || meet(q_out, need * 4, k, kv_bytes) || meet(q_out, need * 4, v, kv_bytes) ||
            meet(q_out, need * 4, inv_freq, head_dim / 2 * 4)) {
            return llmtie_fail(LLMTIE_ERR_INVALID, "the rotated query overlaps the rows the call reads");
        }
    }
    Spans spans;
    for (size_t b = 0; b < batch; b++) {
        const int n = cu_seqlens[b + 1] - cu_seqlens[b];
        if (n == 0) continue;
        TRY(check_cache(caches[b], cap[b], past[b] < 0 ? -1 : (long long)past[b] + n));
        if (pos[b] < 0 || (long long)pos[b] + n > 0x7fffffffll) {
            return llmtie_fail(LLMTIE_ERR_INVALID, "rows at position %d", pos[b]);
        }
        const size_t size = cache_bytes(kv_heads, head_dim, (size_t)cap[b]), kv_bytes = total * kv_heads * head_dim * 4;
        TRY(check_clear("the key rows", k, kv_bytes, caches[b], size));
        TRY(check_clear("the value rows", v, kv_bytes, caches[b], size));
        if (inv_freq) TRY(check_clear("the inverse frequencies", inv_freq, head_dim / 2 * 4, caches[b], size));
        if (turn_q) {
            TRY(check_clear("the queries", q, total * heads * head_dim * 4, caches[b], size));
            TRY(check_clear("the rotated queries", q_out, total * heads * head_dim * 4, caches[b], size));
        }
        spans.emplace_back((uintptr_t)caches[b], size);
    }
    TRY(check_apart(spans));
    for (size_t b0 = 0; b0 < batch;) {
        Q8AppendParams p;
        memset(&p, 0, sizeof(p));
        for (; b0 < batch && p.nseq < LLMTIE_Q8_MAX_SEQ; b0++) {
            const int n = cu_seqlens[b0 + 1] - cu_seqlens[b0];
            if (n == 0) continue;
            Q8AppendSeq &s = p.seq[p.nseq++];
            s.base = (unsigned char *)caches[b0];
            s.nb = cap[b0] / kQ8Block;
            s.past = past[b0];
            s.n = n;
            s.row0 = cu_seqlens[b0];
            s.pos = pos[b0];
            s.item0 = p.items;
            const int rows = past[b0] % kQ8Block + n, blocks = (rows + kQ8Block - 1) / kQ8Block;
            p.items += blocks - (blocks > 1 && rows % kQ8Block != 0 ? 1 : 0);
        }
        if (p.nseq == 0) break;
        p.q = turn_q ? q : nullptr;
        p.q_out = q_out;
        p.k = k;
        p.v = v;
        p.inv_freq = inv_freq;
        p.heads = (int)heads;
        p.kv_heads = (int)kv_heads;
        LaunchScope ls(g, "rope_append_q8");
        const cudaError_t e = launch_q8_append(g->stream, p, (int)head_dim, g->sm_count);
        if (e != cudaSuccess) return llmtie_driver_fail("rope_append_q8", e);
        TRY(ls.done());
    }
    return LLMTIE_OK;
}
NO_MEMORY_IS_AN_ERROR

extern "C" llmtie_status llmtie_cache_read_q8(llmtie_gpu *g, const void *const *caches, const int32_t *cap,
                                              const int32_t *live, const int32_t *first, const int32_t *cu_seqlens,
                                              size_t batch, size_t kv_heads, size_t head_dim, uint16_t *k_out,
                                              size_t k_len, uint16_t *v_out, size_t v_len)
{
    TRY(check_geometry(g, batch, kv_heads, head_dim));
    if (!cu_seqlens || !caches || !cap || !live || !first) return llmtie_fail(LLMTIE_ERR_INVALID, "null sequence table");
    if (batch == 0) return LLMTIE_OK;
    size_t total;
    TRY(check_rows(cu_seqlens, batch, &total));
    if (k_len < total * kv_heads * head_dim || v_len < total * kv_heads * head_dim) {
        return overrun(total * kv_heads * head_dim, std::min(k_len, v_len));
    }
    if (total > (size_t)cu_seqlens[0] && (!k_out || !v_out)) return llmtie_fail(LLMTIE_ERR_INVALID, "null output pointer");
    if (((uintptr_t)k_out & 15u) != 0) return llmtie_misaligned("the keys read", k_out, 16);
    if (((uintptr_t)v_out & 15u) != 0) return llmtie_misaligned("the values read", v_out, 16);
    if (meet(k_out, total * kv_heads * head_dim * 2, v_out, total * kv_heads * head_dim * 2)) {
        return llmtie_fail(LLMTIE_ERR_INVALID, "the keys and the values go to the same rows");
    }
    for (size_t b = 0; b < batch; b++) {
        const int n = cu_seqlens[b + 1] - cu_seqlens[b];
        if (n == 0) continue;
        TRY(check_cache(caches[b], cap[b], live[b]));
        if (first[b] < 0 || (long long)first[b] + n > live[b]) {
            return llmtie_fail(LLMTIE_ERR_CACHE_OVERRUN, "reading to %lld of a cache that holds %d", (long long)first[b] + n, live[b]);
        }
        const size_t size = cache_bytes(kv_heads, head_dim, (size_t)cap[b]), bytes = total * kv_heads * head_dim * 2;
        TRY(check_clear("the keys read", k_out, bytes, caches[b], size));
        TRY(check_clear("the values read", v_out, bytes, caches[b], size));
    }
    for (size_t b0 = 0; b0 < batch;) {
        Q8ReadParams p;
        memset(&p, 0, sizeof(p));
        for (; b0 < batch && p.nseq < LLMTIE_Q8_MAX_SEQ; b0++) {
            const int n = cu_seqlens[b0 + 1] - cu_seqlens[b0];
            if (n == 0) continue;
            p.seq[p.nseq++] = {(const unsigned char *)caches[b0], cap[b0] / kQ8Block, live[b0], first[b0], n, cu_seqlens[b0], p.items};
            p.items += (first[b0] + n - 1) / kQ8Block - first[b0] / kQ8Block + 1;
        }
        if (p.nseq == 0) break;
        p.k = k_out;
        p.v = v_out;
        p.kv_heads = (int)kv_heads;
        LaunchScope ls(g, "cache_read_q8");
        const cudaError_t e = launch_q8_read(g->stream, p, (int)head_dim);
        if (e != cudaSuccess) return llmtie_driver_fail("cache_read_q8", e);
        TRY(ls.done());
    }
    return LLMTIE_OK;
}

extern "C" llmtie_status llmtie_cache_rewind_q8(llmtie_gpu *g, void *const *caches, const int32_t *cap,
                                                const int32_t *live, const int32_t *to, size_t batch, size_t kv_heads,
                                                size_t head_dim)
try {
    TRY(check_geometry(g, batch, kv_heads, head_dim));
    if (!caches || !cap || !live || !to) return llmtie_fail(LLMTIE_ERR_INVALID, "null sequence table");
    Spans spans;
    for (size_t b = 0; b < batch; b++) {
        TRY(check_cache(caches[b], cap[b], live[b]));
        if (to[b] < 0 || to[b] > live[b]) {
            return llmtie_fail(LLMTIE_ERR_CACHE_OVERRUN, "cutting a cache that holds %d to %d", live[b], to[b]);
        }
        spans.emplace_back((uintptr_t)caches[b], cache_bytes(kv_heads, head_dim, (size_t)cap[b]));
    }
    TRY(check_apart(spans));
    for (size_t b0 = 0; b0 < batch;) {
        Q8RewindParams p;
        memset(&p, 0, sizeof(p));
        for (; b0 < batch && p.nseq < LLMTIE_Q8_MAX_SEQ; b0++) {
            // a cut at a block's start needs no tail, one inside the tail has it
            if (to[b0] % kQ8Block == 0 || to[b0] / kQ8Block == live[b0] / kQ8Block) continue;
            p.seq[p.nseq++] = {(unsigned char *)caches[b0], cap[b0] / kQ8Block, to[b0]};
        }
        if (p.nseq == 0) break;
        p.kv_heads = (int)kv_heads;
        LaunchScope ls(g, "cache_rewind_q8");
        const cudaError_t e = launch_q8_rewind(g->stream, p, (int)head_dim);
        if (e != cudaSuccess) return llmtie_driver_fail("cache_rewind_q8", e);
        TRY(ls.done());
    }
    return LLMTIE_OK;
}
NO_MEMORY_IS_AN_ERROR

extern "C" llmtie_status llmtie_cache_evict_q8(llmtie_gpu *g, const void *const *src, const int32_t *src_cap,
                                               void *const *dst, const int32_t *dst_cap, const int32_t *live,
                                               const int32_t *keep, size_t batch, size_t keep_first, size_t keep_recent,
                                               size_t kv_heads, size_t head_dim, int32_t *index, size_t index_len)
try {
    TRY(check_geometry(g, batch, kv_heads, head_dim));
    if (!src || !src_cap || !dst || !dst_cap || !live || !keep) return llmtie_fail(LLMTIE_ERR_INVALID, "null sequence table");
    Spans writes, reads;
    int most = 0;
    for (size_t b = 0; b < batch; b++) {
        TRY(check_cache(src[b], src_cap[b], live[b]));
        const int full = live[b] / kQ8Block;
        if (keep[b] < 0 || (full > keep[b] && (keep_first > (size_t)keep[b] || keep_recent > (size_t)keep[b] - keep_first))) {
            return llmtie_fail(LLMTIE_ERR_INVALID, "keeping %d blocks of which the first %zu and the last %zu stay", keep[b],
                               keep_first, keep_recent);
        }
        const int kept = std::min(full, keep[b]);
        most = std::max(most, kept);
        TRY(check_cache(dst[b], dst_cap[b], (long long)kept * kQ8Block + live[b] % kQ8Block));
        writes.emplace_back((uintptr_t)dst[b], cache_bytes(kv_heads, head_dim, (size_t)dst_cap[b]));
        if (dst[b] != src[b]) {
            reads.emplace_back((uintptr_t)src[b], cache_bytes(kv_heads, head_dim, (size_t)src_cap[b]));
        } else if (dst_cap[b] != src_cap[b]) {
            return llmtie_fail(LLMTIE_ERR_INVALID, "a cache shortened in place keeps its capacity of %d, not %d", src_cap[b],
                               dst_cap[b]);
        }
    }
    TRY(check_apart(writes, reads));
    const size_t numbers = batch * kv_heads * (size_t)most;
    if (index && index_len < numbers) return overrun(numbers, index_len);
    for (const Spans *spans : {&writes, &reads}) {
        for (const auto &s : *spans) TRY(check_clear("the blocks' numbers", index, numbers * 4, (const void *)s.first, s.second));
    }
    for (size_t b0 = 0; b0 < batch; b0 += LLMTIE_Q8_MAX_SEQ) {
        Q8EvictParams p;
        memset(&p, 0, sizeof(p));
        p.nseq = (int)std::min<size_t>(LLMTIE_Q8_MAX_SEQ, batch - b0);
        for (int b = 0; b < p.nseq; b++) {
            Q8EvictSeq &s = p.seq[b];
            s.src = (const unsigned char *)src[b0 + b];
            s.dst = (unsigned char *)dst[b0 + b];
            s.src_nb = src_cap[b0 + b] / kQ8Block;
            s.dst_nb = dst_cap[b0 + b] / kQ8Block;
            s.full = live[b0 + b] / kQ8Block;
            s.tail = live[b0 + b] % kQ8Block;
            s.keep = std::min(s.full, (int)keep[b0 + b]);
            // (where nothing goes, everything is kept whatever these say)
            s.first = s.keep < s.full ? (int)keep_first : 0;
            s.recent = s.keep < s.full ? (int)keep_recent : 0;
        }
        p.kv_heads = (int)kv_heads;
        p.max_keep = most;
        p.user_stride = most;
        p.user_index = index ? index + b0 * kv_heads * (size_t)most : nullptr;
        cudaError_t err;
        p.index = (int *)workspace_reserve(g->ws_q8, (size_t)p.nseq * kv_heads * std::max(most, 1) * sizeof(int), g->stream, &err);
        if (!p.index) return llmtie_driver_fail("allocating", err);
        LaunchScope ls(g, "cache_evict_q8");
        const cudaError_t e = launch_q8_evict(g->stream, p, (int)head_dim, g->sm_count);
        if (e != cudaSuccess) return llmtie_driver_fail("cache_evict_q8", e);
        if (most > 0) g->launches++;   // two kernels in that launcher then
        TRY(ls.done());
    }
    return LLMTIE_OK;
}
NO_MEMORY_IS_AN_ERROR

extern "C" llmtie_status llmtie_cache_grow_q8(llmtie_gpu *g, const void *src, size_t src_len, void *dst, size_t dst_len,
                                              size_t kv_heads, size_t head_dim, size_t old_cap, size_t new_cap,
                                              size_t live)
{
    TRY(check_geometry(g, 1, kv_heads, head_dim));
    if (live > old_cap || new_cap < old_cap || !fits_i32(new_cap)) {
        return llmtie_fail(LLMTIE_ERR_CACHE_OVERRUN, "appending at %zu to a cache with room for %zu", std::max(live, old_cap),
                           std::min(new_cap, old_cap));
    }
    const int32_t oc = (int32_t)old_cap, nc = (int32_t)new_cap, n = (int32_t)live, keep = n / kQ8Block;
    TRY(check_cache(src, oc, n));
    TRY(check_cache(dst, nc, n));
    if (src_len < cache_bytes(kv_heads, head_dim, old_cap)) return overrun(cache_bytes(kv_heads, head_dim, old_cap), src_len);
    if (dst_len < cache_bytes(kv_heads, head_dim, new_cap)) return overrun(cache_bytes(kv_heads, head_dim, new_cap), dst_len);
    if (src == dst) return llmtie_fail(LLMTIE_ERR_INVALID, "a cache cannot grow in place");
    if (n == 0) return LLMTIE_OK;
    return llmtie_cache_evict_q8(g, &src, &oc, &dst, &nc, &n, &keep, 1, 0, 0, kv_heads, head_dim, nullptr, 0);
}

extern "C" llmtie_status llmtie_decode_batched_q8(llmtie_gpu *g, const float *q, size_t q_len, void *const *caches,
                                                  const int32_t *live, const int32_t *cap, size_t batch, size_t heads,
                                                  size_t kv_heads, size_t head_dim, float scale, int32_t weigh,
                                                  llmtie_decode_scratch *scratch, void *out, size_t out_len,
                                                  int32_t out_f16)
try {
    TRY(check_geometry(g, batch, kv_heads, head_dim));
    if (!scratch) return llmtie_fail(LLMTIE_ERR_INVALID, "null decode scratch");
    if (!caches || !live || !cap) return llmtie_fail(LLMTIE_ERR_INVALID, "null sequence table");
    if (heads % kv_heads != 0 || heads / kv_heads > 8 || heads == 0) return llmtie_unsupported(head_dim, heads, kv_heads);
    const size_t n = heads * head_dim;
    if (q_len < batch * n) return overrun(batch * n, q_len);
    if (out_len < batch * n) return overrun(batch * n, out_len);
    if (batch == 0) return LLMTIE_OK;
    if (!q || !out) return llmtie_fail(LLMTIE_ERR_INVALID, "null query or output");
    if (((uintptr_t)q & 15u) != 0) return llmtie_misaligned("the query", q, 16);
    if (((uintptr_t)out & 15u) != 0) return llmtie_misaligned("the output", out, 16);
    if (meet(q, batch * n * 4, out, batch * n * (out_f16 ? 2 : 4))) return llmtie_fail(LLMTIE_ERR_INVALID, "the output overlaps the query");
    Spans spans;
    for (size_t b = 0; b < batch; b++) {
        TRY(check_cache(caches[b], cap[b], live[b]));
        const size_t size = cache_bytes(kv_heads, head_dim, (size_t)cap[b]);
        TRY(check_clear("the output", out, batch * n * (out_f16 ? 2 : 4), caches[b], size));
        if (weigh) {
            TRY(check_clear("the query", q, batch * n * 4, caches[b], size));
            spans.emplace_back((uintptr_t)caches[b], size);
        }
    }
    TRY(check_apart(spans));
    std::vector<DecodeQ8Seq> jobs(batch);
    for (size_t b = 0; b < batch; b++) {
        jobs[b] = {(unsigned char *)caches[b], cap[b] / kQ8Block, live[b] / kQ8Block, live[b], (int)b, 1};
    }
    return run_jobs(g, jobs, q, out, out_f16, heads, kv_heads, head_dim, scale, 1, weigh, scratch);
}
NO_MEMORY_IS_AN_ERROR

extern "C" llmtie_status llmtie_decode_plan_q8(const int32_t *live, size_t batch, size_t kv_heads, size_t head_dim,
                                               int32_t sm_count, int32_t resident8, int32_t resident16, int32_t *grid,
                                               int32_t *cluster, int64_t *ns)
{
    if ((head_dim != 64 && head_dim != 128) || kv_heads == 0 || kv_heads > 4096) return llmtie_unsupported(head_dim, kv_heads, kv_heads);
    if (!live || !grid || !cluster || !ns || batch > LLMTIE_Q8_MAX_SEQ || sm_count <= 0) {
        return llmtie_fail(LLMTIE_ERR_INVALID, "a malformed plan request");
    }
    int units[LLMTIE_Q8_MAX_SEQ];
    for (size_t b = 0; b < batch; b++) {
        if (live[b] < 0) return llmtie_fail(LLMTIE_ERR_CACHE_OVERRUN, "a context of %d", live[b]);
        units[b] = (int)(((long long)live[b] + kQ8Block - 1) / kQ8Block);
    }
    const int clusters[2] = {resident8, resident16};
    DecodeQ8Plan plan;
    plan_decode_q8(plan, units, (int)batch, (int)kv_heads, (int)head_dim, sm_count, clusters);
    *grid = plan.grid;
    *cluster = plan.cluster;
    *ns = (int64_t)(plan.us * 1000.0);
    return LLMTIE_OK;
}

extern "C" llmtie_status llmtie_flash_attn_q8(llmtie_gpu *g, const float *q, size_t q_len, const int32_t *cu_seqlens,
                                              size_t batch, const void *const *caches, const int32_t *past,
                                              const int32_t *cap, size_t heads, size_t kv_heads, size_t head_dim,
                                              float scale, int32_t causal, void *out, size_t out_len, int32_t out_f16)
try {
    TRY(check_geometry(g, batch, kv_heads, head_dim));
    if (!cu_seqlens || !caches || !past || !cap) return llmtie_fail(LLMTIE_ERR_INVALID, "null sequence table");
    if (heads % kv_heads != 0 || heads == 0 || heads > 65535) return llmtie_unsupported(head_dim, heads, kv_heads);
    if (batch == 0) return LLMTIE_OK;
    size_t total;
    TRY(check_rows(cu_seqlens, batch, &total));
    const size_t n = heads * head_dim;
    if (q_len < total * n || out_len < total * n) return overrun(total * n, std::min(q_len, out_len));
    if (total > (size_t)cu_seqlens[0] && (!q || !out)) return llmtie_fail(LLMTIE_ERR_INVALID, "null query or output");
    if (((uintptr_t)q & 15u) != 0) return llmtie_misaligned("the query", q, 16);
    if (((uintptr_t)out & 15u) != 0) return llmtie_misaligned("the output", out, 16);
    if (meet(q, total * n * 4, out, total * n * (out_f16 ? 2 : 4))) return llmtie_fail(LLMTIE_ERR_INVALID, "the output overlaps the query");
    for (size_t b = 0; b < batch; b++) {
        const int rows = cu_seqlens[b + 1] - cu_seqlens[b];
        if (rows == 0) continue;
        TRY(check_cache(caches[b], cap[b], past[b] < 0 ? -1 : (long long)past[b] + rows));
        TRY(check_clear("the output", out, total * n * (out_f16 ? 2 : 4), caches[b], cache_bytes(kv_heads, head_dim, (size_t)cap[b])));
    }
    // Sequences of few rows may go through the decode kernel, which reads their codes
    // as they lie, as a job for every eight rows of a group: where that is estimated to
    // take less than unpacking them, 13 us for a launch and a microsecond for every 77
    // cache blocks (155 at head_dim 64) as measured. (8 x 512 tokens, 32 / 8 heads x
    // 128: 8 rows 9 against 26 us, 32 rows 31 against 27.)
    const size_t group = heads / kv_heads;
    constexpr int kMostJobs = 16;
    std::vector<DecodeQ8Seq> jobs;
    std::vector<char> few(batch, 0);
    double unpacked = 0.0, decoded = 0.0;
    bool others = false;
    for (size_t b = 0; b < batch; b++) {
        const int rows = cu_seqlens[b + 1] - cu_seqlens[b], each = group <= 8 ? (int)(8 / group) : 0;
        if (rows == 0) continue;
        if (each == 0 || (rows + each - 1) / each > kMostJobs) {
            others = true;                                  // (there is such a launch anyway)
            continue;
        }
        few[b] = 1;
        unpacked += (double)((past[b] + rows + kQ8Block - 1) / kQ8Block) * (double)kv_heads / (head_dim == 128 ? 77.0 : 155.0);
        for (int r = 0; r < rows; r += each) {
            const int n = std::min(each, rows - r);
            jobs.push_back({(unsigned char *)caches[b], cap[b] / kQ8Block, (past[b] + rows) / kQ8Block,
                            past[b] + (causal ? r + n : rows), cu_seqlens[b] + r, n});
        }
    }
    for (size_t j = 0; j < jobs.size(); j += LLMTIE_Q8_MAX_SEQ) {
        DecodeQ8Plan plan;
        TRY(plan_jobs(g, jobs, j, kv_heads, head_dim, plan));
        decoded += plan.us;
    }
    if (decoded > unpacked + (others ? 0.0 : 13.0)) {
        jobs.clear();
        std::fill(few.begin(), few.end(), 0);
    }
    if (!jobs.empty()) {
        if (!g->q8_scratch) TRY(llmtie_decode_scratch_new(g, &g->q8_scratch));
        TRY(run_jobs(g, jobs, q, out, out_f16, heads, kv_heads, head_dim, scale, causal, 0, g->q8_scratch));
    }
    // A launch of the attention kernel takes LLMTIE_TC_MAX_SEQ sequences; a
    // sequence of more than kRows rows is as many of them as it takes, over the
    // same keys.
    constexpr int kRows = 16384;
    constexpr size_t kMostUnpacked = (size_t)1 << 30;   // for more than eight sequences
    for (size_t b = 0, done = 0; b < batch;) {
        Q8UnpackParams up;
        PrefillParams pp;
        memset(&up, 0, sizeof(up));
        memset(&pp, 0, sizeof(pp));
        size_t bytes = 0;
        size_t at[LLMTIE_TC_MAX_SEQ];       // where the sequence's keys lie in the workspace
        while (b < batch && pp.nseq < LLMTIE_TC_MAX_SEQ) {
            const int rows = cu_seqlens[b + 1] - cu_seqlens[b];
            if (rows == 0 || few[b]) {
                b++;
                continue;
            }
            const int live = past[b] + rows;
            const size_t cap16 = ((size_t)live + 7) / 8 * 8, half = (kv_heads * cap16 * head_dim * 2 + 255) / 256 * 256;
            if (up.nseq >= 8 && bytes + 2 * half > kMostUnpacked) break;
            Q8UnpackSeq &u = up.seq[up.nseq++];
            u.base = (const unsigned char *)caches[b];
            u.nb = cap[b] / kQ8Block;
            u.live = live;
            u.cap16 = (int)cap16;
            u.item0 = up.items;
            up.items += (live + q8_unpack_tokens((int)head_dim) - 1) / q8_unpack_tokens((int)head_dim);
            const size_t place = bytes;
            u.k = (uint16_t *)place;             // (offsets until the workspace is known)
            u.v = (uint16_t *)(place + half);
            bytes += 2 * half;
            while (done < (size_t)rows && pp.nseq < LLMTIE_TC_MAX_SEQ) {
                const int take = (int)std::min<size_t>(kRows, rows - done);
                PrefillSeq &s = pp.seq[pp.nseq];
                at[pp.nseq++] = up.nseq - 1;
                s.row0 = cu_seqlens[b] - cu_seqlens[0] + (int)done;
                s.tq = take;
                s.past = past[b] + (int)done;
                s.cap = (int)cap16;
                s.tk = live;
                done += take;
            }
            if (done == (size_t)rows) {
                b++;
                done = 0;
            }
        }
        if (pp.nseq == 0) break;
        cudaError_t err;
        char *work = (char *)workspace_reserve(g->ws_q8, bytes, g->stream, &err);
        if (!work) return llmtie_driver_fail("allocating", err);
        for (int i = 0; i < up.nseq; i++) {
            up.seq[i].k = (uint16_t *)(work + (size_t)up.seq[i].k);
            up.seq[i].v = (uint16_t *)(work + (size_t)up.seq[i].v);
        }
        for (int i = 0; i < pp.nseq; i++) {
            pp.seq[i].k = up.seq[at[i]].k;
            pp.seq[i].v = up.seq[at[i]].v;
        }
        up.kv_heads = (int)kv_heads;
        {
            LaunchScope ls(g, "q8_unpack");
            const cudaError_t e = launch_q8_unpack(g->stream, up, (int)head_dim);
            if (e != cudaSuccess) return llmtie_driver_fail("q8_unpack", e);
            TRY(ls.done());
        }
        const size_t row0 = (size_t)cu_seqlens[0] * n;
        pp.q = q + row0;
        pp.q_stride = (long long)n;
        pp.out = out_f16 ? (void *)((uint16_t *)out + row0) : (void *)((float *)out + row0);
        pp.out_stride = (long long)n;
        pp.out_f16 = out_f16 ? 1 : 0;
        pp.heads = (int)heads;
        pp.kv_heads = (int)kv_heads;
        pp.causal = causal ? 1 : 0;
        // (the kernel takes its maxima before it scales: a scale that is not positive goes into q)
        pp.q_scale = scale < 0.0f ? -1.0f : scale == 0.0f ? 0.0f : 1.0f;
        pp.sl2 = scale == 0.0f ? kLog2e : fabsf(scale) * kLog2e;
        const bool tc = llmtie_use_tc(pp, (int)head_dim);
        static const bool no_pdl = getenv("LLMTIE_B200_NO_PDL") != nullptr;
        pp.after_prepass = (tc && !no_pdl && !g->kprof) ? 1 : 0;
        WaitCtl w = llmtie_next_wait_ctl(g);
        w.part = &g->ws_q8_part;
        LaunchScope ls(g, tc ? "flash_attn_q8_tc" : "flash_attn_q8");
        err = tc ? launch_prefill_tc(g->stream, pp, (int)head_dim, w) : launch_prefill_mma(g->stream, pp, (int)head_dim);
        if (err != cudaSuccess) return llmtie_driver_fail("flash_attn_q8", err);
        TRY(ls.done());
    }
    return LLMTIE_OK;
}
NO_MEMORY_IS_AN_ERROR
