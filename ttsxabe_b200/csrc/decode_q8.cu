// Split-KV decode over the 8-bit cache (kv_q8.cuh): one query row a head, or
// the few of a short prompt (as long as a group's are no more than eight); the
// codes go into the tensor cores as they lie in memory.
//
// Mathematics. With q of a row as 16-bit fixed point, q = f (256 H + L), H and L
// int8, and a block's keys k = s_k c, the scores are f s_k (256 H.c + L.c): two
// int8 products, exact in 32 bits. The probabilities of a block are taken
// relative to the block's own maximum, p = 2^(s - m_blk) in [0, 1], and held as
// 16-bit fixed point too, p = (256 P + Q) / 65535 with P and Q unsigned bytes:
// their product with the value codes is exact as well, and is folded into the
// f32 accumulator with the factor s_v 2^(m_blk - m) / 65535. So nothing is
// converted code by code, every rounding is 2^-16 of a row's or a block's
// largest value, and a key far below another block's maximum keeps its
// precision.
//
// Tiles. One warp takes one cache block of 32 tokens: mma.m16n8k32 with the
// query's H rows as rows 0-7 and its L rows as rows 8-15 of A (up to eight
// query rows of a group), four key tiles of eight tokens as B; the result
// fragment holds a row's H and L sums in one thread, and, with the tokens
// dealt to the tiles' columns as below, exactly the eight tokens whose bytes
// that thread needs of the A fragment of the second product. No shuffle but
// the two of the block's maximum, no conversion of codes, no trip of the
// probabilities through shared memory.
//
// The kernel is bound by reading the cache: each warp keeps a ring of its own
// blocks in flight (cp.async.bulk, an mbarrier a stage; two stages, since with
// three the queue at the memory makes every other load wait: 344 against 301 us
// for 8 x 131072 keys of 8 heads x 128, which is 7.1 TB/s; up to 320 on other B200s). A pair
// (sequence, KV head) is taken by a cluster of blocks of the grid that merge
// through distributed shared memory, or by several, whose results the last to
// arrive merges row by row, or the grid is cut by work and the last block to
// arrive merges (see plan_decode_q8, and there what each costs). The
// tensor pipe is 20 % busy, so there is no more to gain from tcgen05 here.
#include "kv_q8.cuh"

#include <math_constants.h>

#include <algorithm>

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 8;             // query rows a pair may have

template <int HD>
struct Geo {
    static constexpr int BLOCK = kQ8Block * HD;          // bytes of a block's keys (or values)
    static constexpr int STAGES = 2;
    static constexpr int RESIDENT = HD == 128 ? 2 : 3;   // blocks of the grid that fit an SM
    static constexpr int STAGE = 2 * BLOCK;              // keys, then values
    static constexpr int RING = kWarps * STAGES * STAGE;
    static constexpr int MERGE = kWarps * kRows * HD * 4;
    static constexpr int SMEM = RING + MERGE;
};

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

// Waits for a phase of the ring, at most p.wait_cycles.
__device__ __forceinline__ bool ring_wait(uint32_t bar, uint32_t parity, int *status, long long cycles)
{
    long long start = 0;
    for (uint32_t it = 0;; it++) {
        uint32_t ok;
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
            "selp.u32 %0, 1, 0, p;\n"
            "}\n"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
        if (ok) return true;
        if (it == 0) start = clock64();
        else if ((it & 15u) == 0 && clock64() - start > cycles) break;
    }
    report_timeout(status, 60);
    return false;
}

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_u8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// One run of a block of the grid: blocks [first, last) of one pair, and its
// tail if the run reaches the pair's end.
struct Run {
    int seq, head;
    int first, last;      // complete blocks
    int units;            // of the whole pair
    int begin;            // its first unit
    bool tail;
    bool whole;           // the pair has no other block of the grid
    int next;             // unit after the run
};

// A pair that several blocks of the grid hold (units 0: none).
struct Shared {
    int seq, head, begin, units;
};
__device__ __forceinline__ Shared pick(bool second, const Shared &a, const Shared &b)
{
    return {second ? b.seq : a.seq, second ? b.head : a.head, second ? b.begin : a.begin, second ? b.units : a.units};
}

__device__ __forceinline__ Run run_at(const DecodeQ8Params &p, int u, int end)
{
    int lo = 0, hi = p.nseq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.unit0[mid] <= u) lo = mid;
        else hi = mid - 1;
    }
    Run r;
    const int live = p.seq[lo].live, full = p.seq[lo].full;
    r.units = (live + 31) >> 5;                                 // (0 only where the block has no units)
    r.seq = lo;
    r.head = (int)((unsigned)(u - p.unit0[lo]) / (unsigned)max(1, r.units));
    r.begin = p.unit0[lo] + r.head * r.units;
    r.first = u - r.begin;
    const int stop = min(r.units, end - r.begin);
    r.tail = stop > full;
    r.last = min(stop, full);
    r.whole = r.first == 0 && stop == r.units;
    r.next = r.begin + stop;
    return r;
}

// The cut is one of virtual units: a pair is its units behind `over` more that
// stand for what a run costs besides its blocks. A block of the grid whose share
// starts among those takes the pair from its first unit, one whose share ends
// there stops at the pair before; a share of nothing else is empty. The first
// `more` blocks take each + 1, the others each.
__device__ __forceinline__ int first_unit(const DecodeQ8Params &p, int block)
{
    const int v = block * p.each + min(block, p.more);
    int lo = 0, hi = p.nseq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.unit0[mid] + p.over * mid * p.kv_heads <= v) lo = mid;
        else hi = mid - 1;
    }
    const int units = (p.seq[lo].live + 31) >> 5;
    if (units == 0) return p.unit0[lo];                         // (only past the last unit)
    const int in = v - p.unit0[lo] - p.over * lo * p.kv_heads;
    const int pair = (int)((unsigned)in / (unsigned)(units + p.over));
    return p.unit0[lo] + pair * units + max(0, in - pair * (units + p.over) - p.over);
}
// The block of the grid that holds unit u, of pair number `pair` of the launch.
__device__ __forceinline__ int block_of(const DecodeQ8Params &p, int u, int pair)
{
    const int v = u + p.over * (pair + 1), seam = p.more * (p.each + 1);
    return v < seam ? (int)((unsigned)v / (unsigned)(p.each + 1)) : p.more + (int)((unsigned)(v - seam) / (unsigned)p.each);
}

template <int HD>
__device__ __forceinline__ void store_row(const DecodeQ8Params &p, long long at, int lane, const float (&o)[HD / 32])
{
    constexpr int V = HD / 32;
    if (p.out_f16) {
        __half2 *d = (__half2 *)((uint16_t *)p.out + at + V * lane);
#pragma unroll
        for (int e = 0; e < V / 2; e++) d[e] = __floats2half2_rn(o[2 * e], o[2 * e + 1]);
    } else {
        float2 *d = (float2 *)((float *)p.out + at + V * lane);
#pragma unroll
        for (int e = 0; e < V / 2; e++) d[e] = make_float2(o[2 * e], o[2 * e + 1]);
    }
}

// By cluster: a pair is cut evenly over the blocks of its p.parts clusters.
__device__ __forceinline__ Run run_of_rank(const DecodeQ8Params &p)
{
    const int over = p.parts * p.cluster, pair = (int)blockIdx.x / over, rank = (int)blockIdx.x - pair * over;
    Run r;
    r.seq = pair / p.kv_heads;
    r.head = pair - r.seq * p.kv_heads;
    const int full = p.seq[r.seq].full;
    r.units = (p.seq[r.seq].live + 31) >> 5;
    r.begin = 0;
    r.first = (int)((long long)r.units * rank / over);
    const int stop = (int)((long long)r.units * (rank + 1) / over);
    r.tail = stop > full && r.first < stop;
    r.last = min(stop, full);
    r.whole = p.cluster == 1;
    r.next = 0;
    return r;
}

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// An address of this block's shared memory in that of cluster rank `rank`.
__device__ __forceinline__ uint32_t peer(uint32_t addr, int rank)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}
__device__ __forceinline__ float2 peer_f2(uint32_t addr)
{
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

// Row `row` of `count` partial results, slots first + skew, first + step, first + 2
// step and so on: in that order, 32 at a time, 16 of their loads in flight.
template <int HD>
__device__ __forceinline__ void merge_parts(const DecodeQ8Params &p, int lane, int count, int first, int step, int skew, int row,
                                            float &M, float &L, float (&o)[HD / 32])
{
    constexpr int V = HD / 32, U = 16;
    M = -CUDART_INF_F;
    L = 0.0f;
#pragma unroll
    for (int e = 0; e < V; e++) o[e] = 0.0f;
    for (int at = 0; at < count; at += 32) {
        const int n = min(32, count - at);
        auto slot = [&](int i) { return first + step * (at + i) + (at + i == 0 ? skew : 0); };
        float2 ml = make_float2(-CUDART_INF_F, 0.0f);
        if (lane < n) ml = __ldcg(&p.part_ml[slot(lane) * kRows + row]);
        float y[U][V];
        auto load = [&](int i0) {
#pragma unroll
            for (int i = 0; i < U; i++) {
                if (i0 + i < n) {
                    const float *src = p.part_o + ((long long)slot(i0 + i) * kRows + row) * HD + V * lane;
                    if constexpr (V == 4) {
                        const float4 z = __ldcg((const float4 *)src);
                        y[i][0] = z.x; y[i][1] = z.y; y[i][2] = z.z; y[i][3] = z.w;
                    } else {
                        const float2 z = __ldcg((const float2 *)src);
                        y[i][0] = z.x; y[i][1] = z.y;
                    }
                }
            }
        };
        load(0);
        float top = ml.x;
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        top = fmaxf(top, M);
        const float keep = M == -CUDART_INF_F ? 0.0f : ex2(M - top);
        const float f = ml.x == -CUDART_INF_F ? 0.0f : ex2(ml.x - top);
        float sum = f * ml.y;
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
        L = fmaf(L, keep, sum);
#pragma unroll
        for (int e = 0; e < V; e++) o[e] *= keep;
        for (int i0 = 0; i0 < n; i0 += U) {
            if (i0) load(i0);
#pragma unroll
            for (int i = 0; i < U; i++) {
                const float fi = __shfl_sync(0xffffffffu, f, (i0 + i) & 31);
                if (i0 + i < n) {
#pragma unroll
                    for (int e = 0; e < V; e++) o[e] = fmaf(fi, y[i][e], o[e]);
                }
            }
        }
        M = top;
    }
}

// PROMPT: a job may hold several queries, the first of which see less than the last.
template <int HD, bool PROMPT>
__global__ void __launch_bounds__(kThreads, Geo<HD>::RESIDENT) decode_q8_kernel(const __grid_constant__ DecodeQ8Params p)
{
    using G = Geo<HD>;
    constexpr int PANELS = HD / 64;
    constexpr int NT = HD / 8;           // value tiles of eight channels
    constexpr int V = HD / 32;           // channels a lane holds of a merged row
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) uint64_t bars[kWarps * G::STAGES];
    __shared__ float m_s[kWarps][kRows], l_s[kWarps][kRows];
    __shared__ int last_s[2];
    __shared__ float2 part_s[kRows];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = p.heads / p.kv_heads;
    // Row `row` of a job: head row % group of the group, at its query row / group.
    auto row_at = [&](int seq, int head, int row) {
        const int pos = row / group;
        return ((long long)(p.seq[seq].row0 + pos) * p.heads + head * group + (row - pos * group)) * HD;
    };
    const int u_begin = p.cluster ? 0 : first_unit(p, (int)blockIdx.x);
    const int u_end = p.cluster ? 0 : first_unit(p, (int)blockIdx.x + 1);
    float *merge = (float *)(smem + G::RING);
    const uint32_t ring0 = smem_u32(smem) + (uint32_t)warp * (G::STAGES * G::STAGE);
    const uint32_t bar0 = smem_u32(&bars[warp * G::STAGES]);
    if (lane == 0) {
        for (int s = 0; s < G::STAGES; s++) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar0 + 8 * s));
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    const int r = lane >> 2, c = lane & 3;
    Run run = p.cluster ? run_of_rank(p) : run_at(p, u_begin, u_end);

    // What a run needs besides its blocks: the query (row r, the 16 channels of
    // chunk c in each panel), and of the tail the warp's eight tokens (keys: token
    // r, the same channels; values: V channels of each). It is asked for in front
    // of the blocks, and for the next run in front of this one's merge: behind a
    // full ring of blocks a load waits for all of them.
    float x[PANELS][16];
    uint4 tk[PANELS][2];
    uint2 tv[8];
    // The scales of the warp's next 32 blocks, a lane each (half of them ahead of
    // use, later on).
    float k_scale, v_scale, k_next = 0.0f, v_next = 0.0f;
    const float *ks, *vs;
    auto load_scales = [&](int blk, float &a, float &b) {
        blk += lane * kWarps;
        if (blk < run.last) {
            a = __ldcg(ks + blk);
            b = __ldcg(vs + blk);
        }
    };
    auto load_run = [&] {
        const DecodeQ8Seq &s = p.seq[run.seq];
        const Q8Layout at = q8_layout(p.kv_heads, HD, s.nb);
        ks = (const float *)(s.base + at.ks) + (long long)run.head * s.nb;
        vs = (const float *)(s.base + at.vs) + (long long)run.head * s.nb;
        load_scales(run.first + warp, k_scale, v_scale);
        const bool mine = r < group * s.n;
        const float *qr = p.q + row_at(run.seq, run.head, mine ? r : 0);
#pragma unroll
        for (int j = 0; j < PANELS; j++) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
                if (mine) y = __ldcg((const float4 *)(qr + 64 * j + 16 * c + 4 * i));
                x[j][4 * i] = y.x; x[j][4 * i + 1] = y.y; x[j][4 * i + 2] = y.z; x[j][4 * i + 3] = y.w;
            }
        }
        const int n = run.tail ? s.live - 32 * s.full - 8 * warp : 0;
        if (n > 0) {
            const uint16_t *kt = (const uint16_t *)(s.base + at.kt) + ((long long)run.head * kQ8Block + 8 * warp) * HD;
            const uint16_t *vt = (const uint16_t *)(s.base + at.vt) + ((long long)run.head * kQ8Block + 8 * warp) * HD;
#pragma unroll
            for (int i = 0; i < 2 * PANELS; i++) {
                tk[i / 2][i % 2] = r < n ? *(const uint4 *)(kt + r * HD + 64 * (i / 2) + 16 * c + 8 * (i % 2)) : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int t = 0; t < 8; t++) {
                tv[t] = make_uint2(0u, 0u);
                if (t < n) {
                    if (V == 4) tv[t] = *(const uint2 *)(vt + t * HD + V * lane);
                    else tv[t].x = *(const uint32_t *)(vt + t * HD + V * lane);
                }
            }
        }
    };

    // The warp's blocks in order, over all runs: `ahead` is what is fetched next.
    Run ahead = run;
    int ahead_blk = ahead.first + warp;
    const unsigned char *ahead_k, *ahead_v;      // of the head's first block
    auto aim = [&] {
        const DecodeQ8Seq &s = p.seq[ahead.seq];
        const Q8Layout at = q8_layout(p.kv_heads, HD, s.nb);
        const long long b = (long long)ahead.head * s.nb;
        ahead_k = s.base + at.k + b * G::BLOCK;
        ahead_v = s.base + at.v + b * G::BLOCK;
    };
    aim();

    // The next kernel of the stream may set itself up; nothing of the one before
    // is read until it has ended.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (p.cluster ? run.units == 0 : u_begin >= u_end) return;   // (a sequence of no tokens; a share that was all charges)
    load_run();

    int issued = 0, used = 0;
    auto skip_done = [&] {
        while (ahead_blk >= ahead.last && ahead.next < u_end) {
            ahead = run_at(p, ahead.next, u_end);
            ahead_blk = ahead.first + warp;
            aim();
        }
        return ahead_blk < ahead.last;
    };
    auto fetch = [&] {
        if (!skip_done()) return;
        if (lane == 0) {
            const int stage = issued % G::STAGES;
            const uint32_t dst = ring0 + (uint32_t)stage * G::STAGE, bar = bar0 + 8 * stage;
            const size_t off = (size_t)ahead_blk * G::BLOCK;
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(G::STAGE) : "memory");
            bulk_load(dst, ahead_k + off, G::BLOCK, bar);
            bulk_load(dst + G::BLOCK, ahead_v + off, G::BLOCK, bar);
        }
        issued++;
        ahead_blk += kWarps;
    };
    for (int s = 0; s < G::STAGES; s++) fetch();

    bool ok = true, is_first = true;
    Shared shared0 = {0, 0, 0, 0}, shared1 = {0, 0, 0, 0};       // of the first run and the last
    for (;;) {
        const DecodeQ8Seq &sq = p.seq[run.seq];
        const Q8Layout at = q8_layout(p.kv_heads, HD, sq.nb);

        const int rows = group * sq.n;
        // the last token that row r sees, and the last that all rows see
        const int lim = p.causal && r < rows ? sq.live - sq.n + r / group : sq.live - 1;
        const int lim_all = p.causal ? sq.live - sq.n : sq.live - 1;
        const int tail_n = run.tail ? min(8, sq.live - 32 * sq.full - 8 * warp) : 0;    // the warp's tokens
        // -- the query as fixed point
        uint32_t qa[PANELS][4], qb[PANELS][4];
        float f_q;
        {
            uint32_t most = 0;
#pragma unroll
            for (int j = 0; j < PANELS; j++) {
#pragma unroll
                for (int i = 0; i < 16; i++) most = max(most, __float_as_uint(x[j][i]) & 0x7fffffffu);
            }
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const float top = __uint_as_float(most);
            // (an infinity or NaN in the row makes every score NaN; a row of nothing
            // above 1e-30 scores nothing)
            const bool some = top > 1e-30f && most < 0x7f800000u;
            f_q = some ? top * (1.0f / 32639.0f) * p.sl2 : (most >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : 0.0f);
            const float inv = some ? 32639.0f / top : 0.0f;
#pragma unroll
            for (int j = 0; j < PANELS; j++) {
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    uint32_t z[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        z[i] = (uint32_t)(some ? max(-32639, min(32639, __float2int_rn(x[j][4 * w + i] * inv))) : 0);
                    }
                    // z = 256 H + L: L its low byte, signed, H what is left
                    qb[j][w] = __byte_perm(__byte_perm(z[0], z[1], 0x0040), __byte_perm(z[2], z[3], 0x0040), 0x5410);
                    qa[j][w] = __byte_perm(__byte_perm(z[0] + 128u, z[1] + 128u, 0x0051),
                                           __byte_perm(z[2] + 128u, z[3] + 128u, 0x0051), 0x5410);
                }
            }
        }

        // -- the warp's part of the tail: what its sums start from. The keys are f16 and
        // so is the query, as two parts again: x / f_q's top = hi + lo to 2^-22, hi as
        // rows 0-7 and lo as rows 8-15 of A, both in the lane that holds x already
        float m = -CUDART_INF_F, l = 0.0f;       // reference maximum of row r; this lane's part of the sum
        float acc[NT][2];
        if (tail_n > 0) {
            if constexpr (PROMPT) {
                // 0 times a value that a row may not see would be NaN if the value is not
                // finite: it becomes a zero behind a key of NaN, as in q8_unpack_kernel
                uint32_t odd = 0;
#pragma unroll
                for (int t = 0; t < 8; t++) {
                    if (__any_sync(0xffffffffu, not_finite(tv[t].x) || not_finite(tv[t].y))) {
                        odd |= 1u << t;
                        tv[t] = make_uint2(0u, 0u);
                    }
                }
                if (odd >> r & 1u) {
#pragma unroll
                    for (int i = 0; i < 2 * PANELS; i++) tk[i / 2][i % 2] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
                }
            }
            const float unit = f_q * 32639.0f, over = f_q != 0.0f ? p.sl2 / unit : 0.0f;   // sl2 top, 1 / top
            float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < PANELS; j++) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t a[4];
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const float y0 = x[j][4 * k + 2 * i] * over, y1 = x[j][4 * k + 2 * i + 1] * over;
                        const __half2 hi = __floats2half2_rn(y0, y1);
                        const __half2 lo = __floats2half2_rn(y0 - __low2float(hi), y1 - __high2float(hi));
                        a[2 * i] = *(const uint32_t *)&hi;
                        a[2 * i + 1] = *(const uint32_t *)&lo;
                    }
                    const uint4 kk = tk[j][k / 2];
                    mma_f16(d, a[0], a[1], a[2], a[3], k % 2 ? kk.z : kk.x, k % 2 ? kk.w : kk.y);
                }
            }
            // row r against tokens 2 c and 2 c + 1
            const int seen = min(tail_n, lim + 1 - 32 * sq.full - 8 * warp);      // of the warp's tokens
            const float s0 = 2 * c < seen ? (d[0] + d[2]) * unit : -CUDART_INF_F;
            const float s1 = 2 * c + 1 < seen ? (d[1] + d[3]) * unit : -CUDART_INF_F;
            m = fmaxf(s0, s1);
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            const float e0 = 2 * c < seen ? ex2(s0 - m) : 0.0f, e1 = 2 * c + 1 < seen ? ex2(s1 - m) : 0.0f;
            l = e0 + e1;
            float *mine = merge + warp * kRows * HD;
            for (int g = 0; g < rows; g++) {
                float o4[V];
#pragma unroll
                for (int i = 0; i < V; i++) o4[i] = 0.0f;
#pragma unroll
                for (int t = 0; t < 8; t++) {
                    const float w = __shfl_sync(0xffffffffu, t % 2 ? e1 : e0, 4 * g + t / 2);
                    const float2 v0 = __half22float2(*(const __half2 *)&tv[t].x);
                    o4[0] = fmaf(w, v0.x, o4[0]);
                    o4[1] = fmaf(w, v0.y, o4[1]);
                    if (V == 4) {
                        const float2 v1 = __half22float2(*(const __half2 *)&tv[t].y);
                        o4[V - 2] = fmaf(w, v1.x, o4[V - 2]);
                        o4[V - 1] = fmaf(w, v1.y, o4[V - 1]);
                    }
                }
                // channels V lane .. of row g, where the fragment layout finds them
#pragma unroll
                for (int i = 0; i < V; i++) mine[g * HD + 8 * ((V * lane / 8) ^ g) + V * lane % 8 + i] = o4[i];
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < NT; i++) {
                const float2 y = r < rows ? *(const float2 *)(mine + r * HD + 8 * (i ^ r) + 2 * c) : make_float2(0.f, 0.f);
                acc[i][0] = y.x;
                acc[i][1] = y.y;
            }
            __syncwarp();
        } else {
#pragma unroll
            for (int i = 0; i < NT; i++) acc[i][0] = acc[i][1] = 0.0f;
        }

        // -- the warp's blocks
        for (int blk = ok ? run.first + warp : run.last; blk < run.last; blk += kWarps) {
            const int stage = used % G::STAGES;
            const uint32_t kb = ring0 + (uint32_t)stage * G::STAGE, vb = kb + G::BLOCK;
            // (given up, the stage's copy may still be in flight, and its barrier in the
            // phase it was armed for: the warp takes and asks for no more blocks)
            ok = ring_wait(bar0 + 8 * stage, (uint32_t)(used / G::STAGES) & 1u, p.status, p.wait_cycles);
            if (!ok) break;
            used++;
            // scores: column n of tile t is token 8 (n / 2) + 2 t + n % 2
            float s[8];
            float mb = -CUDART_INF_F;
            const int turn = (blk - run.first - warp) / kWarps & 31;
            const float sk = __shfl_sync(0xffffffffu, k_scale, turn);
            float sv = __shfl_sync(0xffffffffu, v_scale, turn);
            if (turn == 15) load_scales(blk + 17 * kWarps, k_next, v_next);
            if (turn == 31) {
                k_scale = k_next;
                v_scale = v_next;
            }
            const float f = f_q * sk;
#pragma unroll
            for (int t = 0; t < 4; t++) {
                int d[4] = {0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < PANELS; j++) {
                    const uint32_t src = kb + (uint32_t)(j * (kQ8Block * 64) + (8 * (r >> 1) + 2 * t + (r & 1)) * 64 + c * 16);
                    uint32_t b0, b1, b2, b3;
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(b0), "=r"(b1), "=r"(b2), "=r"(b3) : "r"(src) : "memory");
                    mma_s8(d, qa[j][0], qb[j][0], qa[j][1], qb[j][1], b0, b1);
                    mma_s8(d, qa[j][2], qb[j][2], qa[j][3], qb[j][3], b2, b3);
                }
                s[2 * t] = (float)(d[0] * 256 + d[2]) * f;          // token 8 c + 2 t of row r
                s[2 * t + 1] = (float)(d[1] * 256 + d[3]) * f;      // and the next
            }
            if (32 * blk + 31 > lim_all) {
                // (a block among a prompt's own rows: the first of them may see nothing of it)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (32 * blk + 8 * c + i > lim) s[i] = -CUDART_INF_F;
                }
                if (PROMPT && 32 * blk > lim) sv = 0.0f;     // (and the block may be of NaN)
            }
#pragma unroll
            for (int i = 0; i < 8; i++) mb = fmaxf(mb, s[i]);
            mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, 1));
            mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, 2));
            // The reference moves only when a block's maximum is far above it
            // (2^16 times): f32 has room for the rest.
            if (__any_sync(0xffffffffu, mb > m + 16.0f)) {
                const float to = mb > m + 16.0f ? mb : m;
                const float a = m == -CUDART_INF_F ? 0.0f : ex2(m - to);
                l *= a;
#pragma unroll
                for (int i = 0; i < NT; i++) {
                    acc[i][0] *= a;
                    acc[i][1] *= a;
                }
                m = to;
            }
            const bool seen = mb != -CUDART_INF_F;
            const float top = seen ? mb : 0.0f;
            float sum = 0.0f;
            uint32_t z[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float e = ex2(s[i] - top);
                sum += e;
                z[i] = __float_as_uint(fmaf(e, 65535.0f, 8388608.0f));
            }
            const float beta = seen ? ex2(mb - m) : 0.0f;
            l = fmaf(beta, sum, l);
            if (p.stats) {
                float whole = sum;
                whole += __shfl_xor_sync(0xffffffffu, whole, 1);
                whole += __shfl_xor_sync(0xffffffffu, whole, 2);
                if (c == 0) {
                    p.stats[(p.stat0[run.seq] + (long long)run.head * sq.full + blk) * kRows + r] = make_float2(mb, whole);
                }
            }
            uint32_t a_hi[2], a_lo[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t x = __byte_perm(z[4 * i], z[4 * i + 1], 0x5410), y = __byte_perm(z[4 * i + 2], z[4 * i + 3], 0x5410);
                a_hi[i] = __byte_perm(x, y, 0x7531);
                a_lo[i] = __byte_perm(x, y, 0x6420);
            }
            const float w = beta * sv * (1.0f / 65535.0f);
#pragma unroll
            for (int i = 0; i < NT; i++) {
                int d[4] = {0, 0, 0, 0};
                uint32_t b0, b1;
                asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(b0), "=r"(b1) : "r"(vb + (uint32_t)((8 * i + r) * kQ8Block + 8 * c)) : "memory");
                mma_u8(d, a_hi[0], a_lo[0], a_hi[1], a_lo[1], b0, b1);
                acc[i][0] = fmaf((float)(d[0] * 256 + d[2]), w, acc[i][0]);
                acc[i][1] = fmaf((float)(d[1] * 256 + d[3]), w, acc[i][1]);
            }
            __syncwarp();   // every lane has read the stage
            fetch();
        }

        // the next run's query and tail are on their way under the merge
        const Run now = run;
        const bool more = now.next < u_end;
        if (more) {
            run = run_at(p, now.next, u_end);
            load_run();
        }

        // -- the run's result: a warp merges rows warp, warp + kWarps of the block's warps'
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (c == 0) {
            m_s[warp][r] = m;
            l_s[warp][r] = l;
        }
        if (r < rows) {
#pragma unroll
            for (int i = 0; i < NT; i++) {
                // (groups of eight channels swizzled by the row: no bank conflicts on either side)
                *(float2 *)(merge + (warp * kRows + r) * HD + 8 * (i ^ r) + 2 * c) = make_float2(acc[i][0], acc[i][1]);
            }
        }
        __syncthreads();
        const int slot = (int)blockIdx.x * 2 + (is_first ? 0 : 1);
        for (int row = warp; row < rows; row += kWarps) {
            float M = -CUDART_INF_F, L = 0.0f, o[V];
#pragma unroll
            for (int e = 0; e < V; e++) o[e] = 0.0f;
#pragma unroll
            for (int k = 0; k < kWarps; k++) M = fmaxf(M, m_s[k][row]);
#pragma unroll
            for (int k = 0; k < kWarps; k++) {
                const float mk = m_s[k][row];
                const float fk = mk == -CUDART_INF_F ? 0.0f : ex2(mk - M);
                L = fmaf(fk, l_s[k][row], L);
#pragma unroll
                for (int e = 0; e < V; e++) {
                    o[e] = fmaf(fk, merge[(k * kRows + row) * HD + 8 * ((V * lane / 8) ^ row) + V * lane % 8 + e], o[e]);
                }
            }
            if (now.whole) {
                const float inv = 1.0f / L;
#pragma unroll
                for (int e = 0; e < V; e++) o[e] *= inv;
                store_row<HD>(p, row_at(now.seq, now.head, row), lane, o);
                if (p.stats && lane == 0) p.fin[((long long)now.seq * p.kv_heads + now.head) * kRows + row] = make_float2(M, inv);
            } else if (p.cluster) {
                // (the ring is empty: there is no other run)
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    *(float2 *)((float *)smem + row * HD + V * lane + e) = make_float2(o[e], o[e + 1]);
                }
                if (lane == 0) part_s[row] = make_float2(M, L);
            } else {
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    *(float2 *)(p.part_o + ((long long)slot * kRows + row) * HD + V * lane + e) = make_float2(o[e], o[e + 1]);
                }
                if (lane == 0) p.part_ml[slot * kRows + row] = make_float2(M, L);
            }
        }
        if (!now.whole) {
            if (is_first) shared0 = {now.seq, now.head, now.begin, now.units};
            else shared1 = {now.seq, now.head, now.begin, now.units};
        }
        if (!more) break;
        is_first = false;
        __syncthreads();   // merge and m_s are free again
    }

    if (p.cluster > 1) {
        // -- by cluster: the blocks' results meet through distributed shared memory, row
        // k of them merged by the block of rank k mod the cluster's size
        const int rank = (int)blockIdx.x % p.cluster, rows = group * p.seq[run.seq].n;
        cluster_sync();
        for (int i = warp; rank + i * p.cluster < rows; i += kWarps) {
            const int row = rank + i * p.cluster;
            const uint32_t ml_at = smem_u32(&part_s[row]), o_at = smem_u32(smem) + (uint32_t)(row * HD + V * lane) * 4;
            float M = -CUDART_INF_F, L = 0.0f, o[V];
#pragma unroll
            for (int e = 0; e < V; e++) o[e] = 0.0f;
            for (int k0 = 0; k0 < p.cluster; k0 += 8) {
                float2 ml[8], y[8][V / 2];
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    if (k0 + k < p.cluster) {
                        ml[k] = peer_f2(peer(ml_at, k0 + k));
#pragma unroll
                        for (int e = 0; e < V / 2; e++) y[k][e] = peer_f2(peer(o_at, k0 + k) + 8 * e);
                    }
                }
                float top = M;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    if (k0 + k < p.cluster) top = fmaxf(top, ml[k].x);
                }
                const float keep = M == -CUDART_INF_F ? 0.0f : ex2(M - top);
                L *= keep;
#pragma unroll
                for (int e = 0; e < V; e++) o[e] *= keep;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    if (k0 + k < p.cluster) {
                        const float f = ml[k].x == -CUDART_INF_F ? 0.0f : ex2(ml[k].x - top);
                        L = fmaf(f, ml[k].y, L);
#pragma unroll
                        for (int e = 0; e < V / 2; e++) {
                            o[2 * e] = fmaf(f, y[k][e].x, o[2 * e]);
                            o[2 * e + 1] = fmaf(f, y[k][e].y, o[2 * e + 1]);
                        }
                    }
                }
                M = top;
            }
            if (p.parts > 1) {
                // a row of a pair that several clusters share: the last to arrive merges
                // them, in their order whoever came last
                const int cluster = (int)blockIdx.x / p.cluster, pair = cluster / p.parts;
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    *(float2 *)(p.part_o + ((long long)cluster * kRows + row) * HD + V * lane + e) = make_float2(o[e], o[e + 1]);
                }
                if (lane == 0) p.part_ml[cluster * kRows + row] = make_float2(M, L);
                __threadfence();
                __syncwarp();
                unsigned seen = 0;
                if (lane == 0) {
                    unsigned *ctr = &p.ctr[pair * kRows + row];
                    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(seen) : "l"(ctr) : "memory");
                    if (seen == (unsigned)(p.parts - 1)) *ctr = 0u;
                }
                seen = __shfl_sync(0xffffffffu, seen, 0);
                if (seen != (unsigned)(p.parts - 1)) continue;
                __threadfence();
                merge_parts<HD>(p, lane, p.parts, pair * p.parts, 1, 0, row, M, L, o);
            }
            const float inv = 1.0f / L;
#pragma unroll
            for (int e = 0; e < V; e++) o[e] *= inv;
            store_row<HD>(p, row_at(run.seq, run.head, row), lane, o);
            if (p.stats && lane == 0) p.fin[((long long)run.seq * p.kv_heads + run.head) * kRows + row] = make_float2(M, inv);
        }
        cluster_sync();   // no block leaves while another reads its results
        if (!ok) {
            for (int i = 0; i < 64; i++) __nanosleep(1000);
        }
        return;
    }

    // -- pairs shared with other blocks of the grid (the first run's and the last's,
    // at most): the last to arrive merges. All arrivals wait until the block's own
    // work is done: an arrival takes as long as the memory is busy.
    __syncthreads();
    if (tid < 2) {
        last_s[tid] = 0;
        const Shared now = pick(tid != 0, shared0, shared1);
        if (now.units > 0) {
            const int pair = now.seq * p.kv_heads + now.head;
            const int b0 = block_of(p, now.begin, pair), b1 = block_of(p, now.begin + now.units - 1, pair);
            // (releases what the barrier ordered before it, acquires the others')
            unsigned *ctr = &p.ctr[pair], seen;
            asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(seen) : "l"(ctr) : "memory");
            last_s[tid] = seen == (unsigned)(b1 - b0);
            if (last_s[tid]) *ctr = 0u;
        }
    }
    __syncthreads();
    // (a warp takes a row of either pair)
    for (int item = warp; item < 2 * kRows; item += kWarps) {
        const int row = item % kRows;
        const Shared now = pick(item >= kRows, shared0, shared1);
        if (!last_s[item >= kRows] || row >= group * p.seq[now.seq].n) continue;
        const int pair = now.seq * p.kv_heads + now.head;
        const int b0 = block_of(p, now.begin, pair), b1 = block_of(p, now.begin + now.units - 1, pair);
        // The contributors in order, whoever came last: the same bits every time. A
        // block's first run has slot 0, and only b0 may hold the pair in its last.
        const int skew = first_unit(p, b0) >= now.begin ? 0 : 1;
        float M, L, o[V];
        merge_parts<HD>(p, lane, b1 + 1 - b0, 2 * b0, 2, skew, row, M, L, o);
        const float inv = 1.0f / L;
#pragma unroll
        for (int e = 0; e < V; e++) o[e] *= inv;
        store_row<HD>(p, row_at(now.seq, now.head, row), lane, o);
        if (p.stats && lane == 0) p.fin[(long long)pair * kRows + row] = make_float2(M, inv);
    }
    if (!ok) {
        // a wait gave up: leave the copies still in flight time to land
        for (int i = 0; i < 64; i++) __nanosleep(1000);
    }
}

// The weights, behind the decode kernel: what the tokens of each complete block got,
// summed over the group's heads, from the block's maximum and sum of each row (in
// `stats`) and the row's own (in `fin`). A thread a cache block, bound by the latency of
// its 64 bytes: with this work in the decode kernel, done for a pair by whichever block
// finished it, 4 x 131072 tokens of 4 KV heads x 128 took 134 us; they take 95, and 86
// without weights. (The next kernel may start once the decode is over, no earlier: a
// decode set up among these blocks is spread badly over the SMs, 66 us for 49 with 30 x
// 15000 tokens of 4 KV heads x 64.)
constexpr int kWeighThreads = 128;
constexpr int kGridRows = 65535;     // a grid has no more (and as many layers): reached at 2^28 tokens
template <int HD>
__global__ void __launch_bounds__(kWeighThreads) q8_weigh_kernel(const __grid_constant__ DecodeQ8Params p)
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int pair = (int)blockIdx.x, seq = pair / p.kv_heads, head = pair - seq * p.kv_heads, group = p.heads / p.kv_heads;
    const DecodeQ8Seq &sq = p.seq[seq];
    const int b = (int)(blockIdx.z * kGridRows + blockIdx.y) * kWeighThreads + (int)threadIdx.x;
    if (b >= sq.full) return;
    const Q8Layout at = q8_layout(p.kv_heads, HD, sq.nb);
    float *weight = (float *)(sq.base + at.w) + (long long)head * sq.nb + b;
    const float2 *st = p.stats + (p.stat0[seq] + (long long)head * sq.full + b) * kRows, *f = p.fin + (long long)pair * kRows;
    float2 y[kRows], z[kRows];
    const float before = *weight;
#pragma unroll
    for (int k = 0; k < kRows; k++) {
        y[k] = k < group ? st[k] : make_float2(0.f, 0.f);
        z[k] = k < group ? f[k] : make_float2(0.f, 0.f);
    }
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kRows; k++) {
        if (k < group) sum = fmaf(ex2(y[k].x - z[k].x) * z[k].y, y[k].y, sum);
    }
    *weight = before + sum;
}

// Sequences that hold no token: zeros.
__global__ void q8_zero_rows_kernel(const __grid_constant__ DecodeQ8Params p, int width)
{
    if (p.seq[blockIdx.x].live) return;
    for (int i = threadIdx.x; i < width; i += blockDim.x) {
        const long long at = (long long)p.seq[blockIdx.x].row0 * width + i;
        if (p.out_f16) ((uint16_t *)p.out)[at] = 0;
        else ((float *)p.out)[at] = 0.0f;
    }
}

const KernelReg reg128("decode_q8_128", (const void *)decode_q8_kernel<128, false>);
const KernelReg reg64("decode_q8_64", (const void *)decode_q8_kernel<64, false>);

}  // namespace

// Once a device: what the kernels may take of it, and how many clusters of 8 and
// of 16 blocks it holds at once.
static cudaError_t configure(int dev, int hd, int (**resident)[2])
{
    static bool done[64] = {false};
    static int clusters[64][2][2];
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!done[dev]) {
        const void *kernel[4] = {(const void *)decode_q8_kernel<128, false>, (const void *)decode_q8_kernel<64, false>,
                                 (const void *)decode_q8_kernel<128, true>, (const void *)decode_q8_kernel<64, true>};
        const int smem[4] = {Geo<128>::SMEM, Geo<64>::SMEM, Geo<128>::SMEM, Geo<64>::SMEM};
        for (int i = 0; i < 4; i++) {
            cudaError_t e = cudaFuncSetAttribute(kernel[i], cudaFuncAttributeMaxDynamicSharedMemorySize, smem[i]);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel[i], cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) return e;
            for (int c = 0; c < 2 && i < 2; c++) {           // (the others take as much of an SM)
                cudaLaunchConfig_t cfg = {};
                cudaLaunchAttribute attr[1];
                cfg.gridDim = dim3(c ? 16 : 8);
                cfg.blockDim = dim3(kThreads);
                cfg.dynamicSmemBytes = (size_t)smem[i];
                attr[0].id = cudaLaunchAttributeClusterDimension;
                attr[0].val.clusterDim.x = c ? 16 : 8;
                attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
                cfg.attrs = attr;
                cfg.numAttrs = 1;
                if (cudaOccupancyMaxActiveClusters(&clusters[dev][i][c], kernel[i], &cfg) != cudaSuccess) {
                    cudaGetLastError();
                    clusters[dev][i][c] = 0;
                }
            }
        }
        done[dev] = true;
    }
    if (resident) *resident = &clusters[dev][hd == 128 ? 0 : 1];
    return cudaSuccess;
}

cudaError_t launch_decode_q8(cudaStream_t st, const DecodeQ8Params &p, int hd, int grid)
{
    int dev = 0;
    cudaGetDevice(&dev);
    const cudaError_t ce = configure(dev, hd, nullptr);
    if (ce != cudaSuccess) return ce;
    bool empty = false, prompt = false;
    for (int b = 0; b < p.nseq; b++) {
        empty = empty || p.seq[b].live == 0;
        prompt = prompt || (p.causal && p.seq[b].n > 1);
    }
    if (empty) {
        q8_zero_rows_kernel<<<p.nseq, 256, 0, st>>>(p, p.heads * hd);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
    }
    if (grid == 0) return cudaSuccess;
    const dim3 blocks((unsigned)grid);
    const auto kernel = hd == 128 ? (prompt ? decode_q8_kernel<128, true> : decode_q8_kernel<128, false>)
                                  : (prompt ? decode_q8_kernel<64, true> : decode_q8_kernel<64, false>);
    const cudaError_t e = launch_dependent(st, blocks, kThreads, hd == 128 ? Geo<128>::SMEM : Geo<64>::SMEM, p.cluster, kernel, p);
    if (e != cudaSuccess || !p.stats) return e;
    int most = 0;
    for (int b = 0; b < p.nseq; b++) most = std::max(most, p.seq[b].full);
    const int rows = (most + kWeighThreads - 1) / kWeighThreads;
    const dim3 all((unsigned)(p.nseq * p.kv_heads), (unsigned)std::min(rows, kGridRows), (unsigned)((rows + kGridRows - 1) / kGridRows));
    return hd == 128 ? launch_dependent(st, all, kWeighThreads, 0, 1, q8_weigh_kernel<128>, p)
                     : launch_dependent(st, all, kWeighThreads, 0, 1, q8_weigh_kernel<64>, p);
}

void plan_decode_q8(DecodeQ8Plan &plan, const int *units, int n, int kv_heads, int hd, int sm_count, const int *clusters)
{
    // Microseconds, as measured (148 SMs): cache blocks a microsecond that the memory
    // gives (6.9 TB/s), a warp's time for one when nothing but the warp itself bounds
    // it, and what a launch costs besides: by a cluster of 1, 2, 4, 8 or 16 blocks of
    // the grid (the last are packed onto half as many SMs), by the cut (whose merge
    // goes through memory, and is long where many blocks share a pair: short
    // launches, and 0.1 us for each block beyond 32), by several clusters a pair, and
    // for a further wave of blocks of the grid.
    const double all = (hd == 128 ? 842.0 : 1684.0) * sm_count / 148, one = hd == 128 ? 0.7 : 0.6;
    constexpr double kCluster[5] = {4.0, 4.5, 5.0, 5.4, 6.3}, kPacked = 1.15, kCut = 7.0, kShort = 16.0, kWave = 3.5,
                     kJoin = 0.1, kParts = 8.3, kPart = 0.11;
    const int most = sm_count * (hd == 128 ? Geo<128>::RESIDENT : Geo<64>::RESIDENT);
    long long total = 0, longest = 0;
    for (int i = 0; i < n; i++) {
        total += (long long)units[i] * kv_heads;
        longest = std::max<long long>(longest, units[i]);
    }
    const long long pairs = (long long)n * kv_heads;
    plan = DecodeQ8Plan{0, 0, 1, 0, 0.0};
    if (total == 0) return;
    // the cut by work: never fewer than four cache blocks, one a warp, for a block of
    // the grid; where a launch is short, as many that what the warps take in turn (0.5
    // us each) and what the merge takes for each block that a pair is spread over (0.04
    // us) is least. Where it is long a run is charged for what it costs besides its
    // cache blocks, about 16 of them.
    long long grid = most;
    int over = 16;
    if (total < 8ll * most) {
        double best = 0.0;
        for (int k = 1; k <= 32; k++) {
            const long long blocks = (total + 4 * k - 1) / (4 * k);
            const double cost = 0.5 * k + 0.04 * (double)blocks / (double)pairs;
            if (blocks <= most && (best == 0.0 || cost < best)) {
                best = cost;
                grid = blocks;
            }
        }
        over = 0;
    }
    const long long share = (total + grid - 1) / grid;
    const double joined = kJoin * std::max(0.0, (double)grid / (double)pairs - 32.0);
    plan = DecodeQ8Plan{(int)grid, 0, 1, over, (over ? kCut : kShort) + std::max((double)total / all, one * (double)((share + 3) / 4)) + joined};
    for (int i = 0, c = 1; i < 5; i++, c *= 2) {
        const long long blocks = pairs * c;
        if (c > 1 && blocks > most) break;
        if (c >= 8 && clusters[c == 16] < pairs) break;
        const double waves = (double)((blocks + most - 1) / most), part = std::max(1.0, (double)blocks / most);
        const double own = one * (double)(((longest + c - 1) / c + 3) / 4) * (c == 16 ? kPacked : 1.0);
        const double cost = kCluster[i] + kWave * (waves - 1.0) + std::max((double)total / all * waves / part, own * waves);
        if (cost < plan.us && blocks <= 0x7fffffff) plan = DecodeQ8Plan{(int)blocks, c, 1, 0, cost};
    }
    // Several clusters of eight for a pair, as many as the device holds at once, and
    // none of them without a block. 131072 tokens, one KV head x 128: 16 us by 29 clusters, 45 by the
    // cut, whose last block has 296 results to merge; 8000 tokens: 12 us by all of them,
    // 9 by one of 16.
    for (long long parts = 2; parts <= 32 && pairs * parts <= clusters[0] && parts * 8 <= longest; parts++) {
        const long long blocks = pairs * parts * 8;
        const double own = one * (double)(((longest + 8 * parts - 1) / (8 * parts) + 3) / 4);
        const double cost = kParts + kPart * (double)parts + std::max((double)total / all * std::max(1.0, 0.8 * most / (double)blocks), own);
        if (cost < plan.us) plan = DecodeQ8Plan{(int)blocks, 8, (int)parts, 0, cost};
    }
}

cudaError_t decode_q8_clusters(int hd, int (&clusters)[2])
{
    int dev = 0;
    cudaGetDevice(&dev);
    int(*held)[2];
    const cudaError_t e = configure(dev, hd, &held);
    if (e == cudaSuccess) {
        clusters[0] = (*held)[0];
        clusters[1] = (*held)[1];
    }
    return e;
}
