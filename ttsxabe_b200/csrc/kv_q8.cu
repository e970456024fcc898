// The movers of the 8-bit KV cache: rows rotated and appended, read back,
// unpacked for the prefill kernel, a cut block put back into the tail, and the
// eviction of blocks by accumulated attention weight.
#include "kv_q8.cuh"

#include <algorithm>

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// Four int8 codes of one word as floats, exactly: a byte biased to unsigned in
// the low mantissa byte of 2^23 is 2^23 + code + 128.
__device__ __forceinline__ void codes_f32(uint32_t w, float (&f)[4])
{
    const uint32_t u = w ^ 0x80808080u;
    f[0] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)) - 8388736.0f;
    f[1] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441)) - 8388736.0f;
    f[2] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442)) - 8388736.0f;
    f[3] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443)) - 8388736.0f;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// The values four codes stand for, rounded to f16.
__device__ __forceinline__ uint2 dequant4(uint32_t w, float scale)
{
    float f[4];
    codes_f32(w, f);
    return make_uint2(pack_half2(f[0] * scale, f[1] * scale), pack_half2(f[2] * scale, f[3] * scale));
}

// A 4 x 4 byte transpose: byte j of r[i] <-> byte i of r[j].
__device__ __forceinline__ void transpose4(uint32_t (&r)[4])
{
    const uint32_t a = __byte_perm(r[0], r[1], 0x5140), b = __byte_perm(r[2], r[3], 0x5140);
    const uint32_t c = __byte_perm(r[0], r[1], 0x7362), d = __byte_perm(r[2], r[3], 0x7362);
    r[0] = __byte_perm(a, b, 0x5410);
    r[1] = __byte_perm(a, b, 0x7632);
    r[2] = __byte_perm(c, d, 0x5410);
    r[3] = __byte_perm(c, d, 0x7632);
}

// The last sequence whose first work item is at or before `item`.
template <typename Seq>
__device__ __forceinline__ int seq_of(const Seq *seq, int nseq, int item)
{
    int lo = 0, hi = nseq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (seq[mid].item0 <= item) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// A kernel of this file may be set up while the one before it in the stream
// still runs; nothing is read or written before that one has ended.
__device__ __forceinline__ void after_previous()
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---- append -------------------------------------------------------------------------
//
// A block of the grid takes the up to 32 new rows of one cache block for a
// chunk of heads: blockIdx.y runs over the chunks of key heads (rotated, then
// quantised or put into the tail), of value heads (the same without the
// rotation), and of query heads (rotated only). The sines and cosines of those
// rows are worked out once, into shared memory, and shared by the chunk's
// heads; the angle is pos * inv_freq[j] in 64 bits, taken in half turns and
// reduced before it is rounded to f32, so that far positions lose nothing.
//
// Bound by memory on long prompts (8192 rows of 32 + 8 + 8 heads x 128: 352 MB in
// 67 us, 5.2 TB/s; the sines are a third of the instructions), by one trip to
// memory and the launch on single rows (2.7 us behind another kernel).
//
// The sequence's first work item also writes its last, incomplete block: the
// tail holds the first rows of the one and receives the rows of the other, and
// one block of the grid does both in order.
template <int HD>
__global__ void __launch_bounds__(kThreads, 3) q8_append_kernel(const __grid_constant__ Q8AppendParams p)
{
    constexpr int LPR = HD / 8;                  // lanes of a row, each with four values of either half
    constexpr int RPW = 32 / LPR;                // rows a warp loads at once
    constexpr int ITER = kQ8Block / (kWarps * RPW);
    constexpr int HALF = HD / 2;
    constexpr int SW = HD / 4 + 1;               // words of a staged row, padded
    __shared__ float2 turn[kQ8Block][HALF];      // (cosine, sine)
    __shared__ uint32_t stage[kQ8Block * SW];
    __shared__ uint32_t red[2][kWarps];

    const int item = blockIdx.x;
    const Q8AppendSeq sq = p.seq[seq_of(p.seq, p.nseq, item)];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int kv_chunks = (p.kv_heads + p.kv_chunk - 1) / p.kv_chunk;
    const bool is_q = (int)blockIdx.y >= 2 * kv_chunks;
    const int which = !is_q && (int)blockIdx.y >= kv_chunks ? 1 : 0;        // values, not keys
    const bool turns = p.inv_freq != nullptr && !which;
    const int r = sq.past & 31;                  // rows of the first block that lie in the tail
    const int total = r + sq.n;
    const int nblk = (total + 31) >> 5;
    const int mine = item - sq.item0;
    const bool rest = mine == 0 && nblk > 1 && (total & 31) != 0;   // the last block too
    const Q8Layout at = q8_layout(p.kv_heads, HD, sq.nb);
    const int c = lane % LPR;
    after_previous();

    for (int pass = 0; pass < (rest ? 2 : 1); pass++) {
        const int j = pass ? nblk - 1 : mine;
        const int t_lo = j == 0 ? r : 0;                       // new rows of this block: [t_lo, t_hi)
        const int t_hi = min(32, total - 32 * j);
        const long long row_of = (long long)sq.row0 + 32 * j - r;   // + t: its packed row
        __syncthreads();   // the pass before is done with `turn`, and with the tail rows it read
        auto fill_turns = [&] {
            const int f = tid % HALF;
            const double each = (double)p.inv_freq[f] * 0.31830988618379067154;
            for (int t = t_lo + tid / HALF; t < t_hi; t += kThreads / HALF) {
                const double half_turns = (double)(sq.pos + 32 * j - r + t) * each;
                float sn, cs;
                sincospif((float)(half_turns - 2.0 * rint(0.5 * half_turns)), &sn, &cs);
                turn[t][f] = make_float2(cs, sn);
            }
            __syncthreads();
        };
        auto rotate4 = [&](int t, float4 &a, float4 &b) {
            const float4 w0 = *(const float4 *)&turn[t][4 * c], w1 = *(const float4 *)&turn[t][4 * c + 2];
            float4 lo, hi;
            rope_rotate(a.x, b.x, w0.x, w0.y, lo.x, hi.x);
            rope_rotate(a.y, b.y, w0.z, w0.w, lo.y, hi.y);
            rope_rotate(a.z, b.z, w1.x, w1.y, lo.z, hi.z);
            rope_rotate(a.w, b.w, w1.z, w1.w, lo.w, hi.w);
            a = lo;
            b = hi;
        };
        if (is_q) {
            const int h0 = ((int)blockIdx.y - 2 * kv_chunks) << p.q_log, mask = (1 << p.q_log) - 1;
            const int rows = (t_hi - t_lo) << p.q_log;
            constexpr int U = 4;                               // rows in flight
            constexpr int STEP = kWarps * RPW;
            const long long base = ((row_of + t_lo) * p.heads + h0) * HD + 4 * c;
            bool ready = false;
            for (int i0 = warp * RPW + lane / LPR; !ready || i0 < rows; i0 += U * STEP) {
                float4 a[U], b[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int i = i0 + u * STEP, h = i & mask;
                    if (i < rows && h0 + h < p.heads) {
                        const float *x = p.q + base + ((long long)(i >> p.q_log) * p.heads + h) * HD;
                        a[u] = *(const float4 *)x;
                        b[u] = *(const float4 *)(x + HALF);
                    }
                }
                if (!ready) {                                  // (the first rows are on their way meanwhile)
                    fill_turns();
                    ready = true;
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int i = i0 + u * STEP, h = i & mask;
                    if (i < rows && h0 + h < p.heads) {
                        rotate4(t_lo + (i >> p.q_log), a[u], b[u]);
                        float *y = p.q_out + base + ((long long)(i >> p.q_log) * p.heads + h) * HD;
                        *(float4 *)y = a[u];
                        *(float4 *)(y + HALF) = b[u];
                    }
                }
            }
            continue;
        }
        const int blk = (sq.past >> 5) + j;
        const bool complete = 32 * (j + 1) <= total;
        const float *src = which ? p.v : p.k;
        const int h0 = ((int)blockIdx.y - (which ? kv_chunks : 0)) * p.kv_chunk;
        const int h1 = min(p.kv_heads, h0 + p.kv_chunk);
        float4 a[ITER], b[ITER];
        auto load = [&](int h) {
#pragma unroll
            for (int it = 0; it < ITER; it++) {
                const int t = (warp * ITER + it) * RPW + lane / LPR;
                if (t >= t_lo && t < t_hi) {
                    const float *x = src + ((row_of + t) * p.kv_heads + h) * HD + 4 * c;
                    a[it] = *(const float4 *)x;
                    b[it] = *(const float4 *)(x + HALF);
                }
            }
        };
        load(h0);
        if (turns) fill_turns();
        for (int h = h0; h < h1; h++) {
            uint16_t *tail = (uint16_t *)(sq.base + (which ? at.vt : at.kt)) + (long long)h * kQ8Block * HD;
            __half2 x[ITER][4];                                // two halves of the row, four values each
            uint32_t most = 0;
#pragma unroll
            for (int it = 0; it < ITER; it++) {
                const int t = (warp * ITER + it) * RPW + lane / LPR;
                uint2 lo16 = make_uint2(0u, 0u), hi16 = lo16;
                if (t >= t_lo && t < t_hi) {
                    if (turns) rotate4(t, a[it], b[it]);
                    lo16 = make_uint2(pack_half2(a[it].x, a[it].y), pack_half2(a[it].z, a[it].w));
                    hi16 = make_uint2(pack_half2(b[it].x, b[it].y), pack_half2(b[it].z, b[it].w));
                    if (!complete) {
                        *(uint2 *)(tail + t * HD + 4 * c) = lo16;
                        *(uint2 *)(tail + t * HD + HALF + 4 * c) = hi16;
                    }
                } else if (complete) {                         // (t < t_lo: a row of the tail)
                    lo16 = *(const uint2 *)(tail + t * HD + 4 * c);
                    hi16 = *(const uint2 *)(tail + t * HD + HALF + 4 * c);
                }
                const uint32_t w[4] = {lo16.x, lo16.y, hi16.x, hi16.y};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    x[it][i] = *(const __half2 *)&w[i];
                    most = max(most, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
                }
            }
            if (h + 1 < h1) load(h + 1);                       // (under this head's arithmetic)
            if (!complete) continue;
            most = __reduce_max_sync(0xffffffffu, most);
            if (lane == 0) red[h & 1][warp] = most;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kWarps; i++) most = max(most, red[h & 1][i]);
            // A block that holds an infinity or NaN reads back as NaN throughout.
            const float top = __half2float(__ushort_as_half((uint16_t)most));
            const float scale = most >= 0x7c00u ? __uint_as_float(0x7fffffffu) : __fdiv_rn(top, 127.0f);
            const float inv = most > 0u && most < 0x7c00u ? __fdiv_rn(127.0f, top) : 0.0f;
            uint32_t *codes = (uint32_t *)(sq.base + (which ? at.v : at.k) +
                                           ((long long)h * sq.nb + blk) * (kQ8Block * HD));
#pragma unroll
            for (int it = 0; it < ITER; it++) {
                const int t = (warp * ITER + it) * RPW + lane / LPR;
                uint32_t word[2];
#pragma unroll
                for (int side = 0; side < 2; side++) {
                    const float2 u = __half22float2(x[it][2 * side]), v = __half22float2(x[it][2 * side + 1]);
                    float y[4] = {u.x, u.y, v.x, v.y};
                    if (inv == 0.0f) y[0] = y[1] = y[2] = y[3] = 0.0f;
                    // rint(y / scale) by the reciprocal, whose product is within 2^-15 of the
                    // quotient (2^-22 of at most 127): only next to a tie is it divided
                    uint32_t q[4];
                    bool near = false;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float t = y[i] * inv, n = t + 12582912.0f;         // the integer in its low bits
                        q[i] = __float_as_uint(n);
                        near = near || fabsf(t - (n - 12582912.0f)) > 0.4999f;
                    }
                    if (near) {
#pragma unroll
                        for (int i = 0; i < 4; i++) q[i] = (uint32_t)__float2int_rn(__fdiv_rn(y[i], scale));
                    }
                    word[side] = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
                }
                if (!which) {
                    // panels of 64 channels: word of token t, channel d in panel d / 64
                    const int other = HD == 128 ? kQ8Block * 64 / 4 : HALF / 4;
                    codes[t * 16 + c] = word[0];
                    codes[t * 16 + c + other] = word[1];
                } else {
                    stage[t * SW + c] = word[0];
                    stage[t * SW + HALF / 4 + c] = word[1];
                }
            }
            if (which) {
                // transposed: a thread turns four tokens x four channels
                __syncthreads();
                const int tq = lane & 7, dq = warp * 4 + (lane >> 3);
                if (dq < HD / 4) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) w[i] = stage[(4 * tq + i) * SW + dq];
                    transpose4(w);
#pragma unroll
                    for (int i = 0; i < 4; i++) codes[(4 * dq + i) * 8 + tq] = w[i];
                }
                // (the next head's maximum is exchanged, with a barrier, before `stage` is written again)
            }
            if (tid == 0) {
                const long long at_b = (long long)h * sq.nb + blk;
                ((float *)(sq.base + (which ? at.vs : at.ks)))[at_b] = scale;
                if (which) ((float *)(sq.base + at.w))[at_b] = 0.0f;
            }
        }
    }
}

// ---- reading back -------------------------------------------------------------------

// Tokens [first, first + n) as f16 rows [kv_heads*hd]: blockIdx = (cache block,
// KV head, keys or values).
template <int HD>
__global__ void __launch_bounds__(kThreads) q8_read_kernel(const __grid_constant__ Q8ReadParams p)
{
    const Q8ReadSeq sq = p.seq[seq_of(p.seq, p.nseq, (int)blockIdx.x)];
    after_previous();
    const int blk = (sq.first >> 5) + (int)blockIdx.x - sq.item0;
    const int h = blockIdx.y, which = blockIdx.z;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Q8Layout at = q8_layout(p.kv_heads, HD, sq.nb);
    const int t0 = 32 * blk;
    const int lo = max(sq.first - t0, 0), hi = min(sq.first + sq.n - t0, 32);
    // row of token t of this block
    uint16_t *out = (which ? p.v : p.k) + (((long long)sq.row0 + t0 - sq.first) * p.kv_heads + h) * HD;
    const long long step = (long long)p.kv_heads * HD;
    if (blk >= sq.live >> 5) {
        const uint16_t *tail = (const uint16_t *)(sq.base + (which ? at.vt : at.kt)) + (long long)h * kQ8Block * HD;
        for (int i = tid; i < kQ8Block * HD / 4; i += kThreads) {
            const int t = i / (HD / 4), d = i % (HD / 4) * 4;
            if (t >= lo && t < hi) *(uint2 *)(out + t * step + d) = *(const uint2 *)(tail + t * HD + d);
        }
        return;
    }
    const long long b = (long long)h * sq.nb + blk;
    const uint4 *codes = (const uint4 *)(sq.base + (which ? at.v : at.k) + b * (kQ8Block * HD));
    const float scale = ((const float *)(sq.base + (which ? at.vs : at.ks)))[b];
    if (!which) {
        // eight channels of a token, so that the lanes of a store write whole sectors
        constexpr int PER = kQ8Block * HD / 8;
#pragma unroll
        for (int i = tid; i < PER; i += kThreads) {
            const uint2 w = ((const uint2 *)codes)[i];
            const int panel = i / (kQ8Block * 8), t = i / 8 % kQ8Block, d = panel * 64 + i % 8 * 8;
            if (t < lo || t >= hi) continue;
            const uint2 w0 = dequant4(w.x, scale), w1 = dequant4(w.y, scale);
            *(uint4 *)(out + t * step + d) = make_uint4(w0.x, w0.y, w1.x, w1.y);
        }
        return;
    }
    const uint4 w = tid < kQ8Block * HD / 16 ? codes[tid] : make_uint4(0u, 0u, 0u, 0u);
    // 16 tokens of a channel in, four channels of four tokens out (rows of eight
    // words padded to ten: neither side meets a bank twice)
    __shared__ uint32_t stage[HD * 10];
    if (tid < kQ8Block * HD / 16) {
        uint32_t *to = stage + tid / 2 * 10 + tid % 2 * 4;
        *(uint2 *)to = make_uint2(w.x, w.y);
        *(uint2 *)(to + 2) = make_uint2(w.z, w.w);
    }
    __syncthreads();
    const int tq = lane & 7, dq = warp * 4 + (lane >> 3);
    if (dq < HD / 4) {
        uint32_t x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = stage[(4 * dq + i) * 10 + tq];
        transpose4(x);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int t = 4 * tq + i;
            if (t >= lo && t < hi) *(uint2 *)(out + t * step + 4 * dq) = dequant4(x[i], scale);
        }
    }
}

// The live tokens as f16 caches that the prefill kernel's tensor maps can be
// laid over. blockIdx = (kUnpack cache blocks, KV head); a thread turns four times
// eight codes of either into 16 bytes (so that the lanes of a store write whole
// sectors), all eight loads in flight. Past the live tokens, up to the
// capacity (the next multiple of eight), lie zeros. A value that is not finite would
// make NaN of every row of a tile, those that may not see its token among them (0
// times it): it becomes a zero behind a key of NaN, which does that to the rows that
// see it and to no others. Bound by memory: 16896 tokens
// of 8 heads x 128, 104 MB, in 16 us (23 with stores of half sectors).
template <int HD>
__global__ void __launch_bounds__(kThreads) q8_unpack_kernel(const __grid_constant__ Q8UnpackParams p)
{
    constexpr int PER = kQ8Block * HD / 8;       // pieces of eight codes of a block
    constexpr int U = 4, kUnpack = U * kThreads / PER;
    const Q8UnpackSeq sq = p.seq[seq_of(p.seq, p.nseq, (int)blockIdx.x)];
    const int blk0 = kUnpack * ((int)blockIdx.x - sq.item0);
    const int h = blockIdx.y, tid = threadIdx.x;
    const int full = sq.live >> 5;
    const Q8Layout at = q8_layout(p.kv_heads, HD, sq.nb);
    const long long b0 = (long long)h * sq.nb;
    const float *ks = (const float *)(sq.base + at.ks) + b0, *vs = (const float *)(sq.base + at.vs) + b0;
    uint16_t *ko = sq.k + (long long)h * sq.cap16 * HD, *vo = sq.v + (long long)h * HD * sq.cap16;
    // (the attention kernel behind this one sets itself up meanwhile)
    after_previous();
    uint2 kc[U], vc[U];
    float ksc[U], vsc[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int i = tid + u * kThreads, blk = blk0 + i / PER, e = i % PER;
        if (blk < full) {
            kc[u] = ((const uint2 *)(sq.base + at.k + (b0 + blk) * (kQ8Block * HD)))[e];
            vc[u] = ((const uint2 *)(sq.base + at.v + (b0 + blk) * (kQ8Block * HD)))[e];
            ksc[u] = ks[blk];
            vsc[u] = vs[blk];
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int i = tid + u * kThreads, blk = blk0 + i / PER, e = i % PER;
        if (blk >= full) continue;
        const int panel = e / (kQ8Block * 8), t = e / 8 % kQ8Block, d = panel * 64 + e % 8 * 8;
        if (vsc[u] != vsc[u]) {
            ksc[u] = vsc[u];
            vsc[u] = 0.0f;
        }
        const uint2 k0 = dequant4(kc[u].x, ksc[u]), k1 = dequant4(kc[u].y, ksc[u]);
        *(uint4 *)(ko + (long long)(32 * blk + t) * HD + d) = make_uint4(k0.x, k0.y, k1.x, k1.y);
        const uint2 v0 = dequant4(vc[u].x, vsc[u]), v1 = dequant4(vc[u].y, vsc[u]);
        *(uint4 *)(vo + (long long)(e / 4) * sq.cap16 + 32 * blk + e % 4 * 8) = make_uint4(v0.x, v0.y, v1.x, v1.y);
    }
    const int tail = sq.live & 31;
    if (tail && full >= blk0 && full < blk0 + kUnpack) {
        // the tail's rows, and zeros up to the capacity, a multiple of eight
        __shared__ uint32_t rows[kQ8Block][HD / 2 + 1];
        const uint4 *kt = (const uint4 *)(sq.base + at.kt) + (long long)h * PER;
        const uint4 *vt = (const uint4 *)(sq.base + at.vt) + (long long)h * PER;
        const int upto = sq.cap16 - 32 * full;
        for (int i = tid; i < PER; i += kThreads) {
            const int t = i / (HD / 8), d = i % (HD / 8);
            const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
            uint4 k = t < tail ? kt[i] : zero, v = t < tail ? vt[i] : zero;
            // (every lane is here; a row's are LANES neighbours)
            constexpr uint32_t LANES = HD / 8;
            const uint32_t odd = __ballot_sync(0xffffffffu, not_finite(v.x) || not_finite(v.y) || not_finite(v.z) || not_finite(v.w));
            if (odd >> (tid % 32 / LANES * LANES) & ((1u << LANES) - 1u)) {
                k = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
                v = zero;
            }
            if (t < upto) ((uint4 *)(ko + (long long)32 * full * HD))[i] = k;
            rows[t][4 * d] = v.x;
            rows[t][4 * d + 1] = v.y;
            rows[t][4 * d + 2] = v.z;
            rows[t][4 * d + 3] = v.w;
        }
        __syncthreads();
        for (int i = tid; i < HD * 4; i += kThreads) {
            const int d = i / 4, t = i % 4 * 8;                  // eight tokens of a channel
            if (t >= upto) continue;
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                w[e] = __byte_perm(rows[t + 2 * e][d / 2], rows[t + 2 * e + 1][d / 2], d % 2 ? 0x7632 : 0x5410);
            }
            *(uint4 *)(vo + (long long)d * sq.cap16 + 32 * full + t) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// The first to % 32 tokens of block to / 32 back into the tail.
template <int HD>
__global__ void __launch_bounds__(kThreads) q8_rewind_kernel(const __grid_constant__ Q8RewindParams p)
{
    const Q8RewindSeq sq = p.seq[blockIdx.y];
    after_previous();
    const int h = blockIdx.x, which = blockIdx.z, tid = threadIdx.x;
    const Q8Layout at = q8_layout(p.kv_heads, HD, sq.nb);
    const long long b = (long long)h * sq.nb + (sq.to >> 5);
    const signed char *codes = (const signed char *)(sq.base + (which ? at.v : at.k) + b * (kQ8Block * HD));
    const float scale = ((const float *)(sq.base + (which ? at.vs : at.ks)))[b];
    uint16_t *tail = (uint16_t *)(sq.base + (which ? at.vt : at.kt)) + (long long)h * kQ8Block * HD;
    for (int i = tid; i < (sq.to & 31) * HD; i += kThreads) {
        const int t = i / HD, d = i % HD;
        const int code = which ? codes[d * kQ8Block + t] : codes[d / 64 * (kQ8Block * 64) + t * 64 + d % 64];
        tail[i] = __half_as_ushort(__float2half_rn((float)code * scale));
    }
}

// ---- eviction -----------------------------------------------------------------------
//
// Which blocks stay: one block of the grid a (sequence, KV head). Among the
// blocks that may go, `room` stay: those above the weight `key`, and of those at
// it the first `ties`. Up to kPickFew blocks every thread counts the weights
// that come before its own; of more the room-th largest is found by its bits,
// eleven at a time (weights are not negative, so their bits order as they do;
// NaN and negative ones count as zero). One walk in order then moves scales and
// weights: a tile is read before anything of it is written, and a kept block
// only ever moves down, so source and destination may be one cache.
constexpr int kPickThreads = 1024;
constexpr int kPickKeys = 8192;              // weights held in shared memory
constexpr int kPickBins = 2048;
constexpr int kPickFew = 512;                // counting 512 takes 3 us, their bits 6; 1024 the other way about

__device__ __forceinline__ uint32_t weight_key(float w) { return w > 0.0f ? __float_as_uint(w) : 0u; }

// Exclusive prefix sum of v over the block; *sum is the total. Every thread calls.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *warp_sum, uint32_t *sum)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();   // what was read of warp_sum before is done with
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    static_assert(kPickThreads == 1024, "a warp sum for every lane");
    uint32_t s = warp_sum[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
    }
    *sum = __shfl_sync(0xffffffffu, s, 31);
    const uint32_t before = __shfl_sync(0xffffffffu, s, max(warp, 1) - 1);
    return (warp ? before : 0u) + x - v;
}

__global__ void __launch_bounds__(kPickThreads) q8_pick_kernel(const __grid_constant__ Q8EvictParams p, int hd)
{
    __shared__ uint32_t hist[kPickBins], warp_sum[32], found[2];
    __shared__ __align__(16) uint32_t keys[kPickKeys];
    const Q8EvictSeq sq = p.seq[blockIdx.y];
    const int h = blockIdx.x, tid = threadIdx.x;
    const Q8Layout a = q8_layout(p.kv_heads, hd, sq.src_nb), z = q8_layout(p.kv_heads, hd, sq.dst_nb);
    const long long sb = (long long)h * sq.src_nb, db = (long long)h * sq.dst_nb;
    const float *w = (const float *)(sq.src + a.w) + sb;
    int *index = p.index + ((long long)blockIdx.y * p.kv_heads + h) * p.max_keep;
    int *user = p.user_index ? p.user_index + ((long long)blockIdx.y * p.kv_heads + h) * p.user_stride : nullptr;
    const int lo = sq.first, hi = sq.full - sq.recent;           // those that may go
    const bool all = sq.keep >= sq.full;
    uint32_t room = all ? 0u : (uint32_t)(sq.keep - sq.first - sq.recent);
    uint32_t key = 0xffffffffu, ties = 0;                        // above key: stays; at it: the first `ties`
    bool chosen = false;                                         // (few blocks: this thread's own stays)
    const bool few = sq.full <= kPickFew;
    after_previous();
    // Everything whose address is known is asked for first: the first tile's
    // weights and scales, and the tail's rows of this head.
    const float *ks = (const float *)(sq.src + a.ks) + sb, *vs = (const float *)(sq.src + a.vs) + sb;
    float wi = 0.0f, kscale = 0.0f, vscale = 0.0f;
    if (tid < sq.full) {
        wi = w[tid];
        kscale = ks[tid];
        vscale = vs[tid];
    }
    if (sq.dst != sq.src) {
        const int n = sq.tail * hd / 8;                          // 16-byte pieces, no more than 512
        const uint4 *kt = (const uint4 *)(sq.src + a.kt) + (long long)h * (kQ8Block * hd / 8);
        const uint4 *vt = (const uint4 *)(sq.src + a.vt) + (long long)h * (kQ8Block * hd / 8);
        if (tid < n) {
            const uint4 x = kt[tid], y = vt[tid];
            ((uint4 *)(sq.dst + z.kt))[(long long)h * (kQ8Block * hd / 8) + tid] = x;
            ((uint4 *)(sq.dst + z.vt))[(long long)h * (kQ8Block * hd / 8) + tid] = y;
        }
    }
    if (!all && room > 0) {
        const bool held = sq.full <= kPickKeys;
        if (held) {
            // (four loads in flight; the first tile's is there already)
            for (int i0 = tid; i0 < (sq.full + 3) / 4 * 4; i0 += 4 * kPickThreads) {
                float x[4];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int i = i0 + u * kPickThreads;
                    x[u] = i == tid ? wi : i >= lo && i < hi ? w[i] : 0.0f;
                }
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int i = i0 + u * kPickThreads;
                    if (i < kPickKeys) keys[i] = i >= lo && i < hi ? weight_key(x[u]) + (few ? 1u : 0u) : 0u;
                }
            }
            __syncthreads();
        }
        if (few) {
            // (keys are one up here, so that 0 stands for blocks that are not to choose from)
            if (tid >= lo && tid < hi) {
                const uint32_t k = keys[tid] + 1u;               // above its own
                const int at = tid / 4 * 4;
                uint32_t ahead = 0;                              // those that go before it
                auto count = [&](int from, int to, uint32_t least) {
                    for (int i = from; i < to; i += 4) {
                        const uint4 y = *(const uint4 *)&keys[i];
                        ahead += (y.x >= least) + (y.y >= least) + (y.z >= least) + (y.w >= least);
                    }
                };
                count(lo / 4 * 4, at, k - 1u);                   // lower ones: as heavy or heavier
                for (int i = at; i < min(at + 4, hi); i++) ahead += i != tid && keys[i] >= (i < tid ? k - 1u : k);
                count(at + 4, hi, k);                            // higher ones: heavier
                chosen = ahead < room;
            }
        } else {
            uint32_t prefix = 0, mask = 0;
            for (int round = 0; round < 3; round++) {
                const int shift = round == 0 ? 21 : round == 1 ? 10 : 0;
                const uint32_t digits = round == 2 ? 1023u : 2047u;
                hist[tid] = 0;
                hist[tid + kPickThreads] = 0;
                __syncthreads();
                for (int i = lo + tid; i < hi; i += kPickThreads) {
                    const uint32_t k = held ? keys[i] : weight_key(w[i]);
                    if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & digits], 1u);
                }
                __syncthreads();
                // digits from the top, two a thread
                const uint32_t d0 = kPickBins - 1 - 2 * tid;
                const uint32_t n0 = hist[d0], n1 = hist[d0 - 1];
                uint32_t sum;
                const uint32_t above = block_scan(n0 + n1, warp_sum, &sum);
                if (above < room && above + n0 >= room) {
                    found[0] = d0;
                    found[1] = room - above;
                } else if (above + n0 < room && above + n0 + n1 >= room) {
                    found[0] = d0 - 1;
                    found[1] = room - above - n0;
                }
                __syncthreads();
                prefix |= found[0] << shift;
                mask |= digits << shift;
                room = found[1];
            }
            key = prefix;
            ties = room;
        }
    }
    uint32_t kept = 0, tied = 0;
    for (int i0 = 0; i0 < sq.full; i0 += kPickThreads) {
        const int i = i0 + tid;
        const bool in = i < sq.full;
        const bool safe = in && (all || i < lo || i >= hi);
        // the next tile's are asked for before this one's are written: they lie above
        const int next = i + kPickThreads;
        float w_next = 0.0f, ks_next = 0.0f, vs_next = 0.0f;
        if (next < sq.full) {
            w_next = w[next];
            ks_next = ks[next];
            vs_next = vs[next];
        }
        const uint32_t k = weight_key(wi);
        const bool sure = safe || (few ? chosen : in && k > key);
        const bool tie = !few && in && !safe && k == key;
        // both counts in one sum: a tile has no more than 1024 of either
        uint32_t sum;
        const uint32_t before = block_scan((sure ? 1u : 0u) | (tie ? 0x10000u : 0u), warp_sum, &sum);
        const uint32_t t_before = min(tied + (before >> 16), ties), t_tile = min(tied, ties);
        const bool stay = sure || (tie && tied + (before >> 16) < ties);
        const uint32_t to = kept + (before & 0xffffu) + t_before - t_tile;
        kept += (sum & 0xffffu) + min(tied + (sum >> 16), ties) - t_tile;
        tied += sum >> 16;
        // (the tile is read: every thread has passed the scan's barriers with its values)
        if (stay) {
            index[to] = i;
            if (user) user[to] = i;
            ((float *)(sq.dst + z.ks))[db + to] = kscale;
            ((float *)(sq.dst + z.vs))[db + to] = vscale;
            ((float *)(sq.dst + z.w))[db + to] = wi;
        }
        wi = w_next;
        kscale = ks_next;
        vscale = vs_next;
    }
}

// Moves the kept blocks' codes. Into another cache every block is a copy of its
// own: blockIdx = (share of the list, keys or values of a head, sequence), a
// pass of the threads takes kThreads * 16 bytes.
//
// In place blockIdx.x is a slice of every block's bytes instead. Slices move by
// the same list and never meet, so each may go at its own pace; within one, a
// group of blocks is read before any of it is written, and later groups lie
// above what it writes, so the next one is on its way meanwhile.
template <int HD>
__global__ void __launch_bounds__(kThreads) q8_move_kernel(const __grid_constant__ Q8EvictParams p, int slices)
{
    constexpr int PIECES = kQ8Block * HD / 16;                   // 16-byte pieces of a block
    after_previous();
    const Q8EvictSeq sq = p.seq[blockIdx.z];
    const int h = blockIdx.y >> 1, which = blockIdx.y & 1;
    const Q8Layout a = q8_layout(p.kv_heads, HD, sq.src_nb), z = q8_layout(p.kv_heads, HD, sq.dst_nb);
    const uint4 *src = (const uint4 *)(sq.src + (which ? a.v : a.k)) + (long long)h * sq.src_nb * PIECES;
    uint4 *dst = (uint4 *)(sq.dst + (which ? z.v : z.k)) + (long long)h * sq.dst_nb * PIECES;
    const int *index = p.index + ((long long)blockIdx.z * p.kv_heads + h) * p.max_keep;
    if (sq.src != sq.dst) {
        constexpr int DEPTH = 8, LANES = kThreads / PIECES;
        const int piece = threadIdx.x % PIECES, sub = threadIdx.x / PIECES;
        const int share = (sq.keep + (int)gridDim.x - 1) / (int)gridDim.x;
        const int j1 = min(sq.keep, (int)(blockIdx.x + 1) * share);
        for (int j0 = (int)blockIdx.x * share; j0 < j1; j0 += LANES * DEPTH) {
            uint4 x[DEPTH];
#pragma unroll
            for (int u = 0; u < DEPTH; u++) {
                const int j = j0 + u * LANES + sub;
                if (j < j1) x[u] = src[(long long)index[j] * PIECES + piece];
            }
#pragma unroll
            for (int u = 0; u < DEPTH; u++) {
                const int j = j0 + u * LANES + sub;
                if (j < j1) dst[(long long)j * PIECES + piece] = x[u];
            }
        }
        return;
    }
    constexpr int DEPTH = 4;
    if ((int)blockIdx.x >= slices) return;
    const int per = PIECES / slices, lanes = kThreads / per;     // blocks a pass of the threads takes
    const int piece = (int)blockIdx.x * per + threadIdx.x % per, sub = threadIdx.x / per;
    uint4 x[2][DEPTH];
    bool go[2][DEPTH];
    auto load = [&](int b, int j0) {
#pragma unroll
        for (int u = 0; u < DEPTH; u++) {
            const int j = j0 + u * lanes + sub;
            go[b][u] = false;
            if (j < sq.keep) {
                const int i = index[j];
                go[b][u] = i != j;
                if (go[b][u]) x[b][u] = src[(long long)i * PIECES + piece];
            }
        }
    };
    auto store = [&](int b, int j0) {
#pragma unroll
        for (int u = 0; u < DEPTH; u++) {
            if (go[b][u]) dst[(long long)(j0 + u * lanes + sub) * PIECES + piece] = x[b][u];
        }
    };
    const int step = lanes * DEPTH;
    load(0, 0);
    for (int j0 = 0; j0 < sq.keep; j0 += 2 * step) {
        load(1, j0 + step);
        __syncthreads();       // group j0 has been read by all
        store(0, j0);
        load(0, j0 + 2 * step);
        __syncthreads();
        store(1, j0 + step);
    }
}

const KernelReg reg_append("q8_append", (const void *)q8_append_kernel<128>);
const KernelReg reg_read("q8_read", (const void *)q8_read_kernel<128>);
const KernelReg reg_unpack("q8_unpack", (const void *)q8_unpack_kernel<128>);
const KernelReg reg_pick("q8_pick", (const void *)q8_pick_kernel);
const KernelReg reg_move("q8_move", (const void *)q8_move_kernel<128>);

}  // namespace

// (every kernel launched here calls after_previous)
template <typename... Params, typename... Args>
static cudaError_t launch(cudaStream_t st, dim3 grid, int threads, void (*kernel)(Params...), Args... args)
{
    return launch_dependent(st, grid, threads, 0, 1, kernel, args...);
}

cudaError_t launch_q8_append(cudaStream_t st, Q8AppendParams &p, int hd, int sm_count)
{
    // Heads share a block of the grid (and its sines and cosines) as long as the
    // launch still has a few blocks for every SM.
    p.kv_chunk = 4;
    p.q_log = 3;
    auto rows = [&] {
        const int kvc = (p.kv_heads + p.kv_chunk - 1) / p.kv_chunk;
        const int qc = p.q ? (p.heads + (1 << p.q_log) - 1) >> p.q_log : 0;
        return 2 * kvc + qc;
    };
    while (p.q_log > 1 && (long long)p.items * rows() < 4ll * sm_count) {
        if (p.kv_chunk > 1) p.kv_chunk /= 2;
        p.q_log--;
    }
    const dim3 grid((unsigned)p.items, (unsigned)rows());
    return hd == 128 ? launch(st, grid, kThreads, q8_append_kernel<128>, p) : launch(st, grid, kThreads, q8_append_kernel<64>, p);
}

cudaError_t launch_q8_read(cudaStream_t st, const Q8ReadParams &p, int hd)
{
    const dim3 grid((unsigned)p.items, (unsigned)p.kv_heads, 2);
    return hd == 128 ? launch(st, grid, kThreads, q8_read_kernel<128>, p) : launch(st, grid, kThreads, q8_read_kernel<64>, p);
}

int q8_unpack_tokens(int hd) { return kQ8Block * (2 * kThreads * 16 / (kQ8Block * hd)); }

cudaError_t launch_q8_unpack(cudaStream_t st, const Q8UnpackParams &p, int hd)
{
    const dim3 grid((unsigned)p.items, (unsigned)p.kv_heads);
    return hd == 128 ? launch(st, grid, kThreads, q8_unpack_kernel<128>, p) : launch(st, grid, kThreads, q8_unpack_kernel<64>, p);
}

cudaError_t launch_q8_rewind(cudaStream_t st, const Q8RewindParams &p, int hd)
{
    const dim3 grid((unsigned)p.kv_heads, (unsigned)p.nseq, 2);
    return hd == 128 ? launch(st, grid, kThreads, q8_rewind_kernel<128>, p) : launch(st, grid, kThreads, q8_rewind_kernel<64>, p);
}

cudaError_t launch_q8_evict(cudaStream_t st, const Q8EvictParams &p, int hd, int sm_count)
{
    const cudaError_t e = launch(st, dim3((unsigned)p.kv_heads, (unsigned)p.nseq), kPickThreads, q8_pick_kernel, p, hd);
    if (e != cudaSuccess || p.max_keep == 0) return e;
    // In place: slices of no less than 256 bytes, until every SM has a few. Into
    // another cache: shares of no less than a pass of eight loads, the same way.
    const int most = kQ8Block * hd / 256, rows = p.kv_heads * 2 * p.nseq;
    bool in_place = false, apart = false;
    for (int b = 0; b < p.nseq; b++) {
        if (p.seq[b].src == p.seq[b].dst) in_place = true;
        else apart = true;
    }
    int slices = 1, shares = 1;
    while (slices < most && (long long)slices * rows < 4ll * sm_count) slices *= 2;
    const int pass = 8 * kThreads * 16 / (kQ8Block * hd);
    while (shares * 2 * pass <= p.max_keep + pass && (long long)shares * rows < 8ll * sm_count) shares *= 2;
    const dim3 grid((unsigned)std::max(in_place ? slices : 1, apart ? shares : 1), (unsigned)p.kv_heads * 2, (unsigned)p.nseq);
    return hd == 128 ? launch(st, grid, kThreads, q8_move_kernel<128>, p, slices) : launch(st, grid, kThreads, q8_move_kernel<64>, p, slices);
}
