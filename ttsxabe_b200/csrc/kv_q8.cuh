// The 8-bit KV cache: where its sections lie, and the launchers of the kernels
// that fill, read, shorten and attend over it.
//
// Tokens lie in blocks of 32. A complete block of one KV head is int8 codes
// with one f32 scale for its keys and one for its values: code = rint(x /
// scale), scale = max|x| / 127 over the block's 32 x hd elements, x the row
// rounded to f16. The tokens of the last, incomplete block stay f16 rows (the
// tail), so that a token is rounded to 8 bits once, together with its block,
// and the codes do not depend on how the tokens arrived (one by one, or in
// prompts cut anywhere).
//
// One buffer holds a layer's cache; its sections, each at a multiple of 128
// bytes, nb = capacity / 32:
//   key codes    [kv][nb][hd/64][32 tokens][64]   panels of 64 channels: eight
//                lanes reading 16 bytes each of two neighbouring rows touch
//                every bank once
//   value codes  [kv][nb][hd][32 tokens]          transposed inside a block, as
//                the product with the probabilities reads them
//   key scales   f32 [kv][nb]
//   value scales f32 [kv][nb]
//   weights      f32 [kv][nb]     accumulated attention weight of each block
//   key tail     f16 [kv][32][hd]
//   value tail   f16 [kv][32][hd]
#pragma once

#include "common.cuh"

#include <stdlib.h>

constexpr int kQ8Block = 32;
#define LLMTIE_Q8_MAX_SEQ 32

struct Q8Layout {
    long long k, v, ks, vs, w, kt, vt, bytes;
};
__host__ __device__ inline Q8Layout q8_layout(int kv_heads, int hd, int nb)
{
    const long long codes = (long long)kv_heads * nb * kQ8Block * hd;
    const long long scales = ((long long)kv_heads * nb * 4 + 127) / 128 * 128;
    const long long tail = (long long)kv_heads * kQ8Block * hd * 2;
    Q8Layout l;
    l.k = 0;
    l.v = codes;
    l.ks = 2 * codes;
    l.vs = l.ks + scales;
    l.w = l.vs + scales;
    l.kt = l.w + scales;
    l.vt = l.kt + tail;
    l.bytes = l.vt + tail;
    return l;
}

// Launches `kernel` as the programmatic dependent of the kernel before it in the
// stream: it may be set up while that one still runs, and waits for its end
// (griddepcontrol.wait) before it reads or writes anything.
template <typename... Params, typename... Args>
inline cudaError_t launch_dependent(cudaStream_t st, dim3 grid, int threads, size_t smem, int cluster, void (*kernel)(Params...),
                                    Args... args)
{
    static const bool no_pdl = getenv("LLMTIE_B200_NO_PDL") != nullptr;   // an A/B switch
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    if (!no_pdl) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = (unsigned)cluster;
        attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
        cfg.numAttrs++;
    }
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Whether either f16 of a word is an infinity or NaN.
__device__ __forceinline__ bool not_finite(uint32_t w)
{
    return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u;
}

// ---- kv_q8.cu ---------------------------------------------------------------

struct Q8AppendSeq {
    unsigned char *base;
    int nb;        // blocks of the cache's capacity
    int past;      // tokens the cache holds
    int n;         // rows this sequence brings (never 0 here)
    int row0;      // its first row in q, k and v
    int pos;       // rotary position of that row
    int item0;     // first of its work items
};
struct Q8AppendParams {
    Q8AppendSeq seq[LLMTIE_Q8_MAX_SEQ];
    int nseq, items;
    const float *q;          // null: no queries to rotate
    float *q_out;            // may be q
    const float *k, *v;
    const float *inv_freq;   // null: the rows come rotated
    int heads, kv_heads;
    int kv_chunk, q_log;     // heads a block of the grid takes: kv_chunk, or 1 << q_log of the query
};
cudaError_t launch_q8_append(cudaStream_t st, Q8AppendParams &p, int hd, int sm_count);

struct Q8ReadSeq {
    const unsigned char *base;
    int nb, live;
    int first, n;      // tokens [first, first + n)
    int row0;          // where they go in the packed outputs
    int item0;
};
struct Q8ReadParams {
    Q8ReadSeq seq[LLMTIE_Q8_MAX_SEQ];
    int nseq, items;
    uint16_t *k, *v;   // f16 [rows][kv_heads*hd]
    int kv_heads;
};
cudaError_t launch_q8_read(cudaStream_t st, const Q8ReadParams &p, int hd);

// The first `live` tokens as f16 caches of capacity cap16 (a multiple of 8):
// keys [kv][cap16][hd], values [kv][hd][cap16], for the prefill kernel.
struct Q8UnpackSeq {
    const unsigned char *base;
    uint16_t *k, *v;
    int nb, live, cap16;
    int item0;
};
struct Q8UnpackParams {
    Q8UnpackSeq seq[LLMTIE_Q8_MAX_SEQ];
    int nseq, items;
    int kv_heads;
};
int q8_unpack_tokens(int hd);    // tokens of a work item
cudaError_t launch_q8_unpack(cudaStream_t st, const Q8UnpackParams &p, int hd);

struct Q8RewindSeq {
    unsigned char *base;
    int nb, to;        // the block of token `to` goes back into the tail
};
struct Q8RewindParams {
    Q8RewindSeq seq[LLMTIE_Q8_MAX_SEQ];
    int nseq;
    int kv_heads;
};
cudaError_t launch_q8_rewind(cudaStream_t st, const Q8RewindParams &p, int hd);

struct Q8EvictSeq {
    const unsigned char *src;
    unsigned char *dst;      // may be src
    int src_nb, dst_nb;
    int full;                // complete blocks in src
    int tail;                // tokens of the tail
    int keep;                // blocks that stay, <= full
    int first, recent;       // blocks at either end that stay whatever their weight
};
struct Q8EvictParams {
    Q8EvictSeq seq[LLMTIE_Q8_MAX_SEQ];
    int nseq;
    int kv_heads;
    int max_keep;
    int *index;              // [seq][kv][max_keep]: which source block each kept one was
    int *user_index;         // the same for the caller (or null), rows user_stride apart
    long long user_stride;
};
cudaError_t launch_q8_evict(cudaStream_t st, const Q8EvictParams &p, int hd, int sm_count);

// f32 inverse frequencies theta^(-2j/hd) (/ freq_div[j]), the bits rope_scaled uses.
void launch_rope_inv_freq(cudaStream_t st, float *out, const float *freq_div, int hd, float theta);

// ---- decode_q8.cu -----------------------------------------------------------

// One job: n queries (n * heads / kv_heads at most eight) of one sequence.
struct DecodeQ8Seq {
    unsigned char *base;     // (the weights are written)
    int nb, full;            // blocks of the capacity, and complete ones (what is past them lies in the tail)
    int live;                // the last query sees that many tokens
    int row0, n;             // its first row in q and out
};
struct DecodeQ8Params {
    DecodeQ8Seq seq[LLMTIE_Q8_MAX_SEQ];
    int unit0[LLMTIE_Q8_MAX_SEQ + 1];                  // first 32-token unit of each sequence
    int each, more, over;                              // the cut over the grid: see first_unit in decode_q8.cu
    int cluster, parts;                                // or: a pair to so many clusters of so many blocks, no cut (0: the cut)
    long long stat0[LLMTIE_Q8_MAX_SEQ];                // first block of each sequence in `stats`
    int nseq, heads, kv_heads;
    int causal;              // query i sees live - n + 1 + i tokens, else all
    const float *q;          // rows [heads*hd]
    void *out;               // the same, f16 or f32
    int out_f16;
    float sl2;               // scale * log2(e)
    float *part_o;           // [block][2][8][hd], or [cluster][8][hd]
    float2 *part_ml;         // [block][2][8], or [cluster][8]
    unsigned *ctr;           // arrivals of each (sequence, KV head), or of each of its rows; zero at rest
    float2 *stats;           // [block of a sequence][8] (maximum, sum), or null: no weights
    float2 *fin;             // [sequence, KV head][8] (maximum, 1 / sum), with them
    int *status;
    long long wait_cycles;
};
cudaError_t launch_decode_q8(cudaStream_t st, const DecodeQ8Params &p, int hd, int grid);
// How a launch over pairs of `units` cache blocks (the tail counts as one), each
// kv_heads times, is laid over the device.
struct DecodeQ8Plan {
    int grid;      // blocks of the grid (0: nothing to do)
    int cluster;   // clusters of so many, or 0: cut by work
    int parts;     // that many of them a pair
    int over;      // what the cut charges a run
    double us;     // about what it takes
};
void plan_decode_q8(DecodeQ8Plan &plan, const int *units, int n, int kv_heads, int hd, int sm_count, const int *clusters);
// How many clusters of 8 and of 16 blocks the current device holds at once.
cudaError_t decode_q8_clusters(int hd, int (&clusters)[2]);
