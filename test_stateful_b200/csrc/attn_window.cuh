// Paged GQA attention with a sliding window and sinks, over the fp16 pool or the 4-bit one.
//
// A query row of context c (its keys are 0 .. c - 1) sees key j when
//     j < c  and  (j >= c - window  or  j < sinks  or  window == 0),
// and gets softmax(q k^T / sqrt(D)) v over those keys; a row that sees none gets zeros.
//
// Row kernel.  One warp walks 16-token blocks, copied ahead of use into a ring of its own in shared
// memory (cp.async, 16 bytes a lane; K and V are separate steps of the ring).  The tensor work is
// mma.sync with the keys on the M side and (query, head) slots on the N side:
//     S^T[16 tokens][8]   += K[16][channels] . Q^T
//     O^T[16 channels][8] += V^T[16][16 tokens] . P^T
// q and the probabilities enter as pairs of a high part and what it leaves, so that they keep 16
// bits or more; movmatrix turns the probabilities from S^T's accumulator layout into the operand
// layout.
// Decode tiles fill few of the eight columns (two query heads a KV head: two).  Over the 4-bit pool
// the columns are shared by KB = 8 / SL blocks of SL slots: q stands in every group of columns, so that
// each lane of a quad finds the scores of one block in its registers and the softmax of KB blocks
// runs at once, a block to a lane; for P V each block takes its own group's columns of P, the opposite
// group's hold the low parts, the rest zero.  The column groups of O add up at the end.
//
// 4-bit pool, K: the nibbles of a word are two words of bytes, x & 0x0f0f0f0f and (x >> 4) & 0x0f0f0f0f: unsigned
// operands of an integer product (m16n8k32).  q is a 22-bit fixed-point number in three signed digits, its unit
// 2^-21 of the slot's largest channel (two digits, 2^-16, moved scores by up to 1e-4 where q has loud channels);
// 64 codes of 15 times it stay below 2^31, so that the sum is exact.  A key's scale multiplies the sum, its zero sum(q).
// V: a nibble masked out of a code word IS a small bf16 number (a subnormal: nibble << 0 = code *
// 2^-133, nibble << 4 = 16 times that), so that no conversion is needed; the powers of two move
// into p and the output, a token's scale into its probability, and its zero is added on the fp32 side.
// The channel order of the contractions is the one in which a lane's words arrive: lane (g, t) takes
// of K tokens g and g + 8 the channels 64 w + 16 t .. + 15, of V tokens 2 t, 2 t + 1, 2 t + 8,
// 2 t + 9 the channels 64 w + 8 g .. + 7.
//
// Bound by (16 heads over 8, D = 128, B200): fp16 by HBM, 64 x 4096 keys 173 us (6.2 TB/s); 4 bits by instructions
// (0.53 of the issue slots, 48% of the integer pipe, 32% of the tensor one) next to HBM, the same keys 68 us
// (4.4 TB/s).  A decode step of one wave by latencies (block ids, first copies, the longest row): 64 streams of 260
// .. 780 keys at 4 bits 18.7 us, under a window of 72 + 4 12.1 us over fp16, 8.6 over 4 bits.
#pragma once

#include <type_traits>

#include "attention.cuh"
#include "kv_q4.cuh"

namespace qtts {

struct WinParams {
    const float* q;  // [R][num_heads][D]
    const uint8_t* kv;
    const int32_t* block_table;  // [num_slots][mbps]
    const int32_t* row_slot;
    const int32_t* row_ctx;
    __nv_bfloat16* out;
    __nv_bfloat16* out_lo;
    int R, S;               // rows; consecutive rows that belong to one stream
    int num_heads, kv_heads;
    int group;              // query heads per KV head
    FastDiv by_group;
    int head_tiles;         // tiles a KV head's query heads are cut into
    int qt, tiles;          // queries per tile, tiles per stream
    int layer, num_layers, num_blocks, num_slots, mbps;
    int max_ctx, window, sinks;
    uint32_t block_bytes, v_offset;  // of one pool block; from a K chunk to its V chunk
    float scale_log2;       // log2(e) / sqrt(D)
};

enum { kWinF16 = 0, kWinQ4 = 1 };

// D += A B, and D = A B for the first of a chain.  Not volatile: the compiler may interleave chains.
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma_f16_first(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.f));
}
__device__ __forceinline__ void mma_u8s8(int (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma_u8s8_first(int (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "r"(0));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// transpose of an 8 x 8 matrix of 16-bit elements held as two per lane
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int N>
__device__ __forceinline__ void lds_words(uint32_t (&w)[N], uint32_t addr) {
    if constexpr (N == 4)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
    else if constexpr (N == 2)
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
    else
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
}
__device__ __forceinline__ float2 lds_half2(uint32_t addr) {
    uint32_t u;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(u) : "r"(addr));
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
__device__ __forceinline__ uint32_t pack_bf2(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// A chunk in shared memory, 16-byte pieces permuted so that the fragment reads meet no bank twice.
//   fp16: rows of 2 D bytes read by ldmatrix; piece c of row r sits at c ^ (r % 8).
//   4 bits: rows of D / 2 bytes; of D = 128 the eight pieces of two rows sit at L ^ 2 (r / 2 % 4):
//   K reads two whole rows a quarter-warp, V one 16-channel stretch of rows 0, 2, 4, 6 (+ 1, + 8).
template <int FMT, int D>
struct WinChunk {
    static constexpr int NW = D / 64;
    static constexpr int BYTES = FMT == kWinQ4 ? Q4Layout<D>::CHUNK : 32 * D;  // of one (block, layer, k|v, head)

    // this lane's copies
    static __device__ __forceinline__ void copy(uint32_t dst, const uint8_t* src, int lane) {
        if constexpr (FMT == kWinQ4) {
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                const int j = lane + 32 * i, sw = D == 128 ? j ^ ((j >> 2) & 6) : j;
                cp_async16(dst + sw * 16, src + j * 16);
            }
            // the (scale, zero) pairs; their 4 NW pieces
            if (lane < 4 * NW) cp_async16(dst + Q4Layout<D>::PARAMS + lane * 16, src + Q4Layout<D>::PARAMS + lane * 16);
        } else {
            constexpr int PR = D / 8;  // pieces per row
#pragma unroll
            for (int i = 0; i < 16 * PR / 32; ++i) {
                const int j = lane + 32 * i, r = j / PR, c = j % PR;
                cp_async16(dst + (r * PR + (c ^ (r & 7))) * 16, src + j * 16);
            }
        }
    }
};

// The 4-bit pool's probabilities carry 2^100 into the bf16 product, whose other factor is code * 2^-133:
// a probability is at most 2^8 and a scale below 2^14, so 2^122 at most, and the products are
// normal numbers down to probabilities of 2^-90.
constexpr float kPScale = 1.2676506002282294e30f;  // 2^100
constexpr float kPUnscale = 8589934592.f;          // 2^133 / 2^100

// fp16 halves of a probability: it is taken relative to 2^-7 of the running maximum, which leaves it below 2^15 (the
// maximum may lag by 2^8) and puts fp16's last step at 2^-31 of the maximum.  Relative to the maximum itself,
// keys below 2^-25 of it would vanish from O but not from the sum: 32000 of them, 1e-3 of the output.
constexpr float kPShift = 7.f;

constexpr int kWinMaxSplits = 16;  // CTAs of a cluster

// ld.shared::cluster that several of may be under way (no memory clobber): the data was published by
// a cluster barrier
__device__ __forceinline__ float ld_dsmem_now(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}

// SL slots a tile, W warps per CTA, NBUF steps of KB chunks in a warp's ring, at least MINB CTAs an SM.
template <int FMT, int D, int SL, int W, int NBUF, int MINB>
__global__ void __launch_bounds__(W * 32, MINB) paged_attn_window_kernel(const WinParams p) {
    using G = WinChunk<FMT, D>;
    constexpr int NW = G::NW, MT = D / 16, KB = 8 / SL;
    constexpr int STEP = KB * G::BYTES, RING = NBUF * STEP;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_ml[W][SL][2];
    __shared__ float s_part[SL][2];  // the CTA's (max, sum) per slot
    // Q^T operand words of (slot, t): high parts to low parts; accumulator -> log2 units; sums of q
    constexpr int NQ = FMT == kWinQ4 ? 2 * NW : MT, QP = FMT == kWinQ4 ? 3 : 2;
    __shared__ __align__(16) uint32_t s_q[SL][4][QP * 2 * NQ];
    __shared__ float s_qf[SL], s_qsum[SL][NW];
    static_assert(SL * D * 4 <= RING, "a warp's partial output replaces its ring");

    griddep_wait();
    griddep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int kb = 2 * t / SL;  // the block of an iteration whose scores this lane holds
    uint32_t splits;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(splits));
    const uint32_t rank = cluster_ctarank();

    // the tile: (query, head) slots of one stream and KV head
    const int tile = blockIdx.x / splits;
    const int head_tile = tile % (p.kv_heads * p.head_tiles), row_tile = tile / (p.kv_heads * p.head_tiles);
    const int kvh = head_tile / p.head_tiles, h0 = (head_tile % p.head_tiles) * SL;
    const int heads = min(SL, p.group - h0);
    const int stream = row_tile / p.tiles, q0 = (row_tile % p.tiles) * p.qt;
    const int nq = min(p.qt, p.S - q0);
    const int row0 = stream * p.S + q0;
    const int slots = nq * heads;

    // q of this warp's slots (warp, warp + W, ...), on its way while the contexts and block ids are read.
    //   4 bits: lane = 16 w + 4 t + 2 e + odd takes the odd or even channels of word (w, t, e)
    //   fp16: lane takes the channel pairs lane and lane + 32
    constexpr int QS = (SL + W - 1) / W;
    float qv[QS][4];
#pragma unroll
    for (int k = 0; k < QS; ++k) {
        const int s = warp + k * W;
        qv[k][0] = qv[k][1] = qv[k][2] = qv[k][3] = 0.f;
        if (s < slots) {
            const float* qr = p.q + ((size_t)(row0 + s / heads) * p.num_heads + kvh * p.group + h0 + s % heads) * D;
            if constexpr (FMT == kWinQ4) {
                if (lane < 16 * NW) {
                    const float4 a = __ldcg(reinterpret_cast<const float4*>(qr + 8 * (lane >> 1)));
                    const float4 b = __ldcg(reinterpret_cast<const float4*>(qr + 8 * (lane >> 1) + 4));
                    qv[k][0] = lane & 1 ? a.y : a.x, qv[k][1] = lane & 1 ? a.w : a.z;
                    qv[k][2] = lane & 1 ? b.y : b.x, qv[k][3] = lane & 1 ? b.w : b.z;
                }
            } else {
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    const float2 a = __ldcg(reinterpret_cast<const float2*>(qr) + lane + 32 * w);
                    qv[k][2 * w] = a.x, qv[k][2 * w + 1] = a.y;
                }
            }
        }
    }

    // contexts: this lane's score columns, and the tile's extremes over rows that see anything
    const int limit = min(p.max_ctx, p.mbps * 16);
    const int window = p.window > 0 ? p.window : 0x7fffffff;
    const int slot = __ldcg(p.row_slot + row0);
    const bool slot_ok = slot >= 0 && slot < p.num_slots;
    int ctx[2];
    int cmax = 0, cmin = 0x7fffffff;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int s = (2 * t + e) % SL;
        ctx[e] = s < slots && slot_ok ? min(max(__ldcg(p.row_ctx + row0 + s / heads), 0), limit) : 0;
        cmax = max(cmax, ctx[e]);
        if (ctx[e] > 0) cmin = min(cmin, ctx[e]);
    }
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
        cmax = max(cmax, __shfl_xor_sync(0xffffffffu, cmax, x));
        cmin = min(cmin, __shfl_xor_sync(0xffffffffu, cmin, x));
    }
    if (!slot_ok && threadIdx.x == 0) record_error(DEV_ERR_ATTN_BOUNDS);
    // blocks that hold a visible key: the sinks', then from the earliest window's start
    const int nb_end = (cmax + 15) >> 4;
    const int nb_sink = min((min(p.sinks, cmax) + 15) >> 4, nb_end);
    const int first = max(nb_sink, cmax > 0 ? max(0, cmin - window) >> 4 : 0);
    const int past_sinks = first - nb_sink;  // what the blocks after the sinks' skip
    const int nb = nb_sink + max(0, nb_end - first);
    // this warp's share of them: [i0, i0 + mine)
    const int workers = (int)splits * W, me = (int)rank * W + warp;
    const int even = nb / workers, rest = nb % workers;
    const int i0 = me * even + min(me, rest), mine = even + (me < rest);

    // ids of the warp's next 32 blocks, one per lane
    const int32_t* table = p.block_table + (size_t)(slot_ok ? slot : 0) * p.mbps;
    const uint8_t* base = p.kv + ((size_t)p.layer * 2 * p.kv_heads + kvh) * G::BYTES;
    const uint32_t ring = smem_u32(smem) + warp * RING;
    int ids = 0;
    bool bad_id = false;  // an id outside the pool came up: its keys are hidden
    auto table_id = [&](int n) {  // of the warp's block n
        const int i = i0 + n;
        return __ldcg(table + (i < nb_sink ? i : i + past_sinks));
    };
    // copy the K (v = 0) or V chunks of blocks n .. n + KB - 1; every lane commits a group, full or empty
    auto issue = [&](int n, int v, uint32_t buf) {
        if (n < mine) {
            if (v == 0 && (n & 31) == 0) {
                ids = n + lane < mine ? table_id(n + lane) : 0;
                const bool out = ids < 0 || ids >= p.num_blocks;
                if (__any_sync(0xffffffffu, out)) bad_id = true;
                if (out) {
                    record_error(DEV_ERR_ATTN_BOUNDS);
                    ids = 0;
                }
            }
            const uint8_t* from = base + (v ? p.v_offset : 0);
#pragma unroll
            for (int k = 0; k < KB; ++k) {
                if (k > 0 && n + k >= mine) break;
                const uint32_t id = (uint32_t)__shfl_sync(0xffffffffu, ids, (n & 31) + k);
                G::copy(buf + k * G::BYTES, from + (uint64_t)id * p.block_bytes, lane);
            }
        }
        cp_async_commit();
    };
    // steps are K, V, K, V, ...; step h lives in buffer h % NBUF, and NBUF - 1 are under way
#pragma unroll
    for (int h = 0; h < NBUF - 1; ++h) issue((h >> 1) * KB, h & 1, ring + h * STEP);

    // Q^T operand, made once per CTA.
    //   fp16: q scaled by a power of two that brings the slot's largest channel to [2^11, 2^12), so
    //   that two fp16 halves hold it whatever its size.
    //   4 bits: q / (largest channel) * 2^21 rounded to an integer, digits of 65536, 256 and 1, the lower two in [-128, 127].
#pragma unroll
    for (int k = 0; k < QS; ++k) {
        const int s = warp + k * W;
        if (s >= SL) break;
        float amax = max_nan(max_nan(fabsf(qv[k][0]), fabsf(qv[k][1])), max_nan(fabsf(qv[k][2]), fabsf(qv[k][3])));
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, x));
        float f;
        if constexpr (FMT == kWinQ4) {
            // a q that is zero everywhere (or below what a reciprocal holds) scores zero; one that is
            // not finite makes its scores NaN through f
            const float up = amax >= 1e-30f ? 2097152.f / amax : 0.f;
            f = amax * (1.f / 2097152.f) * p.scale_log2;
            if (!(amax < INFINITY)) f = __int_as_float(0x7fffffff);
            float sum = (qv[k][0] + qv[k][1]) + (qv[k][2] + qv[k][3]);
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            uint32_t hi = 0, mid = 0, lo = 0;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int x = __float2int_rn(qv[k][c] * up), y = (x + 128) >> 8, h = (y + 128) >> 8;
                hi |= (uint32_t)(h & 255) << (8 * c);
                mid |= (uint32_t)((y - 256 * h) & 255) << (8 * c);
                lo |= (uint32_t)((x - 256 * y) & 255) << (8 * c);
            }
            const int w = lane >> 4;
            if (w < NW) {
                uint32_t* dst = &s_q[s][(lane >> 2) & 3][2 * (2 * w + (lane & 1)) + ((lane >> 1) & 1)];
                dst[0] = hi;
                dst[2 * NQ] = mid;
                dst[4 * NQ] = lo;
                if ((lane & 15) == 0) s_qsum[s][w] = sum * p.scale_log2;
            }
        } else {
            const int ex = max((int)(__float_as_uint(amax) >> 23), 12);
            const float up = __uint_as_float((uint32_t)(265 - ex) << 23);
            f = __uint_as_float((uint32_t)(ex - 11) << 23) * p.scale_log2;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                uint32_t hi, lo;
                split_h2(qv[k][2 * w] * up, qv[k][2 * w + 1] * up, hi, lo);
                const int pair = lane + 32 * w;  // channels 16 i + 8 h + 2 t: word 2 i + h of t
                s_q[s][pair & 3][pair >> 2] = hi;
                s_q[s][pair & 3][2 * NQ + (pair >> 2)] = lo;
            }
        }
        if (lane == 0) s_qf[s] = f;
    }
    __syncthreads();
    uint32_t qh[NQ][2], qm[FMT == kWinQ4 ? NQ : 1][2], ql[NQ][2];  // of column g: slot g % SL
    float sf[2], qsum[NW][2];          // of this lane's score columns
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            qh[i][h] = s_q[g % SL][t][2 * i + h];
            if constexpr (FMT == kWinQ4) qm[i][h] = s_q[g % SL][t][2 * NQ + 2 * i + h];
            ql[i][h] = s_q[g % SL][t][2 * NQ * (QP - 1) + 2 * i + h];
        }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        sf[e] = s_qf[(2 * t + e) % SL];
#pragma unroll
        for (int w = 0; w < NW; ++w) qsum[w][e] = FMT == kWinQ4 ? s_qsum[(2 * t + e) % SL][w] : 0.f;
    }

    float o[MT][4];  // FMT q4: row tile 4 w + k holds channels 64 w + 8 g + 2 k (c 0, 1) and + 1 (c 2, 3)
    float zacc[NW][2], l[2] = {0.f, 0.f};
    // running maximum of the two columns' slots, and what probabilities are relative to (the maximum, or 2^-7 of it
    // over fp16; 0 until a key is seen)
    float m[2] = {-INFINITY, -INFINITY}, mu[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < MT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) zacc[w][0] = zacc[w][1] = 0.f;

    uint32_t buf = ring;      // of the step at hand
    uint32_t ahead = ring + (NBUF - 1) * STEP;  // ... and of the one that is issued at it
    auto turn = [&](int n, int v) {  // begin step (n, v): its chunks are there, the last step's buffer is free
        cp_async_wait<NBUF - 2>();
        __syncwarp();
        issue(n + (NBUF - 1 + v) / 2 * KB, (NBUF - 1 + v) & 1, ahead);
    };
    auto next_step = [&]() {
        ahead = buf;
        buf = buf + STEP == ring + RING ? ring : buf + STEP;
    };

    // one iteration's blocks (n .. n + n_here - 1); MASKED: some row does not see all of them.
    // j0: first token of this lane's block; present: it is there and in the pool
    auto blocks = [&](auto masked, const int n, const int n_here, const int j0, const bool present) {
        constexpr bool MASKED = decltype(masked)::value;
        auto sees = [&](int i) {  // score i: token g + 8 (i / 2) of block kb, column 2 t + i % 2
            const int j = j0 + g + 8 * (i >> 1), c = ctx[i & 1];
            return present && j < c && (j >= c - window || j < p.sinks);
        };

        // S^T, relative to mu
        float s[4];
        if constexpr (FMT == kWinQ4) {
            int acc[NW][4];
            constexpr int KI = KB > 1 ? 2 : 1;  // blocks whose chains of instructions run interleaved
#pragma unroll
            for (int k0 = 0; k0 < KB; k0 += KI) {
                if (MASKED && k0 > 0 && k0 >= n_here) break;
                uint32_t kw[KI][2][2 * NW];  // tokens g and g + 8
                const int row = g * (D / 2) + t * 8 * NW;
                const int sw = D == 128 ? row ^ (((g >> 1) & 3) << 5) : row;
#pragma unroll
                for (int k = 0; k < KI; ++k) {
                    lds_words(kw[k][0], buf + (k0 + k) * G::BYTES + sw);
                    lds_words(kw[k][1], buf + (k0 + k) * G::BYTES + sw + 8 * (D / 2));
                }
                int d[KI][NW][4];
                uint32_t a[2][KI][NW][4];  // even and odd nibbles
#pragma unroll
                for (int k = 0; k < KI; ++k)
#pragma unroll
                    for (int w = 0; w < NW; ++w)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t x = kw[k][i & 1][(i >> 1) * NW + w];
                            a[0][k][w][i] = x & 0x0f0f0f0fu;
                            a[1][k][w][i] = (x >> 4) & 0x0f0f0f0fu;
                        }
#pragma unroll
                for (int step = 0; step < 6; ++step)  // high digits of both nibbles, then lower ones
#pragma unroll
                    for (int k = 0; k < KI; ++k)
#pragma unroll
                        for (int w = 0; w < NW; ++w) {
                            if (step == 2 || step == 4)
#pragma unroll
                                for (int i = 0; i < 4; ++i) d[k][w][i] *= 256;
                            if (step == 0) mma_u8s8_first(d[k][w], a[0][k][w], qh[2 * w]);
                            else mma_u8s8(d[k][w], a[step & 1][k][w], (step < 2 ? qh : step < 4 ? qm : ql)[2 * w + (step & 1)]);
                        }
#pragma unroll
                for (int k = 0; k < KI; ++k)
#pragma unroll
                    for (int w = 0; w < NW; ++w)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (k0 + k == 0 || kb == k0 + k) acc[w][i] = d[k][w][i];
            }
            float2 kp[NW][2];
#pragma unroll
            for (int w = 0; w < NW; ++w)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    kp[w][h] = lds_half2(buf + kb * G::BYTES + Q4Layout<D>::PARAMS + w * 64 + (g + 8 * h) * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float d = (float)acc[0][i] * kp[0][i >> 1].x;
                float z = fmaf(qsum[0][i & 1], kp[0][i >> 1].y, -mu[i & 1]);
                if constexpr (NW == 2) {
                    d = fmaf((float)acc[1][i], kp[1][i >> 1].x, d);
                    z = fmaf(qsum[1][i & 1], kp[1][i >> 1].y, z);
                }
                s[i] = fmaf(d, sf[i & 1], z);
            }
        } else {
            float acc[4][4];  // independent chains: even and odd steps, each half of q
            const int r = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                uint32_t a[4];
                const int c = 2 * i + (lane >> 4);
                ldsm_x4(buf + (r * (D / 8) + (c ^ (r & 7))) * 16, a);
                if (i < 2) mma_f16_first(acc[i & 1], a, qh[i]), mma_f16_first(acc[2 + (i & 1)], a, ql[i]);
                else mma_f16(acc[i & 1], a, qh[i]), mma_f16(acc[2 + (i & 1)], a, ql[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                s[i] = fmaf((acc[0][i] + acc[1][i]) + (acc[2][i] + acc[3][i]), sf[i & 1], -mu[i & 1]);
        }
        if constexpr (MASKED) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!sees(i)) s[i] = -INFINITY;
        }

        // softmax in the log2 domain; the running maximum moves only when a score passes it by 8, so that
        // probabilities stay below 2^8 (fp16: 2^15)
        constexpr float kShift = FMT == kWinF16 ? kPShift : 0.f;
        bool grow = false;
#pragma unroll
        for (int e = 0; e < 2; ++e) grow |= fmaxf(s[e], s[2 + e]) > (m[e] == -INFINITY ? -INFINITY : 8.f + kShift);
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float mn = fmaxf(s[e], s[2 + e]) + mu[e];
#pragma unroll
                for (int x = SL / 2; x < 32; x <<= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, x));
                mn = fmaxf(mn, m[e]);
                const float corr = mn == -INFINITY ? 1.f : ex2_approx(m[e] - mn);
                const float to = mn == -INFINITY ? 0.f : mn - kShift;
                s[e] += mu[e] - to;
                s[2 + e] += mu[e] - to;
                m[e] = mn;
                mu[e] = to;
                l[e] *= corr;
#pragma unroll
                for (int w = 0; w < NW; ++w) zacc[w][e] *= corr;
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    o[i][e] *= corr;
                    o[i][2 + e] *= corr;
                }
            }
        }
        float pr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            pr[i] = ex2_approx(s[i]);
            l[i & 1] += pr[i];
        }

        next_step();
        turn(n, 1);
        if constexpr (MASKED && FMT == kWinF16) {
            // a key that some row does not see must not reach it through 0 * V: what is not finite in
            // such a row of V is set to zero, and the rows that do see it become NaN
            const int r = lane >> 1, j = j0 + r;
            const bool all = present && j < cmin && (j >= cmax - window || j < p.sinks);
            bool bad = false;
            if (!all) {
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    const uint32_t at = buf + (r * (D / 8) + (((lane & 1) * (D / 16) + c) ^ (r & 7))) * 16;
                    uint32_t u[4];
                    lds_words(u, at);
                    bool here = false;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        if ((u[x] & 0x7c00u) == 0x7c00u) u[x] &= 0xffff0000u, here = true;
                        if ((u[x] & 0x7c000000u) == 0x7c000000u) u[x] &= 0x0000ffffu, here = true;
                    }
                    if (here)
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(u[0]), "r"(u[1]), "r"(u[2]),
                                     "r"(u[3])
                                     : "memory");
                    bad |= here;
                }
            }
            const unsigned rows = __ballot_sync(0xffffffffu, bad);
            if (rows) {
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (((rows >> (2 * (g + 8 * (i >> 1)))) & 3) && sees(i)) l[i & 1] = __int_as_float(0x7fffffff);
            }
        }

        // O^T += V^T P^T
        if constexpr (FMT == kWinQ4) {
            uint32_t ph[NW][2], pl[NW][2];  // P^T operands of the KB blocks: column g belongs to block g / SL
#pragma unroll
            for (int w = 0; w < NW; ++w) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float2 vp = lds_half2(buf + kb * G::BYTES + Q4Layout<D>::PARAMS + w * 64 + (g + 8 * h) * 4);
                    const float sc = vp.x * kPScale;
                    float x[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float pe = pr[2 * h + e];
                        x[e] = pe * sc;
                        if constexpr (MASKED) {  // the parameters of a hidden key may be anything
                            if (sees(2 * h + e)) zacc[w][e] = fmaf(pe, vp.y, zacc[w][e]);
                            else x[e] = 0.f;
                        } else {
                            zacc[w][e] = fmaf(pe, vp.y, zacc[w][e]);
                        }
                    }
                    // bf16 halves: the first cuts x off (the rest is exact in fp32), the second rounds the
                    // rest: 16 bits together.  To nearest, as cutting off would be a bias that stays when a
                    // long row's values average out (32749 keys: 1e-3 of the output)
                    const uint32_t hi = prmt(__float_as_uint(x[0]), __float_as_uint(x[1]), 0x7632);
                    const float r0 = x[0] - __uint_as_float(hi << 16), r1 = x[1] - __uint_as_float(hi & 0xffff0000u);
                    ph[w][h] = movmatrix_t(hi);
                    pl[w][h] = movmatrix_t(pack_bf2(r0, r1));
                    if constexpr (KB > 1) pl[w][h] = __shfl_xor_sync(0xffffffffu, pl[w][h], 16);  // to column g ^ 4
                }
            }
#pragma unroll
            for (int k = 0; k < KB; ++k) {
                if (MASKED && k > 0 && k >= n_here) break;
                const uint32_t vs = buf + k * G::BYTES;
                uint32_t v[4][NW];  // tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 2 * t + (i & 1) + 8 * (i >> 1), at = r * (D / 2) + g * 4 * NW;
                    lds_words(v[i], vs + (D == 128 ? at ^ (t << 5) : at));
                }
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    uint32_t b[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        b[h] = ph[w][h];
                        if constexpr (KB > 1) b[h] = g / SL == k ? ph[w][h] : (g ^ 4) / SL == k ? pl[w][h] : 0u;
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {  // nibbles 0-3, 4-7 of two tokens side by side
                        const uint32_t x = prmt(v[0][w], v[1][w], h ? 0x7632 : 0x5410);
                        const uint32_t y = prmt(v[2][w], v[3][w], h ? 0x7632 : 0x5410);
                        const uint32_t a1[4] = {x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u};
                        const uint32_t a2[4] = {(x >> 8) & 0x000f000fu, (x >> 8) & 0x00f000f0u, (y >> 8) & 0x000f000fu,
                                                (y >> 8) & 0x00f000f0u};
                        mma_bf16(o[4 * w + 2 * h], a1, b);
                        mma_bf16(o[4 * w + 2 * h + 1], a2, b);
                        if constexpr (KB == 1) {
                            mma_bf16(o[4 * w + 2 * h], a1, pl[w]);
                            mma_bf16(o[4 * w + 2 * h + 1], a2, pl[w]);
                        }
                    }
                }
            }
        } else {
            uint32_t ph[2], pl[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                split_h2(pr[2 * h], pr[2 * h + 1], ph[h], pl[h]);
                ph[h] = movmatrix_t(ph[h]);
                pl[h] = movmatrix_t(pl[h]);
            }
            const int r = (lane & 7) + (lane >> 4) * 8;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                uint32_t a[4];
                const int c = 2 * i + ((lane >> 3) & 1);
                ldsm_x4_t(buf + (r * (D / 8) + (c ^ (r & 7))) * 16, a);
                mma_f16(o[i], a, ph);
                mma_f16(o[i], a, pl);
            }
        }
    };

    for (int n = 0; n < mine; n += KB) {
        turn(n, 0);
        const int i = i0 + n + kb;
        const int j0 = (i < nb_sink ? i : i + past_sinks) * 16;
        bool present = n + kb < mine;
        const bool whole = present && j0 + 16 <= cmin && (j0 >= cmax - window || j0 + 16 <= p.sinks) && !bad_id;
        if (__all_sync(0xffffffffu, whole)) {
            blocks(std::false_type{}, n, KB, j0, true);
        } else {
            if (bad_id && present) {
                const int id = table_id(n + kb);
                present = id >= 0 && id < p.num_blocks;
            }
            blocks(std::true_type{}, n, min(KB, mine - n), j0, present);
        }
        next_step();
    }
    cp_async_wait<0>();
    __syncwarp();  // the ring becomes the warp's partial output

    // fold: lanes and column groups, then warps of the CTA, then CTAs of the cluster
    float* part = reinterpret_cast<float*>(smem + warp * RING);  // [SL][D]
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int sl = (2 * t + e) % SL;
        // a row without keys in a tile of rows that have some: whole blocks scored its q unmasked, so its sum may
        // be anything and its maximum infinite (inf - inf would make the folds' factors NaN)
        if (ctx[e] == 0) l[e] = 0.f, m[e] = -INFINITY;
#pragma unroll
        for (int x = SL / 2; x < 32; x <<= 1) {
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], x);
#pragma unroll
            for (int w = 0; w < NW; ++w) zacc[w][e] += __shfl_xor_sync(0xffffffffu, zacc[w][e], x);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            float lo = o[i][e], hi = o[i][2 + e];  // rows g and g + 8 of the tile
#pragma unroll
            for (int x = SL / 2; x < 4; x <<= 1) {
                lo += __shfl_xor_sync(0xffffffffu, lo, x);
                hi += __shfl_xor_sync(0xffffffffu, hi, x);
            }
            int d0 = 16 * i + g, d1 = d0 + 8;
            if constexpr (FMT == kWinQ4) {
                lo = fmaf(lo, kPUnscale, zacc[i >> 2][e]);
                hi = fmaf(hi, kPUnscale * 0.0625f, zacc[i >> 2][e]);
                d0 = 64 * (i >> 2) + 8 * g + 2 * (i & 3), d1 = d0 + 1;
            }
            if (kb == 0) part[sl * D + d0] = lo, part[sl * D + d1] = hi;
        }
        if (g == 0 && kb == 0) s_ml[warp][sl][0] = m[e], s_ml[warp][sl][1] = l[e];
    }
    __syncthreads();
    const float* parts = reinterpret_cast<const float*>(smem);
    constexpr int kPartStride = RING / 4;
    auto store = [&](int e, float v) {
        const int r = e / D, d = e % D;
        const size_t idx = ((size_t)(row0 + r / heads) * p.num_heads + kvh * p.group + h0 + r % heads) * D + d;
        const __nv_bfloat16 hi = __float2bfloat16_rn(v);
        p.out[idx] = hi;
        if (p.out_lo) p.out_lo[idx] = __float2bfloat16_rn(v - __bfloat162float(hi));
    };
    for (int e = threadIdx.x; e < slots * D; e += W * 32) {
        const int r = e / D, d = e % D;
        float mx = s_ml[0][r][0];
#pragma unroll
        for (int w = 1; w < W; ++w) mx = fmaxf(mx, s_ml[w][r][0]);
        float sum = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float mw = s_ml[w][r][0], lw = s_ml[w][r][1];
            if (mw != -INFINITY) {  // a warp without keys holds nothing
                const float f = ex2_approx(mw - mx);
                sum += lw * f;
                acc += parts[w * kPartStride + e] * f;
            } else if (lw != 0.f) {  // nothing but NaN scores
                sum = lw;
            }
        }
        if (splits == 1) {
            store(e, sum == 0.f ? 0.f : acc / sum);
        } else {
            reinterpret_cast<float*>(smem)[e] = acc;  // only this thread reads or writes the element
            if (d == 0) s_part[r][0] = mx, s_part[r][1] = sum;
        }
    }
    if (splits == 1) return;
    cluster_sync();
    // a warp takes 32 channels of a slot; lane c fetches CTA c's (max, sum), every lane its channel of
    // every CTA, all loads under way at once
    for (int j = (int)rank * W + warp; j < slots * (D / 32); j += (int)splits * W) {
        const int r = j / (D / 32), e = j * 32 + lane;
        float mc = -INFINITY, lc = 0.f;
        if (lane < (int)splits) {
            mc = ld_dsmem_now(map_to_rank(smem_u32(&s_part[r][0]), lane));
            lc = ld_dsmem_now(map_to_rank(smem_u32(&s_part[r][1]), lane));
        }
        float v[kWinMaxSplits];
#pragma unroll
        for (int c = 0; c < kWinMaxSplits; ++c)
            if (c < (int)splits) v[c] = ld_dsmem_now(map_to_rank(smem_u32(parts + e), c));
        const float mx = warp_max(mc);
        const float f = mc == -INFINITY ? 0.f : ex2_approx(mc - mx);
        // a CTA without keys holds nothing (0 f), one of nothing but NaN scores a sum that is not zero
        const float sum = warp_sum(mc == -INFINITY && lc != 0.f ? lc : lc * f);
        float acc = 0.f;
#pragma unroll
        for (int c = 0; c < kWinMaxSplits; ++c) {
            const float fc = __shfl_sync(0xffffffffu, f, c);
            if (c < (int)splits && fc != 0.f) acc = fmaf(v[c], fc, acc);
        }
        store(e, sum == 0.f ? 0.f : acc / sum);
    }
    cluster_sync();  // no CTA leaves while another reads its shared memory
}

template <int FMT, int D, int SL, int W, int MINB>
inline int launch_window_rows_w(const WinParams& p, long long tiles, int splits, cudaStream_t st) {
    // 4 bits: three steps of KB chunks (one iteration's K and V ahead of the step at hand); with one
    // block a step, six, for the same bytes under way.  fp16: four steps of one 4 KB chunk.
    constexpr int NBUF = FMT == kWinQ4 ? (SL == 8 ? 6 : 3) : 4;
    constexpr int smem = W * NBUF * (8 / SL) * WinChunk<FMT, D>::BYTES;
    constexpr auto kernel = paged_attn_window_kernel<FMT, D, SL, W, NBUF, MINB>;
    QTTS_CHECK_CUDA((func_attr_once<kernel>(smem, true)));
    QTTS_CHECK_CUDA(launch_pdl(kernel, dim3((unsigned)(tiles * splits)), dim3(W * 32), smem, st, dim3(splits, 1, 1), p));
    return QTTS_OK;
}

// How a tile's keys are shared.  16 warps fit an SM over the 4-bit pool, 12 over fp16; all variants
// fill it, with fewer and larger CTAs the fewer tiles there are: warps of one CTA fold cheaper than
// CTAs of a cluster.  Beyond the tiles that half-SM CTAs cover, a cluster splits a tile while every
// warp keeps three blocks.  Measured (us, 16 heads over 8, rows x context, B200, K and V from HBM), warps x splits:
//   4 bits  1 x 4000:  8 x 8 8.0    4 x 16 8.1   8 x 16 9.4   8 x 4 9.9    2 x 16 9.3
//          16 x 520:   8 x 1 7.8    4 x 1 8.7    4 x 2 9.4    8 x 2 10.2   4 x 4 10.1
//          64 x 520:   4 x 1 16.1   2 x 1 16.3   8 x 1 19.9   4 x 2 23.0
//         128 x 520:   2 x 1 26.1   4 x 1 28.3   8 x 1 36.4
//   fp16    1 x 4000:  6 x 8 10.2   3 x 16 10.5  6 x 16 10.6  6 x 4 14.2
//          16 x 520:   6 x 1 10.3   6 x 2 11.2   3 x 2 12.0   3 x 1 12.1
//          64 x 520:   3 x 1 26.9   2 x 1 27.7   6 x 1 28.9   3 x 2 33.2
//         128 x 520:   3 x 1 48.8   2 x 1 58.0   6 x 1 53.8
template <int FMT, int D, int SL>
inline int launch_window_rows(WinParams p, cudaStream_t st) {
    using G = WinChunk<FMT, D>;
    constexpr int WL = FMT == kWinQ4 ? 8 : 6;  // warps of a half-SM CTA
    p.head_tiles = ceil_div(p.group, SL);
    p.qt = p.group >= SL ? 1 : SL / p.group;
    if (p.qt > p.S) p.qt = p.S;
    p.tiles = ceil_div(p.S, p.qt);
    const long long block_bytes = (long long)p.num_layers * 2 * p.kv_heads * G::BYTES;
    QTTS_REQUIRE(block_bytes < (1ll << 31), "paged attention: %lld bytes per block", block_bytes);
    p.block_bytes = (uint32_t)block_bytes;
    p.v_offset = (uint32_t)(p.kv_heads * G::BYTES);
    const long long tiles = (long long)(p.R / p.S) * p.tiles * p.kv_heads * p.head_tiles;
    QTTS_REQUIRE(tiles * kWinMaxSplits < (1ll << 31), "paged attention: %lld tiles", tiles);
    const int slots = 2 * num_sms();
    if (tiles > slots) {
        if constexpr (FMT == kWinQ4) {
            if (tiles > 2 * slots) return launch_window_rows_w<FMT, D, SL, 2, 8>(p, tiles, 1, st);
            return launch_window_rows_w<FMT, D, SL, 4, 4>(p, tiles, 1, st);
        }
        return launch_window_rows_w<FMT, D, SL, 3, 4>(p, tiles, 1, st);
    }
    // blocks one tile walks, at most
    const int limit = p.max_ctx < p.mbps * 16 ? p.max_ctx : p.mbps * 16;
    long long keys = limit;
    if (p.window > 0 && (long long)p.window + p.sinks + p.qt + 32 < keys) keys = (long long)p.window + p.sinks + p.qt + 32;
    int splits = 1;
    while (splits < kWinMaxSplits && tiles * splits * 2 <= slots && keys >= 2ll * splits * WL * 3 * 16) splits *= 2;
    return launch_window_rows_w<FMT, D, SL, WL, 2>(p, tiles, splits, st);
}

template <int FMT, int D>
inline int launch_window_attention(const WinParams& p, cudaStream_t st) {
    // the fp16 pool's blocks are four times the bytes for the same work, so that eight columns for
    // one block cost it nothing; 4 bits: as few slots as the rows need, more blocks at once
    if constexpr (FMT == kWinQ4) {
        const int slots = p.S > 1 ? 8 : p.group;
        if (slots <= 2) return launch_window_rows<FMT, D, 2>(p, st);
        if (slots <= 4) return launch_window_rows<FMT, D, 4>(p, st);
    }
    return launch_window_rows<FMT, D, 8>(p, st);
}

}  // namespace qtts
