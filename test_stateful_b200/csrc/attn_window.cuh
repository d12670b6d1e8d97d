// Paged GQA attention with a sliding window and sinks, over the fp16 pool or the 4-bit one.
//
// A query row of context c (its keys are 0 .. c - 1) sees key j when
//     j < c  and  (j >= c - window  or  j < sinks  or  window == 0),
// and gets softmax(q k^T / sqrt(D)) v over those keys; a row that sees none gets zeros.
//
// Row kernel.  One warp walks 16-token blocks, copied ahead of use into a ring of its own in shared
// memory (cp.async, 16 bytes a lane).  The tensor work is mma.sync m16n8k16 with the keys on the M
// side and (query, head) slots on the N side:
//     S^T[16 tokens][8]   += K[16][16 channels] . Q^T       D/16 instructions a block
//     O^T[16 channels][8] += V^T[16][16 tokens] . P^T       D/16 instructions a block
// Four slots fill the eight columns: columns 0-3 carry the operand's high half, 4-7 what rounding
// took from it, so that q and the probabilities keep 16 bits or more at no extra instructions;
// lanes t and t ^ 2 of a quad hold the two halves of the same scores.  movmatrix turns the
// probabilities from S^T's accumulator layout into the operand layout.
//
// 4-bit pool: a nibble masked out of a code word IS a small fp16 or bf16 number (a subnormal:
// nibble << 0 = code * 2^-24 or 2^-133, nibble << 4 = 16 times that), so that no conversion is
// needed; the powers of two move into q and the output, a token's scale into the score (K) and the
// probability (V), and its zero multiplies sum(q) and p on the fp32 side.  The channel order of the
// contractions is the one in which a lane's words arrive: lane (g, t) takes of K tokens g and g + 8
// the channels 64 w + 16 t .. + 15, of V tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9 the channels
// 64 w + 8 g .. + 7.
#pragma once

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
    int head_tiles;         // tiles a KV head's query heads are cut into
    int qt, tiles;          // queries per tile, tiles per stream
    int layer, num_layers, num_blocks, num_slots, mbps;
    int max_ctx, window, sinks;
    float scale_log2;       // log2(e) / sqrt(D)
};

enum { kWinF16 = 0, kWinQ4 = 1 };

__device__ __forceinline__ void mma_16816_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// A block's stage in shared memory: the K chunk, then the V chunk, 16-byte pieces permuted so that
// the fragment reads meet no bank twice.
//   fp16: rows of 2 D bytes read by ldmatrix; piece c of row r sits at c ^ (r % 8).
//   4 bits: rows of D / 2 bytes; of D = 128 the eight pieces of two rows sit at L ^ 2 (r / 2 % 4):
//   K reads two whole rows a quarter-warp, V one 16-channel stretch of rows 0, 2, 4, 6 (+ 1, + 8).
template <int FMT, int D>
struct WinStage {
    static constexpr int NW = D / 64;
    static constexpr int CHUNK = FMT == kWinQ4 ? Q4Layout<D>::CHUNK : 32 * D;  // bytes of one (block, layer, k|v, head)
    static constexpr int BYTES = 2 * CHUNK;

    // this lane's copies of one block
    static __device__ __forceinline__ void copy(uint32_t dst, const uint8_t* k, const uint8_t* v, int lane) {
        if constexpr (FMT == kWinQ4) {
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                const int j = lane + 32 * i, sw = D == 128 ? j ^ ((j >> 2) & 6) : j;
                cp_async16(dst + sw * 16, k + j * 16);
                cp_async16(dst + CHUNK + sw * 16, v + j * 16);
            }
            constexpr int PP = 4 * NW;  // pieces of (scale, zero) pairs
            if (lane < 2 * PP) {
                const int off = Q4Layout<D>::PARAMS + (lane & (PP - 1)) * 16;
                cp_async16(dst + off + (lane < PP ? 0 : CHUNK), (lane < PP ? k : v) + off);
            }
        } else {
            constexpr int PR = D / 8;  // pieces per row
#pragma unroll
            for (int i = 0; i < 16 * PR / 32; ++i) {
                const int j = lane + 32 * i, r = j / PR, c = j % PR;
                const int sw = r * PR + (c ^ (r & 7));
                cp_async16(dst + sw * 16, k + j * 16);
                cp_async16(dst + CHUNK + sw * 16, v + j * 16);
            }
        }
    }
};

// The 4-bit pool's probabilities carry 2^100 into the bf16 product, whose other factor is code * 2^-133:
// a probability is at most 2^8 and a scale below 2^14, so 2^122 at most, and the products are
// normal numbers down to probabilities of 2^-90.
constexpr float kPScale = 1.2676506002282294e30f;  // 2^100
constexpr float kPUnscale = 8589934592.f;          // 2^133 / 2^100

// NB: column groups of four slots.  W warps per CTA, ST stages per warp.
template <int FMT, int D, int NB, int W, int ST>
__global__ void __launch_bounds__(W * 32) paged_attn_window_kernel(const WinParams p) {
    using G = WinStage<FMT, D>;
    constexpr int NW = G::NW, MT = D / 16, SL = 4 * NB;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_ml[W][SL][2];
    __shared__ float s_part[SL][2];  // the CTA's (max, sum) per slot
    static_assert(SL * D * 4 <= ST * G::BYTES, "a warp's partial output replaces its ring");

    griddep_wait();
    griddep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
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

    // contexts: this lane's slots, and the tile's extremes over rows that see anything
    const int limit = min(p.max_ctx, p.mbps * 16);
    const int window = p.window > 0 ? p.window : 0x7fffffff;
    const int slot = __ldg(p.row_slot + row0);
    const bool slot_ok = slot >= 0 && slot < p.num_slots;
    int ctx[NB][2];
    int cmax = 0, cmin = 0x7fffffff;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int s = 4 * b + 2 * (t & 1) + e;
            ctx[b][e] = s < slots && slot_ok ? min(max(__ldg(p.row_ctx + row0 + s / heads), 0), limit) : 0;
            cmax = max(cmax, ctx[b][e]);
            if (ctx[b][e] > 0) cmin = min(cmin, ctx[b][e]);
        }
    cmax = max(cmax, __shfl_xor_sync(0xffffffffu, cmax, 1));
    cmin = min(cmin, __shfl_xor_sync(0xffffffffu, cmin, 1));
    if (!slot_ok && threadIdx.x == 0) record_error(DEV_ERR_ATTN_BOUNDS);
    // blocks that hold a visible key: the sinks', then from the earliest window's start
    const int nb_end = (cmax + 15) >> 4;
    const int nb_sink = min((min(p.sinks, cmax) + 15) >> 4, nb_end);
    const int first = max(nb_sink, cmax > 0 ? max(0, cmin - window) >> 4 : 0);
    const int nb = nb_sink + max(0, nb_end - first);
    const int stride = (int)splits * W;
    const int i0 = (int)rank * W + warp;
    const int mine = i0 < nb ? (nb - i0 + stride - 1) / stride : 0;
    auto block_no = [&](int n) {  // the warp's n-th block
        const int i = i0 + n * stride;
        return i < nb_sink ? i : first + (i - nb_sink);
    };

    // ids of the warp's next 32 blocks, one per lane; an id outside the pool hides its keys
    const int32_t* table = p.block_table + (size_t)(slot_ok ? slot : 0) * p.mbps;
    const size_t block_stride = (size_t)p.num_layers * 2 * p.kv_heads * G::CHUNK;
    const uint8_t* base = p.kv + ((size_t)p.layer * 2 * p.kv_heads + kvh) * G::CHUNK;
    const size_t v_off = (size_t)p.kv_heads * G::CHUNK;
    const uint32_t ring = smem_u32(smem) + warp * ST * G::BYTES;
    int ids = -1;
    auto issue = [&](int n) {  // copy block n into its stage; every lane commits a group, full or empty
        if (n < mine) {
            if ((n & 31) == 0) {
                ids = -1;
                if (n + lane < mine) {
                    const int b = __ldg(table + block_no(n + lane));
                    if (b >= 0 && b < p.num_blocks) ids = b;
                    else record_error(DEV_ERR_ATTN_BOUNDS);
                }
            }
            const int id = __shfl_sync(0xffffffffu, ids, n & 31);
            if (id >= 0) {
                const uint8_t* c = base + (size_t)id * block_stride;
                G::copy(ring + (n % ST) * G::BYTES, c, c + v_off, lane);
            }
            cp_async_commit();
            return id >= 0;
        }
        cp_async_commit();
        return false;
    };
    uint32_t present = 0;  // bit n % 32: block n is in the pool
#pragma unroll
    for (int n = 0; n < ST - 1; ++n)
        if (issue(n)) present |= 1u << n;

    // Q^T operand.  Each slot's q is scaled by a power of two that brings its largest channel to
    // [2^11, 2^12), so that fp16 halves hold it whatever its size; the upper nibbles' channels take
    // 1/16.  Lane (g, t) holds column g: slot g % 4 of each column group, high (g < 4) or low half.
    uint32_t qb[NB][MT][2];
    float sf[NB][2], qsum[NB][NW][2];  // of this lane's score columns: accumulator -> log2 units, sum of q
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int s = 4 * b + (g & 3);
        const bool valid = s < slots;
        const float* qr = p.q + ((size_t)(row0 + (valid ? s / heads : 0)) * p.num_heads + kvh * p.group + h0 +
                                 (valid ? s % heads : 0)) * D;
        float v[NW][16], sum[NW], amax = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            sum[w] = 0.f;
#pragma unroll
            for (int c = 0; c < (FMT == kWinQ4 ? 4 : 8); ++c) {
                if constexpr (FMT == kWinQ4) {
                    const float4 u = valid ? __ldg(reinterpret_cast<const float4*>(qr + 64 * w + 16 * t + 4 * c))
                                           : make_float4(0.f, 0.f, 0.f, 0.f);
                    v[w][4 * c] = u.x, v[w][4 * c + 1] = u.y, v[w][4 * c + 2] = u.z, v[w][4 * c + 3] = u.w;
                } else {
                    const float2 u = valid ? __ldg(reinterpret_cast<const float2*>(qr + 64 * w + 2 * t + 8 * c))
                                           : make_float2(0.f, 0.f);
                    v[w][2 * c] = u.x, v[w][2 * c + 1] = u.y;
                }
            }
#pragma unroll
            for (int c = 0; c < 16; ++c) {
                amax = fmaxf(amax, fabsf(v[w][c]));
                sum[w] += v[w][c];
            }
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int ex = max((int)(__float_as_uint(amax) >> 23), 12);
        const float up = __uint_as_float((uint32_t)(265 - ex) << 23);
        float f = __uint_as_float((uint32_t)(ex - 11) << 23) * p.scale_log2;
        if constexpr (FMT == kWinQ4) f *= 16777216.f;  // 2^24
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // column 2 t + e belongs to lane (2 (t % 2) + e, any)
            const int src = 4 * (2 * (t & 1) + e);
            sf[b][e] = __shfl_sync(0xffffffffu, f, src);
        }
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            sum[w] += __shfl_xor_sync(0xffffffffu, sum[w], 1);
            sum[w] += __shfl_xor_sync(0xffffffffu, sum[w], 2);
#pragma unroll
            for (int e = 0; e < 2; ++e)
                qsum[b][w][e] = __shfl_sync(0xffffffffu, sum[w], 4 * (2 * (t & 1) + e)) * p.scale_log2;
#pragma unroll
            for (int s4 = 0; s4 < 4; ++s4) {
                float x[4];
                if constexpr (FMT == kWinQ4) {  // nibbles (2 h, 2 h + 4), (2 h + 1, 2 h + 5) of word s4 / 2, h = s4 % 2
                    const int c = 8 * (s4 >> 1) + 2 * (s4 & 1);
                    x[0] = v[w][c] * up, x[1] = v[w][c + 4] * up;
                    x[2] = v[w][c + 1] * (up * 0.0625f), x[3] = v[w][c + 5] * (up * 0.0625f);
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c) x[c] = v[w][4 * s4 + c] * up;
                }
                uint32_t hi, lo;
                split_h2(x[0], x[1], hi, lo);
                qb[b][4 * w + s4][0] = g < 4 ? hi : lo;
                split_h2(x[2], x[3], hi, lo);
                qb[b][4 * w + s4][1] = g < 4 ? hi : lo;
            }
        }
    }

    float o[NB][MT][4];  // FMT q4: row tile 4 w + k holds channels 64 w + 8 g + 2 k (c 0, 1) and + 1 (c 2, 3)
    float zacc[NB][NW][2], m[NB][2], l[NB][2];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int i = 0; i < MT; ++i) o[b][i][0] = o[b][i][1] = o[b][i][2] = o[b][i][3] = 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            m[b][e] = -INFINITY;
            l[b][e] = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) zacc[b][w][e] = 0.f;
        }
    }
    const uint32_t lo_mask = t < 2 ? 0u : 0xffff0000u;  // lanes of the low columns keep x - high(x)

    for (int n = 0; n < mine; ++n) {
        cp_async_wait<ST - 2>();
        __syncwarp();  // every lane's copies of block n are there, and every lane is done with block n - 1
        {
            const bool in = issue(n + ST - 1);
            const uint32_t bit = 1u << ((n + ST - 1) & 31);
            present = in ? present | bit : present & ~bit;
        }
        const uint32_t ks = ring + (n % ST) * G::BYTES, vs = ks + G::CHUNK;
        if (!((present >> (n & 31)) & 1)) continue;
        const int j0 = block_no(n) * 16;

        // S^T
        float s[NB][4];
        if constexpr (FMT == kWinQ4) {
            uint32_t kg[2 * NW], kh[2 * NW];  // tokens g, g + 8: word 2 w' + ... as stored (e * NW + w)
            const int row = g * (D / 2) + t * 8 * NW;
            const int sw = D == 128 ? row ^ (((g >> 1) & 3) << 5) : row;
            lds_words(kg, ks + sw);
            lds_words(kh, ks + sw + 8 * (D / 2));
            float acc[NB][NW][4];
#pragma unroll
            for (int w = 0; w < NW; ++w) {
#pragma unroll
                for (int b = 0; b < NB; ++b) acc[b][w][0] = acc[b][w][1] = acc[b][w][2] = acc[b][w][3] = 0.f;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t x = kg[e * NW + w], y = kh[e * NW + w];
                    const uint32_t a1[4] = {x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u};
                    const uint32_t a2[4] = {(x >> 8) & 0x000f000fu, (y >> 8) & 0x000f000fu, (x >> 8) & 0x00f000f0u,
                                            (y >> 8) & 0x00f000f0u};
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        mma_16816(acc[b][w], a1, qb[b][4 * w + 2 * e][0], qb[b][4 * w + 2 * e][1]);
                        mma_16816(acc[b][w], a2, qb[b][4 * w + 2 * e + 1][0], qb[b][4 * w + 2 * e + 1][1]);
                    }
                }
            }
            float2 kp[NW][2];
#pragma unroll
            for (int w = 0; w < NW; ++w)
#pragma unroll
                for (int h = 0; h < 2; ++h) kp[w][h] = lds_half2(ks + Q4Layout<D>::PARAMS + w * 64 + (g + 8 * h) * 4);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float d = acc[b][0][i] * kp[0][i >> 1].x, z = qsum[b][0][i & 1] * kp[0][i >> 1].y;
                    if constexpr (NW == 2) {
                        d = fmaf(acc[b][1][i], kp[1][i >> 1].x, d);
                        z = fmaf(qsum[b][1][i & 1], kp[1][i >> 1].y, z);
                    }
                    d += __shfl_xor_sync(0xffffffffu, d, 2);
                    s[b][i] = fmaf(d, sf[b][i & 1], z);
                }
        } else {
            float acc[NB][2][4];  // two chains
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[b][0][i] = acc[b][1][i] = 0.f;
            const int r = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                uint32_t a[4];
                const int c = 2 * i + (lane >> 4);
                ldsm_x4(ks + (r * (D / 8) + (c ^ (r & 7))) * 16, a);
#pragma unroll
                for (int b = 0; b < NB; ++b) mma_16816(acc[b][i & 1], a, qb[b][i][0], qb[b][i][1]);
            }
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float d = acc[b][0][i] + acc[b][1][i];
                    d += __shfl_xor_sync(0xffffffffu, d, 2);
                    s[b][i] = d * sf[b][i & 1];
                }
        }

        // the mask, where the block is not visible to every row as a whole
        const bool whole = j0 + 16 <= cmin && (j0 >= cmax - window || j0 + 16 <= p.sinks);
        auto sees = [&](int b, int i) {  // row of score i: token g + 8 (i / 2), column 2 t + i % 2
            const int j = j0 + g + 8 * (i >> 1), c = ctx[b][i & 1];
            return j < c && (j >= c - window || j < p.sinks);
        };
        if (!whole) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!sees(b, i)) s[b][i] = -INFINITY;
            if constexpr (FMT == kWinF16) {
                // a key that some row does not see must not reach it through 0 * V: what is not
                // finite in such a row of V is set to zero, and the rows that do see it become NaN
                const int r = lane >> 1, j = j0 + r;
                const bool all = j < cmin && (j >= cmax - window || j < p.sinks);
                bool bad = false;
                if (!all) {
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) {
                        const uint32_t at = vs + (r * (D / 8) + (((lane & 1) * (D / 16) + c) ^ (r & 7))) * 16;
                        uint32_t u[4];
                        lds_words(u, at);
                        bool here = false;
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            if ((u[x] & 0x7c00u) == 0x7c00u) u[x] &= 0xffff0000u, here = true;
                            if ((u[x] & 0x7c000000u) == 0x7c000000u) u[x] &= 0x0000ffffu, here = true;
                        }
                        if (here)
                            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(u[0]), "r"(u[1]),
                                         "r"(u[2]), "r"(u[3])
                                         : "memory");
                        bad |= here;
                    }
                }
                const unsigned rows = __ballot_sync(0xffffffffu, bad);
                if (rows) {
                    __syncwarp();
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (((rows >> (2 * (g + 8 * (i >> 1)))) & 3) && sees(b, i))
                                l[b][i & 1] = __int_as_float(0x7fffffff);
                }
            }
        }

        // softmax in the log2 domain; the running maximum moves only when a score passes it by
        // 8, so that probabilities stay below 2^8
        bool grow = false;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) grow |= fmaxf(s[b][e], s[b][2 + e]) > m[b][e] + 8.f;
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float mn = fmaxf(m[b][e], fmaxf(s[b][e], s[b][2 + e]));
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, x));
                    const float corr = mn == -INFINITY ? 1.f : ex2_approx(m[b][e] - mn);
                    m[b][e] = mn;
                    l[b][e] *= corr;
#pragma unroll
                    for (int w = 0; w < NW; ++w) zacc[b][w][e] *= corr;
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        o[b][i][e] *= corr;
                        o[b][i][2 + e] *= corr;
                    }
                }
        }
        float pr[NB][4];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float mu = m[b][i & 1] == -INFINITY ? 0.f : m[b][i & 1];
                pr[b][i] = ex2_approx(s[b][i] - mu);
                l[b][i & 1] += pr[b][i];
            }

        // O^T += V^T P^T
        if constexpr (FMT == kWinQ4) {
            uint32_t v[4][NW];  // tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 2 * t + (i & 1) + 8 * (i >> 1), at = r * (D / 2) + g * 4 * NW;
                lds_words(v[i], vs + (D == 128 ? at ^ (t << 5) : at));
            }
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                uint32_t pb[NB][2];
                float2 vp[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) vp[h] = lds_half2(vs + Q4Layout<D>::PARAMS + w * 64 + (g + 8 * h) * 4);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    float x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float z = pr[b][i] * vp[i >> 1].y;
                        x[i] = pr[b][i] * (vp[i >> 1].x * kPScale);
                        if (!whole && !sees(b, i)) x[i] = z = 0.f;
                        zacc[b][w][i & 1] += z;
                        x[i] -= __uint_as_float(__float_as_uint(x[i]) & lo_mask);
                    }
                    // bf16 by cutting off: exact for the high half, 2^-16 of x for the low one
                    pb[b][0] = movmatrix_t(prmt(__float_as_uint(x[0]), __float_as_uint(x[1]), 0x7632));
                    pb[b][1] = movmatrix_t(prmt(__float_as_uint(x[2]), __float_as_uint(x[3]), 0x7632));
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {  // nibbles 0-3, 4-7 of two tokens side by side
                    const uint32_t x = prmt(v[0][w], v[1][w], h ? 0x7632 : 0x5410);
                    const uint32_t y = prmt(v[2][w], v[3][w], h ? 0x7632 : 0x5410);
                    const uint32_t a1[4] = {x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u};
                    const uint32_t a2[4] = {(x >> 8) & 0x000f000fu, (x >> 8) & 0x00f000f0u, (y >> 8) & 0x000f000fu,
                                            (y >> 8) & 0x00f000f0u};
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        mma_16816_bf16(o[b][4 * w + 2 * h], a1, pb[b][0], pb[b][1]);
                        mma_16816_bf16(o[b][4 * w + 2 * h + 1], a2, pb[b][0], pb[b][1]);
                    }
                }
            }
        } else {
            uint32_t pb[NB][2];
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t hi, lo;
                    split_h2(pr[b][2 * h], pr[b][2 * h + 1], hi, lo);
                    pb[b][h] = movmatrix_t(t < 2 ? hi : lo);
                }
            const int r = (lane & 7) + (lane >> 4) * 8;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                uint32_t a[4];
                const int c = 2 * i + ((lane >> 3) & 1);
                ldsm_x4_t(vs + (r * (D / 8) + (c ^ (r & 7))) * 16, a);
#pragma unroll
                for (int b = 0; b < NB; ++b) mma_16816(o[b][i], a, pb[b][0], pb[b][1]);
            }
        }
    }
    cp_async_wait<0>();
    __syncwarp();  // the ring becomes the warp's partial output

    // fold: halves and lanes, then warps of the CTA, then CTAs of the cluster
    float* part = reinterpret_cast<float*>(smem + warp * ST * G::BYTES);  // [SL][D]
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int sl = 4 * b + 2 * (t & 1) + e;
            if (ctx[b][e] == 0) l[b][e] = 0.f;  // a row without keys in a tile of rows that have some
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
                l[b][e] += __shfl_xor_sync(0xffffffffu, l[b][e], x);
#pragma unroll
                for (int w = 0; w < NW; ++w) zacc[b][w][e] += __shfl_xor_sync(0xffffffffu, zacc[b][w][e], x);
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                float lo = o[b][i][e], hi = o[b][i][2 + e];  // rows g and g + 8 of the tile
                lo += __shfl_xor_sync(0xffffffffu, lo, 2);
                hi += __shfl_xor_sync(0xffffffffu, hi, 2);
                int d0 = 16 * i + g, d1 = d0 + 8;
                if constexpr (FMT == kWinQ4) {
                    lo = fmaf(lo, kPUnscale, zacc[b][i >> 2][e]);
                    hi = fmaf(hi, kPUnscale * 0.0625f, zacc[b][i >> 2][e]);
                    d0 = 64 * (i >> 2) + 8 * g + 2 * (i & 3), d1 = d0 + 1;
                }
                if (t < 2) part[sl * D + d0] = lo, part[sl * D + d1] = hi;
            }
            if (lane < 2) s_ml[warp][sl][0] = m[b][e], s_ml[warp][sl][1] = l[b][e];
        }
    __syncthreads();
    const float* parts = reinterpret_cast<const float*>(smem);
    constexpr int kPartStride = ST * G::BYTES / 4;
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
            const float v = sum == 0.f ? 0.f : acc / sum;
            const size_t idx = ((size_t)(row0 + r / heads) * p.num_heads + kvh * p.group + h0 + r % heads) * D + d;
            const __nv_bfloat16 hi = __float2bfloat16_rn(v);
            p.out[idx] = hi;
            if (p.out_lo) p.out_lo[idx] = __float2bfloat16_rn(v - __bfloat162float(hi));
        } else {
            reinterpret_cast<float*>(smem)[e] = acc;  // only this thread reads or writes the element
            if (d == 0) s_part[r][0] = mx, s_part[r][1] = sum;
        }
    }
    if (splits == 1) return;
    cluster_sync();
    for (int e = (int)rank * W * 32 + threadIdx.x; e < slots * D; e += (int)splits * W * 32) {
        const int r = e / D, d = e % D;
        const uint32_t a_o = smem_u32(parts + e), a_m = smem_u32(&s_part[r][0]), a_l = smem_u32(&s_part[r][1]);
        float mx = -INFINITY;
        for (uint32_t c = 0; c < splits; ++c) mx = fmaxf(mx, ld_dsmem_f32(map_to_rank(a_m, c)));
        float sum = 0.f, acc = 0.f;
        for (uint32_t c = 0; c < splits; ++c) {
            const float mc = ld_dsmem_f32(map_to_rank(a_m, c)), lc = ld_dsmem_f32(map_to_rank(a_l, c));
            if (mc != -INFINITY) {
                const float f = ex2_approx(mc - mx);
                sum += lc * f;
                acc += ld_dsmem_f32(map_to_rank(a_o, c)) * f;
            } else if (lc != 0.f) {
                sum = lc;
            }
        }
        const float v = sum == 0.f ? 0.f : acc / sum;
        const size_t idx = ((size_t)(row0 + r / heads) * p.num_heads + kvh * p.group + h0 + r % heads) * D + d;
        const __nv_bfloat16 hi = __float2bfloat16_rn(v);
        p.out[idx] = hi;
        if (p.out_lo) p.out_lo[idx] = __float2bfloat16_rn(v - __bfloat162float(hi));
    }
    cluster_sync();  // no CTA leaves while another reads its shared memory
}

template <int FMT, int D, int NB>
inline int launch_window_rows(WinParams p, cudaStream_t st) {
    constexpr int W = 4, ST = FMT == kWinQ4 ? 4 : 2, SL = 4 * NB;
    constexpr int smem = W * ST * WinStage<FMT, D>::BYTES;
    p.head_tiles = ceil_div(p.group, SL);
    p.qt = p.group >= SL ? 1 : SL / p.group;
    if (p.qt > p.S) p.qt = p.S;
    p.tiles = ceil_div(p.S, p.qt);
    const long long tiles = (long long)(p.R / p.S) * p.tiles * p.kv_heads * p.head_tiles;
    // keys one tile walks, at most
    const int limit = p.max_ctx < p.mbps * 16 ? p.max_ctx : p.mbps * 16;
    long long keys = limit;
    if (p.window > 0 && (long long)p.window + p.sinks + p.qt + 32 < keys) keys = (long long)p.window + p.sinks + p.qt + 32;
    const int blocks = (int)((keys + 15) / 16);
    int splits = 1;
    while (splits < 16 && tiles * splits * 2 <= 4 * num_sms() && blocks >= 2 * W * splits * 2) splits *= 2;
    QTTS_REQUIRE(tiles * splits < (1ll << 31), "paged attention: %lld tiles", tiles);
    constexpr auto kernel = paged_attn_window_kernel<FMT, D, NB, W, ST>;
    QTTS_CHECK_CUDA((func_attr_once<kernel>(smem, true)));
    QTTS_CHECK_CUDA(launch_pdl(kernel, dim3((unsigned)(tiles * splits)), dim3(W * 32), smem, st, dim3(splits, 1, 1), p));
    return QTTS_OK;
}

template <int FMT, int D>
inline int launch_window_attention(const WinParams& p, cudaStream_t st) {
    // eight slots a tile where they can be filled: a block is then read once for twice the rows
    if (p.group > 4 || (p.S > 1 && p.S * p.group > 4)) return launch_window_rows<FMT, D, 2>(p, st);
    return launch_window_rows<FMT, D, 1>(p, st);
}

}  // namespace qtts
