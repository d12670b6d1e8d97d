// Paged GQA attention with a sliding window and sinks, over the fp16 pool or the 4-bit one.
//
// A query row of context c (its keys are 0 .. c - 1) sees key j when
//     j < c  and  (j >= c - window  or  j < sinks  or  window == 0),
// and gets softmax(q k^T / sqrt(D)) v over those keys; a row that sees none gets zeros.
//
// One warp walks 16-token blocks.  The tensor work is mma.sync m16n8k16 with the queries on the M
// side: the 16 rows are 8 (query, head) slots twice, the high halves of the operand in rows 0-7 and
// what rounding took from them in rows 8-15, so that q and the probabilities keep 16 bits or more at
// no extra instructions, and the accumulator's two row halves of a lane add up to the exact sum.
//     S[16][8 tokens]  += Q[16][16 channels] . K^T      2 x D/16 instructions a block
//     O[16][8 channels] += P[16][16 tokens] . V         D/8 instructions a block
// S's accumulator layout is P's operand layout, so nothing moves between lanes but the rare
// update of the running maximum.  K and V go from global memory to registers in operand order; the
// channel and token orders of the two contractions are permuted to make each lane's share
// contiguous: lane (g, t) holds of K token 4 (g / 2) + 2 j + g % 2 (j = 0, 1) 16 channels of each
// 64 (4 bits: 16 t .. + 15; fp16: 8 t .. + 7 and 32 + 8 t .. + 7, whole 32-byte sectors a load), and
// of V tokens 4 t .. 4 t + 3 the channels 64 w + 8 g .. + 7.
//
// 4-bit pool: a nibble masked out of a code word IS a small fp16 or bf16 number (a subnormal:
// nibble << 0 = code * 2^-24 or 2^-133, nibble << 4 = 16 times that), so that no conversion is
// needed; the powers of two move into q and the output, a token's scale into the score (K) and the
// probability (V), and its zero multiplies sum(q) and p on the fp32 side.
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
    int head_tiles;         // ceil(group / 8)
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

// N 32-bit words at a 4 N-byte aligned address
template <int N>
__device__ __forceinline__ void ld_words(uint32_t* w, const uint8_t* src) {
    if constexpr (N == 4) {
        const uint4 u = *reinterpret_cast<const uint4*>(src);
        w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    } else if constexpr (N == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(src);
        w[0] = u.x, w[1] = u.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(src);
    }
}

template <int FMT, int D>
struct WinLayout {
    static constexpr int NW = D / 64;
    static constexpr int CHUNK = FMT == kWinQ4 ? Q4Layout<D>::CHUNK : 16 * D * 2;  // bytes of one (block, layer, k|v, head)
    static constexpr int KW = FMT == kWinQ4 ? 2 * NW : 8 * NW;  // K words per lane and token
    static constexpr int VW = FMT == kWinQ4 ? NW : 4 * NW;      // V words per lane and token
    static constexpr int PW = FMT == kWinQ4 ? 4 * NW : 1;       // (scale, zero) words per lane: 4 tokens a group
};

// One block's share of a lane.
template <int FMT, int D>
struct KFrag {
    using L = WinLayout<FMT, D>;
    uint32_t w[2][L::KW];
    uint32_t prm[L::PW];
    __device__ __forceinline__ void load(const uint8_t* chunk, int g, int t) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int tok = 4 * (g >> 1) + 2 * j + (g & 1);
            if constexpr (FMT == kWinQ4) {
                ld_words<2 * L::NW>(w[j], chunk + tok * (D / 2) + t * 8 * L::NW);
            } else {
#pragma unroll
                for (int c = 0; c < 2 * L::NW; ++c)
                    ld_words<4>(w[j] + 4 * c, chunk + tok * D * 2 + c * 64 + t * 16);
            }
        }
        if constexpr (FMT == kWinQ4) {
#pragma unroll
            for (int x = 0; x < L::NW; ++x) ld_words<4>(prm + 4 * x, chunk + Q4Layout<D>::PARAMS + x * 64 + t * 16);
        }
    }
};

template <int FMT, int D>
struct VFrag {
    using L = WinLayout<FMT, D>;
    uint32_t w[4][L::VW];
    uint32_t prm[L::PW];
    __device__ __forceinline__ void load(const uint8_t* chunk, int g, int t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (FMT == kWinQ4) {
                ld_words<L::NW>(w[i], chunk + (4 * t + i) * (D / 2) + g * 4 * L::NW);
            } else {
#pragma unroll
                for (int x = 0; x < L::NW; ++x) ld_words<4>(w[i] + 4 * x, chunk + (4 * t + i) * D * 2 + x * 128 + g * 16);
            }
        }
        if constexpr (FMT == kWinQ4) {
#pragma unroll
            for (int x = 0; x < L::NW; ++x) ld_words<4>(prm + 4 * x, chunk + Q4Layout<D>::PARAMS + x * 64 + t * 16);
        }
    }
};

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }
__device__ __forceinline__ float2 unpack_h2(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
__device__ __forceinline__ uint32_t pack_bf2(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Two values as high and low bf16 halves: hi cuts x off (the rest is exact in fp32), lo = bf16(x - hi): 16 bits
__device__ __forceinline__ void split_bf16(float a, float b, uint32_t& hi, uint32_t& lo) {
    const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
    hi = prmt(ua, ub, 0x7632);
    lo = pack_bf2(a - __uint_as_float(ua & 0xffff0000u), b - __uint_as_float(ub & 0xffff0000u));
}

// The 4-bit pool's probabilities carry 2^100 into the bf16 product, whose other factor is code * 2^-133:
// a probability is at most 2^8 and a scale below 2^14, so 2^122 at most, and the products are
// normal numbers down to probabilities of 2^-90.
constexpr float kPScale = 1.2676506002282294e30f;  // 2^100

template <int FMT, int D, int W>
__global__ void __launch_bounds__(W * 32) paged_attn_window_kernel(const WinParams p) {
    using L = WinLayout<FMT, D>;
    constexpr int NW = L::NW, NT = D / 8;
    __shared__ float s_o[W][8][D];
    __shared__ float s_ml[W][8][2];
    __shared__ float s_part[8][2];  // the CTA's (max, sum) per slot

    griddep_wait();
    griddep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    uint32_t splits;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(splits));
    const uint32_t rank = cluster_ctarank();

    // the tile: up to 8 (query, head) slots of one stream and KV head
    const int tile = blockIdx.x / splits;
    const int head_tile = tile % (p.kv_heads * p.head_tiles), row_tile = tile / (p.kv_heads * p.head_tiles);
    const int kvh = head_tile / p.head_tiles, h8 = (head_tile % p.head_tiles) * 8;
    const int heads = min(8, p.group - h8);
    const int stream = row_tile / p.tiles, q0 = (row_tile % p.tiles) * p.qt;
    const int nq = min(p.qt, p.S - q0);
    const int row0 = stream * p.S + q0;
    const int slots = nq * heads;

    // contexts: this lane's slot, and the tile's extremes over rows that see anything
    const int limit = min(p.max_ctx, p.mbps * 16);
    const int window = p.window > 0 ? p.window : 0x7fffffff;
    const int slot = __ldg(p.row_slot + row0);
    const bool slot_ok = slot >= 0 && slot < p.num_slots;
    int my_ctx = 0;
    if (g < slots && slot_ok) my_ctx = min(max(__ldg(p.row_ctx + row0 + g / heads), 0), limit);
    int cmax = my_ctx, cmin = my_ctx > 0 ? my_ctx : 0x7fffffff;
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
        cmax = max(cmax, __shfl_xor_sync(0xffffffffu, cmax, o));
        cmin = min(cmin, __shfl_xor_sync(0xffffffffu, cmin, o));
    }
    if (!slot_ok && threadIdx.x == 0) record_error(DEV_ERR_ATTN_BOUNDS);
    // blocks that hold a visible key: the sinks', then from the earliest window's start
    const int nb_end = (cmax + 15) >> 4;
    const int nb_sink = min((min(p.sinks, cmax) + 15) >> 4, nb_end);
    const int first = max(nb_sink, cmax > 0 ? max(0, cmin - window) >> 4 : 0);
    const int nb = nb_sink + max(0, nb_end - first);
    const int stride = (int)splits * W;
    const int i0 = (int)rank * W + warp;

    // Q operand.  Each slot's q is scaled by a power of two that brings its largest channel to
    // [2^11, 2^12), so that fp16 halves hold it whatever its size; odd nibble positions take 1/16.
    uint32_t qa[NW][4][4];
    float qsum[NW];   // sum of a group's channels, for the 4-bit zeros (log2 units)
    float sf;         // accumulator -> log2 units
    {
        float v[NW][16];
        float amax = 0.f;
        const bool valid = g < slots;
        const float* qr = p.q + ((size_t)(row0 + (valid ? g / heads : 0)) * p.num_heads + kvh * p.group + h8 +
                                 (valid ? g % heads : 0)) * D;
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
                const int ch = FMT == kWinQ4 ? 16 * t + 4 * c : 32 * (c >> 1) + 8 * t + 4 * (c & 1);
                if (valid) u = __ldg(reinterpret_cast<const float4*>(qr + 64 * w + ch));
                v[w][4 * c] = u.x, v[w][4 * c + 1] = u.y, v[w][4 * c + 2] = u.z, v[w][4 * c + 3] = u.w;
                amax = fmaxf(amax, fmaxf(fmaxf(fabsf(u.x), fabsf(u.y)), fmaxf(fabsf(u.z), fabsf(u.w))));
            }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int ex = max((int)(__float_as_uint(amax) >> 23), 12);
        const float up = __uint_as_float((uint32_t)(265 - ex) << 23), down = __uint_as_float((uint32_t)(ex - 11) << 23);
        sf = down * p.scale_log2;
        if constexpr (FMT == kWinQ4) sf *= 16777216.f;  // 2^24
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            float s = 0.f;
#pragma unroll
            for (int c = 0; c < 16; ++c) s += v[w][c];
            s += __shfl_xor_sync(0xffffffffu, s, 1);
            s += __shfl_xor_sync(0xffffffffu, s, 2);
            qsum[w] = s * p.scale_log2;
#pragma unroll
            for (int c = 0; c < 16; ++c) v[w][c] *= up;
#pragma unroll
            for (int s4 = 0; s4 < 4; ++s4) {  // channel quadruple of K words: see the loop below
                if constexpr (FMT == kWinQ4) {
                    const int b = 8 * (s4 >> 1) + 2 * (s4 & 1);  // nibbles (2h, 2h + 4) and (2h + 1, 2h + 5)
                    split_h2(v[w][b], v[w][b + 4], qa[w][s4][0], qa[w][s4][1]);
                    split_h2(v[w][b + 1] * 0.0625f, v[w][b + 5] * 0.0625f, qa[w][s4][2], qa[w][s4][3]);
                } else {
                    split_h2(v[w][4 * s4], v[w][4 * s4 + 1], qa[w][s4][0], qa[w][s4][1]);
                    split_h2(v[w][4 * s4 + 2], v[w][4 * s4 + 3], qa[w][s4][2], qa[w][s4][3]);
                }
            }
        }
    }

    float o[NT][4];
    float zacc[NW];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) zacc[w] = 0.f;

    // block numbers and ids of the warp's next 32 blocks, one per lane
    const int32_t* table = p.block_table + (size_t)(slot_ok ? slot : 0) * p.mbps;
    const size_t head_stride = (size_t)L::CHUNK;
    const size_t block_stride = (size_t)p.num_layers * 2 * p.kv_heads * head_stride;
    const uint8_t* base = p.kv + ((size_t)p.layer * 2 * p.kv_heads + kvh) * head_stride;
    const size_t v_off = (size_t)p.kv_heads * head_stride;
    int ids = -1;
    auto block_no = [&](int i) { return i < nb_sink ? i : first + (i - nb_sink); };
    auto load_ids = [&](int n) {  // ids of the warp's blocks n .. n + 31
        const int i = i0 + (n + lane) * stride;
        ids = -1;
        if (i < nb) {
            const int b = __ldg(table + block_no(i));
            if (b >= 0 && b < p.num_blocks) ids = b;
            else record_error(DEV_ERR_ATTN_BOUNDS);
        }
    };
    const int mine = i0 < nb ? (nb - i0 + stride - 1) / stride : 0;

    KFrag<FMT, D> kf;
    VFrag<FMT, D> vf;
    int id = -1;
    if (mine > 0) {
        load_ids(0);
        id = __shfl_sync(0xffffffffu, ids, 0);
        const uint8_t* c = base + (size_t)max(id, 0) * block_stride;
        kf.load(c, g, t);
        vf.load(c + v_off, g, t);
    }
    for (int n = 0; n < mine; ++n) {
        const int blk = block_no(i0 + n * stride);
        const bool present = id >= 0;  // an id outside the pool hides its keys
        // the next block's id and address
        int id_next = -1;
        if (n + 1 < mine) {
            if (((n + 1) & 31) == 0) load_ids(n + 1);
            id_next = __shfl_sync(0xffffffffu, ids, (n + 1) & 31);
        }
        const uint8_t* c_next = base + (size_t)max(id_next, 0) * block_stride;

        // S
        float s[2][2];
        if constexpr (FMT == kWinQ4) {
            float acc[2][NW][4];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    float (&a)[4] = acc[j][w];
                    a[0] = a[1] = a[2] = a[3] = 0.f;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t x = kf.w[j][e * NW + w], y = x >> 8;
                        mma_16816(a, qa[w][2 * e], x & 0x000f000fu, x & 0x00f000f0u);
                        mma_16816(a, qa[w][2 * e + 1], y & 0x000f000fu, y & 0x00f000f0u);
                    }
                }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float d = 0.f, z = 0.f;
#pragma unroll
                    for (int w = 0; w < NW; ++w) {
                        const float2 sz = unpack_h2(kf.prm[4 * w + 2 * j + e]);
                        d = fmaf(acc[j][w][e] + acc[j][w][2 + e], sz.x, d);
                        z = fmaf(qsum[w], sz.y, z);
                    }
                    s[j][e] = fmaf(d, sf, z);
                }
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < NW; ++w)
#pragma unroll
                    for (int s4 = 0; s4 < 4; ++s4)
                        mma_16816(a, qa[w][s4], kf.w[j][8 * w + 2 * s4], kf.w[j][8 * w + 2 * s4 + 1]);
                s[j][0] = (a[0] + a[2]) * sf;
                s[j][1] = (a[1] + a[3]) * sf;
            }
        }
        if (n + 1 < mine) kf.load(c_next, g, t);

        // the mask, where the block is not visible to every row as a whole
        const int j0 = blk * 16;
        const bool whole = present && j0 + 16 <= cmin && (j0 >= cmax - window || j0 + 16 <= p.sinks);
        bool seen[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = j0 + 4 * t + i;
            seen[i] = whole || (present && j < my_ctx && (j >= my_ctx - window || j < p.sinks));
        }
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!seen[i]) s[i >> 1][i & 1] = -INFINITY;
            if constexpr (FMT == kWinF16) {
                // a key that some row does not see must not reach it through 0 * V: what is not
                // finite is taken out of V, and the rows that do see it become NaN
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = j0 + 4 * t + i;
                    const bool all = present && j < cmin && (j >= cmax - window || j < p.sinks);
                    bool bad = false;
                    if (!all) {
#pragma unroll
                        for (int x = 0; x < L::VW; ++x) {
                            uint32_t u = vf.w[i][x];
                            if ((u & 0x7c00u) == 0x7c00u) u &= 0xffff0000u, bad = true;
                            if ((u & 0x7c000000u) == 0x7c000000u) u &= 0x0000ffffu, bad = true;
                            vf.w[i][x] = u;
                        }
                    }
                    const unsigned b = __ballot_sync(0xffffffffu, bad) & (0x11111111u << t);
                    if (b && seen[i]) l = __int_as_float(0x7fffffff);
                }
            }
        }

        // softmax in the log2 domain; the running maximum moves only when a score passes it by
        // 8, so that probabilities stay below 2^8
        const float top = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
        if (__any_sync(0xffffffffu, top > m + 8.f)) {
            float mn = fmaxf(m, top);
            mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 1));
            mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 2));
            const float corr = mn == -INFINITY ? 1.f : ex2_approx(m - mn);
            m = mn;
            l *= corr;
#pragma unroll
            for (int w = 0; w < NW; ++w) zacc[w] *= corr;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                o[i][0] *= corr;
                o[i][1] *= corr;
                o[i][2] *= corr;
                o[i][3] *= corr;
            }
        }
        const float mu = m == -INFINITY ? 0.f : m;
        float pr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            pr[i] = ex2_approx(s[i >> 1][i & 1] - mu);
            l += pr[i];
        }

        // O += P V
        if constexpr (FMT == kWinQ4) {
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                float ps[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float2 sz = unpack_h2(vf.prm[4 * w + i]);
                    if (!whole && !seen[i]) sz = make_float2(0.f, 0.f);
                    ps[i] = pr[i] * (sz.x * kPScale);
                    zacc[w] = fmaf(pr[i], sz.y, zacc[w]);
                }
                uint32_t a[4];
                split_bf16(ps[0], ps[1], a[0], a[1]);
                split_bf16(ps[2], ps[3], a[2], a[3]);
                const uint32_t x0 = prmt(vf.w[0][w], vf.w[1][w], 0x5410), x1 = prmt(vf.w[2][w], vf.w[3][w], 0x5410);
                const uint32_t y0 = prmt(vf.w[0][w], vf.w[1][w], 0x7632), y1 = prmt(vf.w[2][w], vf.w[3][w], 0x7632);
                mma_16816_bf16(o[8 * w + 0], a, x0 & 0x000f000fu, x1 & 0x000f000fu);
                mma_16816_bf16(o[8 * w + 1], a, x0 & 0x00f000f0u, x1 & 0x00f000f0u);
                mma_16816_bf16(o[8 * w + 2], a, (x0 >> 8) & 0x000f000fu, (x1 >> 8) & 0x000f000fu);
                mma_16816_bf16(o[8 * w + 3], a, (x0 >> 8) & 0x00f000f0u, (x1 >> 8) & 0x00f000f0u);
                mma_16816_bf16(o[8 * w + 4], a, y0 & 0x000f000fu, y1 & 0x000f000fu);
                mma_16816_bf16(o[8 * w + 5], a, y0 & 0x00f000f0u, y1 & 0x00f000f0u);
                mma_16816_bf16(o[8 * w + 6], a, (y0 >> 8) & 0x000f000fu, (y1 >> 8) & 0x000f000fu);
                mma_16816_bf16(o[8 * w + 7], a, (y0 >> 8) & 0x00f000f0u, (y1 >> 8) & 0x00f000f0u);
            }
        } else {
            uint32_t a[4];
            split_h2(pr[0], pr[1], a[0], a[1]);
            split_h2(pr[2], pr[3], a[2], a[3]);
#pragma unroll
            for (int x = 0; x < 4 * NW; ++x) {
                mma_16816(o[2 * x], a, prmt(vf.w[0][x], vf.w[1][x], 0x5410), prmt(vf.w[2][x], vf.w[3][x], 0x5410));
                mma_16816(o[2 * x + 1], a, prmt(vf.w[0][x], vf.w[1][x], 0x7632), prmt(vf.w[2][x], vf.w[3][x], 0x7632));
            }
        }
        if (n + 1 < mine) vf.load(c_next + v_off, g, t);
        id = id_next;
    }

    // fold: warps of the CTA, then CTAs of the cluster
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (my_ctx == 0) l = 0.f;  // a row without keys in a tile of rows that have some
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        zacc[w] += __shfl_xor_sync(0xffffffffu, zacc[w], 1);
        zacc[w] += __shfl_xor_sync(0xffffffffu, zacc[w], 2);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float a = o[8 * w + i][0] + o[8 * w + i][2], b = o[8 * w + i][1] + o[8 * w + i][3];
            if constexpr (FMT == kWinQ4) {
                const float f = (i & 1) ? 0.0625f * 8589934592.f : 8589934592.f;  // 2^133 / 2^100
                a = fmaf(a, f, zacc[w]);
                b = fmaf(b, f, zacc[w]);
            }
            if (g < slots) {
                s_o[warp][g][64 * w + 16 * t + i] = a;
                s_o[warp][g][64 * w + 16 * t + 8 + i] = b;
            }
        }
    }
    if (g < slots && t == 0) {
        s_ml[warp][g][0] = m;
        s_ml[warp][g][1] = l;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < slots * D; e += W * 32) {
        const int r = e / D, d = e % D;
        float mx = s_ml[0][r][0];
#pragma unroll
        for (int w = 1; w < W; ++w) mx = fmaxf(mx, s_ml[w][r][0]);
        float sum = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float mw = s_ml[w][r][0];
            const float f = mw == -INFINITY ? 0.f : ex2_approx(mw - mx);
            if (mw != -INFINITY) {  // a warp without keys holds nothing
                sum += s_ml[w][r][1] * f;
                acc += s_o[w][r][d] * f;
            } else if (s_ml[w][r][1] != 0.f) {
                sum = s_ml[w][r][1];
            }
        }
        if (splits == 1) {
            const float v = sum == 0.f ? 0.f : acc / sum;
            const size_t idx = ((size_t)(row0 + r / heads) * p.num_heads + kvh * p.group + h8 + r % heads) * D + d;
            const __nv_bfloat16 hi = __float2bfloat16_rn(v);
            p.out[idx] = hi;
            if (p.out_lo) p.out_lo[idx] = __float2bfloat16_rn(v - __bfloat162float(hi));
        } else {
            s_o[0][r][d] = acc;  // this thread is the only one that reads or writes the element
            if (d == 0) s_part[r][0] = mx, s_part[r][1] = sum;
        }
    }
    if (splits == 1) return;
    cluster_sync();
    for (int e = (int)rank * W * 32 + threadIdx.x; e < slots * D; e += (int)splits * W * 32) {
        const int r = e / D, d = e % D;
        const uint32_t a_o = smem_u32(&s_o[0][r][d]), a_m = smem_u32(&s_part[r][0]), a_l = smem_u32(&s_part[r][1]);
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
        const size_t idx = ((size_t)(row0 + r / heads) * p.num_heads + kvh * p.group + h8 + r % heads) * D + d;
        const __nv_bfloat16 hi = __float2bfloat16_rn(v);
        p.out[idx] = hi;
        if (p.out_lo) p.out_lo[idx] = __float2bfloat16_rn(v - __bfloat162float(hi));
    }
    cluster_sync();  // no CTA leaves while another reads its shared memory
}

template <int FMT, int D>
inline int launch_window_attention(WinParams p, cudaStream_t st) {
    constexpr int W = 4;
    p.head_tiles = ceil_div(p.group, 8);
    p.qt = p.group >= 8 ? 1 : 8 / p.group;
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
    auto kernel = paged_attn_window_kernel<FMT, D, W>;
    QTTS_CHECK_CUDA((func_attr_once<paged_attn_window_kernel<FMT, D, W>>(0, true)));
    QTTS_CHECK_CUDA(launch_pdl(kernel, dim3((unsigned)(tiles * splits)), dim3(W * 32), 0, st, dim3(splits, 1, 1), p));
    return QTTS_OK;
}

}  // namespace qtts
