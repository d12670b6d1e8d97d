// Prompt chunks under a window with sinks, over the fp16 pool or the 4-bit one, on the tcgen05 pipe.
//
// One CTA takes 128 rows (row = query * group + head: the query heads of one KV head for consecutive
// queries of a stream) through tiles of four 16-token blocks, only those that hold a key some row sees:
//     S[128][64]  = Q K^T      TMEM, two buffers
//     P           = 2^(S - m)  TMEM, two buffers: one thread per row writes it as fp16 pairs, high and low halves
//     O[128][D]  += P V        TMEM
// Warps 0-3 are the softmax, warps 4-7 bring K and 8-11 V (one block a warp: cp.async for fp16; 4 bits
// are turned into fp16 pairs on the way through registers), warp 12 issues the products, S one tile ahead of P
// V.  K and V tiles are panels of 64 channels, 128-byte rows with the 128-byte swizzle; V is read in place as an
// MN-major operand.
//
// q enters as fp16 after a scaling by a power of two that brings the row's largest channel to
// [2^11, 2^12), and P relative to 2^-7 of the running maximum, both as pairs of a high half and what it leaves: 22
// bits, as the row kernel has, so that the form a call goes through is not seen in its output's low half.
// (Single halves, 2^-11 of q, move a score by up to 2^-11 sum |q k| / sqrt(D): with loud channels more than
// the bf16 output rounds off.)  4-bit values are pairs too, to 2^-18 of their group's largest.  Products of two
// low parts are left out.  Sums, maxima and O are fp32.
//
// Bound by, a tile of D = 128: fp16 by 128 x 64 exponentials (512 cycles at 16 a cycle and SM) and what the
// softmax does around them, next to some 1600 cycles of products (57 an instruction of N = 64 for S, 88 of
// N = 128 for P V), and by the copies of K and V; 4 bits by the products, three for two (2400 cycles; without the
// third 19.0 us for 20.7), and K and V made fp16 beside them.  A launch adds some 8 us before its first
// products and after its last.  16 heads over 8, D = 128, B200: 8 x 128 rows after 384, 4 bits 20.7 us (182
// TFLOP/s; 16.7 in single halves), fp16 25.1 (K and V from HBM); 2 x 500 rows under a window of 256, fp16 21.1 us
// (102 TFLOP/s; 19.6).  4 bits with the scales on P and on S instead, codes alone in the products: 38.8.
// Every wait is bounded.
#pragma once

#include "attn_window.cuh"

namespace qtts {

constexpr int kChunkThreads = 416;  // 4 softmax warps, 4 for K, 4 for V, 1 issuing warp

// 32 lanes x 32 bits, 64 consecutive columns, both loads under way before the wait
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float (&v)[64]) {
    uint32_t r[64];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t* q = r + 32 * h;
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
            "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
            : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]), "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7]),
              "=r"(q[8]), "=r"(q[9]), "=r"(q[10]), "=r"(q[11]), "=r"(q[12]), "=r"(q[13]), "=r"(q[14]), "=r"(q[15]),
              "=r"(q[16]), "=r"(q[17]), "=r"(q[18]), "=r"(q[19]), "=r"(q[20]), "=r"(q[21]), "=r"(q[22]), "=r"(q[23]),
              "=r"(q[24]), "=r"(q[25]), "=r"(q[26]), "=r"(q[27]), "=r"(q[28]), "=r"(q[29]), "=r"(q[30]), "=r"(q[31])
            : "r"(taddr + 32 * h));
    }
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}

// 32 lanes x 32 bits, 16 consecutive columns; tmem_st_wait() after the last of several
__device__ __forceinline__ void tmem_st16_now(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
        "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

template <int FMT, int D>
struct ChunkLayout {
    static constexpr int NW = D / 64;
    static constexpr int NP = FMT == kWinQ4 ? 2 : 1;  // fp16 numbers a value of K or V is held in
    static constexpr int ST = FMT == kWinQ4 ? 2 : 4;  // stages of fp16 tiles
    static constexpr int RAW = FMT == kWinQ4 ? 3 : 0; // tiles of codes on their way (cp.async), not yet turned into fp16
    static constexpr int PANEL = 64 * 128;            // 64 keys x 64 channels
    static constexpr int PART_KV = NW * PANEL;        // high or low parts of K or V
    static constexpr int STAGE = 2 * NP * PART_KV;    // K's parts, V's parts
    static constexpr int QHALF = NW * 128 * 128;      // NW panels of 128 rows
    static constexpr int Q = 0;                       // high halves, low halves
    static constexpr int RING = Q + 2 * QHALF;
    static constexpr int CODES = RING + ST * STAGE;   // [K, V][warp][RAW] chunks
    static constexpr int SMEM = CODES + 4 * RAW * 2 * WinChunk<FMT, D>::BYTES + 1024;
    static constexpr int PART = D + 4;                // floats per row of a partial output (no bank met twice)
    static constexpr int ROWB = 2 * D + 16;           // bytes per row of a bf16 output
    static_assert(128 * PART * 4 <= ST * STAGE && 2 * 128 * ROWB <= ST * STAGE, "outputs replace the ring");
    // TMEM columns: S (two buffers of 64), O, P (two buffers of 32 for the high halves of 64 keys, 32 for the low)
    static constexpr uint32_t TS = 0, TO = 128, TP = 256, TCOLS = 512;
    static_assert(SMEM + 4096 <= 227 * 1024, "tile exceeds shared memory");
};

template <int FMT, int D>
__global__ void __launch_bounds__(kChunkThreads, 1) paged_attn_chunk_kernel(const WinParams p) {
    using L = ChunkLayout<FMT, D>;
    using G = WinChunk<FMT, D>;
    constexpr int NW = L::NW, ST = L::ST;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t k_full[ST], v_full[ST], empty[ST], s_full[2], p_full[2], pv_done[2], q_full;
    __shared__ uint32_t s_tmem;
    __shared__ int s_lim[4][2];                                 // contexts' extremes per softmax warp
    __shared__ __align__(16) uint8_t s_bad[ST][128];            // per key and half: V had a value that is not finite
    __shared__ __align__(4) uint8_t s_here[ST][4];              // per block: it is there and in the pool
    __shared__ __align__(4) uint8_t s_some_bad[ST][4];          // per block: some key is bad
    __shared__ float s_part[128][2];                            // (max, sum) per row
    __shared__ float s_sf[128];                                 // accumulator -> log2 units, per row

    griddep_wait();
    griddep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t splits;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(splits));
    const uint32_t rank = cluster_ctarank();

    const int tile = blockIdx.x / splits;
    const int kvh = tile % p.kv_heads, row_tile = tile / p.kv_heads;
    const int stream = row_tile / p.tiles, q0 = (row_tile % p.tiles) * p.qt;
    const int nq = min(p.qt, p.S - q0), rows = nq * p.group;
    const int row0 = stream * p.S + q0;
    const size_t head0 = (size_t)row0 * p.num_heads + kvh * p.group;  // q and out row (head) of tile row 0
    auto head_row = [&](int row) { return head0 + (uint32_t)(p.by_group.div(row) * (p.num_heads - p.group) + row); };
    // Q, on its way while the contexts are read: warps 0-11 take every twelfth row (D = 64: pair of rows),
    // four channels a lane
    constexpr int RPI = 128 / D, LPR = 32 / RPI;  // rows per step, lanes per row
    auto q_row = [&](int k) { return (warp + 12 * k) * RPI + lane / LPR; };
    float4 q_now[6], q_next[6];
#pragma unroll
    for (int k = 0; k < 12; ++k) {
        float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
        if (warp < 12 && q_row(k) < rows) u = __ldcg(reinterpret_cast<const float4*>(p.q + head_row(q_row(k)) * D) + lane % LPR);
        if (k < 6) q_now[k] = u;
        else q_next[k - 6] = u;
    }
    const int limit = min(p.max_ctx, p.mbps * 16);
    const int window = p.window > 0 ? p.window : 0x7fffffff;
    const int slot = __ldcg(p.row_slot + row0);
    const bool slot_ok = slot >= 0 && slot < p.num_slots;
    if (!slot_ok && threadIdx.x == 0) record_error(DEV_ERR_ATTN_BOUNDS);

    const int r = threadIdx.x;  // softmax threads: the row
    int ctx = 0;
    if (warp < 4) {
        if (r < rows && slot_ok) ctx = min(max(__ldcg(p.row_ctx + row0 + p.by_group.div(r)), 0), limit);
        int hi = ctx, lo = ctx > 0 ? ctx : 0x7fffffff;
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) {
            hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, x));
            lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, x));
        }
        if (lane == 0) s_lim[warp][0] = hi, s_lim[warp][1] = lo;
    }
    if (warp == 12) {
        if (lane == 0) {
            for (int i = 0; i < ST; ++i) {
                mbar_init(&k_full[i], 128);
                mbar_init(&v_full[i], 128);
                mbar_init(&empty[i], 1);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(&s_full[i], 1);
                mbar_init(&p_full[i], 128);
                mbar_init(&pv_done[i], 1);
            }
            mbar_init(&q_full, 384);
            fence_mbar_init();
        }
        __syncwarp();
        tmem_alloc(&s_tmem, L::TCOLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    int cmax = 0, cmin = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < 4; ++i) cmax = max(cmax, s_lim[i][0]), cmin = min(cmin, s_lim[i][1]);
    const int nb_end = (cmax + 15) >> 4;
    const int nb_sink = min((min(p.sinks, cmax) + 15) >> 4, nb_end);
    const int first = max(nb_sink, cmax > 0 ? max(0, cmin - window) >> 4 : 0);
    const int past_sinks = first - nb_sink;
    const int nb = nb_sink + max(0, nb_end - first);
    const int all_tiles = (nb + 3) >> 2;
    const int even = all_tiles / (int)splits, rest = all_tiles % (int)splits;
    const int t0 = (int)rank * even + min((int)rank, rest), nt = even + ((int)rank < rest);  // this CTA's tiles
    auto first_key = [&](int pos) { return (pos < nb_sink ? pos : pos + past_sinks) * 16; };
    auto is_whole = [&](int j0) { return j0 + 16 <= cmin && (j0 >= cmax - window || j0 + 16 <= p.sinks); };

    // tiles [whole0, whole1) of all hold only blocks that every row sees whole (if they are in the pool)
    const int below_all = cmin >> 4;  // blocks that end at or before every row's context
    int whole0 = 0, whole1 = min(nb, below_all >= first ? nb_sink + below_all - first : min(nb_sink, below_all)) >> 2;
    if (cmax > window) {  // blocks from the latest window's start on, or all within the sinks
        const int from = nb_sink + max(0, ((cmax - window + 15) >> 4) - first);
        whole0 = (from + 3) >> 2;
        if (from <= nb_sink && (nb_sink == 0 || nb_sink * 16 <= p.sinks)) whole0 = 0;
    }

    bool ok = true;  // a wait that ran out ends the thread's loop
    // ---------------------------------------------------------------------- loading warps: where they are
    const int is_v = (warp - 4) >> 2, w4 = warp & 3, pt = threadIdx.x & 127, key = pt >> 1, half = pt & 1, off = key & 15;
    uint64_t* full = is_v ? v_full : k_full;
    const int32_t* table = p.block_table + (size_t)(slot_ok ? slot : 0) * p.mbps;
    const uint8_t* base = p.kv + ((size_t)p.layer * 2 * p.kv_heads + kvh) * G::BYTES + (is_v ? p.v_offset : 0);
    int ids = -1;
    auto block_id = [&](int i) {  // of this warp's block of tile i; -1: none, or outside the pool
        if ((i & 31) == 0) {      // 32 tiles' ids, one per lane
            const int pos = (t0 + i + lane) * 4 + w4;
            ids = -1;
            if (i + lane < nt && pos < nb) {
                ids = __ldcg(table + (first_key(pos) >> 4));
                if (ids < 0 || ids >= p.num_blocks) {
                    record_error(DEV_ERR_ATTN_BOUNDS);
                    ids = -1;
                }
            }
        }
        return __shfl_sync(0xffffffffu, ids, i & 31);
    };
    uint32_t valid = 0;  // bit i % 32: tile i's block is there
    // V of a key that some row does not see: what is not finite is set to zero and noted
    auto hidden = [&](int i, bool in) {
        const int j0 = first_key((t0 + i) * 4 + w4), j = j0 + off;
        return !(in && (is_whole(j0) || (j < cmin && (j >= cmax - window || j < p.sinks))));
    };
    auto clean = [&](uint4& u) {
        uint32_t* o = &u.x;
        bool bad = false;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            if ((o[x] & 0x7c00u) == 0x7c00u) o[x] &= 0xffff0000u, bad = true;
            if ((o[x] & 0x7c000000u) == 0x7c000000u) o[x] &= 0x0000ffffu, bad = true;
        }
        return bad;
    };
    // The stage of tile i >= ST has been read.  4 bits: K's, with two stages and two S, once S of tile i - 2 is there; as
    // softmax may still be at that tile, it waits for nothing of K's loaders (k_full could be two phases on).
    auto wait_empty = [&](int i) {
        uint64_t* read = FMT == kWinQ4 && !is_v ? &s_full[i & 1] : &empty[i % ST];
        ok = mbar_wait(read, (uint32_t)(i / ST - 1) & 1u, DEV_ERR_ATTN_WAIT);
        ok = __all_sync(0xffffffffu, ok);
    };
    // 4 bits: codes through the warp's own ring, RAW - 1 tiles ahead
    const uint32_t raw = smem_u32(smem + L::CODES) + (warp - 4) * L::RAW * G::BYTES;
    // fp16: 16-byte piece c of this thread's half row of a tile
    auto piece = [&](int st, int c) {
        const int ch = half * (D / 16) + c;  // of D / 8
        return smem + L::RING + st * L::STAGE + is_v * L::NP * L::PART_KV + (ch >> 3) * L::PANEL + key * 128 + (((ch & 7) ^ (key & 7)) << 4);
    };
    auto fetch = [&](int i) {  // tile i's copies, a group
        const int id = i < nt ? block_id(i) : -1;
        valid = id >= 0 ? valid | (1u << (i & 31)) : valid & ~(1u << (i & 31));
        const uint8_t* src = base + (uint64_t)(uint32_t)max(id, 0) * p.block_bytes;
        if constexpr (FMT == kWinQ4) {
            if (id >= 0) {
                const uint32_t dst = raw + (i % L::RAW) * G::BYTES;
#pragma unroll
                for (int c = 0; c < G::BYTES / 16; c += 32)
                    if (c + lane < G::BYTES / 16) cp_async16(dst + (c + lane) * 16, src + (c + lane) * 16);
            }
        } else if (i < nt) {
            const int st = i % ST;
            if (!is_v && lane == 0) s_here[st][w4] = id >= 0;
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
                if (id >= 0) cp_async16(smem_u32(piece(st, c)), src + off * (2 * D) + half * D + 16 * c);
                else *reinterpret_cast<uint4*>(piece(st, c)) = make_uint4(0, 0, 0, 0);
            }
        }
        cp_async_commit();
    };
    constexpr int AHEAD = FMT == kWinQ4 ? L::RAW - 1 : ST - 1;
    if (warp >= 4 && warp < 12)
        for (int i = 0; i < AHEAD; ++i) fetch(i);

    // ---------------------------------------------------------------------- Q to shared memory
    if (warp < 12) {
        const int c = lane % LPR;
#pragma unroll 1
        for (int k0 = 0; k0 < 12; k0 += 6) {
#pragma unroll
            for (int k = 0; k < 6; ++k) {
                const int row = q_row(k0 + k);
                if (row >= 128) break;
                const float4 u = q_now[k];
                // magnitudes order as integers do; NaN is above infinity
                uint32_t top = max(max(__float_as_uint(u.x) & 0x7fffffffu, __float_as_uint(u.y) & 0x7fffffffu),
                                   max(__float_as_uint(u.z) & 0x7fffffffu, __float_as_uint(u.w) & 0x7fffffffu));
                top = __reduce_max_sync(RPI == 1 ? 0xffffffffu : 0xffffu << (lane & 16), top);
                const int ex = max((int)(top >> 23), 12);
                const float up = __uint_as_float((uint32_t)(265 - ex) << 23);
                uint2 h[2];  // high and low halves
                split_h2(u.x * up, u.y * up, h[0].x, h[1].x);
                split_h2(u.z * up, u.w * up, h[0].y, h[1].y);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint2& x = h[half];
                    if constexpr (FMT == kWinQ4) {
                        // the channel order in which nibbles come apart (below): 0 4 1 5 2 6 3 7 of each eight.
                        // An even lane holds 0 1 2 3 and makes 0 4 1 5, the odd one beside it 4 5 6 7 and 2 6 3 7
                        const uint32_t other = __shfl_xor_sync(0xffffffffu, lane & 1 ? x.x : x.y, 1);
                        x = lane & 1 ? make_uint2(prmt(other, x.y, 0x5410), prmt(other, x.y, 0x7632))
                                     : make_uint2(prmt(x.x, other, 0x5410), prmt(x.x, other, 0x7632));
                    }
                    *reinterpret_cast<uint2*>(smem + L::Q + half * L::QHALF + (c >> 4) * 16384 +
                                              sw128_off(row, (c & 15) * 4)) = x;
                }
                if (c == 0) s_sf[row] = __uint_as_float((uint32_t)(ex - 11) << 23) * (FMT == kWinQ4 ? 2.f * p.scale_log2 : p.scale_log2);
            }
#pragma unroll
            for (int k = 0; k < 6; ++k) q_now[k] = q_next[k];
        }
        fence_proxy_async_smem();
        mbar_arrive(&q_full);
    }

    float m = -INFINITY, mu = 0.f, l = 0.f;
    if (warp < 4) {
        // ------------------------------------------------------------------ softmax
        ok = __all_sync(0xffffffffu, mbar_wait(&q_full, 0, DEV_ERR_ATTN_WAIT));  // (for s_sf)
        const float sf = s_sf[r];
        const uint32_t lanes = tmem + ((uint32_t)warp << 21);
        for (int i = 0; i < nt && ok; ++i) {
            const int st = i % ST, pos = (t0 + i) * 4;
            ok = mbar_wait(&s_full[i & 1], (uint32_t)(i >> 1) & 1u, DEV_ERR_ATTN_WAIT) &&
                 mbar_wait(FMT == kWinQ4 ? &v_full[st] : &k_full[st], (uint32_t)(i / ST) & 1u, DEV_ERR_ATTN_WAIT);  // (for s_here)
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            float v[64];
            tmem_ld64(lanes + L::TS + (i & 1) * 64, v);
            const uint32_t here = *reinterpret_cast<const uint32_t*>(s_here[st]);
            const bool whole = here == 0x01010101u && t0 + i >= whole0 && t0 + i < whole1;
            if (!whole) {
                ok = mbar_wait(&v_full[st], (uint32_t)(i / ST) & 1u, DEV_ERR_ATTN_WAIT);  // (for s_bad)
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int j0 = first_key(pos + b);
                    const bool there = (here >> (8 * b)) & 1;
                    if (there && is_whole(j0)) continue;
                    // bit k: the row sees key j0 + k
                    auto below = [&](int j) { return (1u << min(max(j - j0, 0), 16)) - 1u; };
                    uint32_t sees = below(ctx) & (~below(max(ctx - window, 0)) | below(p.sinks));
                    if (!there) sees = 0;
                    if (s_some_bad[st][b]) {
                        for (int k = 0; k < 16; ++k)  // its V was taken out: the row becomes NaN
                            if (((sees >> k) & 1) && *reinterpret_cast<const uint16_t*>(s_bad[st] + 32 * b + 2 * k))
                                l = __int_as_float(0x7fffffff);
                    }
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        if (!(sees & (1u << k))) v[16 * b + k] = -INFINITY;
                }
            }
            float t8[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) t8[k] = v[k];
#pragma unroll
            for (int k = 8; k < 64; ++k) t8[k & 7] = fmaxf(t8[k & 7], v[k]);
            // sf > 0; -inf stays
            const float top = sf * fmaxf(fmaxf(fmaxf(t8[0], t8[1]), fmaxf(t8[2], t8[3])),
                                         fmaxf(fmaxf(t8[4], t8[5]), fmaxf(t8[6], t8[7])));
            // the running maximum moves only when a score passes it by 8; P, relative to 2^-7 of it, stays below 2^15
            if (__any_sync(0xffffffffu, top > (m == -INFINITY ? -INFINITY : m + 8.f))) {
                const float mn = fmaxf(m, top);
                const float corr = mn == -INFINITY ? 1.f : ex2_approx(m - mn);
                m = mn;
                mu = mn == -INFINITY ? 0.f : mn - kPShift;
                l *= corr;
                if (i > 0) {  // O holds P V of tiles 0 .. i - 1 once the last is done
                    ok = mbar_wait(&pv_done[(i - 1) & 1], (uint32_t)((i - 1) >> 1) & 1u, DEV_ERR_ATTN_WAIT);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D; c += 16) {
                        float x[16];
                        tmem_ld16(lanes + L::TO + c, x);
#pragma unroll
                        for (int k = 0; k < 16; ++k) x[k] *= corr;
                        tmem_st16(lanes + L::TO + c, x);
                    }
                }
            }
            float s4[4] = {0.f, 0.f, 0.f, 0.f};
            const uint32_t to_p = lanes + L::TP + (i & 1) * 64;
#pragma unroll
            for (int c = 0; c < 2; ++c) {  // 32 keys: 16 columns of two each
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const float a = ex2_approx(fmaf(v[32 * c + 2 * k], sf, -mu));
                    const float b = ex2_approx(fmaf(v[32 * c + 2 * k + 1], sf, -mu));
                    s4[k & 3] += a + b;
                    split_h2(a, b, hi[k], lo[k]);
                }
                tmem_st16_now(to_p + 16 * c, hi);
                tmem_st16_now(to_p + 32 + 16 * c, lo);
            }
            tmem_st_wait();
            l += (s4[0] + s4[1]) + (s4[2] + s4[3]);
            tc_fence_before();
            mbar_arrive(&p_full[i & 1]);
        }
        if (ok && nt > 0) ok = mbar_wait(&pv_done[(nt - 1) & 1], (uint32_t)((nt - 1) >> 1) & 1u, DEV_ERR_ATTN_WAIT);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
    } else if (warp < 12) {
        // ------------------------------------------------------------------ K (is_v 0) or V: block `w4` of each tile
        if constexpr (FMT == kWinQ4) {
            // Nibbles (0, 4), (1, 5), (2, 6), (3, 7) of a word as two fp16 pairs, high + low = half of code * scale +
            // zero (half, so that values past 65504 fit).  With g = 2^-9 of the power of two below the group's
            // largest value M, scale and zero are multiples of g (sh, zh) and what those leave (sl, zl): the high
            // part is exact, a multiple of g / 2 below 2^11 of them, and the low part, below 4 g, rounds: the value
            // is off by at most 2^-18 of M (2^-23 where M is below 2^-5).
            auto values = [&](uint32_t x, __half2 sh, __half2 sl, __half2 zh, __half2 zl, uint4& hi, uint4& lo) {
                uint32_t *oh = &hi.x, *ol = &lo.x;
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    // 512 + code / 2 is an fp16 number with the nibble in its low bits
                    const uint32_t a = ((x >> (4 * h)) & 0x000f000fu) | 0x60006000u;
                    const __half2 c = __hsub2_rn(*reinterpret_cast<const __half2*>(&a), __floats2half2_rn(512.f, 512.f));
                    const __half2 v = __hfma2(c, sh, zh), l = __hfma2(c, sl, zl);
                    oh[h] = *reinterpret_cast<const uint32_t*>(&v);
                    ol[h] = *reinterpret_cast<const uint32_t*>(&l);
                }
            };
            // a thread's words: i = 4 half + k / NW of group k % NW (k < 4 NW), of a row of D / 8 words
            uint8_t* to = smem + L::RING + is_v * L::NP * L::PART_KV + key * 128;
            const uint32_t from = raw + off * (D / 2) + half * 16 * NW;
            for (int i = 0; i < nt; ++i) {
                const int st = i % ST;
                cp_async_wait<L::RAW - 2>();
                __syncwarp();  // tile i's codes are there, and every lane is done with the ring's slot of tile i - 1
                fetch(i + L::RAW - 1);
                const bool in = (valid >> (i & 31)) & 1;
                uint32_t x[NW][4] = {};
                const bool check = is_v && hidden(i, in);
                bool bad = false;
                __half2 sh[NW], sl[NW], zh[NW], zl[NW];  // scales; zeros' halves
#pragma unroll
                for (int c = 0; c < NW; ++c) sh[c] = sl[c] = zh[c] = zl[c] = __floats2half2_rn(0.f, 0.f);
                if (in) {
                    const uint32_t slot_at = (i % L::RAW) * G::BYTES;
#pragma unroll
                    for (int c = 0; c < NW; ++c) {
                        lds_words(x[c], from + slot_at + 16 * c);
                        float2 prm = lds_half2(raw + slot_at + Q4Layout<D>::PARAMS + c * 64 + off * 4);
                        // what a key that some row does not see may hold: not what a write leaves
                        const float top = fmaxf(fabsf(prm.y), fabsf(fmaf(15.f, prm.x, prm.y)));  // M
                        if (check && !(fabsf(prm.x) <= 8736.f && top < 100000.f)) prm = make_float2(0.f, 0.f), bad = true;
                        // adding 1.5 * 2^23 g rounds to a multiple of g (2^-23 at least: halves stay fp16 numbers)
                        const uint32_t e = max((int)(__float_as_uint(top) >> 23), 113);
                        const float magic = __uint_as_float(((e + 14) << 23) | 0x400000u);
                        const float s0 = __fsub_rn(__fadd_rn(prm.x, magic), magic), z0 = __fsub_rn(__fadd_rn(prm.y, magic), magic);
                        sh[c] = __float2half2_rn(s0);
                        sl[c] = __float2half2_rn(prm.x - s0);
                        zh[c] = __float2half2_rn(0.5f * z0);
                        zl[c] = __float2half2_rn(0.5f * (prm.y - z0));
                    }
                }
                if (i >= ST) {
                    wait_empty(i);
                    if (!ok) break;
                }
                if (is_v && lane == 0) s_here[st][w4] = in;
#pragma unroll
                for (int c = 0; c < 4 * NW; ++c) {  // channels 64 w + 8 ii .. + 7, w = c % NW
                    const int ii = 4 * half + c / NW;
                    uint4 u[2];
                    values(x[c >> 2][c & 3], sh[c % NW], sl[c % NW], zh[c % NW], zl[c % NW], u[0], u[1]);
#pragma unroll
                    for (int part = 0; part < 2; ++part)
                        *reinterpret_cast<uint4*>(to + st * L::STAGE + part * L::PART_KV + (c % NW) * L::PANEL +
                                                  ((ii ^ (key & 7)) << 4)) = u[part];
                }
                if (is_v) {
                    s_bad[st][pt] = bad;
                    const bool any = __any_sync(0xffffffffu, bad);
                    if (lane == 0) s_some_bad[st][w4] = any;
                }
                fence_proxy_async_smem();
                mbar_arrive(&full[st]);
            }
        } else {
            for (int i = 0; i < nt; ++i) {
                const int st = i % ST;
                cp_async_wait<ST - 2>();
                if (is_v) {
                    bool bad = false;
                    if (hidden(i, (valid >> (i & 31)) & 1)) {
#pragma unroll
                        for (int c = 0; c < D / 16; ++c) {
                            uint4 u = *reinterpret_cast<const uint4*>(piece(st, c));
                            if (clean(u)) *reinterpret_cast<uint4*>(piece(st, c)) = u, bad = true;
                        }
                    }
                    s_bad[st][pt] = bad;
                    const bool any = __any_sync(0xffffffffu, bad);
                    if (lane == 0) s_some_bad[st][w4] = any;
                }
                fence_proxy_async_smem();
                mbar_arrive(&full[st]);
                // the next tile takes the stage of i - 1, whose products need nothing past tile i
                if (i >= 1 && i + ST - 1 < nt) {
                    wait_empty(i + ST - 1);
                    if (!ok) break;
                }
                fetch(i + ST - 1);
            }
        }
        cp_async_wait<0>();
    } else {
        // ------------------------------------------------------------------ products
        // The whole warp walks the loop and one lane issues, so that descriptors stay uniform values.
        const bool lead = elect_one();
        const uint32_t idesc_s = make_idesc_f16(128, 64), idesc_o = make_idesc_f16(128, D) | (1u << 16);  // V is MN-major
        // descriptors of the buffers' starts; a step's is an addition to the address field (16-byte units)
        const uint64_t q_desc = make_sw128_desc(smem_u32(smem + L::Q)), k_desc = make_sw128_desc(smem_u32(smem + L::RING)),
                       v_desc = make_sw128_mn_desc(smem_u32(smem + L::RING + L::NP * L::PART_KV), L::PANEL);
        auto issue_s = [&](int i) {
            // (every lane has waited before one issues: K's next tile may follow the products at once)
            if (!__all_sync(0xffffffffu, mbar_wait(&k_full[i % ST], (uint32_t)(i / ST) & 1u, DEV_ERR_ATTN_WAIT))) return false;
            tc_fence_after();
            const uint64_t kd = k_desc + (uint32_t)((i % ST) * (L::STAGE >> 4));
            const uint32_t d = tmem + L::TS + (i & 1) * 64;
            if (lead) {
#pragma unroll
                for (int t = 0; t < 1 + L::NP; ++t)  // both halves of q times K, the high one times K's low parts
#pragma unroll
                    for (int kk = 0; kk < 4 * NW; ++kk)
                        umma_bf16(d, q_desc + ((t & 1) * (L::QHALF >> 4) + (kk >> 2) * (16384 >> 4) + 2 * (kk & 3)),
                                  kd + ((t >> 1) * (L::PART_KV >> 4) + (kk >> 2) * (L::PANEL >> 4) + 2 * (kk & 3)), idesc_s,
                                  (t | kk) ? 1u : 0u);
                umma_commit(&s_full[i & 1]);
            }
            return true;
        };
        if (nt > 0) ok = __all_sync(0xffffffffu, mbar_wait(&q_full, 0, DEV_ERR_ATTN_WAIT)) && issue_s(0);
        for (int i = 0; i < nt && ok; ++i) {
            if (i + 1 < nt) ok = issue_s(i + 1);
            ok = ok && mbar_wait(&p_full[i & 1], (uint32_t)(i >> 1) & 1u, DEV_ERR_ATTN_WAIT);
            ok = ok && mbar_wait(&v_full[i % ST], (uint32_t)(i / ST) & 1u, DEV_ERR_ATTN_WAIT);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint64_t vd = v_desc + (uint32_t)((i % ST) * (L::STAGE >> 4));
            const uint32_t pt0 = tmem + L::TP + (i & 1) * 64;
            if (lead) {
#pragma unroll
                for (int t = 0; t < 1 + L::NP; ++t)  // both halves of P times V, the high one times V's low parts
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        umma_ts_f16(tmem + L::TO, pt0 + (t & 1) * 32 + kk * 8,
                                    vd + (t >> 1) * (L::PART_KV >> 4) + kk * (2048 >> 4), idesc_o,
                                    (i > 0 || t > 0 || kk > 0) ? 1u : 0u);
                umma_commit(&empty[i % ST]);
                umma_commit(&pv_done[i & 1]);
            }
            __syncwarp();
        }
        if (!__all_sync(0xffffffffu, ok) && lead) {  // every product issued so far ends before TMEM is given back
            __shared__ uint64_t drain;
            mbar_init(&drain, 1);
            fence_mbar_init();
            umma_commit(&drain);
            mbar_wait(&drain, 0, DEV_ERR_DRAIN);
        }
    }

    // ---------------------------------------------------------------------- out
    // a row without keys in a tile of rows that have some: whole tiles scored its q unmasked, so its sum may be
    // anything and its maximum infinite (inf - inf would make the fold's factor NaN)
    if (ctx == 0) l = 0.f, m = -INFINITY;
    float* part = reinterpret_cast<float*>(smem + L::RING);
    auto out_at = [&](int row, int d) { return head_row(row) * D + d; };
    __syncwarp();
    if (warp < 4) {
        const uint32_t lanes = tmem + ((uint32_t)warp << 21) + L::TO;
        const bool sum = ok && nt > 0 && l != 0.f;  // else zeros (NaN counts as a sum)
        const float inv = (FMT == kWinQ4 ? 2.f : 1.f) * (splits == 1 ? 1.f / l : 1.f);  // (4 bits: V is halved)
        uint8_t* staged = smem + L::RING;  // [row][ROWB] bf16, then the low halves
        s_part[r][0] = m;
        s_part[r][1] = ok ? l : 0.f;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
            float x[32], y[32];
            tmem_ld32(lanes + c, x);
#pragma unroll
            for (int k = 0; k < 32; ++k) {
                // 4 bits: position 8 n + k of V holds channel 8 n + k / 2 + 4 (k % 2)
                const int ch = FMT == kWinQ4 ? (k & 24) + ((k & 7) >> 1) + 4 * (k & 1) : k;
                y[ch] = sum ? x[k] * inv : 0.f;
            }
            if (splits > 1) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    *reinterpret_cast<float4*>(part + r * L::PART + c + 4 * k) =
                        make_float4(y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]);
            } else {
                uint8_t* at = staged + r * L::ROWB + 2 * c;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t hi[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) hi[j] = pack_bf2(y[8 * k + 2 * j], y[8 * k + 2 * j + 1]);
                    *reinterpret_cast<uint4*>(at + 16 * k) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if (p.out_lo) {
                        uint32_t lo[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            lo[j] = pack_bf2(y[8 * k + 2 * j] - __uint_as_float(hi[j] << 16),
                                             y[8 * k + 2 * j + 1] - __uint_as_float(hi[j] & 0xffff0000u));
                        *reinterpret_cast<uint4*>(at + 128 * L::ROWB + 16 * k) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 12) tmem_dealloc(tmem, L::TCOLS);
    if (splits == 1) {
        // whole rows leave shared memory
        for (int k = threadIdx.x; k < rows * (D / 8); k += kChunkThreads) {
            const int row = k / (D / 8), c = k % (D / 8);
            const size_t at = out_at(row, 8 * c);
            const uint8_t* from = smem + L::RING + row * L::ROWB + 16 * c;
            *reinterpret_cast<uint4*>(p.out + at) = *reinterpret_cast<const uint4*>(from);
            if (p.out_lo)
                *reinterpret_cast<uint4*>(p.out_lo + at) = *reinterpret_cast<const uint4*>(from + 128 * L::ROWB);
        }
        return;
    }
    cluster_sync();
    // four channels a lane, a row (D = 64: two) a warp; every CTA's part is fetched at once
    for (int j = (int)rank * (kChunkThreads / 32) + warp; j * RPI < rows; j += (int)splits * (kChunkThreads / 32)) {
        const int row = min(j * RPI + lane / LPR, rows - 1), d = (lane % LPR) * 4;
        const uint32_t at_o = smem_u32(part + row * L::PART + d), at_m = smem_u32(&s_part[row][0]);
        float4 v[8];
        float mc[8], lc[8], mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            mc[c] = -INFINITY;
            lc[c] = 0.f;
            if (c < (int)splits) {
                mc[c] = ld_dsmem_now(map_to_rank(at_m, c));
                lc[c] = ld_dsmem_now(map_to_rank(at_m + 4, c));
                v[c] = ld_dsmem_f32x4(map_to_rank(at_o, c));
            }
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) mx = fmaxf(mx, mc[c]);
        float sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            // a CTA without keys holds nothing, one of nothing but NaN scores a sum that is not zero
            if (mc[c] == -INFINITY) {
                sum += lc[c];
            } else {
                const float f = ex2_approx(mc[c] - mx);
                sum = fmaf(lc[c], f, sum);
                acc.x = fmaf(v[c].x, f, acc.x), acc.y = fmaf(v[c].y, f, acc.y);
                acc.z = fmaf(v[c].z, f, acc.z), acc.w = fmaf(v[c].w, f, acc.w);
            }
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const float x = acc.x * inv, y = acc.y * inv, z = acc.z * inv, w = acc.w * inv;
        const uint2 hi = make_uint2(pack_bf2(x, y), pack_bf2(z, w));
        *reinterpret_cast<uint2*>(p.out + out_at(row, d)) = hi;
        if (p.out_lo)
            *reinterpret_cast<uint2*>(p.out_lo + out_at(row, d)) =
                make_uint2(pack_bf2(x - __uint_as_float(hi.x << 16), y - __uint_as_float(hi.x & 0xffff0000u)),
                           pack_bf2(z - __uint_as_float(hi.y << 16), w - __uint_as_float(hi.y & 0xffff0000u)));
    }
    cluster_sync();  // no CTA leaves while another reads its shared memory
}

// CTAs of clusters of `splits` that are on the card at once (the clusters of eight are fewer than its SMs hold CTAs,
// as a cluster stays within a GPC: 16 of them ran as two waves).  Asked once per kernel, device and size.
template <int FMT, int D>
inline int chunk_clusters(int splits) {
    constexpr auto kernel = paged_attn_chunk_kernel<FMT, D>;
    static std::atomic<int> known[64][4];
    int dev = 0, n = 0, at = 0;
    while ((1 << at) < splits) ++at;  // 1, 2, 4, 8
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (dev < 64 && (n = known[dev][at].load(std::memory_order_relaxed)) > 0) return n;
    if (func_attr_once<kernel>(ChunkLayout<FMT, D>::SMEM) != cudaSuccess) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(splits);
    cfg.blockDim = dim3(kChunkThreads);
    cfg.dynamicSmemBytes = ChunkLayout<FMT, D>::SMEM;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = splits, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    if (dev < 64) known[dev][at].store(n, std::memory_order_relaxed);
    return n;
}

// How a call would go through 128-row tiles: queries a tile, tiles of a stream and of all, the CTAs that share a
// tile's keys (while all clusters are on the card at once and a CTA keeps two tiles), 64-key tiles a CTA walks.
struct ChunkPlan {
    int qt, stream_tiles, splits, walk;
    long long tiles;
};
// keys that a tile of `q` queries reads, at most
inline long long window_keys(const WinParams& p, int q) {
    const long long limit = p.max_ctx < p.mbps * 16 ? p.max_ctx : p.mbps * 16, seen = (long long)p.window + p.sinks + q + 32;
    return p.window > 0 && seen < limit ? seen : limit;
}
template <int FMT, int D>
inline ChunkPlan plan_chunk(const WinParams& p) {
    ChunkPlan c;
    c.qt = 128 / p.group < p.S ? 128 / p.group : p.S;
    c.stream_tiles = ceil_div(p.S, c.qt);
    c.tiles = (long long)(p.R / p.S) * c.stream_tiles * p.kv_heads;
    const long long keys = window_keys(p, c.qt);
    c.splits = 1;
    while (c.splits < 8 && keys >= 2ll * c.splits * 2 * 64 && c.tiles <= chunk_clusters<FMT, D>(c.splits * 2)) c.splits *= 2;
    c.walk = (int)((keys + 64 * c.splits - 1) / (64 * c.splits));
    return c;
}

// Whether rows go through 128-row tiles (QTTS_WINDOW_TILES=0 / 1 forces it where either form can run): the shorter of
// two estimates in us, fitted to 192 measured pairs (four head layouts, both pools, 1 to 16 streams of 16 to 1000 rows, 0
// to 8000 keys before them; the pick is within 11% of the better form, once 19%).
//   tiles:      waves (8 + c a 64-key tile of a CTA), 3 more for a cluster; c = 1.4 (4 bits), 2.3 (fp16), D = 64: 1.0, 1.2
//   8-row tiles: 5 + 6.6e-6 D a (tile, 16-key block) pair + 3e-3 (4 bits) or 8e-3 (fp16) a tile
// Measured (us, 16 heads over 8, D = 128, streams x rows + past, tiles / 8-row tiles, B200, K and V from HBM):
//   4 bits  1 x 64 + 500   14.8 / 9.2     1 x 128 + 500  15.1 / 13.3   1 x 256 + 500  16.3 / 23.4
//           8 x 16 + 500   16.5 / 12.8    8 x 32 + 500   17.5 / 19.8   8 x 64 + 500   19.4 / 35.5
//           2 x 64         10.2 / 7.1     8 x 64         10.3 / 12.9   1 x 1000 + 4000 119 / 370
//           1 x 16 + 8000  33.3 / 19.5    1 x 32 + 8000  34.0 / 30.4   1 x 64 + 8000  36.2 / 52.8
//   fp16    1 x 64 + 500   15.8 / 13.9    1 x 128 + 500  16.1 / 15.0   1 x 256 + 500  17.6 / 25.1
//           8 x 16 + 500   18.9 / 14.6    8 x 32 + 500   19.8 / 21.9   8 x 64 + 500   21.6 / 41.9
//           2 x 64         10.3 / 8.6     8 x 64         10.5 / 20.2   1 x 1000 + 4000 191 / 374
//           1 x 16 + 8000  45.2 / 21.2    1 x 32 + 8000  45.7 / 31.1   1 x 64 + 8000  47.9 / 52.1
// The keys are max_ctx's (contexts are on the device): a bound far above them picks the wrong form at times.
template <int FMT, int D>
inline bool use_chunk_kernel(const WinParams& p, const ChunkPlan& c) {
    static const int forced = [] {
        const char* v = getenv("QTTS_WINDOW_TILES");
        return v && (v[0] == '0' || v[0] == '1') ? v[0] - '0' : -1;
    }();
    if (forced >= 0) return forced == 1;
    const long long heads = (long long)(p.R / p.S) * p.kv_heads;
    const long long row_tiles = heads * (p.group >= 8 ? (long long)p.S * ceil_div(p.group, 8) : ceil_div(p.S, 8 / p.group));
    const double waves = c.splits > 1 ? 1. : (double)((c.tiles + num_sms() - 1) / num_sms());
    const double a_tile = FMT == kWinQ4 ? (D == 128 ? 1.4 : 1.0) : (D == 128 ? 2.3 : 1.2);
    const double tiles_us = waves * (8. + a_tile * c.walk) + (c.splits > 1 ? 3. : 0.);
    const double rows_us = 5. + 6.6e-6 * D * ((double)row_tiles * (double)(window_keys(p, 8) / 16.)) +
                           (FMT == kWinQ4 ? 3e-3 : 8e-3) * (double)row_tiles;
    return tiles_us < rows_us;
}

template <int FMT, int D>
inline int launch_chunk_attention(WinParams p, const ChunkPlan& c, cudaStream_t st) {
    using L = ChunkLayout<FMT, D>;
    using G = WinChunk<FMT, D>;
    p.qt = c.qt;
    p.tiles = c.stream_tiles;
    const long long block_bytes = (long long)p.num_layers * 2 * p.kv_heads * G::BYTES;
    QTTS_REQUIRE(block_bytes < (1ll << 31), "paged attention: %lld bytes per block", block_bytes);
    p.block_bytes = (uint32_t)block_bytes;
    p.v_offset = (uint32_t)(p.kv_heads * G::BYTES);
    QTTS_REQUIRE(c.tiles * 8 < (1ll << 31), "paged attention: %lld tiles", c.tiles);
    constexpr auto kernel = paged_attn_chunk_kernel<FMT, D>;
    QTTS_CHECK_CUDA((func_attr_once<kernel>(L::SMEM)));
    QTTS_CHECK_CUDA(launch_pdl(kernel, dim3((unsigned)(c.tiles * c.splits)), dim3(kChunkThreads), L::SMEM, st,
                               dim3(c.splits, 1, 1), p));
    return QTTS_OK;
}

// Decode rows, and chunks in the form that suits them.
template <int FMT, int D>
inline int launch_attention(const WinParams& p, cudaStream_t st) {
    const bool either = p.S > 1 && p.group <= 128 &&
                        ((reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.out_lo)) & 15) == 0;
    if (either) {
        const ChunkPlan c = plan_chunk<FMT, D>(p);
        if (use_chunk_kernel<FMT, D>(p, c)) return launch_chunk_attention<FMT, D>(p, c, st);
    }
    return launch_window_attention<FMT, D>(p, st);
}

}  // namespace qtts
