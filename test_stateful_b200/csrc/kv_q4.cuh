// 4-bit paged KV cache: quantising K/V rows as they are written, and reading them back.
//
// A group is 64 channels of one token and head.  With lo, hi its smallest and largest value
// (saturated to fp16's range, +-65504):
//   zero  = fp16(lo)
//   scale = fp16(fl(fl(hi - lo) * fl(1/15)))
//   code  = the integer in [0, 15] nearest to fl(x - zero) / scale, ties to even (0 when scale = 0)
//   value = code * scale + zero
// fl() is fp32 rounding; the quotient is taken exactly, so that the codes do not depend on how a
// division rounds.  A NaN makes its group read back as NaN (zero = NaN, scale = 0, codes 0).  A group that
// spans nearly all of fp16 can have values past 65504 (up to 65600, as scale was rounded): in fp16 they are 65504.
//
// Pool: [num_blocks][layers][2][kv_heads] chunks of 16 tokens.  A chunk is 16 rows of
// head_dim / 2 bytes of codes, then head_dim / 64 arrays of 16 (scale, zero) fp16 pairs.  A row's
// 32-bit words alternate between its groups (word NG * i + w holds channels 64 w + 8 i .. + 7,
// channel 0 in the low nibble), so that one 16- or 8-byte load of the attention kernel brings a
// lane channels of every group.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace qtts {

template <int D>
struct Q4Layout {
    static constexpr int NG = D / 64;                // groups per row
    static constexpr int ROW = D / 2;                // bytes of codes per token
    static constexpr int PARAMS = 16 * ROW;          // offset of the (scale, zero) pairs
    static constexpr int CHUNK = PARAMS + NG * 64;   // bytes per (block, layer, k|v, head)
};

// n / d for n < 2^31 as a multiply-high and a shift (one per row instead of a hardware division)
struct FastDiv {
    uint32_t mul, shift, d;
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return d == 1 ? n : __umulhi(n, mul) >> shift; }
};
inline FastDiv make_fastdiv(uint32_t d) {
    FastDiv f = {0, 0, d};
    if (d > 1) {
        uint32_t l = 0;
        while ((1u << l) < d) ++l;  // 2^(l-1) < d <= 2^l
        // m = ceil(2^(31+l) / d) < 2^32 is exact for n < 2^31 (the excess e = m d - 2^(31+l) is below
        // d <= 2^l, so n e < 2^(31+l) and the quotient is never one too high)
        f.mul = (uint32_t)(((1ull << (31 + l)) + d - 1) / d);
        f.shift = l - 1;
    }
    return f;
}

struct Q4IoParams {
    uint8_t* cache;
    const void *k_in, *v_in;            // write: rows in
    void *k_out, *v_out;                // read: rows out
    int ks[3], vs[3];                   // element strides of (token, layer, head)
    uint32_t block_bytes;               // of a pool block
    int num_blocks, num_layers, kv_heads, first_layer;
    int n;                              // tokens
    const int32_t* mapping;             // position of each token (block * 16 + offset) ...
    const int32_t* blocks;              // ... or the block id of each 16 tokens
    FastDiv rows, heads;                // rows of one token (layers * 2 * heads), heads
    uint32_t total;                     // ceil(n / 16) * 16 * rows
};

// Inputs are read through L2 (__ldcg): a kernel launched with programmatic dependent launch begins
// before its predecessor has written them, so they are not read-only for the kernel's life.
template <typename T>
__device__ __forceinline__ float q4_to_float(T x);
template <>
__device__ __forceinline__ float q4_to_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ float q4_to_float<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float q4_to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T q4_from_float(float x);
template <>
__device__ __forceinline__ float q4_from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half q4_from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 q4_from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// min / max that return NaN when either argument is NaN
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Smallest and largest of a group's 64 values, sixteen in each of the row's four threads; NaN if any is.
// 16-bit types go two to an instruction, and as the pair (min, -max) through the shuffles.
template <typename T>
__device__ __forceinline__ float2 group_range(const T (&x)[16], unsigned peers) {
    if constexpr (sizeof(T) == 4) {
        float lo = x[0], hi = x[0];
#pragma unroll
        for (int c = 1; c < 16; ++c) lo = min_nan(lo, x[c]), hi = max_nan(hi, x[c]);
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            lo = min_nan(lo, __shfl_xor_sync(peers, lo, o));
            hi = max_nan(hi, __shfl_xor_sync(peers, hi, o));
        }
        return make_float2(lo, hi);
    } else {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        const T2* v = reinterpret_cast<const T2*>(x);
        T2 mn = v[0], mx = v[0];
#pragma unroll
        for (int c = 1; c < 8; ++c) mn = __hmin2_nan(mn, v[c]), mx = __hmax2_nan(mx, v[c]);
        T2 r;
        r.x = __hmin_nan(mn.x, mn.y);
        r.y = __hneg(__hmax_nan(mx.x, mx.y));
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            const uint32_t u = __shfl_xor_sync(peers, *reinterpret_cast<const uint32_t*>(&r), o);
            r = __hmin2_nan(r, *reinterpret_cast<const T2*>(&u));
        }
        return make_float2(q4_to_float<T>(r.x), -q4_to_float<T>(r.y));
    }
}

// Where thread group `flat` works: rows are ordered 16 tokens innermost, then head, k|v, layer, then
// the next 16 tokens, so that consecutive rows of a whole block fill a chunk.
struct Q4Row {
    int token, layer, kv, head;
};
__device__ __forceinline__ Q4Row q4_row(const Q4IoParams& p, uint32_t flat) {
    const uint32_t t16 = flat & 15, rest = flat >> 4;
    const uint32_t tg = p.rows.div(rest);
    const uint32_t row = rest - tg * p.rows.d;
    const uint32_t lk = p.heads.div(row);
    return {(int)(tg * 16 + t16), (int)(lk >> 1), (int)(lk & 1), (int)(row - lk * p.heads.d)};
}

// Chunk address of a row's token, or NULL for a position outside the pool.
template <int D>
__device__ __forceinline__ uint8_t* q4_chunk(const Q4IoParams& p, const Q4Row& r, int* off) {
    int blk;
    if (p.mapping) {
        const int m = __ldcg(p.mapping + r.token);
        if (m < 0) return nullptr;
        blk = m >> 4;
        *off = m & 15;
    } else {
        blk = __ldcg(p.blocks + (r.token >> 4));
        *off = r.token & 15;
    }
    if (blk < 0 || blk >= p.num_blocks) return nullptr;
    const uint32_t in_block = (uint32_t)(((p.first_layer + r.layer) * 2 + r.kv) * p.kv_heads + r.head) * Q4Layout<D>::CHUNK;
    return p.cache + (uint64_t)(uint32_t)blk * p.block_bytes + in_block;
}

// Element offset of a row from its K or V base.
__device__ __forceinline__ long long q4_offset(const Q4IoParams& p, const Q4Row& r) {
    const int st0 = r.kv ? p.vs[0] : p.ks[0], st1 = r.kv ? p.vs[1] : p.ks[1], st2 = r.kv ? p.vs[2] : p.ks[2];
    return (long long)r.token * st0 + (long long)r.layer * st1 + (long long)r.head * st2;
}

// The code of d = x - zero by exact remainders; rare, and so a call.
__device__ __noinline__ float q4_exact_code(float d, float scale, float inv15) {
    float k = rintf(__saturatef(d * inv15) * 15.f);
    // e = d - k scale is exact wherever it is near scale / 2
    const float e = __fmaf_rn(-k, scale, d), h = 0.5f * scale;
    const bool odd = (int)k & 1;
    if (e > h || (e == h && odd)) k += 1.f;
    else if (e < -h || (e == -h && odd)) k -= 1.f;
    return fminf(fmaxf(k, 0.f), 15.f);
}

// Four threads a row: thread i takes words i and i + 4 of every group w, the channels 64 w + 8 i .. + 7
// and 64 w + 32 + 8 i .. + 7 (64 contiguous bytes of a 16-bit row per load of the four, and the group's
// scale and zero worked out by four threads instead of eight: 30 -> 21 us for 501 tokens of 28 layers).
constexpr int kQ4Threads = 128, kQ4RowsPerCta = kQ4Threads / 4;

// Bound by instructions and the wait for the rows they work on (0.71 of the issue slots), not by HBM: 501 tokens
// of 28 layers 19.3 us in fp16 (3.8 TB/s), 20.7 in bf16, 22.9 in fp32 (5.7 TB/s; 8 heads, D = 128, rows and pools
// from HBM); a step's 64 tokens of one layer, each in a block of its own, 3.3 us.
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kQ4Threads) kv_write_q4_kernel(const Q4IoParams p) {
    using L = Q4Layout<D>;
    griddep_wait();
    griddep_launch();
    const uint32_t flat = blockIdx.x * kQ4RowsPerCta + (threadIdx.x >> 2);
    const int i = threadIdx.x & 3;
    const bool in_range = flat < p.total;
    const Q4Row r = q4_row(p, in_range ? flat : 0);
    int off = 0;
    uint8_t* chunk = in_range && r.token < p.n ? q4_chunk<D>(p, r, &off) : nullptr;
    const unsigned peers = 0xfu << (threadIdx.x & 28);  // the row's four threads go together
    if (!chunk) return;
    const T* src = reinterpret_cast<const T*>(r.kv ? p.v_in : p.k_in) + q4_offset(p, r) + 8 * i;
    __align__(16) T x[L::NG][16];
#pragma unroll
    for (int w = 0; w < L::NG; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (VEC) {
                const uint4* s4 = reinterpret_cast<const uint4*>(src + 64 * w + 32 * h);
#pragma unroll
                for (int c = 0; c < (int)sizeof(T) / 2; ++c) reinterpret_cast<uint4*>(x[w] + 8 * h)[c] = __ldcg(s4 + c);
            } else {
#pragma unroll
                for (int c = 0; c < 8; ++c) x[w][8 * h + c] = src[64 * w + 32 * h + c];
            }
        }
    uint32_t word[2][L::NG];
#pragma unroll
    for (int w = 0; w < L::NG; ++w) {
        const float2 range = group_range<T>(x[w], peers);
        const bool nan = range.x != range.x;
        // of zeros of both signs, +0
        const float lo = __fadd_rn(fminf(fmaxf(range.x, -65504.f), 65504.f), 0.f);
        const float hi = fminf(fmaxf(range.y, -65504.f), 65504.f);
        // The values saturate as the range does: where fp16(lo) rounds up near 65504, a larger value is not 15 steps
        // away.  16-bit types step so far there that it always is, and below -65504 the code is 0 either way.
        if constexpr (sizeof(T) == 4) {
            if (range.y > 65504.f) {
#pragma unroll
                for (int c = 0; c < 16; ++c) x[w][c] = fminf(x[w][c], 65504.f);
            }
        }
        const __half zero_h = nan ? __ushort_as_half(0x7fff) : __float2half_rn(lo);
        const __half scale_h = nan ? __float2half_rn(0.f)
                                   : __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
        const float zero = __half2float(zero_h), scale = __half2float(scale_h);
        // t = (x - zero) / (15 scale), saturated to [0, 1] (NaN -> 0), then 15 t rounded to an integer
        // by adding 2^23 + 2^22.  The approximate reciprocal (2^-23) and the product that x - zero is folded
        // into put 15 t off by at most 5.4e-6 + 2^-24 |zero| / scale; where it lands within that (and a
        // margin) of a border the code is decided by exact remainders.
        constexpr float kMagic = 12582912.f;
        const float inv = scale > 0.f ? __fdividef(1.f, scale) : 0.f, inv15 = inv * (1.0f / 15.0f), shift = -zero * inv15;
        const float near = 0.5f - (8e-6f + 2.4e-7f * fabsf(zero) * inv);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float code[8], worst = 0.f;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const float t = __saturatef(__fmaf_rn(q4_to_float<T>(x[w][8 * h + c]), inv15, shift));
                code[c] = __fmaf_rn(t, 15.f, kMagic) - kMagic;
                worst = fmaxf(worst, fabsf(__fmaf_rn(t, 15.f, -code[c])));
            }
            if (worst > near) {  // about one value in 3000 of a normal fp16 row lies exactly on a border
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const float f = q4_to_float<T>(x[w][8 * h + c]);
                    const float t = __saturatef(__fmaf_rn(f, inv15, shift));
                    if (fabsf(__fmaf_rn(t, 15.f, -code[c])) > near)
                        code[c] = q4_exact_code(__fsub_rn(f, zero), scale, inv15);
                }
            }
            // four codes to an exact 16-bit integer in fp32, two of those to a word
            float half_word[2];
#pragma unroll
            for (int k = 0; k < 2; ++k)
                half_word[k] = __fmaf_rn(__fmaf_rn(__fmaf_rn(code[4 * k + 3], 16.f, code[4 * k + 2]), 16.f, code[4 * k + 1]),
                                         16.f, code[4 * k]) + kMagic;
            word[h][w] = __byte_perm(__float_as_uint(half_word[0]), __float_as_uint(half_word[1]), 0x5410);
        }
        if (i == w)  // one thread of the row writes each group's parameters
            *reinterpret_cast<__half2*>(chunk + L::PARAMS + w * 64 + off * 4) = __halves2half2(scale_h, zero_h);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint8_t* dst = chunk + off * L::ROW + (i + 4 * h) * 4 * L::NG;
        if constexpr (L::NG == 2) *reinterpret_cast<uint2*>(dst) = make_uint2(word[h][0], word[h][1]);
        else *reinterpret_cast<uint32_t*>(dst) = word[h][0];
    }
}

// Bound by HBM: 501 tokens of 28 layers 13.9 us to fp16 (5.3 TB/s), 13.6 to bf16, 35 to fp32 (3.7 TB/s: 64-byte
// pieces of rows), 1000 tokens 26.3 to fp16 (5.6 TB/s; 8 heads, D = 128, pools from HBM).
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kQ4Threads) kv_read_q4_kernel(const Q4IoParams p) {
    using L = Q4Layout<D>;
    griddep_wait();
    griddep_launch();
    const uint32_t flat = blockIdx.x * kQ4RowsPerCta + (threadIdx.x >> 2);
    const int i = threadIdx.x & 3;
    if (flat >= p.total) return;
    const Q4Row r = q4_row(p, flat);
    if (r.token >= p.n) return;
    int off = 0;
    const uint8_t* chunk = q4_chunk<D>(p, r, &off);
    T* dst = reinterpret_cast<T*>(r.kv ? p.v_out : p.k_out) + q4_offset(p, r) + 8 * i;
    uint32_t word[2][L::NG] = {};
    __half2 prm[L::NG];
#pragma unroll
    for (int w = 0; w < L::NG; ++w) prm[w] = __halves2half2(__float2half(0.f), __float2half(0.f));
    if (chunk) {  // a position outside the pool reads as zeros
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint8_t* src = chunk + off * L::ROW + (i + 4 * h) * 4 * L::NG;
            if constexpr (L::NG == 2) {
                const uint2 u = *reinterpret_cast<const uint2*>(src);
                word[h][0] = u.x;
                word[h][1] = u.y;
            } else {
                word[h][0] = *reinterpret_cast<const uint32_t*>(src);
            }
        }
#pragma unroll
        for (int w = 0; w < L::NG; ++w)
            prm[w] = *reinterpret_cast<const __half2*>(chunk + L::PARAMS + w * 64 + off * 4);
    }
#pragma unroll
    for (int w = 0; w < L::NG; ++w)
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2) {
            const uint32_t wd = word[h2][w];
            __align__(16) T y[8];
            if constexpr (std::is_same<T, __half>::value) {
                // 1024 + code and 1024 + 16 code are fp16 numbers with the nibble in their low bits; code *
                // scale + zero is then one rounding of the exact value
                const __half2 scale = __low2half2(prm[w]), zero = __high2half2(prm[w]);
                const __half2 k1024 = __floats2half2_rn(1024.f, 1024.f), k16 = __floats2half2_rn(0.0625f, 0.0625f),
                              k64 = __floats2half2_rn(-64.f, -64.f), k65504 = __floats2half2_rn(65504.f, 65504.f);
                uint32_t v[4];  // channels (0, 4), (1, 5), (2, 6), (3, 7)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t u = wd >> (8 * h);
                    const uint32_t a = (u & 0x000f000fu) | 0x64006400u, b = (u & 0x00f000f0u) | 0x64006400u;
                    const __half2 ca = __hsub2(*reinterpret_cast<const __half2*>(&a), k1024);
                    const __half2 cb = __hfma2(*reinterpret_cast<const __half2*>(&b), k16, k64);
                    const __half2 va = __hmin2_nan(__hfma2(ca, scale, zero), k65504);
                    const __half2 vb = __hmin2_nan(__hfma2(cb, scale, zero), k65504);
                    v[2 * h] = *reinterpret_cast<const uint32_t*>(&va);
                    v[2 * h + 1] = *reinterpret_cast<const uint32_t*>(&vb);
                }
                *reinterpret_cast<uint4*>(y) = make_uint4(__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410),
                                                          __byte_perm(v[0], v[1], 0x7632), __byte_perm(v[2], v[3], 0x7632));
            } else {
                const float scale = __low2float(prm[w]), zero = __high2float(prm[w]);
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    y[c] = q4_from_float<T>(__fmaf_rn((float)((wd >> (4 * c)) & 15u), scale, zero));
            }
            T* to = dst + 64 * w + 32 * h2;
            if constexpr (VEC) {
#pragma unroll
                for (int c = 0; c < (int)sizeof(T) / 2; ++c)
                    reinterpret_cast<uint4*>(to)[c] = reinterpret_cast<const uint4*>(y)[c];
            } else {
#pragma unroll
                for (int c = 0; c < 8; ++c) to[c] = y[c];
            }
        }
}

// 16-byte accesses: the base and every stride must keep rows 16-byte aligned
inline bool q4_vec_ok(const void* k, const void* v, const int* ks, const int* vs, int elem) {
    if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) return false;
    for (int s = 0; s < 3; ++s)
        if (((unsigned)ks[s] * elem) & 15 || ((unsigned)vs[s] * elem) & 15) return false;
    return true;
}

template <typename T, int D, bool WRITE>
inline int launch_q4_io(const Q4IoParams& p, cudaStream_t st) {
    const bool vec = q4_vec_ok(WRITE ? p.k_in : p.k_out, WRITE ? p.v_in : p.v_out, p.ks, p.vs, (int)sizeof(T));
    const dim3 grid((p.total + kQ4RowsPerCta - 1) / kQ4RowsPerCta), block(kQ4Threads);
    if constexpr (WRITE) {
        if (vec) QTTS_LAUNCH((kv_write_q4_kernel<T, D, true>), grid, block, 0, st, p);
        else QTTS_LAUNCH((kv_write_q4_kernel<T, D, false>), grid, block, 0, st, p);
    } else {
        if (vec) QTTS_LAUNCH((kv_read_q4_kernel<T, D, true>), grid, block, 0, st, p);
        else QTTS_LAUNCH((kv_read_q4_kernel<T, D, false>), grid, block, 0, st, p);
    }
    return QTTS_OK;
}

template <bool WRITE>
inline int run_q4_io(Q4IoParams p, int layers, int head_dim, int dtype, cudaStream_t st) {
    const long long per_token = (long long)layers * 2 * p.kv_heads;
    QTTS_REQUIRE(per_token <= (1 << 20), "q4 cache: %lld rows per token", per_token);
    const long long block_bytes = (long long)p.num_layers * 2 * p.kv_heads * 9 * head_dim;
    QTTS_REQUIRE(block_bytes < (1ll << 31), "q4 cache: %lld bytes per block", block_bytes);
    p.block_bytes = (uint32_t)block_bytes;
    p.rows = make_fastdiv((uint32_t)per_token);
    p.heads = make_fastdiv((uint32_t)p.kv_heads);
    // row numbers stay below 2^31: longer inputs go in several launches
    const int step = (int)(((1ll << 30) / per_token) & ~15ll);
    const int n = p.n, elem = dtype == QTTS_F32 ? 4 : 2;
    for (int t0 = 0; t0 < n; t0 += step) {
        Q4IoParams c = p;
        c.n = n - t0 < step ? n - t0 : step;
        c.total = (uint32_t)((c.n + 15) / 16 * 16 * per_token);
        if (c.mapping) c.mapping += t0;
        if (c.blocks) c.blocks += t0 / 16;
        const long long ko = (long long)t0 * p.ks[0] * elem, vo = (long long)t0 * p.vs[0] * elem;
        if (WRITE) {
            c.k_in = (const char*)p.k_in + ko;
            c.v_in = (const char*)p.v_in + vo;
        } else {
            c.k_out = (char*)p.k_out + ko;
            c.v_out = (char*)p.v_out + vo;
        }
        int rc = QTTS_OK;
        if (dtype == QTTS_F16) rc = head_dim == 128 ? launch_q4_io<__half, 128, WRITE>(c, st) : launch_q4_io<__half, 64, WRITE>(c, st);
        else if (dtype == QTTS_BF16) rc = head_dim == 128 ? launch_q4_io<__nv_bfloat16, 128, WRITE>(c, st) : launch_q4_io<__nv_bfloat16, 64, WRITE>(c, st);
        else rc = head_dim == 128 ? launch_q4_io<float, 128, WRITE>(c, st) : launch_q4_io<float, 64, WRITE>(c, st);
        if (rc) return rc;
    }
    return QTTS_OK;
}

}  // namespace qtts
