// Appending to the 8-bit key/value cache: position rotation, scales and codes in one pass over the step's rows.  Included by cache8.cu.
//
// One block of threads per (16 positions, sequence, share of the heads).  The cosines and sines of the block's positions are made once, in
// shared memory, for all heads: the angle pos * freq and its remainder in units of half turns in 64 bits (in 32 the angle of position 100000
// is off by 0.004), the rest by sincospif.  A warp takes a head's 16 rows of keys or values into registers -- four coordinates per lane, and the
// four it is rotated with -- finds the largest magnitude, and with it the scale, before it rounds: keys and values are read once.
//
// With |x| <= a over the block's new rows the exponent is the smallest E with a <= 448 2^E; a block that an earlier step began keeps the
// larger of its old exponent and this, and its old codes are requantised only where it grows.
#pragma once

#include "cache8.cuh"

namespace smol {
namespace c8 {

constexpr int kAppendThreads = 256;

template <class T> __device__ __forceinline__ float as_float(T v);
template <> __device__ __forceinline__ float as_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float as_float<bf16>(bf16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T as_elem(float v);
template <> __device__ __forceinline__ float as_elem<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 as_elem<bf16>(float v) { return __float2bfloat16_rn(v); }

// elements c .. c + 3 of a row of n; vec: whole aligned groups of four
__device__ __forceinline__ float4 load_four(const float* p, int c, int n, bool vec) {
    if (vec) return c < n ? *reinterpret_cast<const float4*>(p + c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    return make_float4(c < n ? p[c] : 0.0f, c + 1 < n ? p[c + 1] : 0.0f, c + 2 < n ? p[c + 2] : 0.0f, c + 3 < n ? p[c + 3] : 0.0f);
}
__device__ __forceinline__ float4 load_four(const bf16* p, int c, int n, bool vec) {
    if (vec) {
        const uint2 u = c < n ? *reinterpret_cast<const uint2*>(p + c) : make_uint2(0u, 0u);
        return make_float4(bf_lo(u.x), bf_hi(u.x), bf_lo(u.y), bf_hi(u.y));
    }
    return make_float4(c < n ? as_float(p[c]) : 0.0f, c + 1 < n ? as_float(p[c + 1]) : 0.0f, c + 2 < n ? as_float(p[c + 2]) : 0.0f, c + 3 < n ? as_float(p[c + 3]) : 0.0f);
}
__device__ __forceinline__ void store_four(float* p, int c, int n, bool vec, float4 v) {
    if (vec) {
        if (c < n) *reinterpret_cast<float4*>(p + c) = v;
        return;
    }
    const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (c + e < n) p[c + e] = x[e];
}
__device__ __forceinline__ void store_four(bf16* p, int c, int n, bool vec, float4 v) {
    if (vec) {
        if (c < n) *reinterpret_cast<uint2*>(p + c) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
        return;
    }
    const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (c + e < n) p[c + e] = __float2bfloat16_rn(x[e]);
}

// Elements c .. c + 3 of a row, rotated by the row's cosines and sines where c is among the leading 2 * pairs.
template <class T>
__device__ __forceinline__ float4 load_rotated(const AppendArgs& A, const T* p, int c, bool vec, const float* cs, const float* sn) {
    float4 v = load_four(p, c, A.c.d, vec);
    if (c >= 2 * A.pairs) return v;
    float x[4] = {v.x, v.y, v.z, v.w}, y[4];
    if (A.half) {
        // coordinate i with i + pairs
        float o[4];
        if (A.pairs % 4 == 0) {
            const float4 w = load_four(p, c < A.pairs ? c + A.pairs : c - A.pairs, A.c.d, vec);
            o[0] = w.x; o[1] = w.y; o[2] = w.z; o[3] = w.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = c + e;
                o[e] = i < 2 * A.pairs ? as_float(p[i < A.pairs ? i + A.pairs : i - A.pairs]) : 0.0f;
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = c + e, j = i < A.pairs ? i : i - A.pairs;
            y[e] = i < 2 * A.pairs ? fmaf(x[e], cs[j], (i < A.pairs ? -o[e] : o[e]) * sn[j]) : x[e];
        }
    } else {
        // coordinate 2i with 2i + 1
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = c + e, j = i / 2;
            y[e] = i < 2 * A.pairs ? fmaf(x[e], cs[j], (e % 2 ? x[e ^ 1] : -x[e ^ 1]) * sn[j]) : x[e];
        }
    }
    return make_float4(y[0], y[1], y[2], y[3]);
}

// W: groups of 128 coordinates a head has at most
template <class T, int W>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendArgs A) {
    __shared__ float turn[2][kBlock][kMaxPairs];
    dep_wait();
    dep_go();
    const int s = blockIdx.y, t0 = A.b.start[s], n = A.b.start[s + 1] - t0, pos0 = A.b.pos0[s];
    const int block = pos0 / kBlock + blockIdx.x, p0 = block * kBlock;
    if (n <= 0) return;
    if (pos0 < 0 || t0 < 0 || t0 + n > A.b.T || n > A.b.max_new) {
        if (threadIdx.x == 0) atomicExch(A.c.err, 2);
        return;
    }
    if (p0 >= pos0 + n) return;
    const int lo = max(pos0 - p0, 0), hi = min(pos0 + n - p0, kBlock);      // new rows of the block
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pg = p0 / A.c.page, page = pg < A.b.max_pages ? A.b.table[(size_t)s * A.b.max_pages + pg] : -1, in_page = p0 - pg * A.c.page;
    for (int i = threadIdx.x; i < (hi - lo) * A.pairs; i += kAppendThreads) {
        const int r = lo + i / A.pairs, j = i % A.pairs;
        const double half_turns = (double)(p0 + r) * (double)A.freq[j] * 0.3183098861837906715;      // the angle over pi
        float sn, cs;
        sincospif((float)(half_turns - 2.0 * rint(0.5 * half_turns)), &sn, &cs);
        turn[0][r][j] = cs * A.mult;
        turn[1][r][j] = sn * A.mult;
    }
    if (A.pairs > 0) __syncthreads();
    const bool held = page >= 0 && page < A.c.n_pages;
    if (!held && threadIdx.x == 0 && blockIdx.z == 0) atomicExch(A.c.err, 1);
    const int units = 2 * A.c.G + A.H, row0 = t0 + p0 - pos0;      // (row0 + r: the step's row of position p0 + r)
    for (int u = blockIdx.z * (kAppendThreads / 32) + warp; u < units; u += gridDim.z * (kAppendThreads / 32)) {
        if (u >= 2 * A.c.G) {
            const int h = u - 2 * A.c.G;
            const T* q = static_cast<const T*>(A.q) + (size_t)h * A.q_head;
            T* to = static_cast<T*>(A.q_out) + (size_t)h * A.o_head;
#pragma unroll 4
            for (int r = lo; r < hi; ++r)
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const int c = 4 * lane + 128 * w;
                    if (c < A.c.d)
                        store_four(to + (size_t)(row0 + r) * A.o_row, c, A.c.d, A.q_vec, load_rotated(A, q + (size_t)(row0 + r) * A.q_row, c, A.q_vec, turn[0][r], turn[1][r]));
                }
            continue;
        }
        if (!held) continue;
        const bool key = u < A.c.G;
        const int g = key ? u : u - A.c.G, width = key ? A.c.d : A.c.dv, ld = key ? A.c.ldk : A.c.ldv;
        const bool vec = key ? A.k_vec : A.v_vec;
        const T* src = key ? static_cast<const T*>(A.k) + (size_t)g * A.k_head : static_cast<const T*>(A.v) + (size_t)g * A.v_head;
        const size_t row = key ? A.k_row : A.v_row;
        float x[kBlock][4 * W];
        uint32_t top = 0;
        bool nan = false;
#pragma unroll
        for (int r = 0; r < kBlock; ++r)
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const int c = 4 * lane + 128 * w;
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (r >= lo && r < hi && c < width) {
                    const T* p = src + (size_t)(row0 + r) * row;
                    v = key ? load_rotated(A, p, c, vec, turn[0][r], turn[1][r]) : load_four(p, c, width, vec);
                }
                x[r][4 * w] = v.x; x[r][4 * w + 1] = v.y; x[r][4 * w + 2] = v.z; x[r][4 * w + 3] = v.w;
            }
#pragma unroll
        for (int r = 0; r < kBlock; ++r)
#pragma unroll
            for (int e = 0; e < 4 * W; ++e) {
                const float v = x[r][e];
                nan |= v != v;
                // (a NaN passes fminf and fmaxf as the other operand: it is kept by the selection)
                x[r][e] = v != v ? v : fminf(fmaxf(v, -kMostValue), kMostValue);
                top = max(top, v != v ? 0u : __float_as_uint(fabsf(x[r][e])));
            }
        top = __reduce_max_sync(0xffffffffu, top);
        nan = __any_sync(0xffffffffu, nan);
        // top = m 2^e, 1 <= m < 2, and 448 = 1.75 2^8
        int E = max((int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), kLeastExp);
        float* scale = (key ? A.c.ks + (size_t)page * A.c.ks_page : A.c.vs + (size_t)page * A.c.vs_page) + g * (A.c.page / kBlock) + in_page / kBlock;
        uint8_t* codes = (key ? A.c.k + (size_t)page * A.c.k_page : A.c.v + (size_t)page * A.c.v_page) + ((size_t)g * A.c.page + in_page) * ld;
        if (lo > 0) {
            const float had = *scale;
            const int Eold = min(max((int)((__float_as_uint(had) >> 23) & 0xffu) - 127, kLeastExp), kMostExp);
            nan |= had < 0.0f;
            if (E > Eold) {
                const float down = pow2(max(Eold - E, -126));      // codes are below 2^9: nothing of them is left long before
                for (int r = 0; r < lo; ++r)
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        const int c = 4 * lane + 128 * w;
                        if (c < ld) {
                            uint32_t* at = reinterpret_cast<uint32_t*>(codes + (size_t)r * ld + c);
                            const float4 v = from_e4m3x4(*at);
                            *at = to_e4m3x4(v.x * down, v.y * down, v.z * down, v.w * down);
                        }
                    }
            }
            E = max(E, Eold);
            __syncwarp();      // every lane has read the scale
        }
        const float up = pow2(-E);
        if (lane == 0) *scale = nan ? -pow2(E) : pow2(E);
#pragma unroll
        for (int r = 0; r < kBlock; ++r)
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const int c = 4 * lane + 128 * w;
                if (r >= lo && r < hi && c < ld)
                    *reinterpret_cast<uint32_t*>(codes + (size_t)r * ld + c) = to_e4m3x4(x[r][4 * w] * up, x[r][4 * w + 1] * up, x[r][4 * w + 2] * up, x[r][4 * w + 3] * up);
            }
    }
}

}  // namespace c8
}  // namespace smol
