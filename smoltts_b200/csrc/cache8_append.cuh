// Appending to the 8-bit key/value cache: position rotation, scales and codes in one pass over the step's rows.  Included by cache8.cu.
//
// One block of threads per (16 positions, sequence, share of the heads).  The cosines and sines of the block's positions are made once, in
// shared memory, for all heads: the angle pos * freq and its remainder in units of half turns in 64 bits (in 32 the angle of position 100000
// is off by 0.004), the rest by sincospif at the nearest float and a first-order step from there.  A warp takes a head's 16 rows into registers, all loads at once: a lane has sixteen coordinates of a row
// that are rotated with one another (eight and the eight they go with, or eight pairs of neighbours), so that nothing is read twice and
// cosines serve both; the largest magnitude, and with it the scale, is known before anything is rounded.
//
// With |x| <= a over the block's new rows the exponent is the smallest E with a <= 448 2^E; a block that an earlier step began keeps the
// larger of its old exponent and this, and its old codes are requantised only where it grows.
//
// What bounds it: the bytes of queries, keys and values.  10671 tokens of 32 query and 8 key/value heads of 128, slices of one projection: 55 us, 4.4 TB/s
// (four coordinates a lane and the four they go with read again: 228); a token of 12 and 4 heads of 64 3.2 us, which is launch and two dependent loads.
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

// Eight elements as they lie in memory, and back.
template <class T> struct Eight;
template <> struct Eight<bf16> {
    uint4 u;
    __device__ __forceinline__ void clear() { u = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ void load(const bf16* p) { u = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void set(const float (&x)[8]) { u = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])); }
    __device__ __forceinline__ void get(float* x) const {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) { x[2 * e] = bf_lo(w[e]); x[2 * e + 1] = bf_hi(w[e]); }
    }
    static __device__ __forceinline__ void put(bf16* p, const float* x) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
    }
};
template <> struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void clear() { a = b = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
    __device__ __forceinline__ void load(const float* p) { a = *reinterpret_cast<const float4*>(p); b = *reinterpret_cast<const float4*>(p + 4); }
    __device__ __forceinline__ void set(const float (&x)[8]) { a = make_float4(x[0], x[1], x[2], x[3]); b = make_float4(x[4], x[5], x[6], x[7]); }
    __device__ __forceinline__ void get(float* x) const {
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
    static __device__ __forceinline__ void put(float* p, const float* x) {
        *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    }
};

__device__ __forceinline__ float max_or_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// A lane's sixteen coordinates of a row: eight from `at`, eight from `to`.
struct Piece {
    int at, to;
    bool turned, apart;      // rotated among themselves; coordinate at + e with to + e rather than neighbours
};
__device__ __forceinline__ Piece piece_of(int piece, int pairs, bool half) {
    // (pairs that are no multiple of eight are rotated element by element, see odd_pairs)
    Piece p;
    p.turned = pairs % 8 == 0 && piece < pairs / 8;
    p.apart = p.turned && half;
    p.at = p.apart ? piece * 8 : piece * 16;
    p.to = p.apart ? p.at + pairs : p.at + 8;
    return p;
}
template <class T>
__device__ __forceinline__ void load_piece(Eight<T> (&x)[2], const T* row, const Piece& p, int width, bool vec) {
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        const int c = z == 0 ? p.at : p.to;
        if (vec) {
            if (c < width) x[z].load(row + c);
            else x[z].clear();
        } else {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = c + e < width ? as_float(row[c + e]) : 0.0f;
            x[z].set(v);
        }
    }
}
// f[0 .. 7] and f[8 .. 15] turned by the row's cosines and sines
__device__ __forceinline__ void turn_piece(float (&f)[16], const Piece& p, const float* cs, const float* sn) {
    if (!p.turned) return;
    const int j = p.apart ? p.at : p.at / 2;      // first pair
#pragma unroll
    for (int e4 = 0; e4 < 2; ++e4) {
        const float4 c4 = *reinterpret_cast<const float4*>(cs + j + 4 * e4), s4 = *reinterpret_cast<const float4*>(sn + j + 4 * e4);
        const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
        auto turn = [](float& x, float& y, float c, float s) {
            const float was = x;
            x = fmaf(x, c, -y * s);
            y = fmaf(y, c, was * s);
        };
        if (p.apart) {
#pragma unroll
            for (int e = 0; e < 4; ++e) turn(f[4 * e4 + e], f[8 + 4 * e4 + e], c[e], s[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) turn(f[8 * e4 + 2 * e], f[8 * e4 + 2 * e + 1], c[e], s[e]);
        }
    }
}
// The same where the pairs are no multiple of eight: coordinates at .. at + 15, the ones they go with read again.
template <class T>
__device__ __noinline__ void odd_pairs(float (&f)[16], const T* row, int at, int pairs, bool half, const float* cs, const float* sn) {
    for (int e = 0; e < 16; ++e) {
        const int i = at + e;
        if (i >= 2 * pairs) break;
        const bool first = half ? i < pairs : i % 2 == 0;
        const int j = half ? (first ? i : i - pairs) : i / 2, o = half ? (first ? i + pairs : i - pairs) : (first ? i + 1 : i - 1);
        const float x = as_float(row[i]), y = as_float(row[o]);
        f[e] = fmaf(x, cs[j], (first ? -y : y) * sn[j]);
    }
}

// PASSES of 16 / PASSES rows, 2 PASSES lanes a row: heads of up to 32 PASSES coordinates.  ODD: pairs that are no multiple of eight
template <class T, int PASSES, bool ODD>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendArgs A) {
    constexpr int LANES = 2 * PASSES, ROWS = 32 / LANES;
    __shared__ __align__(16) float turn[2][kBlock][kMaxPairs + 4];
    dep_wait();
    dep_go();
    const int s = blockIdx.y;
    const Sequence Q(A.b, s, A.c.err);
    const int t0 = Q.t0, n = Q.n, pos0 = Q.pos0, block = pos0 / kBlock + blockIdx.x;
    if (n == 0) return;
    if (pos0 < 0 || n > A.b.max_new) {
        if (threadIdx.x == 0) atomicExch(A.c.err, 2);
        return;
    }
    if (block > (pos0 + n - 1) / kBlock) return;      // (before there is a position: behind the last it may be no number)
    const int p0 = block * kBlock;
    const int lo = max(pos0 - p0, 0), hi = min(pos0 + n - p0, kBlock);      // new rows of the block
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, piece = lane % LANES, sub = lane / LANES;
    const int pg = p0 / A.c.page, page = pg < A.b.max_pages ? A.b.table[(size_t)s * A.b.max_pages + pg] : -1, in_page = p0 - pg * A.c.page;
    for (int i = threadIdx.x; i < (hi - lo) * A.pairs; i += kAppendThreads) {
        const int r = lo + i / A.pairs, j = i % A.pairs;
        const double half_turns = (double)(p0 + r) * (double)A.freq[j] * 0.3183098861837906715;      // the angle over pi
        const double at = half_turns - 2.0 * rint(0.5 * half_turns);
        const float near = (float)at, rest = (float)((at - (double)near) * 3.141592653589793);      // (a rounding of the angle of up to 2^-25 pi is twice that of the cosine)
        float sn, cs;
        sincospif(near, &sn, &cs);
        turn[0][r][j] = fmaf(-sn, rest, cs) * A.mult;
        turn[1][r][j] = fmaf(cs, rest, sn) * A.mult;
    }
    if (A.pairs > 0) __syncthreads();
    const bool held = page >= 0 && page < A.c.n_pages;
    if (!held && threadIdx.x == 0 && blockIdx.z == 0) atomicExch(A.c.err, 1);
    const int units = 2 * A.c.G + A.H, row0 = t0 + p0 - pos0;      // (row0 + r: the step's row of position p0 + r)
    for (int u = blockIdx.z * (kAppendThreads / 32) + warp; u < units; u += gridDim.z * (kAppendThreads / 32)) {
        // keys, values, queries
        const bool key = u < A.c.G, value = !key && u < 2 * A.c.G, query = u >= 2 * A.c.G;
        const int g = key ? u : value ? u - A.c.G : u - 2 * A.c.G, width = value ? A.c.dv : A.c.d;
        const bool vec = key ? A.k_vec : value ? A.v_vec : A.q_vec;
        const T* src = key ? static_cast<const T*>(A.k) + (size_t)g * A.k_head : value ? static_cast<const T*>(A.v) + (size_t)g * A.v_head : static_cast<const T*>(A.q) + (size_t)g * A.q_head;
        const size_t row = key ? A.k_row : value ? A.v_row : A.q_row;
        const Piece p = piece_of(piece, value ? 0 : A.pairs, A.half);
        Eight<T> x[PASSES][2];
#pragma unroll
        for (int y = 0; y < PASSES; ++y) {
            const int r = y * ROWS + sub;
            if (r >= lo && r < hi) load_piece(x[y], src + (size_t)(row0 + r) * row, p, width, vec);
            else { x[y][0].clear(); x[y][1].clear(); }
        }
        if (query) {
#pragma unroll
            for (int y = 0; y < PASSES; ++y) {
                const int r = y * ROWS + sub;
                if (r < lo || r >= hi) continue;
                float f[16];
                x[y][0].get(f);
                x[y][1].get(f + 8);
                if (!ODD) turn_piece(f, p, turn[0][r], turn[1][r]);
                if (ODD) odd_pairs(f, src + (size_t)(row0 + r) * row, p.at, A.pairs, A.half, turn[0][r], turn[1][r]);
                T* to = static_cast<T*>(A.q_out) + (size_t)g * A.o_head + (size_t)(row0 + r) * A.o_row;
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    const int c = z == 0 ? p.at : p.to;
                    if (vec) {
                        if (c < width) Eight<T>::put(to + c, f + 8 * z);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (c + e < width) to[c + e] = as_elem<T>(f[8 * z + e]);
                    }
                }
            }
            continue;
        }
        if (!held) continue;
        float f[PASSES][16], top = 0.0f;
#pragma unroll
        for (int y = 0; y < PASSES; ++y) {
            const int r = y * ROWS + sub;
            x[y][0].get(f[y]);
            x[y][1].get(f[y] + 8);
            if (key) {
                if (!ODD) turn_piece(f[y], p, turn[0][r], turn[1][r]);      // (rows that are not new: zeros whatever they are turned by, once that is cleared below)
                if (ODD && r >= lo && r < hi) odd_pairs(f[y], src + (size_t)(row0 + r) * row, p.at, A.pairs, A.half, turn[0][r], turn[1][r]);
                if (r < lo || r >= hi) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) f[y][e] = 0.0f;
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) top = max_or_nan(top, fabsf(f[y][e]));
        }
        uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));      // (a NaN's are the largest)
        bool nan = false;
        if (bits > __float_as_uint(kMostValue)) {
            // infinities, NaNs, magnitudes beyond what scales are made for
            top = 0.0f;
#pragma unroll
            for (int y = 0; y < PASSES; ++y)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float v = f[y][e];
                    nan |= v != v;
                    f[y][e] = v != v ? v : fminf(fmaxf(v, -kMostValue), kMostValue);
                    top = v != v ? top : fmaxf(top, fabsf(f[y][e]));
                }
            nan = __any_sync(0xffffffffu, nan);
            bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
        }
        // bits: m 2^e, 1 <= m < 2, and 448 = 1.75 2^8
        int E = max((int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), kLeastExp);
        const int ld = key ? A.c.ldk : A.c.ldv;
        float* scale = (key ? A.c.ks + (size_t)page * A.c.ks_page : A.c.vs + (size_t)page * A.c.vs_page) + g * (A.c.page / kBlock) + in_page / kBlock;
        uint8_t* codes = (key ? A.c.k + (size_t)page * A.c.k_page : A.c.v + (size_t)page * A.c.v_page) + ((size_t)g * A.c.page + in_page) * ld;
        if (lo > 0) {
            const float had = *scale;
            const int Eold = min(max((int)((__float_as_uint(had) >> 23) & 0xffu) - 127, kLeastExp), kMostExp);
            nan |= had < 0.0f;
            if (E > Eold) {
                const float down = pow2(max(Eold - E, -126));      // codes are below 2^9: nothing of them is left long before
#pragma unroll 1
                for (int r = sub; r < lo; r += ROWS)
                    if (piece * 16 < ld) {
                        uint4* at = reinterpret_cast<uint4*>(codes + (size_t)r * ld + piece * 16);
                        const uint4 w = *at;
                        auto again = [&](uint32_t c) {
                            const float4 v = from_e4m3x4(c);
                            return to_e4m3x4(v.x * down, v.y * down, v.z * down, v.w * down);
                        };
                        *at = make_uint4(again(w.x), again(w.y), again(w.z), again(w.w));
                    }
            }
            E = max(E, Eold);
            __syncwarp();      // every lane has read the scale
        }
        const float up = pow2(-E);
        if (lane == 0) *scale = nan ? -pow2(E) : pow2(E);
#pragma unroll
        for (int y = 0; y < PASSES; ++y) {
            const int r = y * ROWS + sub;
            if (r < lo || r >= hi) continue;
            uint32_t w[4];
#pragma unroll
            for (int z = 0; z < 4; ++z) w[z] = to_e4m3x4(f[y][4 * z] * up, f[y][4 * z + 1] * up, f[y][4 * z + 2] * up, f[y][4 * z + 3] * up);
            uint8_t* to = codes + (size_t)r * ld;
            if (p.at < ld) *reinterpret_cast<uint2*>(to + p.at) = make_uint2(w[0], w[1]);
            if (p.to < ld) *reinterpret_cast<uint2*>(to + p.to) = make_uint2(w[2], w[3]);
        }
    }
}

}  // namespace c8
}  // namespace smol
