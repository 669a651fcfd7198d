// A key/value cache in 8 bits (sm_100a): what its kernels and their launches share.
//
// A page holds, per key/value head, `page` rows of e4m3 codes for the keys (ldk bytes each, the head size rounded up to 16, zeros behind it)
// and likewise for the values (ldv).  Sixteen positions that follow one another are a block: one scale per block and head, keys and values
// each their own.  A scale is a power of two, so that a value is its code times an exact factor, and a scale that grows while its block
// fills shifts the codes already there instead of rounding them anew (only those that fall below the smallest normal code lose bits).
// A negative scale marks a block that holds a NaN: its magnitude is the scale, and attention then looks at the codes themselves.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace smol {
namespace c8 {

constexpr int kBlock = 16;                       // positions of a scale
constexpr int kLeastExp = -110, kMostExp = 92;   // exponents of a scale: a code times a scale is a normal fp32 number
constexpr float kMostValue = 1.2676506e30f;      // 2^100: magnitudes above are clamped
constexpr int kMaxDim = 256;
constexpr int kMaxPairs = 128;
constexpr int kPositions = 0x7fffffff - 127;     // positions are below this: a step of 128 rounded up from there is still an int

struct Cache {
    uint8_t *k, *v;                  // codes: page * k_page + (head * page_size + position) * ldk + coordinate
    float *ks, *vs;                  // scales: page * ks_page + head * (page_size / 16) + block
    size_t k_page, v_page;           // bytes from a page to the next
    size_t ks_page, vs_page;         // floats from a page to the next
    int n_pages, page, G, d, dv, ldk, ldv;
    int32_t* err;                    // set where a block table names a page outside the pool
};

// rows start[s] .. start[s + 1] - 1 are sequence s's next positions, from pos0[s] on
struct Batch {
    const int32_t *start, *pos0, *table;
    const int32_t* kv_len;           // attention: keys of the sequence (nullptr: up to the row's own position)
    int S, T, max_pages, max_new, max_len;
};
// Sequence s as the arrays have it, which are looked at here before anything is made of them: rows that lie in the step, positions that are numbers.  Otherwise it has
// no rows, and the batch's error is reported.
struct Sequence {
    int t0, n, pos0;
    __device__ __forceinline__ Sequence(const Batch& b, int s, int32_t* err) : t0(b.start[s]), pos0(b.pos0[s]) {
        const int t1 = b.start[s + 1];
        const bool fits = t0 >= 0 && t1 >= t0 && t1 <= b.T && pos0 <= kPositions - (t1 - t0);
        n = fits ? t1 - t0 : 0;
        if (!fits && threadIdx.x == 0) atomicExch(err, 2);
    }
};

struct AppendArgs {
    Cache c;
    Batch b;
    const void *k, *v, *q;
    void* q_out;
    size_t k_row, k_head, v_row, v_head, q_row, q_head, o_row, o_head;      // strides in elements
    int H;                           // query heads (0: none)
    const float* freq;
    int pairs, half;
    float mult;
    int k_vec, v_vec, q_vec;         // rows are whole groups of eight elements, on 16-byte boundaries
};

struct AttendArgs {
    Cache c;
    Batch b;
    const void* q;
    void* out;
    size_t q_row, q_head, o_row, o_head;
    int H, window, first;
    float scale, softcap;
    const float *sink, *slope, *r1, *r2;
    const float* gate;               // [T] rows of gate_row floats: the result is multiplied by sigmoid(gate[t][h * dv + c]) (nullptr: not)
    size_t gate_row;
    float out_scale;
    float* part;                     // shares of the keys: unnormalised results [T * H][n_splits][dv rounded up to 4], then (maximum, denominator, e of the results, which are in units of 2^(maximum + e), -) [T * H][n_splits]
    int n_splits;
    int q_vec, o_vec;                // rows are whole groups of four elements that a load takes (1), of eight on 16-byte boundaries (2)
    int held;                        // positions that a row of the block table names
    int rows_over, rows_most;        // only sequences of more than rows_over and at most rows_most query rows per key/value head
};

constexpr int kMaxSplits = 128;
__host__ __device__ inline size_t part_floats(const AttendArgs& A, int splits) { return (size_t)A.b.T * A.H * splits * ((A.c.dv + 3) / 4 * 4); }
__device__ __forceinline__ float4* part_stats(const AttendArgs& A) { return reinterpret_cast<float4*>(A.part + part_floats(A, A.n_splits)); }

// what a score goes through in either attention kernel is the plain scaled product
inline bool plain_scores(const AttendArgs& A) { return A.softcap == 0.0f && !A.slope && !A.r1; }

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3), hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}
__device__ __forceinline__ float4 from_e4m3x4(uint32_t w) {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3), b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    const float2 x = __half22float2(__half2(a)), y = __half22float2(__half2(b));
    return make_float4(x.x, x.y, y.x, y.y);
}
// Codes as f16 times 2^-8: sign, exponent and mantissa move to their places, the difference of the exponents' biases stays behind (exact, codes
// below the smallest normal one included).  The NaN code comes out as 480.
// bytes 1 and 3 of w
__device__ __forceinline__ uint32_t odd_codes(uint32_t w) { return (w & 0x80008000u) | ((w >> 1) & 0x3f803f80u); }
// bytes 0 and 2 of w
__device__ __forceinline__ uint32_t even_codes(uint32_t w) { return ((w << 8) & 0x80008000u) | ((w << 7) & 0x3f803f80u); }
constexpr float kCodeUnit = 256.0f;

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float log2_fast(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// log2 of a scale, a normal number above 0: its exponent, exactly.  (A scale that is no power of two, which only a caller who makes scales can bring, takes the function.)
__device__ __forceinline__ float scale_log2(float s) {
    const uint32_t bits = __float_as_uint(s);
    if ((bits & 0x7fffffu) != 0) return log2f(s);
    return __uint_as_float(0x4b000000u | bits >> 23) - (8388608.0f + 127.0f);      // (2^23 and the exponent: fewer instructions than a conversion)
}

// Launches on `st`; 0 or a CUDA error.  `launches` counts them.
cudaError_t append(const AppendArgs& A, bool f32, int n_sms, int* launches, cudaStream_t st);
// Bytes of workspace attend needs for these sizes, and the most it needs for results of dv columns on any device of up to 256 SMs.
size_t attend_bytes(const AttendArgs& A, bool f32, int n_sms);
size_t attend_bytes_most(int dv);
cudaError_t attend(AttendArgs A, bool f32, int n_sms, void* workspace, int* launches, cudaStream_t st);
// What a caller that fills the structs itself leaves to be worked out: whether rows are whole, aligned pieces; the positions that a block table's row names.
void note_alignment(AppendArgs& A, bool f32);
void note_alignment(AttendArgs& A, bool f32);

constexpr float kLog2e = 1.4426950408889634f;

}  // namespace c8
}  // namespace smol
