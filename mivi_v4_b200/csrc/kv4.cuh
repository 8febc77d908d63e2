// A cache whose rows are held in 4 bits: the layout, and the arithmetic between a row and what is held of it.
//
// A row is one token's key or value of one kv head, x of hd elements.  It is held as hd codes of 4 bits and two bfloat16 numbers:
//     zero = bf16(min x), step = bf16(max(0, max x - zero) / 15), code = clamp(rint((x - zero) / step), 0, 15) (0 if step is 0)
// and stands for zero + step * code.  A row with an element that is not finite has step = zero = NaN and stands for NaN throughout.
// Both numbers are bfloat16: its range is the one of the rows (half precision's is not), and its 8 bits cost little, because the
// codes are worked out against the rounded numbers: the largest element may miss its code by 15 * 2^-8 steps, the smallest by 2^-8
// of its own size, as it would in a bfloat16 cache.
//
// Of one kv head in one page (P rows) the pool holds P * (hd + 8) bytes in one piece, so that a copy of it is one run of memory:
//     keys' codes [P][hd / 2], values' codes [P][hd / 2], then (key step, key zero, value step, value zero) [P][4] bfloat16;
// element d of a row lies in byte d / 2, the even one in the low four bits.
#pragma once
#include "common.cuh"

#define KV4_MAX_HEAD_DIM 256

// bytes of one kv head in one page
__host__ __device__ __forceinline__ size_t kv4_head_bytes(int page_size, int hd) { return (size_t)page_size * (hd + 8); }

struct Kv4Params { float ks, kz, vs, vz; };

__device__ __forceinline__ Kv4Params kv4_params(uint2 r) {
    return {__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y << 16), __uint_as_float(r.y & 0xffff0000u)};
}
// A value row that is not finite makes whoever sees it not finite; so does a key row.  Attention kernels let it in by the score alone,
// where what a query does not see is left out by a select, and take the value as 0: 0 * NaN would reach the queries that do not see it.
__device__ __forceinline__ void kv4_poison(Kv4Params& p) {
    if (!(fabsf(p.vs) < INFINITY)) { p.ks = NAN; p.vs = 0.f; p.vz = 0.f; }
}

// A step as bfloat16: the next lower one where zero + 15 steps would pass the largest float.
__device__ __forceinline__ float kv4_round_step(float exact, float zero) {
    const float step = __bfloat162float(__float2bfloat16_rn(exact));
    return fmaf(15.f, step, zero) == INFINITY ? __uint_as_float(__float_as_uint(step) - 0x10000u) : step;
}
// The step of a row whose largest element is hi, zero being bf16 of its smallest: (hi - zero) times 1 / 15, in 32 bits.  (Halves: the difference
// may pass the largest float.)
__device__ __forceinline__ float kv4_step(float hi, float zero) {
    return kv4_round_step(2.f * (fmaxf(0.5f * hi - 0.5f * zero, 0.f) * (1.f / 15.f)), zero);
}
__device__ __forceinline__ unsigned kv4_code(float x, float zero, float step) {
    if (step <= 0.f) return 0u;
    return (unsigned)fminf(fmaxf(rintf((0.5f * x - 0.5f * zero) / (0.5f * step)), 0.f), 15.f);
}
__device__ __forceinline__ unsigned kv4_pack_params(float step, float zero) {
    return (__float_as_uint(step) >> 16) | (__float_as_uint(zero) & 0xffff0000u);
}
// 8 codes of a word, in order
__device__ __forceinline__ void kv4_unpack8(unsigned w, float step, float zero, float* out) {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = fmaf((float)((w >> (4 * i)) & 15u), step, zero);
}
