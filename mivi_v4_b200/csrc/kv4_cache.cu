// The 4-bit cache (kv4.cuh): rows quantised as they are written, rows and pages read back, and attention over it for every head
// size and dtype.
//
// Formulas of the preparation and of attention as in attention.cu and attention_decode.cu (reference:
// crates/mivi-model/src/transformer.rs:81-110, 114-167, 293-298; rotation crates/mivi-core/src/rope.rs:59-61, 219-229).
#include "kv4.cuh"

MV_GUARD_SETTER(kv4_cache)

// ------------------------------------------------- q/k norm, rotation, quantised append
// Block = one token: nh query heads, then nkv key heads, then nkv value heads, as they lie in a row of the fused projection.  A head's row
// lies in LPH lanes, four neighbouring elements each (CH times), so a warp takes 32 / LPH heads of a kind a round; its rows are asked for
// before the token's angles are worked out.  The projection's rows, 4 bytes an element, are what cannot be avoided; the rest is
// instructions, kept few: angles once a block, weights and turns of a lane's elements once a warp, quotients as products (below).
//
// Keys are worked out in 64 bits, from the sum of squares to the code: a code is a decision, and 32 bits move one in a million of them to the
// other side of its border (by a step, 0.3 of the row's mean square).  A key then stands in the cache as the formulas say, whatever the
// order of a sum.  The angle takes 64 bits anyway: a product of 32 bits is off by 2^-25 of it, a thousandth at position 32,768.  Queries,
// which are rounded to the model's dtype and decide nothing, take 32 bits from there; values are used as they come.
//
// Measured, 32 / 8 heads of 64: 8 tokens 3.9 us; 2,048 tokens 13.9 us, 34.7 MB in and out at 2.5 TB/s; 4,373 of 24 / 8 heads, pairs half a row
// apart, 28 us.  (A cache in bfloat16 is written in 2.3, 9.2 and 56 us.)  What bounds it is instructions: some 215 for two heads' rows, issued
// in 0.68 of the clocks.
constexpr int KP_ROUNDS = 4;

// Sine and cosine of the angle a in 64 bits: a less the nearest multiple of a quarter turn, then their series.  Within pi / 4 the first terms left
// out are x^17 / 17! and x^18 / 18!, below 2^-54.  (Off by 2^-52 of a on top, that is by the quarter turn's own last place times their
// number.)
__device__ __forceinline__ double2 kv4_turn(double a) {
    const double k = rint(a * 0.6366197723675814);               // 2 / pi
    const double x = fma(k, -1.5707963267948966, a), z = x * x;
    double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;
    s = fma(s, z, 1.0 / 6227020800.0);
    c = fma(c, z, -1.0 / 87178291200.0);
    s = fma(s, z, -1.0 / 39916800.0);
    c = fma(c, z, 1.0 / 479001600.0);
    s = fma(s, z, 1.0 / 362880.0);
    c = fma(c, z, -1.0 / 3628800.0);
    s = fma(s, z, -1.0 / 5040.0);
    c = fma(c, z, 1.0 / 40320.0);
    s = fma(s, z, 1.0 / 120.0);
    c = fma(c, z, -1.0 / 720.0);
    s = fma(s, z, -1.0 / 6.0);
    c = fma(c, z, 1.0 / 24.0);
    s = fma(s * z, x, x);
    c = fma(fma(c, z, -0.5), z, 1.0);
    const int quarter = (int)((long long)k & 3);
    const double cc = quarter & 1 ? s : c, ss = quarter & 1 ? c : s;
    return make_double2(quarter == 1 || quarter == 2 ? -cc : cc, quarter & 2 ? -ss : ss);
}
// 1 / sqrt(x) and 1 / x in 64 bits by Newton's steps from 32-bit ones (each doubles the places); x in the normal range of 32 bits, or the
// 32-bit value is kept (0, infinity, not a number).
__device__ __forceinline__ double kv4_rsqrt(double x) {
    const float f = rsqrtf((float)x);
    double r = (double)f;
    if (!(f > 1e-18f && f < 1e18f)) return r;
    r = r * fma(-0.5 * x * r, r, 1.5);
    return r * fma(-0.5 * x * r, r, 1.5);
}
__device__ __forceinline__ double kv4_inverse(float x) {
    double r = (double)(1.0f / x);
    if (!(x > 1e-37f && x < 1e37f)) return 1.0 / (double)x;
    return r * fma(-(double)x, r, 2.0);
}

template <int LPH, int CH, typename T>
__global__ void __launch_bounds__(256, CH == 1 ? 4 : 2)
kv4_prepare_kernel(const float* __restrict__ qkv, const float* __restrict__ wq, const float* __restrict__ wk, float eps,
                   const float* __restrict__ inv_freq, int half_split, const int* __restrict__ positions,
                   const int* __restrict__ seq_of, const int* __restrict__ page_table, int table_stride, int page_shift,
                   unsigned char* __restrict__ pool, T* __restrict__ q_out, int nh, int nkv, int hd, double per_hd) {
    mv_pdl_begin();
    __shared__ double2 turn[KV4_MAX_HEAD_DIM / 2];               // cosine and sine of the token's angles
    __shared__ float2 turn32[KV4_MAX_HEAD_DIM / 2];
    constexpr int HPW = 32 / LPH;
    const int n = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & (LPH - 1), hsel = lane / LPH;
    const int warps = blockDim.x >> 5, slots = nh + 2 * nkv, half = hd >> 1, chunks = hd >> 2, shift = half >> 2;
    // rounds of one kind of head each; a warp's first: of queries its own number, of keys too, of values the next free warps'
    const int rq = (nh + HPW - 1) / HPW, rk = (nkv + HPW - 1) / HPW;
    const int first_v = (warp + warps - rk % warps) % warps;
    const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
    const float* rows = qkv + (size_t)n * slots * hd;
    auto load = [&](float4 (&to)[CH], int slot0, int h, int count) {        // head h of ``count`` that begin at slot0
#pragma unroll
        for (int c = 0; c < CH; ++c)
            to[c] = h < count && sub + LPH * c < chunks ? *reinterpret_cast<const float4*>(rows + (size_t)(slot0 + h) * hd + 4 * (sub + LPH * c)) : none;
    };
    float4 qx[KP_ROUNDS][CH], kx[CH], vx[CH];
#pragma unroll
    for (int u = 0; u < KP_ROUNDS; ++u) load(qx[u], 0, (warp + u * warps) * HPW + hsel, nh);
    load(kx, nh, warp * HPW + hsel, nkv);
    load(vx, nh + nkv, first_v * HPW + hsel, nkv);
    const int pos = positions[n];
    const int page = page_table[(size_t)seq_of[n] * table_stride + (pos >> page_shift)];
    if (inv_freq)
        for (int i = threadIdx.x; i < half; i += blockDim.x) {
            const double2 d = kv4_turn((double)pos * (double)inv_freq[i]);
            turn[i] = d;
            turn32[i] = make_float2((float)d.x, (float)d.y);
        }
    __syncthreads();
    const int page_size = 1 << page_shift, at = pos & (page_size - 1);
    const bool writes = mv_page_ok(page);
    unsigned char* const where = pool + (size_t)(writes ? page : 0) * nkv * kv4_head_bytes(page_size, hd);
    // which angle an element turns by, and whether it is its pair's first: pairs (2i, 2i + 1), or (i, i + half) with the other one in
    // the chunk ``shift`` on or back
    auto angle_of = [&](int c, int e) {
        const int i = min(sub + LPH * c, chunks - 1);
        return half_split ? 4 * (i < shift ? i : i - shift) + e : 2 * i + (e >> 1);
    };
    auto partner = [&](auto here, auto there, int c) {           // element of the pair's other chunk: in array 0 or array CH - 1
        const int i = sub + LPH * c, j = i < shift ? i + shift : i - shift, from = (lane & ~(LPH - 1)) | (j & (LPH - 1));
        const auto a = __shfl_sync(0xffffffffu, here, from);
        const auto b = CH == 2 ? __shfl_sync(0xffffffffu, there, from) : a;
        return CH == 2 && j / LPH != 0 ? b : a;
    };
    auto rotate = [&](auto (&y)[CH][4], const auto (&cs)[CH][4], const auto (&sn)[CH][4]) {
        if (!half_split) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const auto a = y[c][e], b = y[c][e + 1];
                    y[c][e] = a * cs[c][e] - b * sn[c][e];
                    y[c][e + 1] = a * sn[c][e] + b * cs[c][e];
                }
        } else {
            auto z = y[0][0];
            decltype(z) w[CH][4];
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) w[c][e] = partner(y[0][e], y[CH - 1][e], c);
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const auto s = sub + LPH * c < shift ? -sn[c][e] : sn[c][e];
                    y[c][e] = w[c][e] * s + y[c][e] * cs[c][e];
                }
        }
    };
    {   // ---- queries
        float w[CH][4], cs[CH][4], sn[CH][4];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            float4 f = make_float4(1.f, 1.f, 1.f, 1.f);
            if (wq && sub + LPH * c < chunks) f = *reinterpret_cast<const float4*>(wq + 4 * (sub + LPH * c));
            w[c][0] = f.x; w[c][1] = f.y; w[c][2] = f.z; w[c][3] = f.w;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 d = inv_freq ? turn32[angle_of(c, e)] : make_float2(1.f, 0.f);
                cs[c][e] = d.x;
                sn[c][e] = d.y;
            }
        }
        for (int r0 = warp; r0 < rq; r0 += KP_ROUNDS * warps) {
            if (r0 != warp)
#pragma unroll
                for (int u = 0; u < KP_ROUNDS; ++u) load(qx[u], 0, (r0 + u * warps) * HPW + hsel, nh);
#pragma unroll
            for (int u = 0; u < KP_ROUNDS; ++u) {
                const int h = (r0 + u * warps) * HPW + hsel;
                if (r0 + u * warps >= rq) break;
                float y[CH][4];
#pragma unroll
                for (int c = 0; c < CH; ++c) { y[c][0] = qx[u][c].x; y[c][1] = qx[u][c].y; y[c][2] = qx[u][c].z; y[c][3] = qx[u][c].w; }
                if (wq) {
                    float ss = 0.f;
#pragma unroll
                    for (int c = 0; c < CH; ++c)
#pragma unroll
                        for (int e = 0; e < 4; ++e) ss = fmaf(y[c][e], y[c][e], ss);
#pragma unroll
                    for (int o = LPH >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    const float m = fmaf(ss, (float)per_hd, eps);
                    float scale = rsqrtf(m);
                    if (scale > 1e-18f && scale < 1e18f) scale = scale * fmaf(-0.5f * m * scale, scale, 1.5f);
#pragma unroll
                    for (int c = 0; c < CH; ++c)
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[c][e] = y[c][e] * scale * w[c][e];
                }
                if (inv_freq) rotate(y, cs, sn);
#pragma unroll
                for (int c = 0; c < CH; ++c)
                    if (h < nh && sub + LPH * c < chunks)
                        mv_store4(q_out + ((size_t)n * nh + h) * hd + 4 * (sub + LPH * c), y[c][0], y[c][1], y[c][2], y[c][3]);
            }
        }
    }
    // ---- a row's ends (rounding keeps the order, so a key's may be looked for in 32 bits), its zero and step, and its way to the pool
    auto hold = [&](const float (&x)[CH][4], int kv, int g, auto step_of, auto code_of) {
        float lo = INFINITY, hi = -INFINITY;
        bool fine = true;
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (sub + LPH * c < chunks)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    lo = fminf(lo, x[c][e]);
                    hi = fmaxf(hi, x[c][e]);
                    fine = fine && fabsf(x[c][e]) < INFINITY;
                }
#pragma unroll
        for (int o = LPH >> 1; o > 0; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        const unsigned group = LPH == 32 ? 0xffffffffu : ((1u << (LPH & 31)) - 1u) << (lane & ~(LPH - 1));
        fine = (__ballot_sync(0xffffffffu, fine) & group) == group;
        // (the lowest floats would round to -infinity)
        float zero = fminf(fmaxf(__bfloat162float(__float2bfloat16_rn(lo)), -3.3895313892515355e38f), 3.3895313892515355e38f);
        float step = step_of(hi, zero);
        unsigned code[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) code[c] = 0u;
        if (step > 0.f && fine) code_of(code, zero, step);
        if (!fine) zero = step = NAN;
        if (g < nkv && writes) {
            unsigned char* base = where + (size_t)g * kv4_head_bytes(page_size, hd);
            unsigned char* codes = base + ((size_t)(kv ? page_size : 0) + at) * half;
#pragma unroll
            for (int c = 0; c < CH; ++c)
                if (sub + LPH * c < chunks) *reinterpret_cast<unsigned short*>(codes + 2 * (sub + LPH * c)) = (unsigned short)code[c];
            if (sub == 0)
                *reinterpret_cast<unsigned*>(base + (size_t)page_size * hd + (size_t)at * 8 + 4 * kv) = kv4_pack_params(step, zero);
        }
    };
    // ---- keys, in 64 bits
    for (int r = warp; r < rk; r += warps) {
        if (r != warp) load(kx, nh, r * HPW + hsel, nkv);
        double y[CH][4];
#pragma unroll
        for (int c = 0; c < CH; ++c) { y[c][0] = kx[c].x; y[c][1] = kx[c].y; y[c][2] = kx[c].z; y[c][3] = kx[c].w; }
        if (wk) {
            double ss = 0.0;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) ss = fma(y[c][e], y[c][e], ss);
#pragma unroll
            for (int o = LPH >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const double scale = kv4_rsqrt(fma(ss, per_hd, (double)eps));
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                float4 f = none;
                if (sub + LPH * c < chunks) f = *reinterpret_cast<const float4*>(wk + 4 * (sub + LPH * c));
                y[c][0] *= scale * f.x; y[c][1] *= scale * f.y; y[c][2] *= scale * f.z; y[c][3] *= scale * f.w;
            }
        }
        if (inv_freq) {
            double cs[CH][4], sn[CH][4];
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const double2 d = turn[angle_of(c, e)];
                    cs[c][e] = d.x;
                    sn[c][e] = d.y;
                }
            rotate(y, cs, sn);
        }
        float x[CH][4];
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[c][e] = (float)y[c][e];
        hold(x, 0, r * HPW + hsel, [&](float hi, float zero) {
            // the largest element in 64 bits, among those that are it in 32
            double top = -INFINITY;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (x[c][e] == hi && y[c][e] > top && sub + LPH * c < chunks) top = y[c][e];
#pragma unroll
            for (int o = LPH >> 1; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
            return kv4_round_step((float)(fmax(top - (double)zero, 0.0) * (1.0 / 15.0)), zero);
        }, [&](unsigned (&code)[CH], float zero, float step) {
            const double per_step = kv4_inverse(step), from = (double)zero;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // to the nearest whole number, ties to the even one: it stands in the low bits of a number of 1.5 * 2^52
                    const double t = fma(y[c][e] - from, per_step, 6755399441055744.0);
                    code[c] |= (unsigned)min(max(__double2loint(t), 0), 15) << (4 * e);
                }
        });
    }
    // ---- values.  A quotient (x - zero) / step, rounded to 32 bits and then to a whole number, is a product by 1 / step rounded once, unless it
    // lies next to a border: then it is divided.
    for (int r = first_v; r < rk; r += warps) {
        if (r != first_v) load(vx, nh + nkv, r * HPW + hsel, nkv);
        float x[CH][4];
#pragma unroll
        for (int c = 0; c < CH; ++c) { x[c][0] = vx[c].x; x[c][1] = vx[c].y; x[c][2] = vx[c].z; x[c][3] = vx[c].w; }
        hold(x, 1, r * HPW + hsel, [](float hi, float zero) { return kv4_step(hi, zero); }, [&](unsigned (&code)[CH], float zero, float step) {
            const float per_step = step > 1e-30f && step < 1e30f ? 2.0f / step : 0.f, from = -0.5f * zero;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float t = fmaf(0.5f, x[c][e], from) * per_step, whole = rintf(t);
                    unsigned v = (unsigned)fminf(fmaxf(whole, 0.f), 15.f);
                    if (fabsf(t - whole) > 0.4999f || per_step == 0.f) v = kv4_code(x[c][e], zero, step);
                    code[c] |= v << (4 * e);
                }
        });
    }
}

// qkv float32 [N, (nh + 2 nkv) * hd]; pool [pages, nkv, page_size * (hd + 8)] bytes.  q_out [N, nh * hd] in q_dtype.  Everything on 16 bytes.
struct Kv4PrepareArgs {
    const float *qkv, *wq, *wk, *inv_freq;
    const int *positions, *seq_of, *page_table;
    void *pool, *q_out;
    cudaStream_t stream;
    int half_split, table_stride, page_size, q_dtype, N, nh, nkv, hd;
    float eps;
};
MV_API int mv_kv4_prepare(const void* record) {
    const auto& [qkv, wq, wk, inv_freq, positions, seq_of, page_table, pool, q_out, stream, half_split, table_stride, page_size, q_dtype, N, nh, nkv, hd,
                eps] = *static_cast<const Kv4PrepareArgs*>(record);
    if (N <= 0) return 0;
    if (hd % 8 || hd < 8 || hd > KV4_MAX_HEAD_DIM || page_size < 1 || (page_size & (page_size - 1)) || nkv < 1 ||
        (((uintptr_t)qkv | (uintptr_t)wq | (uintptr_t)wk | (uintptr_t)q_out | (uintptr_t)pool) & 15))
        return (int)cudaErrorInvalidValue;
    int page_shift = 0;
    while ((1 << page_shift) < page_size) ++page_shift;
    // Few tokens: a warp a round, for the least latency; many: four warps a token, which share its angles.
    const int lph = hd <= 32 ? 8 : hd <= 64 ? 16 : 32, hpw = 32 / lph;
    const int rounds = (nh + hpw - 1) / hpw + 2 * ((nkv + hpw - 1) / hpw);
    const int warps = N >= 296 ? (rounds < 4 ? rounds : 4) : (rounds < 8 ? rounds : 8);
#define MV_GO(LPH, CH, T)                                                                                                                  \
    mv_launch(kv4_prepare_kernel<LPH, CH, T>, dim3(N), 32 * warps, 0, stream, qkv, wq, wk, eps, inv_freq, half_split, positions, seq_of,   \
              page_table, table_stride, page_shift, (unsigned char*)pool, (T*)q_out, nh, nkv, hd, 1.0 / hd)
#define MV_HD(T)                                                                                                                           \
    do {                                                                                                                                   \
        if (hd <= 32) MV_GO(8, 1, T);                                                                                                      \
        else if (hd <= 64) MV_GO(16, 1, T);                                                                                                \
        else if (hd <= 128) MV_GO(32, 1, T);                                                                                               \
        else MV_GO(32, 2, T);                                                                                                              \
    } while (0)
    if (q_dtype == MV_DT_BF16) MV_HD(__nv_bfloat16);
    else MV_HD(float);
#undef MV_HD
#undef MV_GO
    return mv_launch_status();
}

// ------------------------------------------------------------------ reading back
// One thread per 8 codes of a row: a word of codes and the row's two numbers in, 8 elements out.  The launch and three loads that wait for one
// another (position, page, codes) are most of it: 8 rows of 8 kv heads of 64 take 1.7 us, 2,048 rows 3.5 us, 4,373 rows 5.5 us (11.5 MB in and out).
template <typename T>
__device__ __forceinline__ void kv4_store8(T* dst, const float* v) {
    mv_store4(dst, v[0], v[1], v[2], v[3]);
    mv_store4(dst + 4, v[4], v[5], v[6], v[7]);
}

template <typename T>
__global__ void __launch_bounds__(256)
kv4_read_kernel(const unsigned char* __restrict__ pool, const int* __restrict__ page_table, int table_stride, int page_shift,
                const int* __restrict__ positions, const int* __restrict__ seq_of, T* __restrict__ k_out, T* __restrict__ v_out, int N,
                int nkv, int hd) {
    mv_pdl_begin();
    const int words = hd >> 3;
    const long long id = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (id >= (long long)N * nkv * 2 * words) return;
    const int w = (int)(id % words);
    const long long rowid = id / words;                          // ((n * 2 + K or V) * nkv + g)
    const int g = (int)(rowid % nkv), kv = (int)(rowid / nkv & 1), n = (int)(rowid / nkv >> 1);
    const int pos = positions[n], page_size = 1 << page_shift, at = pos & (page_size - 1);
    const int page = mv_read_page(page_table[(size_t)seq_of[n] * table_stride + (pos >> page_shift)]);
    const unsigned char* base = pool + ((size_t)page * nkv + g) * kv4_head_bytes(page_size, hd);
    const unsigned codes = *reinterpret_cast<const unsigned*>(base + ((size_t)(kv ? page_size : 0) + at) * (hd >> 1) + 4 * w);
    const unsigned pr = *reinterpret_cast<const unsigned*>(base + (size_t)page_size * hd + (size_t)at * 8 + 4 * kv);
    float v[8];
    kv4_unpack8(codes, __uint_as_float(pr << 16), __uint_as_float(pr & 0xffff0000u), v);
    kv4_store8((kv ? v_out : k_out) + ((size_t)n * nkv + g) * hd + 8 * w, v);
}

struct Kv4ReadArgs {
    const void* pool;
    const int *page_table, *positions, *seq_of;
    void *k_out, *v_out;
    cudaStream_t stream;
    int table_stride, page_size, dtype, N, nkv, hd;
};
MV_API int mv_kv4_read(const void* record) {
    const auto& [pool, page_table, positions, seq_of, k_out, v_out, stream, table_stride, page_size, dtype, N, nkv, hd] =
        *static_cast<const Kv4ReadArgs*>(record);
    if (N <= 0) return 0;
    if (hd % 8 || page_size < 1 || (page_size & (page_size - 1))) return (int)cudaErrorInvalidValue;
    int page_shift = 0;
    while ((1 << page_shift) < page_size) ++page_shift;
    const unsigned blocks = (unsigned)(((long long)N * nkv * 2 * (hd >> 3) + 255) / 256);
    if (dtype == MV_DT_BF16)
        mv_launch(kv4_read_kernel<__nv_bfloat16>, dim3(blocks), 256, 0, stream, (const unsigned char*)pool, page_table, table_stride,
                  page_shift, positions, seq_of, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, N, nkv, hd);
    else
        mv_launch(kv4_read_kernel<float>, dim3(blocks), 256, 0, stream, (const unsigned char*)pool, page_table, table_stride, page_shift,
                  positions, seq_of, (float*)k_out, (float*)v_out, N, nkv, hd);
    return mv_launch_status();
}

// The pages that the queries of a step read, one after the other into a pool in the model's dtype, with a page table for it: for the
// attention kernels of many query tokens, which read a key once for hundreds of queries.  Sequence b's queries lie at positions
// starts[b] .. starts[b] + cu[b + 1] - cu[b] - 1; with a window only the pages from its first query's first key on are read, and the
// table's entries before them are 0.  Rows that no query sees come out as zeros, so that nothing of them can reach a product.
// grid (W, nkv, n_seqs): one block a kv head of a page.
template <typename T>
__global__ void __launch_bounds__(256)
kv4_read_pages_kernel(const unsigned char* __restrict__ pool, const int* __restrict__ page_table, int table_stride, int page_shift,
                      const int* __restrict__ cu, const int* __restrict__ starts, int window, T* __restrict__ out,
                      int* __restrict__ out_table, int W, int nkv, int hd) {
    mv_pdl_begin();
    const int i = blockIdx.x, g = blockIdx.y, b = blockIdx.z;
    const int page_size = 1 << page_shift;
    __shared__ int base_of;
    if (threadIdx.x < 32) {                                      // pages that the sequences before b take
        int sum = 0;
        for (int s = threadIdx.x; s < b; s += 32) {
            const int st = starts[s], end = st + cu[s + 1] - cu[s];
            const int first = window > 0 ? max(0, st - window + 1) >> page_shift : 0;
            sum += ((end + page_size - 1) >> page_shift) - first;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (threadIdx.x == 0) base_of = sum;
    }
    __syncthreads();
    const int st = starts[b], end = st + cu[b + 1] - cu[b];
    const int first = window > 0 ? max(0, st - window + 1) : 0, first_page = first >> page_shift;
    const bool live = i >= first_page && (i << page_shift) < end;
    const int dst_page = live ? base_of + i - first_page : 0;
    if (g == 0 && threadIdx.x == 0) out_table[(size_t)b * W + i] = dst_page;
    if (!live) return;
    const int page = mv_read_page(page_table[(size_t)b * table_stride + i]);
    const unsigned char* base = pool + ((size_t)page * nkv + g) * kv4_head_bytes(page_size, hd);
    T* dst = out + ((size_t)dst_page * 2 * nkv + g) * page_size * hd;
    const int words = hd >> 3;
    for (int id = threadIdx.x; id < page_size * words; id += blockDim.x) {
        const int r = id / words, w = id - r * words;
        const int t = (i << page_shift) + r;
        float k[8], v[8];
        if (t >= first && t < end) {
            Kv4Params p = kv4_params(*reinterpret_cast<const uint2*>(base + (size_t)page_size * hd + (size_t)r * 8));
            kv4_poison(p);
            kv4_unpack8(*reinterpret_cast<const unsigned*>(base + (size_t)r * (hd >> 1) + 4 * w), p.ks, p.kz, k);
            kv4_unpack8(*reinterpret_cast<const unsigned*>(base + ((size_t)page_size + r) * (hd >> 1) + 4 * w), p.vs, p.vz, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) k[e] = v[e] = 0.f;
        }
        kv4_store8(dst + (size_t)r * hd + 8 * w, k);
        kv4_store8(dst + ((size_t)nkv * page_size + r) * hd + 8 * w, v);
    }
}

MV_API int mv_kv4_read_pages(const void* pool, const int* page_table, int table_stride, int page_size, const int* cu, const int* starts,
                             int window, void* out, int dtype, int* out_table, int W, int n_seqs, int nkv, int hd, cudaStream_t stream) {
    if (n_seqs <= 0 || W <= 0) return 0;
    if (hd % 8 || page_size < 1 || (page_size & (page_size - 1)) || n_seqs > 65535 || nkv > 65535) return (int)cudaErrorInvalidValue;
    int page_shift = 0;
    while ((1 << page_shift) < page_size) ++page_shift;
    const dim3 grid(W, nkv, n_seqs);
    if (dtype == MV_DT_BF16)
        mv_launch(kv4_read_pages_kernel<__nv_bfloat16>, grid, 256, 0, stream, (const unsigned char*)pool, page_table, table_stride,
                  page_shift, cu, starts, window, (__nv_bfloat16*)out, out_table, W, nkv, hd);
    else
        mv_launch(kv4_read_pages_kernel<float>, grid, 256, 0, stream, (const unsigned char*)pool, page_table, table_stride, page_shift, cu,
                  starts, window, (float*)out, out_table, W, nkv, hd);
    return mv_launch_status();
}

// ------------------------------------------------------------------ attention of single query tokens
// Block = (query token, kv head x tile of GT query heads, split of the keys), 4 warps; a warp takes runs of 32 keys in turn.  In a run
// each lane scores one key: with x = zero + step * code, q.x = step * (q.code) + zero * sum(q), so the codes are never turned into
// elements one by one.  Then the lanes are dealt out to (key, 8 elements of the values) and add p * value.  Running maximum and sum per
// head; warps are merged in shared memory, splits in split order by the block that finishes last (ticket counter, left at 0).
//
// For float32, and for pages of fewer than 16 tokens, which the kernel on mma.sync does not take.  Instructions bound it: a key's 64 elements are
// 64 multiply-adds a head for its score and as many for its value, on the lanes that have a key.  16 / 8 heads of 64 in float32, 4 sequences
// of 100 to 900 rows: 12 us.
template <typename T, int GT>
__global__ void __launch_bounds__(128)
attention_kv4_kernel(const T* __restrict__ q, const unsigned char* __restrict__ pool, const int* __restrict__ page_table,
                     int table_stride, int page_shift, const int* __restrict__ positions, const int* __restrict__ seq_of,
                     T* __restrict__ o, float* __restrict__ part_o, float* __restrict__ part_ml, int* __restrict__ tickets, int nh,
                     int nkv, int hd, float scale, int window, int head_tiles) {
    mv_pdl_begin();
    extern __shared__ float smem[];
    float* qs = smem;                                            // [GT][hd]
    float* ms = qs + GT * hd;                                    // [4][GT] running maxima, then
    float* ls = ms + 4 * GT;                                     // [4][GT] sums
    float* os = ls + 4 * GT;                                     // [4][GT][hd]
    __shared__ int is_last;
    const int splits = gridDim.x, split = blockIdx.x, n = blockIdx.z;
    const int g = blockIdx.y / head_tiles, tile = blockIdx.y - g * head_tiles;
    const int G = nh / nkv, h0 = tile * GT, heads = min(GT, G - h0);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pos = positions[n], page_size = 1 << page_shift;
    const int* table = page_table + (size_t)seq_of[n] * table_stride;
    const size_t head_bytes = kv4_head_bytes(page_size, hd);
    const int lo_key = window > 0 ? max(0, pos - window + 1) : 0;
    const int run0 = lo_key >> 5, runs = (pos >> 5) + 1 - run0;
    const int per = (runs + splits - 1) / splits, r_lo = run0 + split * per, r_hi = min(run0 + runs, r_lo + per);
    for (int i = threadIdx.x; i < GT * hd; i += 128) {
        const int h = i / hd;
        qs[i] = h < heads ? mv_to_f32(q[((size_t)n * nh + g * G + h0) * hd + i]) * scale : 0.f;
    }
    for (int i = threadIdx.x; i < 4 * GT * hd; i += 128) os[i] = 0.f;
    __syncthreads();
    float qsum[GT];
#pragma unroll
    for (int h = 0; h < GT; ++h) {
        float s = 0.f;
        for (int d = lane; d < hd; d += 32) s += qs[h * hd + d];
        qsum[h] = mv_warp_sum(s);
    }
    const int words = hd >> 3, lanes_k = 32 / words;             // keys that the lanes take at a time for the values
    const int vk = lane / words, vw = lane - vk * words;
    float m[GT], l[GT], acc[GT][8];
#pragma unroll
    for (int h = 0; h < GT; ++h) {
        m[h] = -INFINITY;
        l[h] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[h][e] = 0.f;
    }
    for (int r = r_lo + warp; r < r_hi; r += 4) {
        const int t = r * 32 + lane;
        const bool seen = t <= pos && t >= lo_key;
        float s[GT], vs = 0.f, vz = 0.f;
        long long vbase = 0;                                     // where this lane's key has its value's codes
        if (seen) {
            const int page = mv_read_page(table[t >> page_shift]), at = t & (page_size - 1);
            const size_t off = ((size_t)page * nkv + g) * head_bytes;
            const unsigned char* base = pool + off;
            Kv4Params p = kv4_params(*reinterpret_cast<const uint2*>(base + (size_t)page_size * hd + (size_t)at * 8));
            kv4_poison(p);
            vs = p.vs;
            vz = p.vz;
            vbase = (long long)off + ((long long)page_size + at) * (hd >> 1);
            const unsigned* kc = reinterpret_cast<const unsigned*>(base + (size_t)at * (hd >> 1));
            float dot[GT];
#pragma unroll
            for (int h = 0; h < GT; ++h) dot[h] = 0.f;
            for (int w = 0; w < words; ++w) {
                float c[8];
                kv4_unpack8(kc[w], 1.f, -8.f, c);
#pragma unroll
                for (int h = 0; h < GT; ++h)
#pragma unroll
                    for (int e = 0; e < 8; ++e) dot[h] = fmaf(c[e], qs[h * hd + 8 * w + e], dot[h]);
            }
#pragma unroll
            for (int h = 0; h < GT; ++h) s[h] = fmaf(p.ks, dot[h], fmaf(8.f, p.ks, p.kz) * qsum[h]);       // (codes less 8: little cancels)
        }
#pragma unroll
        for (int h = 0; h < GT; ++h) {
            if (!seen) s[h] = -INFINITY;
            const float mx = fmaxf(m[h], mv_warp_max(s[h]));
            const float corr = m[h] == -INFINITY ? 0.f : expf(m[h] - mx);
            m[h] = mx;
            // (mx is -infinity only where every score so far is -infinity or NaN: then a score that is seen gives NaN, as it should)
            s[h] = seen ? expf(s[h] - mx) : 0.f;
            l[h] = l[h] * corr + s[h];
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[h][e] *= corr;
        }
        for (int k0 = 0; k0 < 32; k0 += lanes_k) {
            const int k = min(k0 + vk, 31);
            const bool mine = vk < lanes_k && k0 + vk < 32;
            const float ks = __shfl_sync(0xffffffffu, vs, k), kz = __shfl_sync(0xffffffffu, vz, k);
            const long long at = __shfl_sync(0xffffffffu, vbase, k);
            const bool kseen = r * 32 + k <= pos && r * 32 + k >= lo_key;
            float v[8];
            if (mine && kseen) kv4_unpack8(*reinterpret_cast<const unsigned*>(pool + at + 4 * vw), ks, kz, v);
#pragma unroll
            for (int h = 0; h < GT; ++h) {
                const float p = __shfl_sync(0xffffffffu, s[h], k);
                if (mine && kseen)
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[h][e] = fmaf(p, v[e], acc[h][e]);
            }
        }
    }
    // the lanes that hold the same elements of other keys add up, in lane order
#pragma unroll
    for (int h = 0; h < GT; ++h) {
        l[h] = mv_warp_sum(l[h]);
        if (lane == 0) { ms[warp * GT + h] = m[h]; ls[warp * GT + h] = l[h]; }
        for (int k = 0; k < lanes_k; ++k) {
            if (vk == k)
#pragma unroll
                for (int e = 0; e < 8; ++e) os[(warp * GT + h) * hd + 8 * vw + e] += acc[h][e];
            __syncwarp();
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < heads * hd; i += 128) {
        const int h = i / hd, d = i - h * hd;
        float M = -INFINITY, L = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, ms[w * GT + h]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = ms[w * GT + h] == -INFINITY ? (ls[w * GT + h] == 0.f ? 0.f : NAN) : expf(ms[w * GT + h] - M);
            L = fmaf(ls[w * GT + h], f, L);
            v = fmaf(os[(w * GT + h) * hd + d], f, v);
        }
        const int hh = g * G + h0 + h;
        if (splits == 1) {
            o[((size_t)n * nh + hh) * hd + d] = mv_from_f32<T>(v / L);
        } else {
            part_o[(((size_t)n * nh + hh) * splits + split) * hd + d] = v;
            if (d == 0) {
                float* ml = part_ml + (((size_t)n * nh + hh) * splits + split) * 2;
                ml[0] = M;
                ml[1] = L;
            }
        }
    }
    if (splits == 1) return;
    __threadfence();
    __syncthreads();
    int* ticket = tickets + (size_t)n * gridDim.y + blockIdx.y;
    if (threadIdx.x == 0) is_last = atomicAdd(ticket, 1) == splits - 1;
    __syncthreads();
    if (!is_last) return;
    __threadfence();
    for (int i = threadIdx.x; i < heads * hd; i += 128) {
        const int h = i / hd, d = i - h * hd, hh = g * G + h0 + h;
        const size_t at = ((size_t)n * nh + hh) * splits;
        float M = -INFINITY, L = 0.f, v = 0.f;
        for (int s = 0; s < splits; ++s) M = fmaxf(M, __ldcg(part_ml + (at + s) * 2));
        for (int s = 0; s < splits; ++s) {
            const float ms_ = __ldcg(part_ml + (at + s) * 2), ls_ = __ldcg(part_ml + (at + s) * 2 + 1);
            const float f = ms_ == -INFINITY ? (ls_ == 0.f ? 0.f : NAN) : expf(ms_ - M);
            L = fmaf(ls_, f, L);
            v = fmaf(__ldcg(part_o + (at + s) * hd + d), f, v);
        }
        o[((size_t)n * nh + hh) * hd + d] = mv_from_f32<T>(v / L);
    }
    if (threadIdx.x == 0) *ticket = 0;
}

// part_o [N, nh, splits, hd], part_ml [N, nh, splits, 2] float32 and tickets [N, nkv * head_tiles] (zero) are used with splits > 1.
struct AttentionKv4Args {
    const void *q, *pool;
    const int *page_table, *positions, *seq_of;
    void* o;
    float *part_o, *part_ml;
    int* tickets;
    cudaStream_t stream;
    int table_stride, page_size, dtype, N, nh, nkv, hd, window, splits, gt, head_tiles;
    float scale;
};
MV_API int mv_attention_kv4(const void* record) {
    const auto& [q, pool, page_table, positions, seq_of, o, part_o, part_ml, tickets, stream, table_stride, page_size, dtype, N, nh, nkv, hd, window, splits,
                gt, head_tiles, scale] = *static_cast<const AttentionKv4Args*>(record);
    if (N <= 0) return 0;
    if (hd % 8 || hd > KV4_MAX_HEAD_DIM || nkv < 1 || nh % nkv || page_size < 1 || (page_size & (page_size - 1)) || splits < 1 ||
        gt * head_tiles < nh / nkv || N > 65535 || nkv * head_tiles > 65535)
        return (int)cudaErrorInvalidValue;
    int page_shift = 0;
    while ((1 << page_shift) < page_size) ++page_shift;
    const dim3 grid(splits, nkv * head_tiles, N);
    // (at most 4 * (5 * 4 * 256 + 8 * 4) bytes: less than any block may have)
#define MV_GO(T, GT)                                                                                                              \
    mv_launch(attention_kv4_kernel<T, GT>, grid, 128, sizeof(float) * (5 * GT * hd + 8 * GT), stream, (const T*)q,                 \
              (const unsigned char*)pool, page_table, table_stride, page_shift, positions, seq_of, (T*)o, part_o, part_ml, tickets, \
              nh, nkv, hd, scale, window, head_tiles)
#define MV_GT(T)                                                                                                                  \
    do {                                                                                                                          \
        if (gt == 1) MV_GO(T, 1);                                                                                                 \
        else if (gt == 2) MV_GO(T, 2);                                                                                            \
        else if (gt == 4) MV_GO(T, 4);                                                                                            \
        else return (int)cudaErrorInvalidValue;                                                                                   \
    } while (0)
    if (dtype == MV_DT_BF16) MV_GT(__nv_bfloat16);
    else MV_GT(float);
#undef MV_GT
#undef MV_GO
    return mv_launch_status();
}
