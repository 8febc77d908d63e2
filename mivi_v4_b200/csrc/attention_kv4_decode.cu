// Attention of few query tokens a sequence over a cache held in 4 bits (kv4.cuh), bfloat16, pages of 16 rows and more: flash decoding whose
// two products are mma.sync on the codes themselves.
//
// What bounds it.  A key and its value of 64 elements are 72 bytes, so at the memory's rate a multiprocessor gets one every three clocks; in
// that time it has to turn 128 codes into operands, score them and weight them.  The work goes by instructions issued, and the design counts
// them: no element is ever worked out.  With x = zero + step * code = (zero + 8 step) + step * (code - 8),
//     q.k = step_k * (q . (code_k - 8)) + (zero_k + 8 step_k) * sum(q)
//     sum_t p_t v_t = sum_t (p_t step_t) (code_t - 8) + sum_t p_t (zero_t + 8 step_t)
// so the products run on whole numbers from -8 to 7, which are exact in half precision and cost 1.2 instructions a pair to make (mask a
// nibble pair into the mantissa of 1024 or 64, subtract), and the rows' numbers meet scores and weights, two an instruction.
//
// Half precision, not bfloat16: its 11 bits hold a bfloat16 query exactly and give the weights eight times bfloat16's precision.  Its range
// is small, so powers of two are taken out: of a query row its largest element's, of the weights p * step the largest step's so far
// (weights whose step is 2^-24 of the largest vanish: so would their values beside the others' in bfloat16).
//
// The scores are computed transposed, S^T = K Q^T, keys on the 16 rows of m16n8k16 and queries (tokens of one sequence x the heads that share
// the kv head) on its 8 columns, so that the usual group of 4 heads fills half of a product and not a quarter.  Sums over K run over elements
// in any order, so a lane takes a row's bytes as they lie (lane t of four: a quarter of the row) and reads its queries to match.  O^T = V^T
// P^T likewise: a lane takes 8 neighbouring elements of four keys.  P^T gets from the accumulators' layout to the operand's by movmatrix.
// Row r of a product is key r ^ (r >> 2 & 1) of its eight: with that order neither the keys' 8-byte nor the values' 4-byte shared loads of
// rows of 32 bytes meet in a bank.
//
// Block = (tile of query columns, kv head, split of the keys), 4 warps, each with tiles of 64 keys of its own, STAGES ahead by bulk copies:
// one of 4,608 bytes where a page has 64 rows, so that few instructions keep memory busy.  Warps merge in shared memory, splits in split
// order by the block that finishes last (ticket counter, left at 0).
#include "kv4.cuh"
#include "tc_common.cuh"

#include <cuda_fp16.h>

MV_GUARD_SETTER(attention_kv4_decode)

namespace {

constexpr int KD_WARPS = 4, KD_KEYS = 64;

__device__ __forceinline__ void bulk_load(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned transpose8x8(unsigned a) {
    unsigned d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// nibbles 0 and 1 of both halves of x as pairs of halves, less 8: 1024 + c - 1032, and (1024 + 16 c) / 16 - 72
__device__ __forceinline__ void centred(unsigned x, unsigned& even, unsigned& odd) {
    unsigned e, o;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(e) : "r"(x));
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(o) : "r"(x));
    asm("sub.f16x2 %0, %1, %2;" : "=r"(even) : "r"(e), "r"(0x64086408u));
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(odd) : "r"(o), "r"(0x2c002c00u), "r"(0xd480d480u));
}
__device__ __forceinline__ unsigned half_pair(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }       // e from -126 to 127

// HDP: head size rounded up to 64, 128 or 256; NT: tiles of 8 query columns
template <int HDP, int NT>
struct KdShape {
    static constexpr int STAGES = HDP == 64 ? 3 : 2, STAGE_BYTES = KD_KEYS * (HDP + 8);
    // (the last row's loads of a head size below HDP reach past the stage)
    static constexpr int RING = KD_WARPS * STAGES * STAGE_BYTES + HDP, MERGE = KD_WARPS * 8 * NT * (HDP + 4) * 4;
    static constexpr int BARS = RING > MERGE ? RING : MERGE, SMEM = BARS + KD_WARPS * STAGES * 8;
};

// HDP: head size rounded up to 64, 128 or 256; EXACT: it is the head size.  NT: tiles of 8 query columns.  A column is token c / heads and
// head h0 + c % heads of the kv head's group, heads = min(group, 8 NT); grid (splits, nkv * head_tiles, N); the block of a token whose
// place in its sequence's run is no multiple of tokens_per_tile has nothing to do.
template <int HDP, bool EXACT, int NT>
__global__ void __launch_bounds__(KD_WARPS * 32, HDP == 64 ? (NT == 1 ? 4 : NT == 2 ? 3 : 2) : (HDP == 128 && NT == 1 ? 3 : 2))
attention_kv4_decode_kernel(const __nv_bfloat16* __restrict__ q, const unsigned char* __restrict__ pool, const int* __restrict__ page_table,
                            int table_stride, int page_shift, const int* __restrict__ positions, const int* __restrict__ seq_of,
                            const int* __restrict__ starts, __nv_bfloat16* __restrict__ o, float* __restrict__ part_o,
                            float* __restrict__ part_ml, int* __restrict__ tickets, int N, int nh, int nkv, int hd_, float scale_log2, int window,
                            int head_tiles, int heads, int tokens_per_tile, int* __restrict__ err) {
    mv_pdl_begin();
    using Shape = KdShape<HDP, NT>;
    constexpr int STAGES = Shape::STAGES, COLS = 8 * NT, MT = HDP / 16, W = HDP / 32;      // W: words of a lane's quarter of a row
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int is_last;
    const int hd = EXACT ? HDP : hd_;
    const int splits = gridDim.x, split = blockIdx.x, n = blockIdx.z;
    const int kvh = blockIdx.y / head_tiles, h0 = (blockIdx.y - kvh * head_tiles) * heads;
    const int group = nh / nkv, live_heads = min(heads, group - h0);
    const int seq = seq_of[n], pos0 = positions[n];
    int tokens = 1;
    if (tokens_per_tile > 1) {
        if ((pos0 - starts[seq]) % tokens_per_tile) return;
        while (tokens < tokens_per_tile && n + tokens < N && seq_of[n + tokens] == seq) ++tokens;
    }
    const int pos_last = pos0 + tokens - 1, lo_key = window > 0 ? max(0, pos0 - window + 1) : 0;
    const int* table = page_table + (size_t)seq * table_stride;
    const int warp = warp_index(), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int page_size = 1 << page_shift;
    const size_t head_bytes = kv4_head_bytes(page_size, hd);
    const int stage_bytes = KD_KEYS * (hd + 8);
    const unsigned ring = smem_u32(smem) + warp * STAGES * Shape::STAGE_BYTES;
    unsigned char* ring_ptr = smem + warp * STAGES * Shape::STAGE_BYTES;
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(smem + Shape::BARS) + warp * STAGES;
    const unsigned bar0 = smem_u32(bars);
    if (lane == 0) {
        for (int s = 0; s < STAGES; ++s) mbar_init(bar0 + 8 * s, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();

    // this warp's tiles: every KD_WARPS-th of the split's
    const int tile0 = lo_key / KD_KEYS, n_tiles = pos_last / KD_KEYS + 1 - tile0;
    const int per = (n_tiles + splits - 1) / splits;
    const int first = tile0 + split * per + warp, past = min(tile0 + n_tiles, tile0 + (split + 1) * per);
    const int mine = first < past ? (past - first + KD_WARPS - 1) / KD_WARPS : 0;
    auto fetch = [&](int i) {                                    // all lanes; lane 0 copies
        const int key0 = (first + i * KD_WARPS) * KD_KEYS;
        if (lane == 0) {
            const unsigned bar = bar0 + 8 * (i % STAGES), dst = ring + (i % STAGES) * Shape::STAGE_BYTES;
            if (page_shift == 6) {
                const int page = mv_read_page(table[key0 >> 6]);
                mbar_expect_tx(bar, (unsigned)stage_bytes);
                bulk_load(dst, pool + ((size_t)page * nkv + kvh) * head_bytes, (unsigned)stage_bytes, bar);
            } else {
                // rows a copy brings, and how many copies hold rows that exist
                const int rows = min(KD_KEYS, page_size);
                const int parts = min(KD_KEYS, pos_last + 1 - key0 + rows - 1) / rows;
                mbar_expect_tx(bar, (unsigned)(parts * rows * (hd + 8)));
                for (int p = 0; p < parts; ++p) {
                    const int key = key0 + p * rows, row = key & (page_size - 1);
                    // (behind a window, pages before the first key seen may be gone: their entry is a page all the same)
                    const int page = mv_read_page(table[key >> page_shift]);
                    const unsigned char* src = pool + ((size_t)page * nkv + kvh) * head_bytes;
                    const unsigned codes = (unsigned)(rows * (hd >> 1));
                    bulk_load(dst + p * codes, src + (size_t)row * (hd >> 1), codes, bar);
                    bulk_load(dst + KD_KEYS * (hd >> 1) + p * codes, src + ((size_t)page_size + row) * (hd >> 1), codes, bar);
                    bulk_load(dst + KD_KEYS * hd + p * rows * 8, src + (size_t)page_size * hd + (size_t)row * 8, (unsigned)(rows * 8), bar);
                }
            }
        }
    };
    for (int i = 0; i < min(mine, STAGES); ++i) fetch(i);

    // queries: column 8 nt + g, elements of lane t's quarter of a row, in the order in which a word's nibbles come out
    unsigned qf[NT][2 * W][2];
    float2 lsc[NT], qsum[NT];                                    // of columns 2t and 2t + 1: factor to log2 units, sum of the row in them
    int2 at_col[NT];                                             // and their positions (-1: no such column)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int c = 8 * nt + g, tok = c / heads, h = c - tok * heads;
        const bool live = tok < tokens && h < live_heads;
        const __nv_bfloat16* row = q + ((size_t)(n + (live ? tok : 0)) * nh + kvh * group + h0 + (live ? h : 0)) * hd;
        float x[HDP / 4], top = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const int d = t * (HDP / 4) + 8 * w;
            if (live && (EXACT || d < hd)) mv_load8(row + d, x + 8 * w);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) x[8 * w + e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < HDP / 4; ++e) top = fmaxf(top, fabsf(x[e]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int ex = top > 0.f ? min(126, max(-126, (int)(__float_as_uint(top) >> 23) - 127)) : 0;
        const float down = pow2f(-ex);
#pragma unroll
        for (int e = 0; e < HDP / 4; ++e) { x[e] *= down; sum += x[e]; }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            qf[nt][2 * w][0] = half_pair(x[8 * w], x[8 * w + 4]);
            qf[nt][2 * w][1] = half_pair(x[8 * w + 1], x[8 * w + 5]);
            qf[nt][2 * w + 1][0] = half_pair(x[8 * w + 2], x[8 * w + 6]);
            qf[nt][2 * w + 1][1] = half_pair(x[8 * w + 3], x[8 * w + 7]);
        }
        const float l = scale_log2 * pow2f(ex);
        sum *= l;
        const int at = live ? pos0 + tok : -1;
        lsc[nt] = make_float2(__shfl_sync(0xffffffffu, l, 8 * t), __shfl_sync(0xffffffffu, l, 8 * t + 4));
        qsum[nt] = make_float2(__shfl_sync(0xffffffffu, sum, 8 * t), __shfl_sync(0xffffffffu, sum, 8 * t + 4));
        at_col[nt] = make_int2(__shfl_sync(0xffffffffu, at, 8 * t), __shfl_sync(0xffffffffu, at, 8 * t + 4));
    }

    float oacc[NT][MT][4];
    float2 m[NT], l[NT], pz[NT];                                 // maxima (log2 units, alike in all rows' lanes), this lane's sums
    int ev = -126;                                               // the weights' power of two
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt] = make_float2(-INFINITY, -INFINITY);
        l[nt] = pz[nt] = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) oacc[nt][i][e] = 0.f;
    }
    const int key_of = g ^ (g >> 2);                             // of row g of a product (bit 2 into bit 0)
    const int vrow0 = (2 * t) ^ (t >> 1), vrow1 = (2 * t + 1) ^ (t >> 1);
    bool ok = true;
    for (int i = 0; i < mine; ++i) {
        ok = mbar_wait_warp(bar0 + 8 * (i % STAGES), (unsigned)(i / STAGES) & 1u, err, 150);
        if (!ok) {                                               // given up: the copies under way land before the block leaves
            for (int j = i + 1; j < min(mine, i + STAGES); ++j) mbar_wait_warp(bar0 + 8 * (j % STAGES), (unsigned)(j / STAGES) & 1u, err, 151);
            break;
        }
        const unsigned char* kt = ring_ptr + (i % STAGES) * Shape::STAGE_BYTES;
        const unsigned char* vt = kt + KD_KEYS * (hd >> 1);
        const uint2* pt = reinterpret_cast<const uint2*>(kt + KD_KEYS * hd);
        const int key0 = (first + i * KD_WARPS) * KD_KEYS;
        // every key of the tile is seen by every column (columns that stand for nothing may see what they like)
        const bool whole = key0 + KD_KEYS - 1 <= pos0 && (window <= 0 || key0 > pos_last - window);

        // ---- scores: 64 keys x 8 NT columns
        float s[NT][4][4];
        float zv[8];
        float sv[8];
        unsigned smax = 0u;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[nt][b][e] = 0.f;
            const unsigned char* r0 = kt + (16 * b + key_of) * (hd >> 1) + t * (HDP / 8);
            const unsigned char* r1 = r0 + 8 * (hd >> 1);
            unsigned w0[W], w1[W];
            if (EXACT && W == 2) {
                const uint2 a = *reinterpret_cast<const uint2*>(r0), c = *reinterpret_cast<const uint2*>(r1);
                w0[0] = a.x; w0[1] = a.y; w1[0] = c.x; w1[1] = c.y;
            } else if (EXACT) {
#pragma unroll
                for (int w = 0; w < W; w += 4) {
                    const uint4 a = *reinterpret_cast<const uint4*>(r0 + 4 * w), c = *reinterpret_cast<const uint4*>(r1 + 4 * w);
                    w0[w] = a.x; w0[w + 1] = a.y; w0[w + 2] = a.z; w0[w + 3] = a.w;
                    w1[w] = c.x; w1[w + 1] = c.y; w1[w + 2] = c.z; w1[w + 3] = c.w;
                }
            } else {
#pragma unroll
                for (int w = 0; w < W; ++w) {                    // (beyond the head size: another row's codes, times queries of 0)
                    w0[w] = *reinterpret_cast<const unsigned*>(r0 + 4 * w);
                    w1[w] = *reinterpret_cast<const unsigned*>(r1 + 4 * w);
                }
            }
#pragma unroll
            for (int w = 0; w < W; ++w) {
                unsigned a0, a1, a2, a3;
                centred(w0[w], a0, a2);
                centred(w1[w], a1, a3);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma16816(s[nt][b], a0, a1, a2, a3, qf[nt][2 * w][0], qf[nt][2 * w][1]);
                centred(w0[w] >> 8, a0, a2);
                centred(w1[w] >> 8, a1, a3);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma16816(s[nt][b], a0, a1, a2, a3, qf[nt][2 * w + 1][0], qf[nt][2 * w + 1][1]);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {                        // rows g and g + 8
                const int key = 16 * b + 8 * j + key_of;
                Kv4Params p = kv4_params(pt[key]);
                kv4_poison(p);
                const float kz = fmaf(8.f, p.ks, p.kz);
                if (!whole && (key0 + key > pos_last || key0 + key < lo_key)) p.vs = p.vz = 0.f;
                sv[2 * b + j] = p.vs;
                zv[2 * b + j] = fmaf(8.f, p.vs, p.vz);
                smax = max(smax, __float_as_uint(p.vs));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    // (the factors first: rows near the largest floats meet queries near the smallest)
                    float2 y = fma2(make_float2(s[nt][b][2 * j], s[nt][b][2 * j + 1]), mul2(make_float2(p.ks, p.ks), lsc[nt]),
                                    mul2(make_float2(kz, kz), qsum[nt]));
                    if (!whole) {
                        const int at = key0 + key;
                        if (at > at_col[nt].x || (window > 0 && at <= at_col[nt].x - window)) y.x = -INFINITY;
                        if (at > at_col[nt].y || (window > 0 && at <= at_col[nt].y - window)) y.y = -INFINITY;
                    }
                    s[nt][b][2 * j] = y.x;
                    s[nt][b][2 * j + 1] = y.y;
                }
            }
        }
        // ---- running maxima, the weights' power of two
        smax = __reduce_max_sync(0xffffffffu, smax);
        const int ev_new = max(ev, max(-126, (int)(smax >> 23) - 127));
        const float ev_corr = ev_new == ev ? 1.f : (ev_new - ev > 126 ? 0.f : pow2f(ev - ev_new));
        ev = ev_new;
        const float down = pow2f(-ev);
#pragma unroll
        for (int j = 0; j < 8; ++j) sv[j] *= down;
        float2 ref[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float2 mx = m[nt];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                mx.x = fmaxf(mx.x, fmaxf(s[nt][b][0], s[nt][b][2]));
                mx.y = fmaxf(mx.y, fmaxf(s[nt][b][1], s[nt][b][3]));
            }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                mx.x = fmaxf(mx.x, __shfl_xor_sync(0xffffffffu, mx.x, d));
                mx.y = fmaxf(mx.y, __shfl_xor_sync(0xffffffffu, mx.y, d));
            }
            ref[nt] = make_float2(mx.x == -INFINITY ? 0.f : mx.x, mx.y == -INFINITY ? 0.f : mx.y);
            const float2 corr = make_float2(m[nt].x == -INFINITY ? 0.f : ex2(m[nt].x - ref[nt].x), m[nt].y == -INFINITY ? 0.f : ex2(m[nt].y - ref[nt].y));
            m[nt] = mx;
            l[nt] = mul2(l[nt], corr);
            pz[nt] = mul2(pz[nt], corr);
            const float2 oc = mul2(corr, make_float2(ev_corr, ev_corr));
            if (__any_sync(0xffffffffu, oc.x != 1.f || oc.y != 1.f))
#pragma unroll
                for (int k = 0; k < MT; ++k) {
                    oacc[nt][k][0] *= oc.x; oacc[nt][k][1] *= oc.y;
                    oacc[nt][k][2] *= oc.x; oacc[nt][k][3] *= oc.y;
                }
        }
        // ---- weights and the values' product, 16 keys at a time
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            unsigned pb[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float2 y = make_float2(s[nt][b][2 * j] - ref[nt].x, s[nt][b][2 * j + 1] - ref[nt].y);
                    const float2 p = make_float2(ex2(y.x), ex2(y.y));        // (ex2(-infinity) is 0: a key that is not seen)
                    l[nt] = add2(l[nt], p);
                    pz[nt] = fma2(p, make_float2(zv[2 * b + j], zv[2 * b + j]), pz[nt]);
                    const float2 w = mul2(p, make_float2(sv[2 * b + j], sv[2 * b + j]));
                    pb[nt][j] = transpose8x8(half_pair(w.x, w.y));
                }
            const unsigned char* v0 = vt + (16 * b + vrow0) * (hd >> 1) + 4 * g;
            const unsigned char* v1 = vt + (16 * b + vrow1) * (hd >> 1) + 4 * g;
#pragma unroll
            for (int u = 0; u < HDP / 64; ++u) {
                const unsigned wa = *reinterpret_cast<const unsigned*>(v0 + 32 * u), wb = *reinterpret_cast<const unsigned*>(v1 + 32 * u);
                const unsigned wc = *reinterpret_cast<const unsigned*>(v0 + 8 * (hd >> 1) + 32 * u);
                const unsigned wd = *reinterpret_cast<const unsigned*>(v1 + 8 * (hd >> 1) + 32 * u);
#pragma unroll
                for (int half = 0; half < 2; ++half) {           // elements 0 .. 3 of the lane's eight, then 4 .. 7
                    const unsigned x0 = __byte_perm(wa, wb, half ? 0x7632 : 0x5410), x1 = __byte_perm(wc, wd, half ? 0x7632 : 0x5410);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        unsigned a0, a1, a2, a3;
                        centred(k ? x0 >> 8 : x0, a0, a1);
                        centred(k ? x1 >> 8 : x1, a2, a3);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma16816(oacc[nt][4 * u + 2 * half + k], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
                    }
                }
            }
        }
        __syncwarp();
        if (i + STAGES < mine) fetch(i + STAGES);
    }

    // ---- the warps' results meet in shared memory (in place of the rings)
    __syncthreads();
    float* xo = reinterpret_cast<float*>(smem);                  // [warp][column][HDP], then maxima and sums [warp][column]
    float* xm = xo + KD_WARPS * COLS * HDP;
    float* xl = xm + KD_WARPS * COLS;
    const float up = pow2f(ev);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
            l[nt].x += __shfl_xor_sync(0xffffffffu, l[nt].x, d);
            l[nt].y += __shfl_xor_sync(0xffffffffu, l[nt].y, d);
            pz[nt].x += __shfl_xor_sync(0xffffffffu, pz[nt].x, d);
            pz[nt].y += __shfl_xor_sync(0xffffffffu, pz[nt].y, d);
        }
        const int c = 8 * nt + 2 * t;
        if (g == 0) {
            xm[warp * COLS + c] = m[nt].x; xm[warp * COLS + c + 1] = m[nt].y;
            xl[warp * COLS + c] = l[nt].x; xl[warp * COLS + c + 1] = l[nt].y;
        }
#pragma unroll
        for (int u = 0; u < HDP / 64; ++u) {
            float* d0 = xo + ((size_t)warp * COLS + c) * HDP + 64 * u + 8 * g;
            float* d1 = d0 + HDP;
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
                const float(&a)[4] = oacc[nt][4 * u + k];
                const float(&b)[4] = oacc[nt][4 * u + k + 1];
                *reinterpret_cast<float4*>(d0 + 2 * k) = make_float4(fmaf(a[0], up, pz[nt].x), fmaf(a[2], up, pz[nt].x), fmaf(b[0], up, pz[nt].x), fmaf(b[2], up, pz[nt].x));
                *reinterpret_cast<float4*>(d1 + 2 * k) = make_float4(fmaf(a[1], up, pz[nt].y), fmaf(a[3], up, pz[nt].y), fmaf(b[1], up, pz[nt].y), fmaf(b[3], up, pz[nt].y));
            }
        }
    }
    __syncthreads();
    // A part: maximum (log2 units), sum, weighted values.  Where nothing was seen the sum is 0 and the part counts nothing; where all
    // that was seen is not a number the sum is not one, and stays so.
    auto share = [](float mx, float sum, float M) { return mx == -INFINITY ? (sum == 0.f ? 0.f : NAN) : ex2(mx - M); };
    const int used = tokens * live_heads;
    for (int e = threadIdx.x; e < used * (hd >> 2); e += KD_WARPS * 32) {
        const int c0 = e / (hd >> 2), d = (e - c0 * (hd >> 2)) * 4;
        const int tok = c0 / live_heads, h = c0 - tok * live_heads, c = tok * heads + h;
        float M = -INFINITY, L = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < KD_WARPS; ++w) M = fmaxf(M, xm[w * COLS + c]);
#pragma unroll
        for (int w = 0; w < KD_WARPS; ++w) {
            const float f = share(xm[w * COLS + c], xl[w * COLS + c], M);
            const float4 x = *reinterpret_cast<const float4*>(xo + ((size_t)w * COLS + c) * HDP + d);
            L = fmaf(xl[w * COLS + c], f, L);
            v.x = fmaf(x.x, f, v.x); v.y = fmaf(x.y, f, v.y); v.z = fmaf(x.z, f, v.z); v.w = fmaf(x.w, f, v.w);
        }
        const size_t row = (size_t)(n + tok) * nh + kvh * group + h0 + h;
        if (splits == 1) {
            const float inv = 1.0f / L;
            mv_store4(o + row * hd + d, v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        } else {
            *reinterpret_cast<float4*>(part_o + (row * splits + split) * hd + d) = v;
            if (d == 0) *reinterpret_cast<float2*>(part_ml + (row * splits + split) * 2) = make_float2(M, L);
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
    for (int e = threadIdx.x; e < used * (hd >> 2); e += KD_WARPS * 32) {
        const int c0 = e / (hd >> 2), d = (e - c0 * (hd >> 2)) * 4;
        const int tok = c0 / live_heads, h = c0 - tok * live_heads;
        const size_t row = (size_t)(n + tok) * nh + kvh * group + h0 + h;
        float M = -INFINITY, L = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s = 0; s < splits; ++s) M = fmaxf(M, __ldcg(part_ml + (row * splits + s) * 2));
        for (int s = 0; s < splits; ++s) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(part_ml + (row * splits + s) * 2));
            const float4 x = __ldcg(reinterpret_cast<const float4*>(part_o + (row * splits + s) * hd + d));
            const float f = share(ml.x, ml.y, M);
            L = fmaf(ml.y, f, L);
            v.x = fmaf(x.x, f, v.x); v.y = fmaf(x.y, f, v.y); v.z = fmaf(x.z, f, v.z); v.w = fmaf(x.w, f, v.w);
        }
        const float inv = 1.0f / L;
        mv_store4(o + row * hd + d, v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    }
    if (threadIdx.x == 0) *ticket = 0;
}

template <int HDP, bool EXACT, int NT, typename... A>
int kd_launch(dim3 grid, cudaStream_t stream, A... args) {
    constexpr auto kernel = attention_kv4_decode_kernel<HDP, EXACT, NT>;
    const cudaError_t e = mv_allow_smem<kernel>(KdShape<HDP, NT>::SMEM);
    if (e != cudaSuccess) return (int)e;
    mv_launch(kernel, grid, KD_WARPS * 32, KdShape<HDP, NT>::SMEM, stream, args...);
    return mv_launch_status();
}

}  // namespace

// bfloat16; pages of 16 rows or more.  nt: tiles of 8 query columns, 1, 2 or 4 (2 at most above heads of 64, 1 above 128).  A tile of columns is
// tokens_per_tile consecutive tokens of one sequence by ``heads`` heads of a kv head's group (tokens_per_tile * heads <= 8 nt; several tokens
// only where heads is the whole group).  part_o [N, nh, splits, hd], part_ml [N, nh, splits, 2] and tickets [N, nkv * head_tiles] (zero)
// are used with splits > 1.
MV_API int mv_attention_kv4_decode(const void* q, const void* pool, const int* page_table, int table_stride, int page_size,
                                   const int* positions, const int* seq_of, const int* starts, void* o, float* part_o, float* part_ml,
                                   int* tickets, int N, int nh, int nkv, int hd, float scale, int window, int splits, int nt, int head_tiles,
                                   int heads, int tokens_per_tile, int* err, cudaStream_t stream) {
    if (N <= 0) return 0;
    if (hd % 8 || hd < 8 || hd > KV4_MAX_HEAD_DIM || nkv < 1 || nh % nkv || page_size < 16 || (page_size & (page_size - 1)) || splits < 1 ||
        N > 65535 || nkv * head_tiles > 65535 || heads < 1 || heads * head_tiles < nh / nkv || tokens_per_tile < 1 ||
        heads * tokens_per_tile > 8 * nt || (tokens_per_tile > 1 && head_tiles > 1) || ((uintptr_t)pool & 15))
        return (int)cudaErrorInvalidValue;
    int page_shift = 0;
    while ((1 << page_shift) < page_size) ++page_shift;
    const dim3 grid(splits, nkv * head_tiles, N);
#define MV_GO(HDP, EXACT, NT)                                                                                                            \
    return kd_launch<HDP, EXACT, NT>(grid, stream, (const __nv_bfloat16*)q, (const unsigned char*)pool, page_table, table_stride, page_shift, \
                                     positions, seq_of, starts, (__nv_bfloat16*)o, part_o, part_ml, tickets, N, nh, nkv, hd,              \
                                     scale * 1.4426950408889634f, window, head_tiles, heads, tokens_per_tile, err)
    if (hd <= 64) {
        if (hd == 64) {
            if (nt == 1) MV_GO(64, true, 1);
            if (nt == 2) MV_GO(64, true, 2);
            if (nt == 4) MV_GO(64, true, 4);
        } else {
            if (nt == 1) MV_GO(64, false, 1);
            if (nt == 2) MV_GO(64, false, 2);
            if (nt == 4) MV_GO(64, false, 4);
        }
    } else if (hd <= 128) {
        if (hd == 128) {
            if (nt == 1) MV_GO(128, true, 1);
            if (nt == 2) MV_GO(128, true, 2);
        } else {
            if (nt == 1) MV_GO(128, false, 1);
            if (nt == 2) MV_GO(128, false, 2);
        }
    } else if (nt == 1) {
        if (hd == 256) MV_GO(256, true, 1);
        MV_GO(256, false, 1);
    }
#undef MV_GO
    return (int)cudaErrorInvalidValue;
}
