// Attention of few query tokens a sequence over a cache held in 4 bits (kv4.cuh), bfloat16, pages of 16 rows and more: flash decoding whose
// two products are mma.sync on the codes themselves.
//
// What bounds it.  A key and its value of 64 elements are 72 bytes, so at the memory's rate a multiprocessor gets one every three clocks; in
// that time it has to turn 128 codes into operands, score them and weight them.  The work goes by instructions issued, and the design counts
// them: no element of a row is ever worked out.  With x = zero + step * code,
//     q.k = step_k (q . code_k) + zero_k sum(q)
//     sum_t p_t v_t = sum_t (p_t step_t) (code_t - 8) + sum_t p_t (zero_t + 8 step_t)
// so the products run on small whole numbers, and the rows' numbers meet scores and weights.
//
// q . code: whole numbers, m16n8k32 of 8-bit operands.  A word of 8 codes becomes two operands in three instructions (mask the even nibbles,
// shift, mask the odd ones).  A query is held as whole numbers of 16 bits, times a power of two of its own (its largest element has 15
// or 16 of them, so what is lost is 2^-16 of that; a bfloat16 element within 2^-7 of it is exact), in two pieces of 8 bits that take
// neighbouring columns: the 4 heads that usually share a kv head fill the 8 columns, and a lane's two accumulators are one score's two
// pieces.  (In half precision a pair of codes costs 1.2 instructions each, twice the products, and half of the columns stay empty: 746
// instructions a tile of 64 keys against some 620 now, both with what a piece costs besides its tiles.)
//
// Weights times values: m16n8k16 in half precision, whose 11 bits a weight needs (whole numbers of 15 bits lose those that lie far below the
// largest).  Codes less 8 are exact in it and cost 1.25 instructions a code: merge two keys' words, mask a nibble of each into the mantissas
// of 1024 or 64, subtract.  Half's range is small, so the weights p * step are taken relative to a power of two: the largest step's so far,
// while no step is below 2^-KD_SPREAD of it.  Where steps lie further apart, the largest step may be a row's that a column does not see or gives no
// weight, beside which the rows that it does weigh would vanish; there each column has a unit of its own, which follows the most that one of
// its rows brings (score and step together).  (p itself is a 32-bit number: below 2^-126 of the best key's it is 0, whatever it would multiply.)
//
// The scores are computed transposed, S^T = K Q^T, keys on a product's 16 rows.  Sums over a row run over elements in any order, so a lane
// takes the row's bytes as they lie (lane t of four: a quarter of it) and reads its queries to match.  O^T = V^T P^T: a lane takes 8
// neighbouring elements of four keys.  P^T gets from the accumulators' layout to the operand's by movmatrix, two sets of 8 keys at a time:
// they come out in the even and odd columns, and each set's product leaves the other's columns at 0, so a head's two columns add up.
// Row r of a product is key r ^ (r >> 2 & 1) of its eight: with that order neither the keys' 8-byte nor the values' 4-byte shared loads of
// rows of 32 bytes meet in a bank.
//
// Block = (tile of query columns, kv head, piece of its keys), 4 warps, each with tiles of 64 keys of its own, STAGES ahead by bulk copies:
// one of 4,608 bytes where a page has 64 rows, so that few instructions keep memory busy.  How long a piece is, and which piece a block
// takes, is worked out on the device from the step's positions (a scan over its tokens): pieces of one length for all sequences, so many
// that the device is filled.  So unequal sequences are balanced, and a recorded launch fits any lengths it is replayed with.  Warps merge
// in shared memory, pieces in order by the block that finishes last (ticket counter, left at 0).
//
// Measured, 32 / 8 heads of 64: 8 sequences of 32,768 rows, 151 MB, 37.9 us, 3.98 TB/s or 0.61 of a copy's rate: instructions are issued in 0.56
// of the clocks, by 14 warps a multiprocessor, which wait for one another's results (fixed latencies) and for loads in equal parts.
// 8 sequences of 512 to 4,096: 10.0 us; one of 301, where there is next to nothing to read: 4.9 us.  (Where steps lie far apart: 43 us for the 32,768.)  (The same 8 of 32,768 in bfloat16, 537 MB,
// take attention_decode_tc.cu 87 us.)
#include "kv4.cuh"
#include "tc_common.cuh"

#include <cuda_fp16.h>

MV_GUARD_SETTER(attention_kv4_decode)

namespace {

// A piece has a tile for every warp at least; up to KD_WHOLE tiles of keys are not cut: a second tile a warp costs less than the meeting of two
// blocks (300 rows of one sequence: 5.0 us whole, 6.6 us in two; 1,000 rows behind a window: 10.8 us in pieces of 8, 9.6 us in pieces of 4).
constexpr int KD_WARPS = 4, KD_KEYS = 64, KD_WHOLE = 8;
// A weight p * step is at most 2^15 in a column's unit (p up to 2^8, the step below 2 of them times 2^6); steps that lie further apart than
// 2^KD_SPREAD are not weighed in one unit.  A score beyond KD_FAR less its maximum is worked out by itself: in one step with the product that
// makes it, the one is rounded and the other is not, and 2^-24 of a score of 2^31 is more than an exponential takes.
constexpr int KD_ROOM = 6, KD_SPREAD = 8, KD_UNIT_MIN = -120;
constexpr float KD_FAR = 1048576.0f;

__device__ __forceinline__ void bulk_load(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void mma_half(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// unsigned by signed bytes
__device__ __forceinline__ void mma_bytes(int (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned transpose8x8(unsigned a) {
    unsigned d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// nibbles 0 and 1 of both halves of x as pairs of halves, less 8: 1024 + c - 1032, and (1024 + 16 c) / 16 - 72 (whole numbers put into the mantissa of a
// known power of two: Kim, Henry, Fahim and Awadalla, "Who Says Elephants Can't Run", 2022)
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

// HDP: head size rounded up to 64, 128 or 256; NT: tiles of 4 query columns (8 of a product)
template <int HDP, int NT>
struct KdShape {
    static constexpr int RESIDENT = HDP == 64 ? (NT == 1 ? 4 : NT == 2 ? 3 : 2) : (HDP == 128 && NT == 1 ? 3 : 2);      // blocks a multiprocessor
    static constexpr int STAGES = HDP == 64 ? 3 : 2, STAGE_BYTES = KD_KEYS * (HDP + 8);
    // (the last row's loads of a head size below HDP reach past the stage)
    static constexpr int RING = KD_WARPS * STAGES * STAGE_BYTES + HDP, MERGE = KD_WARPS * 4 * NT * (HDP + 4) * 4;
    static constexpr int BARS = RING > MERGE ? RING : MERGE, SMEM = BARS + KD_WARPS * STAGES * 8;
};

// EXACT: HDP is the head size.  The N rows are those from n0 of the step on (cu counts from its first).  A column is token c / heads and head h0 + c % heads of the kv head's group, heads = min(group, 4 NT).  Only a token
// whose place in its sequence's run is a multiple of tokens_per_tile begins a tile.  Block b works on kv head and head tile b % pairs of
// piece b / pairs, counted over the tiles of columns.  piece: tiles of 64 keys in one; 0: such that there are ``blocks`` of them.
template <int HDP, bool EXACT, int NT>
__global__ void __launch_bounds__(KD_WARPS * 32, KdShape<HDP, NT>::RESIDENT)
attention_kv4_decode_kernel(const __nv_bfloat16* __restrict__ q, const unsigned char* __restrict__ pool, const int* __restrict__ page_table,
                            int table_stride, int page_shift, const int* __restrict__ positions, const int* __restrict__ seq_of,
                            const int* __restrict__ cu, int n0, const int* __restrict__ starts, __nv_bfloat16* __restrict__ o,
                            float* __restrict__ part_o, float* __restrict__ part_ml, int* __restrict__ tickets, int N, int tiles, int nh, int nkv, int hd_, float scale_log2, int window,
                            int head_tiles, int heads, int tokens_per_tile, int piece, int blocks, int* __restrict__ err) {
    mv_pdl_begin();
    using Shape = KdShape<HDP, NT>;
    constexpr int STAGES = Shape::STAGES, COLS = 4 * NT, MT = HDP / 16, W = HDP / 32;      // W: words of a lane's quarter of a row
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int scan[KD_WARPS], found[6], is_last;
    const int hd = EXACT ? HDP : hd_;
    const int warp = warp_index(), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int pairs = nkv * head_tiles;

    // ---- which tile of columns, which piece of its keys
    // of row r: its sequence and position, the tokens of the tile of columns that begins with it (0: none does) and their tiles of keys
    int row_seq, row_pos, row_tokens;
    auto tiles_at = [&](int r) {
        if (r >= N) return 0;
        row_seq = seq_of[r];
        row_pos = positions[r];
        row_tokens = 1;
        if (tokens_per_tile > 1) {
            const int in_tile = (row_pos - starts[row_seq]) % tokens_per_tile;
            if (in_tile && r) return 0;                          // (the launch's first row begins one wherever it stands)
            row_tokens = min(tokens_per_tile - in_tile, min(N, cu[row_seq + 1] - n0) - r);
        }
        return (row_pos + row_tokens - 1) / KD_KEYS + 1 - (window > 0 ? max(0, row_pos - window + 1) / KD_KEYS : 0);
    };
    auto block_sum = [&](int v, int& before) {                   // of one number a thread; before: of the threads before this one
        int inc = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += x;
        }
        __syncthreads();
        if (lane == 31) scan[warp] = inc;
        __syncthreads();
        int base = 0, all = 0;
#pragma unroll
        for (int w = 0; w < KD_WARPS; ++w) {
            if (w < warp) base += scan[w];
            all += scan[w];
        }
        before = base + inc - v;
        return all;
    };
    int n, part, parts, seq, pos0, tokens;
    {
        int before, mine = tiles_at(threadIdx.x);                // (of the first 128 rows; usually all there are)
        const bool given = piece > 0;
        if (!given) {
            long long all = block_sum(mine, before);
            if (N > KD_WARPS * 32) {
                for (int r0 = KD_WARPS * 32; r0 < N; r0 += KD_WARPS * 32) all += block_sum(tiles_at(r0 + threadIdx.x), before);
                mine = tiles_at(threadIdx.x);
            }
            // (half a piece a tile of columns is lost where its keys end: as many blocks are left to it)
            const int aim = max(blocks / 2, blocks - (tiles * pairs + 1) / 2);
            piece = max(KD_WARPS, (int)((all * pairs + aim - 1) / aim));
        }
        if (threadIdx.x == 0) found[0] = -1;
        const int want = blockIdx.x / pairs;
        int base = 0;
        for (int r0 = 0; r0 < N && base <= want; r0 += KD_WARPS * 32) {
            if (r0) mine = tiles_at(r0 + threadIdx.x);
            const int count = mine <= KD_WHOLE && !given ? (int)(mine > 0) : (mine + piece - 1) / piece;
            const int all = block_sum(count, before);
            if (want >= base + before && want < base + before + count) {
                found[0] = r0 + threadIdx.x;
                found[1] = want - base - before;
                found[2] = count;
                found[3] = row_seq;
                found[4] = row_pos;
                found[5] = row_tokens;
            }
            base += all;
        }
        __syncthreads();
        n = found[0];
        part = found[1];
        parts = found[2];
        seq = found[3];
        pos0 = found[4];
        tokens = found[5];
    }
    if (n < 0) return;
    const int pair = blockIdx.x % pairs, kvh = pair / head_tiles, h0 = (pair - kvh * head_tiles) * heads;
    const int group = nh / nkv, live_heads = min(heads, group - h0);
    const int pos_last = pos0 + tokens - 1, lo_key = window > 0 ? max(0, pos0 - window + 1) : 0;
    const int* table = page_table + (size_t)seq * table_stride;
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

    // this warp's tiles: every KD_WARPS-th of the piece's
    const int tile0 = lo_key / KD_KEYS, n_tiles = pos_last / KD_KEYS + 1 - tile0;
    const int first = tile0 + part * piece + warp, past = tile0 + (parts == 1 ? n_tiles : min(n_tiles, (part + 1) * piece));
    const int mine = first < past ? (past - first + KD_WARPS - 1) / KD_WARPS : 0;
    // where the first page of a tile lies: asked for a tile early, so that the copy need not wait for the page table
    auto page_of = [&](int i) { return i < mine ? mv_read_page(table[(first + i * KD_WARPS) * KD_KEYS >> page_shift]) : 0; };
    auto fetch = [&](int i, int page) {                          // lane 0
        const int key0 = (first + i * KD_WARPS) * KD_KEYS;
        const unsigned bar = bar0 + 8 * (i % STAGES), dst = ring + (i % STAGES) * Shape::STAGE_BYTES;
        const unsigned char* src = pool + ((size_t)page * nkv + kvh) * head_bytes;
        if (page_shift == 6) {
            mbar_expect_tx(bar, (unsigned)stage_bytes);
            bulk_load(dst, src, (unsigned)stage_bytes, bar);
        } else {
            // rows a copy brings, and how many copies hold rows that exist
            const int rows = min(KD_KEYS, page_size);
            const int copies = min(KD_KEYS, pos_last + 1 - key0 + rows - 1) / rows;
            const unsigned codes = (unsigned)(rows * (hd >> 1));
            mbar_expect_tx(bar, (unsigned)(copies * rows * (hd + 8)));
            for (int p = 0; p < copies; ++p) {
                const int row = (key0 + p * rows) & (page_size - 1);
                // (behind a window, pages before the first key seen may be gone: their entry is a page all the same)
                if (p) src = pool + ((size_t)mv_read_page(table[(key0 + p * rows) >> page_shift]) * nkv + kvh) * head_bytes;
                bulk_load(dst + p * codes, src + (size_t)row * (hd >> 1), codes, bar);
                bulk_load(dst + KD_KEYS * (hd >> 1) + p * codes, src + ((size_t)page_size + row) * (hd >> 1), codes, bar);
                bulk_load(dst + KD_KEYS * hd + p * rows * 8, src + (size_t)page_size * hd + (size_t)row * 8, (unsigned)(rows * 8), bar);
            }
        }
    };
#pragma unroll
    for (int i = 0; i < STAGES; ++i)
        if (i < mine) {
            const int page = page_of(i);
            if (lane == 0) fetch(i, page);
        }

    // Queries: of column 4 nt + g / 2 the high (g even) or low piece, elements of lane t's quarter of a row, the even and the odd ones of a word
    unsigned qf[NT][W][2];
    float lsc[NT], qsum[NT], unit[NT];                           // of column 4 nt + t: factor to log2 units, sum of the row and 1 in its units
    int at_col[NT];                                              // and its position (-1: no such column)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int c = 4 * nt + (g >> 1), tok = c / heads, h = c - tok * heads;
        const bool live = tok < tokens && h < live_heads;
        const __nv_bfloat16* row = q + ((size_t)(n + (live ? tok : 0)) * nh + kvh * group + h0 + (live ? h : 0)) * hd;
        uint4 raw[HDP / 32];                                     // two bfloat16 a word
        __nv_bfloat162 big = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const int d = t * (HDP / 4) + 8 * w;
            raw[w] = live && (EXACT || d < hd) ? *reinterpret_cast<const uint4*>(row + d) : make_uint4(0u, 0u, 0u, 0u);
            const unsigned x[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) big = __hmax2_nan(big, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&x[e])));
        }
        // (not a number, where one of the elements is none: the row's scores are none then)
        float top = __bfloat162float(__hmax_nan(__low2bfloat16(big), __high2bfloat16(big)));
        const float t1 = __shfl_xor_sync(0xffffffffu, top, 1);
        top = top > t1 || top != top ? top : t1;
        const float t2 = __shfl_xor_sync(0xffffffffu, top, 2);
        top = top > t2 || top != top ? top : t2;
        const bool fine = top < INFINITY;
        // the largest element times 2^up: at least 2^13, and at most 127 * 256, so that its pieces are bytes
        int up = top > 0.f && fine ? 14 - ((int)(__float_as_uint(top) >> 23) - 127) : 0;
        float up0 = pow2f(up >> 1), up1 = pow2f(up - (up >> 1));
        if (top * up0 * up1 > 32512.f) { --up; up1 *= 0.5f; }
        if (!fine) up0 = 0.f;
        // Added to 1.5 * 2^23 a number from -2^22 to 2^22 is rounded to a whole one, which stands in the low bits.  Its low piece, from -128 to
        // 127, is its lowest byte; its high piece the next one, once 128 is added.
        const unsigned piece_of = g & 1 ? 0x6240u : 0x7351u, round = g & 1 ? 0u : 128u;
        unsigned sum = 0u;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const unsigned x[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
#pragma unroll
            for (int odd = 0; odd < 2; ++odd) {
                unsigned v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float f = __uint_as_float(odd ? x[e] & 0xffff0000u : x[e] << 16);
                    v[e] = __float_as_uint(fmaf(f * up0, up1, 12582912.f));
                    sum += v[e];
                    v[e] += round;
                }
                // bytes 0 (or 1) of v[0], v[1] and of v[2], v[3], then one of each after the other
                const unsigned lo = __byte_perm(v[0], v[1], piece_of), hi = __byte_perm(v[2], v[3], piece_of);
                qf[nt][w][odd] = __byte_perm(lo, hi, 0x5410);
            }
        }
        sum -= (unsigned)(HDP / 4) * 0x4b400000u;
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        // A score is (q . code) step + sum(q) zero, below 2^25 times a row's numbers: for queries below 2^34 it is taken times 2^-30, so
        // that rows near the largest floats do not pass them; larger ones meet rows so small that 2^-30 of their numbers would be lost.
        const int spare = up > -20 ? -30 : 0;
        const int ex = -up - spare;
        const float f = fine ? scale_log2 * pow2f(max(-126, min(127, ex))) : NAN;
        const float sm = (float)(int)sum * pow2f(spare);
        const int at = live ? pos0 + tok : -1;
        // lane t scores column 4 nt + t, whose pieces lie in the lanes of g = 2t and 2t + 1
        lsc[nt] = __shfl_sync(0xffffffffu, f, 8 * t);
        qsum[nt] = __shfl_sync(0xffffffffu, sm, 8 * t);
        unit[nt] = pow2f(__shfl_sync(0xffffffffu, spare, 8 * t));
        at_col[nt] = __shfl_sync(0xffffffffu, at, 8 * t);
    }

    float oacc[NT][MT][4];
    float m[NT], l[NT], pz[NT];                                  // maxima (log2 units, alike in all rows' lanes), this lane's sums
    // the power of two of the largest step so far, times 2^-KD_ROOM: the unit of all columns' weights, until steps lie far apart (wide); of each
    // column's unit the inverse; this lane's least step so far
    int ev = KD_UNIT_MIN;
    float down[NT];
    unsigned low = 0xffffffffu;
    bool wide = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        down[nt] = pow2f(-KD_UNIT_MIN);
        m[nt] = -INFINITY;
        l[nt] = pz[nt] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) oacc[nt][i][e] = 0.f;
    }
    const int key_of = g ^ (g >> 2);                             // of row g of a product (bit 2 into bit 0)
    const int vrow0 = (2 * t) ^ (t >> 1), vrow1 = (2 * t + 1) ^ (t >> 1);
    bool ok = true;
    for (int i = 0; i < mine; ++i) {
        const int next_page = page_of(i + STAGES);
        ok = mbar_wait_warp(bar0 + 8 * (i % STAGES), (unsigned)(i / STAGES) & 1u, err, 150);
        if (!ok) {                                               // given up: the copies under way land before the block leaves
            for (int j = i + 1; j < min(mine, i + STAGES); ++j) mbar_wait_warp(bar0 + 8 * (j % STAGES), (unsigned)(j / STAGES) & 1u, err, 151);
            break;
        }
        const unsigned char* kt = ring_ptr + (i % STAGES) * Shape::STAGE_BYTES;
        const unsigned char* vt = kt + KD_KEYS * (hd >> 1);
        const uint2* pt = reinterpret_cast<const uint2*>(kt + KD_KEYS * hd);
        const int key0 = (first + i * KD_WARPS) * KD_KEYS;

        // ---- scores, in units of the columns' own: 64 keys x 4 NT columns; s[nt][r]: key 8 r + key_of
        float s[NT][8], sv[8], zv[8];
        unsigned smax = 0u, smin = 0xffffffffu;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            int dot[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) dot[nt][e] = 0;
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
            for (int w = 0; w < W; ++w)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    mma_bytes(dot[nt], w0[w] & 0x0f0f0f0fu, w1[w] & 0x0f0f0f0fu, (w0[w] >> 4) & 0x0f0f0f0fu, (w1[w] >> 4) & 0x0f0f0f0fu,
                              qf[nt][w][0], qf[nt][w][1]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {                        // rows g and g + 8
                const Kv4Params p = kv4_params(pt[16 * b + 8 * j + key_of]);
                sv[2 * b + j] = p.vs;
                zv[2 * b + j] = fmaf(8.f, p.vs, p.vz);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    s[nt][2 * b + j] = fmaf((float)(dot[nt][2 * j] * 256 + dot[nt][2 * j + 1]), p.ks * unit[nt], p.kz * qsum[nt]);
            }
        }
#pragma unroll
        for (int r = 0; r < 8; r += 2) {
            smax = __vimax3_u32(smax, __float_as_uint(sv[r]), __float_as_uint(sv[r + 1]));
            smin = __vimin3_u32(smin, __float_as_uint(sv[r]), __float_as_uint(sv[r + 1]));
        }
        // ---- at the edges: keys that some column, or none, sees
        if (key0 + KD_KEYS - 1 > pos0 || (window > 0 && key0 <= pos_last - window)) {
            smax = 0u;
            smin = 0xffffffffu;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const int at = key0 + 8 * r + key_of;
                if (at > pos_last || at < lo_key) sv[r] = zv[r] = 0.f;
                else smin = min(smin, __float_as_uint(sv[r]));
                smax = max(smax, __float_as_uint(sv[r]));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    if (at > at_col[nt] || (window > 0 && at <= at_col[nt] - window)) s[nt][r] = -INFINITY;
            }
        }
        // ---- the weights' power of two
        smax = __reduce_max_sync(0xffffffffu, smax);
        if (smax > 0x7f7fffffu) {
            // A value row that is not finite: whoever sees it gets a score that is not, and the row counts as 0 (0 * NaN would reach
            // the columns that do not see it).
            smax = 0u;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                if (!(sv[r] < INFINITY)) {
                    sv[r] = zv[r] = 0.f;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        if (s[nt][r] != -INFINITY) s[nt][r] = NAN;
                }
                smax = max(smax, __float_as_uint(sv[r]));
            }
            smax = __reduce_max_sync(0xffffffffu, smax);
        }
        // (where no step is 2^KD_SPREAD times another, a column's best key has a weight within that of the largest there can be, whichever rows
        // the column sees: its others keep 11 bits down to 2^-12 of it, and lose what is below 2^-23 of it)
        low = min(low, smin);
        const int ev_new = max(ev, (int)(smax >> 23) - 127 - KD_ROOM);
        // (and weights beyond 2^118, which times 2^8 could pass the largest float, are taken relative to the maximum at once)
        if (__any_sync(0xffffffffu, low < (unsigned)(ev_new + KD_ROOM - KD_SPREAD + 127) << 23) || ev_new + KD_ROOM > 117) wide = true;
        if (ev_new != ev && !wide) {                             // (as a rule only in the first tiles)
            const float f = ev_new - ev > 126 ? 0.f : pow2f(ev - ev_new);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                down[nt] = pow2f(-ev_new);
#pragma unroll
                for (int k = 0; k < MT; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) oacc[nt][k][e] *= f;
            }
        }
        ev = ev_new;
        // ---- maxima: a column's reference moves when a score passes it by 2^8, for all columns of the warp together
        bool moves = wide;
        float mx[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            mx[nt] = s[nt][0];
#pragma unroll
            for (int r = 1; r < 8; ++r) mx[nt] = fmaxf(mx[nt], s[nt][r]);
            mx[nt] *= lsc[nt];
            moves = moves || mx[nt] > m[nt] + 8.f;
        }
        if (__any_sync(0xffffffffu, moves)) {
            bool far = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) mx[nt] = fmaxf(mx[nt], __shfl_xor_sync(0xffffffffu, mx[nt], d));
                mx[nt] = fmaxf(mx[nt], m[nt]);
                far = far || (fabsf(mx[nt]) > KD_FAR && fabsf(mx[nt]) < INFINITY);
            }
            wide = __any_sync(0xffffffffu, wide || far);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float corr = m[nt] == -INFINITY ? 0.f : ex2(m[nt] - mx[nt]);
                float of = corr;
                if (wide) {
                    // the column's own unit: the most that a row which it sees can bring, its weight times its step, is 2^14 of it or less; it never
                    // falls, relative to 1
                    const float from = mx[nt] == -INFINITY ? 0.f : mx[nt];
                    float my = -INFINITY;
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        s[nt][r] = __fmul_rn(s[nt][r], lsc[nt]) - from;
                        if (sv[r] > 0.f) my = fmaxf(my, s[nt][r] + (float)((int)(__float_as_uint(sv[r]) >> 23) - 126));
                    }
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) my = fmaxf(my, __shfl_xor_sync(0xffffffffu, my, d));
                    const int unit = 127 - (int)(__float_as_uint(down[nt]) >> 23);
                    const int to = max((int)ceilf(fmaxf(my, -400.f)) - 14, (int)ceilf(fmaxf((float)unit + (m[nt] - mx[nt]), -400.f)));
                    const int unit_new = min(max(to, KD_UNIT_MIN), 121);
                    of = m[nt] == -INFINITY ? 0.f : ex2(m[nt] - mx[nt] + (float)(unit - unit_new));
                    down[nt] = pow2f(-unit_new);
                }
                m[nt] = mx[nt];
                l[nt] *= corr;
                pz[nt] *= corr;
                // (a head's two columns of the accumulators are this lane's)
#pragma unroll
                for (int k = 0; k < MT; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) oacc[nt][k][e] *= of;
            }
        }
        // ---- weights and the values' product, 32 keys at a time
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            unsigned pe[NT][2], po[NT][2];                       // even columns: the first 16 keys; odd ones: the second 16
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                // (0 while a column has seen nothing: its weights come out as 0; wide: the scores are relative to it already)
                const float ref = wide || m[nt] == -INFINITY ? 0.f : -m[nt], to_log2 = wide ? 1.f : lsc[nt];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float w[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const int r = 4 * b + 2 * k + j;
                        const float p = ex2(fmaf(s[nt][r], to_log2, ref));  // (ex2(-infinity) is 0: a key that is not seen)
                        l[nt] += p;
                        pz[nt] = fmaf(p, zv[r], pz[nt]);
                        w[k] = p * sv[r] * down[nt];
                    }
                    const unsigned x = transpose8x8(half_pair(w[0], w[1]));
                    pe[nt][j] = g & 1 ? 0u : x;
                    po[nt][j] = g & 1 ? x : 0u;
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const unsigned char* v0 = vt + (32 * b + 16 * k + vrow0) * (hd >> 1) + 4 * g;
                const unsigned char* v1 = vt + (32 * b + 16 * k + vrow1) * (hd >> 1) + 4 * g;
#pragma unroll
                for (int u = 0; u < HDP / 64; ++u) {
                    const unsigned wa = *reinterpret_cast<const unsigned*>(v0 + 32 * u), wb = *reinterpret_cast<const unsigned*>(v1 + 32 * u);
                    const unsigned wc = *reinterpret_cast<const unsigned*>(v0 + 8 * (hd >> 1) + 32 * u);
                    const unsigned wd = *reinterpret_cast<const unsigned*>(v1 + 8 * (hd >> 1) + 32 * u);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {                // elements 2 e and 2 e + 1 of the lane's eight
                        const unsigned x0 = __byte_perm(wa, wb, e >> 1 ? 0x7632 : 0x5410) >> (e & 1 ? 8 : 0);
                        const unsigned x1 = __byte_perm(wc, wd, e >> 1 ? 0x7632 : 0x5410) >> (e & 1 ? 8 : 0);
                        unsigned a0, a1, a2, a3;
                        centred(x0, a0, a1);
                        centred(x1, a2, a3);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            mma_half(oacc[nt][4 * u + e], a0, a1, a2, a3, k ? po[nt][0] : pe[nt][0], k ? po[nt][1] : pe[nt][1]);
                    }
                }
            }
        }
        __syncwarp();
        if (lane == 0 && i + STAGES < mine) fetch(i + STAGES, next_page);
    }

    // ---- the warps' results meet in shared memory (in place of the rings)
    __syncthreads();
    float* xo = reinterpret_cast<float*>(smem);                  // [warp][column][HDP], then maxima and sums [warp][column]
    float* xm = xo + KD_WARPS * COLS * HDP;
    float* xl = xm + KD_WARPS * COLS;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const float up = 1.0f / down[nt];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
            l[nt] += __shfl_xor_sync(0xffffffffu, l[nt], d);
            pz[nt] += __shfl_xor_sync(0xffffffffu, pz[nt], d);
        }
        const int c = 4 * nt + t;
        if (g == 0) {
            xm[warp * COLS + c] = m[nt];
            xl[warp * COLS + c] = l[nt];
        }
#pragma unroll
        for (int u = 0; u < HDP / 64; ++u) {
            float* to = xo + ((size_t)warp * COLS + c) * HDP + 64 * u + 8 * g;
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
                const float(&a)[4] = oacc[nt][4 * u + k];
                const float(&b)[4] = oacc[nt][4 * u + k + 1];
                *reinterpret_cast<float4*>(to + 2 * k) = make_float4(fmaf(a[0] + a[1], up, pz[nt]), fmaf(a[2] + a[3], up, pz[nt]),
                                                                     fmaf(b[0] + b[1], up, pz[nt]), fmaf(b[2] + b[3], up, pz[nt]));
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
        if (parts == 1) {
            const float inv = 1.0f / L;
            mv_store4(o + row * hd + d, v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        } else {
            const size_t at = (size_t)blockIdx.x * COLS + c;
            *reinterpret_cast<float4*>(part_o + at * hd + d) = v;
            if (d == 0) *reinterpret_cast<float2*>(part_ml + at * 2) = make_float2(M, L);
        }
    }
    if (parts == 1) return;
    __syncthreads();
    int* ticket = tickets + (size_t)n * pairs + pair;
    if (threadIdx.x == 0) {
        __threadfence();                                         // (the barrier before it makes it stand for the whole block)
        is_last = atomicAdd(ticket, 1) == parts - 1;
        __threadfence();
    }
    __syncthreads();
    if (!is_last) return;
    for (int e = threadIdx.x; e < used * (hd >> 2); e += KD_WARPS * 32) {
        const int c0 = e / (hd >> 2), d = (e - c0 * (hd >> 2)) * 4;
        const int tok = c0 / live_heads, h = c0 - tok * live_heads;
        const size_t row = (size_t)(n + tok) * nh + kvh * group + h0 + h;
        const size_t at0 = (size_t)(blockIdx.x - part * pairs) * COLS + tok * heads + h, step = (size_t)pairs * COLS;
        float M = -INFINITY, L = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s = 0; s < parts; ++s) M = fmaxf(M, __ldcg(part_ml + (at0 + s * step) * 2));
        for (int s = 0; s < parts; ++s) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(part_ml + (at0 + s * step) * 2));
            const float4 x = __ldcg(reinterpret_cast<const float4*>(part_o + (at0 + s * step) * hd + d));
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

// bfloat16; pages of 16 rows or more.  nt: tiles of 4 query columns, 1, 2 or 4 (2 at most above heads of 128).  A tile of columns is
// tokens_per_tile consecutive tokens of one sequence by ``heads`` heads of a kv head's group (tokens_per_tile * heads <= 4 nt; several tokens
// only where heads is the whole group).  The keys are cut into pieces of ``piece`` tiles of 64 (0: such that there are about ``blocks``
// pieces in all); ``grid`` bounds the pieces times kv heads and head tiles: blocks + N * nkv * head_tiles where piece is 0.
// part_o [grid, 4 nt, hd] and part_ml [grid, 4 nt, 2] float32, tickets [N, nkv * head_tiles] (zero).
struct AttentionKv4DecodeArgs {
    const void *q, *pool;
    const int *page_table, *positions, *seq_of, *cu, *starts;
    void* o;
    float *part_o, *part_ml;
    int *tickets, *err;
    cudaStream_t stream;
    int table_stride, page_size, n0, N, tiles, nh, nkv, hd, window, nt, head_tiles, heads, tokens_per_tile, piece, blocks, grid;
    float scale;
};
MV_API int mv_attention_kv4_decode(const void* record) {
    const auto& [q, pool, page_table, positions, seq_of, cu, starts, o, part_o, part_ml, tickets, err, stream, table_stride, page_size, n0, N, tiles, nh, nkv, hd,
                window, nt, head_tiles, heads, tokens_per_tile, piece, blocks, grid, scale] = *static_cast<const AttentionKv4DecodeArgs*>(record);
    if (N <= 0) return 0;
    if (hd % 8 || hd < 8 || hd > KV4_MAX_HEAD_DIM || nkv < 1 || nh % nkv || page_size < 16 || (page_size & (page_size - 1)) || blocks < 1 ||
        grid < 1 || piece < 0 || heads < 1 || heads * head_tiles < nh / nkv || tokens_per_tile < 1 ||
        heads * tokens_per_tile > 4 * nt || (tokens_per_tile > 1 && head_tiles > 1) || ((uintptr_t)pool & 15))
        return (int)cudaErrorInvalidValue;
    int page_shift = 0;
    while ((1 << page_shift) < page_size) ++page_shift;
#define MV_GO(HDP, EXACT, NT)                                                                                                            \
    return kd_launch<HDP, EXACT, NT>(dim3(grid), stream, (const __nv_bfloat16*)q, (const unsigned char*)pool, page_table, table_stride,   \
                                     page_shift, positions, seq_of, cu, n0, starts, (__nv_bfloat16*)o, part_o, part_ml, tickets, N, tiles, nh, nkv, hd, \
                                     scale * 1.4426950408889634f, window, head_tiles, heads, tokens_per_tile, piece, blocks, err)
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
            if (nt == 4) MV_GO(128, true, 4);
        } else {
            if (nt == 1) MV_GO(128, false, 1);
            if (nt == 2) MV_GO(128, false, 2);
            if (nt == 4) MV_GO(128, false, 4);
        }
    } else if (hd == 256) {
        if (nt == 1) MV_GO(256, true, 1);
        if (nt == 2) MV_GO(256, true, 2);
    } else {
        if (nt == 1) MV_GO(256, false, 1);
        if (nt == 2) MV_GO(256, false, 2);
    }
#undef MV_GO
    return (int)cudaErrorInvalidValue;
}
