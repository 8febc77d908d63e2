// Attention of many query tokens a sequence over a cache held in 4 bits (kv4.cuh), on the fifth-generation tensor cores: bfloat16, heads of up to 64,
// pages of any size, optional window.  Flash attention whose two products are tcgen05.mma in half precision with their results in tensor
// memory; the codes become operands on their way into shared memory, so nothing of the cache is written out in between.
//
// Half precision, not bfloat16 (which both operands of a product would have to be): rows read back in bfloat16 are off by 2^-8, weights too,
// and the result by 0.004 where its own rounding is 0.0017; with 11 bits it is 0.0017.  Half's range is small, so powers of two are taken
// out: of a query row its largest element's, of every 32 keys, and of every 32 values, their largest element's (from the rows' numbers:
// a row's ends are zero and zero + 15 steps).  Those of the keys go into the factor of the exponential, those of the values into the
// exponent of the weights, relative to a power of two of the query's own: the most that a row it sees brings so far, score and size together
// (a row that it does not see, or gives no weight, would push the others' weights below half's range).  Where the rows of 32 lie further apart
// than 2^KQ_SPREAD, each has powers of two of its own: such a key block is uneven, and the softmax warps take its scores one by one.
//
// A tile is 256 query rows of one kv head, as two halves of 128 rows: rows are tokens by the heads that share the kv head, so its keys are
// turned into operands once for all of them, a run of a few dozen tokens fills a half, and little is spent on keys that only some rows see.
// One block a multiprocessor at most, and two ways to share the work out (``attention_kv4_prefill_plan`` takes the quicker): whole tiles and kv
// heads, the longest first, where there are enough of them; or to each block the same share of all tiles' and kv heads' key blocks
// (128 keys of a tile, and some for a tile's beginning and end), where a block begins and ends in the middle of a tile's keys and the block
// that finishes a tile last puts its parts together.  2,048 tokens of a prompt, 32 / 8 heads: 49 us whole, 66 us in shares; 700 and 400 tokens
// behind 6,000 and 12,000: 210 us whole (the longest tiles alone), 163 us in shares.
//
//   warps 0 - 3    operands, a key a thread: codes and numbers of a key block, a block ahead in registers, into rings of three stages each in the
//                  128-byte swizzle.  A word's eight codes come out as pairs (0, 4), (1, 5), (2, 6), (3, 7) by masking them into the mantissa of
//                  1024 or 64 and a subtraction; they are left in that order, in which queries are stored too and results are read.
//   warps 4 - 11   queries to shared memory, then softmax, four warps a half, a row a thread: as in attention_prefill_tc.cu;
//   warp 12        products, for either half: S = Q K^T (128 x 128 x 64), O += P V (128 x 64 x 128); S(j + 1) runs under the softmax of S(j);
//   warp 13        what the block works on next, up to four tiles ahead (warps 14 and 15 only fill the warpgroup that gives its registers away).
//
// What bounds it: a key block of a tile takes 3,900 clocks of a multiprocessor, of which the 32,768 exponentials are 2,400 (16 a clock at best;
// measured 9.4 clocks a warp's instruction with two warps a scheduler), and a row's way from scores to weights is some 3,700 when
// nothing is in its way.  So the two warps of a scheduler, one of either half, take turns at the exponentials: the one's wait
// for its scores, maximum and rescaling run under the other's exponentials (without turns they move in step: 228 us where it is 206).  Products take
// some 1,300 clocks (shared memory's 160 KB of operands), the operands' warps some 350 instructions each; without either nothing changes.
// (Tried: a quarter of the exponentials as a cubic on the multiply-add pipes, 197 us for 161; sixteen softmax warps, half a row a thread, 2.7 us
// a key block.)  Every wait on an mbarrier is bounded.
//
// Same mathematics as attention_prefill.cu (reference: crates/mivi-model/src/transformer.rs:114-167, 293-298).
#include "kv4.cuh"
#include "tc_common.cuh"

#include <cuda_fp16.h>

MV_GUARD_SETTER(attention_kv4_prefill)

namespace {

constexpr int KQ_THREADS = 512, KQ_WARPS = KQ_THREADS / 32, MMA_WARP = 12, SEGMENT_WARP = 13;
constexpr int BQ = 128, TILES = 2, ROWS = BQ * TILES, BKV = 128, HD = 64;
constexpr int Q_BYTES = BQ * HD * 2, KV_BYTES = BKV * HD * 2, P_BYTES = BQ * BKV * 2;
constexpr int STAGES = 3, EXPS = 8, KQ_MOST = 1024;              // most sequences, and most tiles, of a launch
constexpr int KQ_EXTRA = 3;                                      // key blocks that a tile's beginning and end count for
constexpr int UNEVEN = 0x7f800000;
// Rows of 32 whose sizes are within KQ_SPREAD powers of two share theirs: the largest's comes to 2^KQ_LIFT, so that a row 2^-12 of it is still 2^15 times the
// least normal half, and whichever row has the weight, its weight is within 2^12 of the largest there can be.
constexpr int KQ_SPREAD = 12, KQ_LIFT = 13;
constexpr int KQ_BARS = TILES * Q_BYTES + 2 * STAGES * KV_BYTES + TILES * P_BYTES, KQ_EXPS = KQ_BARS + 272, KQ_SEGS = KQ_EXPS + EXPS * 32, KQ_TABLES = KQ_SEGS + 4 * 96,
              KQ_OWN = KQ_TABLES + (3 * KQ_MOST + 4) * 4, KQ_SMEM = KQ_OWN + EXPS * BKV * 4 + 1024;
static_assert(KQ_SMEM <= 227 * 1024 - 512, "shared memory");
constexpr unsigned S_COL0 = 0, O_COL0 = 256;                     // of half t: S 128 t on, O 64 t on
static_assert(KQ_OWN % 16 == 0, "read 16 bytes at a time");
// A row's weights are at most 2^(RESCALE_ABOVE + WEIGHT_ROOM) in its unit, which half precision holds; beside the largest so far they keep their
// 11 bits down to 2^-21 of it, and what is below 2^-32 of it is lost.
constexpr float RESCALE_ABOVE = 8.0f, WEIGHT_ROOM = 7.0f;
// Scores are sums of products below 2^(8 + KQ_LIFT) times a factor.  Where that is more than FAR a score's difference from its maximum is worked out by itself,
// as for keys that are uneven: in one step with the factor, the one is rounded and the other is not, and weights pass half's range.
constexpr float FAR = 2.0f;

enum { B_Q = 0, B_KFULL = B_Q + TILES, B_KEMPTY = B_KFULL + STAGES, B_VFULL = B_KEMPTY + STAGES, B_VEMPTY = B_VFULL + STAGES,
       B_SFULL = B_VEMPTY + STAGES, B_PFULL = B_SFULL + TILES, B_PVDONE = B_PFULL + TILES, B_SFREE = B_PVDONE + TILES, B_SEGFULL = B_SFREE + TILES, B_SEGEMPTY = B_SEGFULL + 4,
       B_PARTS = B_SEGEMPTY + 4, B_LAST, B_COUNT };
static_assert(B_COUNT * 8 + 8 <= 272, "barrier area");

// MN-major operand (values: rows are keys, 128 bytes = 64 elements a row), 128-byte swizzle: 8-row groups 1024 bytes apart
__device__ __forceinline__ unsigned long long smem_desc_mn(unsigned addr) {
    unsigned long long d = 0;
    d |= (unsigned long long)((addr & 0x3ffffu) >> 4);
    d |= (unsigned long long)1 << 16;
    d |= (unsigned long long)(1024 >> 4) << 32;
    d |= (unsigned long long)1 << 46;
    d |= (unsigned long long)2 << 61;
    return d;
}
// kind::f16 with both operands in half precision, float32 results, both K-major
__device__ __forceinline__ unsigned instr_desc_half(int m, int n) { return (1u << 4) | ((unsigned)(n >> 3) << 17) | ((unsigned)(m >> 4) << 24); }
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }       // e from -126 to 127
__device__ __forceinline__ int exponent(unsigned bits) { return max(-126, min(126, (int)(bits >> 23) - 127)); }
// the unit of a row's halves: 2^-KQ_LIFT of its largest element's power of two
__device__ __forceinline__ int unit_of(unsigned bits) { return max(-126, (int)(bits >> 23) - 127 - KQ_LIFT); }

// The 8 codes of a word as four pairs of halves, each step * code + zero (rounded once); the codes by way of the mantissa, as in
// attention_kv4_decode.cu
__device__ __forceinline__ uint4 elements(unsigned w, unsigned step, unsigned zero) {
    unsigned e[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const unsigned x = i ? w >> 8 : w;
        unsigned a, b;
        asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(a) : "r"(x));         // 1024 + c
        asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(b) : "r"(x));         // 1024 + 16 c
        asm("sub.f16x2 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(0x64006400u));
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(b) : "r"(b), "r"(0x2c002c00u), "r"(0xd400d400u));
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(e[2 * i]) : "r"(a), "r"(step), "r"(zero));
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(e[2 * i + 1]) : "r"(b), "r"(step), "r"(zero));
    }
    return make_uint4(e[0], e[1], e[2], e[3]);
}
__device__ __forceinline__ unsigned twice(float x) {
    const __half2 h = __float2half2_rn(x);
    return *reinterpret_cast<const unsigned*>(&h);
}

// three at once
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// x / d of whole numbers from 0 to 2^20, with 1 / d rounded: off by less than 2^-2 before it is cut off, and half of 1 / d is added
__device__ __forceinline__ int quotient(int x, float per) { return (int)(((float)x + 0.5f) * per); }

// A run of key blocks of one tile and kv head, as one block works on it
struct Segment {
    int seq, row0, nq, token0;                                   // the tile: its first of the sequence's rows (token * group + head), how many, that row's token
    int pos0, last, first_key;                                   // position of its first and last row, first key that one of them sees
    int kvh, kb, n;                                              // first block of 128 keys and how many (0: the block's share ends in what counts for a beginning)
    int unit, parts, c1, length;                                 // tile and kv head; blocks that work on it, the first of them; share of the whole
    int nb[TILES], first[TILES], past[TILES];                    // of either half of the rows: key blocks, position of the first and last row
    int row_base;                                                // q's row of the sequence's first token
};
static_assert(sizeof(Segment) <= 96, "segment ring");

// EXACT: the head size is 64; else it is hd_, below that, and operands' columns behind it meet zeros of the queries or are not read
template <bool EXACT>
__global__ void __launch_bounds__(KQ_THREADS, 1)
attention_kv4_prefill_kernel(const __nv_bfloat16* __restrict__ q, const unsigned char* __restrict__ pool, const int* __restrict__ page_table,
                             int table_stride, int page_shift, const int* __restrict__ cu, const int* __restrict__ starts,
                             __nv_bfloat16* __restrict__ o, float* __restrict__ part_o, float* __restrict__ part_ml,
                             int* __restrict__ tickets, int n_seqs, int nh, int nkv, int hd_, float scale_log2, int window, int whole, int* __restrict__ err) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ int scan[KQ_WARPS], is_last;
    __shared__ volatile int raising[TILES][4];                   // a warp of a half is at its exponentials
    if (threadIdx.x < 8) raising[threadIdx.x >> 2][threadIdx.x & 3] = 0;
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const unsigned q_s = smem_u32(smem);
    const unsigned k_s = q_s + TILES * Q_BYTES, v_s = k_s + STAGES * KV_BYTES, p_s = v_s + STAGES * KV_BYTES;
    unsigned char* k_ptr = smem + TILES * Q_BYTES;
    unsigned char* v_ptr = k_ptr + STAGES * KV_BYTES;
    unsigned char* p_ptr = v_ptr + STAGES * KV_BYTES;
    unsigned long long* bars = (unsigned long long*)(smem + KQ_BARS);
    unsigned* tmem_holder = (unsigned*)(bars + B_COUNT);
    Segment* segs = reinterpret_cast<Segment*>(smem + KQ_SEGS);  // the segments to come, a ring of four (worked out by a warp of its own)
    int2* exps = reinterpret_cast<int2*>(smem + KQ_EXPS);        // [key block][32 keys]: powers of two of the keys, of the values (a float, or UNEVEN)
    int* own = reinterpret_cast<int*>(smem + KQ_OWN);            // [key block][key]: the same of each key where they are uneven, 16 bits each
    int* seq_first = reinterpret_cast<int*>(smem + KQ_TABLES);   // [sequence + 1]: its first tile
    int* before = seq_first + KQ_MOST + 1;                       // [tile + 1]: key blocks of the tiles before it
    int* seq_of_tile = before + KQ_MOST + 1;
    const unsigned bar0 = smem_u32(bars);
    auto bar = [&](int i) { return bar0 + 8u * (unsigned)i; };
    const int warp = warp_index(), lane = threadIdx.x & 31, tid = threadIdx.x;
    const int group = nh / nkv, hd = EXACT ? HD : hd_;
    const float per_group = 1.0f / (float)group;

    if (tid == 0) {
        for (int t = 0; t < TILES; ++t) mbar_init(bar(B_Q + t), 4);
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(bar(B_KFULL + s), 4);
            mbar_init(bar(B_KEMPTY + s), 1);
            mbar_init(bar(B_VFULL + s), 4);
            mbar_init(bar(B_VEMPTY + s), 1);
        }
        for (int t = 0; t < TILES; ++t) {
            mbar_init(bar(B_SFULL + t), 1);
            mbar_init(bar(B_PFULL + t), 4);
            mbar_init(bar(B_PVDONE + t), 1);
            mbar_init(bar(B_SFREE + t), 4);
        }
        for (int k = 0; k < 4; ++k) {
            mbar_init(bar(B_SEGFULL + k), 1);
            mbar_init(bar(B_SEGEMPTY + k), 13);
        }
        mbar_init(bar(B_PARTS), 8);
        mbar_init(bar(B_LAST), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem_base = *tmem_holder;
    mv_pdl_wait();

    // ---- the row of all key blocks: first tile of every sequence, then key blocks before every tile
    auto block_scan = [&](int v, int& all) {                     // sum of the threads before this one
        int inc = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += x;
        }
        __syncthreads();
        if (lane == 31) scan[warp] = inc;
        __syncthreads();
        int base = 0;
        all = 0;
        for (int w = 0; w < KQ_WARPS; ++w) {
            if (w < warp) base += scan[w];
            all += scan[w];
        }
        return base + inc - v;
    };
    int n_tiles = 0, n_blocks = 0;
    for (int b0 = 0; b0 < n_seqs; b0 += KQ_THREADS) {
        const int b = b0 + tid;
        int all;
        const int mine = b < n_seqs ? ((cu[b + 1] - cu[b]) * group + ROWS - 1) / ROWS : 0;
        const int at = n_tiles + block_scan(mine, all);
        if (b < n_seqs) seq_first[b] = at;
        n_tiles += all;
    }
    if (tid == 0) seq_first[n_seqs] = n_tiles;
    __syncthreads();
    n_tiles = min(n_tiles, KQ_MOST);
    // rows of tile i of sequence b, from its first one on
    auto place = [&](int b, int i, Segment& g) {
        const int rows = (cu[b + 1] - cu[b]) * group;
        g.seq = b;
        g.row0 = i * ROWS;
        g.nq = min(ROWS, rows - g.row0);
        g.token0 = quotient(g.row0, per_group);
        g.pos0 = starts[b] + g.token0;
        g.last = starts[b] + quotient(g.row0 + g.nq - 1, per_group);
        g.first_key = window > 0 ? max(0, g.pos0 - window + 1) : 0;
    };
    for (int i0 = 0; i0 < n_tiles; i0 += KQ_THREADS) {
        const int i = i0 + tid;
        int nb = 0, b = 0;
        if (i < n_tiles) {
            int lo = 0, hi = n_seqs;                             // the last sequence whose first tile is at most i (none is empty)
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (seq_first[mid] <= i) lo = mid;
                else hi = mid;
            }
            b = lo;
            Segment g;
            place(b, i - seq_first[b], g);
            nb = g.last / BKV + 1 - g.first_key / BKV;
        }
        int all;
        const int at = n_blocks + block_scan(nb, all);
        if (i < n_tiles) {
            before[i] = at;
            seq_of_tile[i] = b;
        }
        n_blocks += all;
    }
    if (tid == 0) before[n_tiles] = n_blocks;
    __syncthreads();
    // shares: block c works on what lies from begin_of(c) to begin_of(c + 1); a tile's kv head takes KQ_EXTRA and its key blocks
    // (a share is one at least: the blocks of a tile are counted, and each of them has a part)
    const int total = (n_blocks + KQ_EXTRA * n_tiles) * nkv, C = whole ? (int)gridDim.x : max(1, min((int)gridDim.x, total));
    const double share_of = (double)total / (double)C, per_share = (double)C / (double)total;
    auto begin_of = [&](int c) { return c >= C ? total : (int)((double)c * share_of); };
    auto block_of = [&](int x) {
        int c = min(C - 1, (int)((double)x * per_share));
        while (begin_of(c) > x) --c;
        while (begin_of(c + 1) <= x) ++c;
        return c;
    };
    auto before_of = [&](int i) { return (before[i] + KQ_EXTRA * i) * nkv; };
    const int units = n_tiles * nkv;
    // whole: where the k-th tile and kv head of this block lies; the last, longest tiles first, and back and forth over the blocks, so that
    // who had the longest of one pass has the shortest of the next
    auto whole_unit = [&](int k, int& tile) {
        const int i = k * C + (k & 1 ? C - 1 - (int)blockIdx.x : (int)blockIdx.x), unit = units - 1 - i;
        if (i >= units) return -1;
        tile = unit / nkv;
        return before_of(tile) + (unit - tile * nkv) * (before[tile + 1] - before[tile] + KQ_EXTRA);
    };
    const int u_first = begin_of(blockIdx.x), u_past = whole ? total : begin_of(blockIdx.x + 1);
    // what lies at u (tile: its tile or an earlier one; moved on)
    auto segment = [&](int u, int& tile) {
        while (tile + 1 < n_tiles && before_of(tile + 1) <= u) ++tile;
        Segment g;
        const int b = seq_of_tile[tile], nb = before[tile + 1] - before[tile], long_ = nb + KQ_EXTRA, rel = u - before_of(tile);
        place(b, tile - seq_first[b], g);
        g.kvh = min(nkv - 1, (int)((float)rel / (float)long_));
        while (g.kvh * long_ > rel) --g.kvh;
        while ((g.kvh + 1) * long_ <= rel) ++g.kvh;
        const int u0 = u - (rel - g.kvh * long_), k0 = max(0, u - u0 - KQ_EXTRA), k1 = max(0, min(u_past, u0 + long_) - u0 - KQ_EXTRA);
        g.kb = g.first_key / BKV + k0;
        g.n = k1 - k0;
        g.length = min(u_past, u0 + long_) - u;
        g.unit = tile * nkv + g.kvh;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            g.first[t] = g.pos0 + quotient(g.row0 + t * BQ, per_group) - g.token0;
            g.past[t] = g.pos0 + quotient(g.row0 + min(g.nq, (t + 1) * BQ) - 1, per_group) - g.token0;
            g.nb[t] = g.nq > t * BQ ? max(0, min(g.n, g.past[t] / BKV + 1 - g.kb)) : 0;
        }
        g.row_base = cu[b];
        g.c1 = whole ? (int)blockIdx.x : block_of(u0 + KQ_EXTRA);
        g.parts = whole ? 1 : block_of(u0 + long_ - 1) - g.c1 + 1;
        return g;
    };
    // the k-th segment, for a warp that then reads it and gives it back with ``next``; null: there is none, or a wait ran out
    auto segment_at = [&](int k) -> const Segment* {
        if (!mbar_wait_warp(bar(B_SEGFULL + (k & 3)), (unsigned)(k >> 2) & 1u, err, 168)) return nullptr;
        return segs[k & 3].n < 0 ? nullptr : segs + (k & 3);
    };
    auto next = [&](int k) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_SEGEMPTY + (k & 3)));
    };

    if (warp < 4) {
        // registers move from this warpgroup and the last to the softmax warps' (128 x 64 + 128 x 32 + 256 x 208 of the 512 x 128 at launch)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        const int page_size = 1 << page_shift, key_of = warp * 32 + lane;
        const size_t head_bytes = kv4_head_bytes(page_size, hd);
        bool ok = true;
        int it = 0;
        for (int k = 0; ok; next(k), ++k) {
            const Segment* sg = segment_at(k);
            if (sg == nullptr) break;
            struct { int first_key, last, kvh, kb, n; } g = {sg->first_key, sg->last, sg->kvh, sg->kb, sg->n};
            const int* table = page_table + (size_t)sg->seq * table_stride;
            // this thread's key of the block, if some row sees it (else zeros): its keys, values and numbers, each fetched again as soon as
            // it is turned into operands
            uint4 kc[2], vc[2];
            uint2 np;
            const unsigned char* from = nullptr;
            int row = 0;
            auto place_of = [&](int kb) {
                const int key = kb * BKV + key_of;
                from = nullptr;
                row = key & (page_size - 1);
                if (key >= g.first_key && key <= g.last)
                    from = pool + ((size_t)mv_read_page(table[key >> page_shift]) * nkv + g.kvh) * head_bytes;
            };
            auto fetch = [&](uint4 (&w)[2], int at) {
                w[0] = w[1] = make_uint4(0u, 0u, 0u, 0u);
                if (from != nullptr) {
                    if (!EXACT) {                                // (a row is at 4 bytes)
                        const unsigned* x = reinterpret_cast<const unsigned*>(from + at + row * (hd >> 1));
                        unsigned c[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) c[i] = 8 * i < hd ? x[i] : 0u;
                        w[0] = make_uint4(c[0], c[1], c[2], c[3]);
                        w[1] = make_uint4(c[4], c[5], c[6], c[7]);
                    } else if (page_shift) {
                        const uint4* x = reinterpret_cast<const uint4*>(from + at + row * (HD / 2));
                        w[0] = x[0];
                        w[1] = x[1];
                    } else {                                     // (pages of one token are 72 bytes a kv head: 8 is all they are aligned to)
                        const uint2* x = reinterpret_cast<const uint2*>(from + at);
                        w[0] = make_uint4(x[0].x, x[0].y, x[1].x, x[1].y);
                        w[1] = make_uint4(x[2].x, x[2].y, x[3].x, x[3].y);
                    }
                }
            };
            auto fetch_numbers = [&]() { np = from != nullptr ? *reinterpret_cast<const uint2*>(from + page_size * hd + row * 8) : make_uint2(0u, 0u); };
            place_of(g.kb);
            fetch_numbers();
            fetch(kc, 0);
            fetch(vc, page_size * (hd >> 1));
            for (int j = 0; j < g.n; ++j, ++it) {
                const int s = it % STAGES;
                const unsigned ph = (unsigned)(it / STAGES) & 1u;
                Kv4Params p = kv4_params(np);
                kv4_poison(p);
                const bool there = from != nullptr;
                if (j + 1 < g.n) {
                    place_of(g.kb + j + 1);
                    fetch_numbers();
                }
                // powers of two of the warp's keys and values (a row that is not finite has no say)
                const float big_k = fmaxf(fabsf(p.kz), fabsf(fmaf(15.f, p.ks, p.kz))), big_v = fmaxf(fabsf(p.vz), fabsf(fmaf(15.f, p.vs, p.vz)));
                const unsigned bits_k = big_k < INFINITY ? __float_as_uint(big_k) : 0u, bits_v = __float_as_uint(big_v);
                const unsigned top_k = __reduce_max_sync(0xffffffffu, bits_k), top_v = __reduce_max_sync(0xffffffffu, bits_v);
                int ek = unit_of(top_k), ev = unit_of(top_v);
                // (a key of zeros scores 0 in any unit; a value of zeros may have the weight that the others' are to be measured by)
                const bool uneven = __any_sync(0xffffffffu, there && ((bits_k != 0u && bits_k + (KQ_SPREAD << 23) < top_k) || bits_v + (KQ_SPREAD << 23) < top_v));
                if (uneven) {
                    ek = unit_of(bits_k);
                    ev = unit_of(bits_v);
                }
                auto put = [&](unsigned char* stage, const uint4 (&w)[2], float step, float zero, float down) {
                    const unsigned st = twice(step * down), z = twice(zero * down);
                    unsigned char* to = stage + key_of * 128;
                    const int x = key_of & 7;
                    const unsigned c[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
                    for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(to + ((i ^ x) << 4)) = elements(c[i], st, z);
                };
                auto hand_over = [&](int b) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(b + s));
                };
                if (!(ok = mbar_wait_warp(bar(B_KEMPTY + s), ph ^ 1u, err, 161))) break;
                if (lane == 0) exps[(it % EXPS) * 4 + warp] = make_int2(ek, uneven ? UNEVEN : __float_as_int((float)ev));
                if (uneven) own[(it % EXPS) * BKV + key_of] = (ek & 0xffff) | (ev << 16);
                put(k_ptr + s * KV_BYTES, kc, p.ks, p.kz, pow2f(-ek));
                if (j + 1 < g.n) fetch(kc, 0);
                hand_over(B_KFULL);
                if (!(ok = mbar_wait_warp(bar(B_VEMPTY + s), ph ^ 1u, err, 162))) break;
                put(v_ptr + s * KV_BYTES, vc, p.vs, p.vz, pow2f(-ev));
                if (j + 1 < g.n) fetch(vc, page_size * (hd >> 1));
                hand_over(B_VFULL);
            }
        }
    } else if (warp >= MMA_WARP) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
        if (warp == MMA_WARP) {
            const unsigned idesc_qk = instr_desc_half(BQ, BKV), idesc_pv = instr_desc_half(BQ, HD) | (1u << 16);
            bool ok = true;
            int it = 0, seen[TILES] = {0, 0}, done[TILES] = {0, 0};   // segments and key blocks of either half of the rows so far
            for (int sk = 0; ok; next(sk), ++sk) {
                const Segment* sg = segment_at(sk);
                if (sg == nullptr) break;
                const int nb[TILES] = {sg->nb[0], sg->nb[1]}, n = sg->n;
#pragma unroll
                for (int t = 0; t < TILES; ++t)
                    if (ok && nb[t] > 0) ok = mbar_wait_warp(bar(B_Q + t), (unsigned)seen[t]++ & 1u, err, 163);
                if (!ok) break;
                // scores of key block j of the segment
                auto scores = [&](int j) {
                    const int s = (it + j) % STAGES;
                    if (!mbar_wait_warp(bar(B_KFULL + s), (unsigned)((it + j) / STAGES) & 1u, err, 164)) return false;
#pragma unroll
                    for (int t = 0; t < TILES; ++t) {
                        if (j >= nb[t]) continue;
                        // its columns are in the softmax warps' registers since the key block before
                        if (done[t] + j > 0 && !mbar_wait_warp(bar(B_SFREE + t), (unsigned)(done[t] + j - 1) & 1u, err, 165)) return false;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const unsigned long long qd = smem_desc(q_s + t * Q_BYTES), kd = smem_desc(k_s + s * KV_BYTES);
                        if (elect_one()) {
#pragma unroll
                            for (int k = 0; k < HD / 16; ++k)
                                mma_f16(tmem_base + S_COL0 + (unsigned)(t * BKV), qd + 2 * k, kd + 2 * k, idesc_qk, k > 0 ? 1u : 0u);
                            mma_commit(bar(B_SFULL + t));
                        }
                    }
                    if (elect_one()) mma_commit(bar(B_KEMPTY + s));
                    return true;
                };
                if (!(ok = scores(0))) break;
                for (int j = 0; j < n; ++j) {
                    if (j + 1 < n && !(ok = scores(j + 1))) break;
                    const int s = (it + j) % STAGES;
                    if (!(ok = mbar_wait_warp(bar(B_VFULL + s), (unsigned)((it + j) / STAGES) & 1u, err, 167))) break;
#pragma unroll
                    for (int t = 0; t < TILES; ++t) {
                        if (!ok || j >= nb[t]) continue;
                        if (!(ok = mbar_wait_warp(bar(B_PFULL + t), (unsigned)(done[t] + j) & 1u, err, 166))) continue;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const unsigned long long pd = smem_desc(p_s + t * P_BYTES), vd = smem_desc_mn(v_s + s * KV_BYTES);
                        if (elect_one()) {
#pragma unroll
                            for (int k = 0; k < BKV / 16; ++k)
                                mma_f16(tmem_base + O_COL0 + (unsigned)(t * HD), pd + (k >> 2) * (BQ * 128 / 16) + (k & 3) * 2, vd + k * 128, idesc_pv,
                                        (j > 0 || k > 0) ? 1u : 0u);
                            mma_commit(bar(B_PVDONE + t));
                        }
                    }
                    if (!ok) break;
                    if (elect_one()) mma_commit(bar(B_VEMPTY + s));
                }
                it += n;
                done[0] += nb[0];
                done[1] += nb[1];
            }
        } else if (warp == SEGMENT_WARP) {
            int u = u_first, tile = 0;
            if (!whole)
                for (int hi = n_tiles; hi - tile > 1;) {
                    const int mid = (tile + hi) >> 1;
                    if (before_of(mid) <= u) tile = mid;
                    else hi = mid;
                }
            for (int k = 0;;) {
                Segment g;
                g.n = -1;
                if (whole) u = whole_unit(k, tile);
                if (u >= 0 && u < u_past) {
                    g = segment(u, tile);
                    u += g.length;
                    if (g.n == 0) continue;
                }
                if (!mbar_wait_warp(bar(B_SEGEMPTY + (k & 3)), (unsigned)(k >> 2 & 1) ^ 1u, err, 160)) break;
                if (lane == 0) segs[k & 3] = g;
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_SEGFULL + (k & 3)));
                ++k;
                if (g.n < 0) break;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int t = (warp - 4) >> 2, quarter = warp & 3;
        const int r = quarter * 32 + lane;                       // this thread's row within its half
        const unsigned lane_addr = (unsigned)(quarter * 32) << 16;
        const unsigned s_addr = tmem_base + lane_addr + S_COL0 + (unsigned)(t * BKV), o_addr = tmem_base + lane_addr + O_COL0 + (unsigned)(t * HD);
        unsigned char* p_row = p_ptr + t * P_BYTES + r * 128;
        unsigned char* q_rows = smem + t * Q_BYTES;
        bool ok = true;
        int it = 0, done = 0, merges = 0;
        for (int k = 0;; next(k), ++k) {
            const Segment* sg = segment_at(k);
            if (sg == nullptr) break;
            const int my_nb = sg->nb[t], parts = sg->parts;
            if (!ok) break;                                      // (a wait ran out: the others' do, too)
            const bool live = t * BQ + r < sg->nq;
            int pos = -1, row_at = -1;                           // the row's position; its place among the rows of q and o
            if (live) {
                const int packed = sg->row0 + t * BQ + r, token = quotient(packed, per_group);
                pos = sg->pos0 + token - sg->token0;
                row_at = (sg->row_base + token) * nh + sg->kvh * group + (packed - token * group);
            }
            // ---- the row's elements to shared memory, as halves in the order of the codes' pairs
            int ex = 0;
            bool fine = true;                                    // the row's elements are finite
            if (my_nb > 0) {                                     // (a half without key blocks is not waited for, and may be segments ahead)
                const uint4* from = reinterpret_cast<const uint4*>(q + (size_t)max(row_at, 0) * hd);
                uint4 raw[8];
                float top = 0.f;
#pragma unroll
                for (int c = 0; c < 8; ++c) raw[c] = live && (EXACT || 8 * c < hd) ? from[c] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const unsigned x[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(x[e] << 16)), fabsf(__uint_as_float(x[e] & 0xffff0000u))));
                }
                // (fmaxf passes over what is not a number)
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const unsigned x[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) fine = fine && (x[e] & 0x7f80u) != 0x7f80u && (x[e] & 0x7f800000u) != 0x7f800000u;
                }
                ex = top > 0.f && fine ? exponent(__float_as_uint(top)) : 0;
                const float down = pow2f(-ex);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const unsigned x[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
                    unsigned w[4];                               // elements (0, 4), (1, 5), (2, 6), (3, 7)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float a = __uint_as_float(e & 1 ? x[e >> 1] & 0xffff0000u : x[e >> 1] << 16);
                        const float b = __uint_as_float(e & 1 ? x[2 + (e >> 1)] & 0xffff0000u : x[2 + (e >> 1)] << 16);
                        const __half2 v = __floats2half2_rn(a * down, b * down);
                        w[e] = *reinterpret_cast<const unsigned*>(&v);
                    }
                    *reinterpret_cast<uint4*>(q_rows + r * 128 + ((c ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_Q + t));
            }
            float m = -INFINITY, l = fine ? 0.f : NAN;           // m: the row's reference, log2 units
            float rel = 0.f;                                     // the accumulator's unit is 2^(rel - WEIGHT_ROOM) of what weights relative to 2^m come to
            int j = 0;
            bool uneven = false;
            auto hand_over = [&]() {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_PFULL + t));
            };
            auto free_scores = [&]() {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_SFREE + t));
            };
            // the row's reference follows its largest score, by 2^RESCALE_ABOVE at least
            auto follow = [&](float mx) {
                if (mx > m + RESCALE_ABOVE) {
                    l *= m == -INFINITY ? 0.f : ex2(m - mx);
                    m = mx;
                }
                return m == -INFINITY ? 0.f : m;
            };
            // the accumulator's unit follows the most that a row brings (relative to 2^m: its weight times its values' power of two); its factor
            auto measure = [&](float most, float m_old) {
                float o_corr = 1.0f;
                if (m != -INFINITY) {                            // (until then all of its weights are 0, and so is its accumulator)
                    rel += m_old - m;                            // (from -infinity: it has no unit yet)
                    if (most > rel + RESCALE_ABOVE) {
                        o_corr = ex2(rel - most);
                        rel = most;
                    }
                }
                return o_corr;
            };
            auto make_room = [&](float o_corr) {
                // P (shared memory) and O (tensor memory) are the key block before's until its product is done
                if (j > 0) {
                    if (!mbar_wait_warp(bar(B_PVDONE + t), (unsigned)(done + j - 1) & 1u, err, 170)) return false;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                }
                if (j > 0 && __any_sync(0xffffffffu, o_corr != 1.0f)) {
#pragma unroll
                    for (int c = 0; c < HD; c += 16) {                  // (16 at a time: the scores lie in 128 registers)
                        unsigned v[16];
                        tmem_ld16(o_addr + (unsigned)c, v);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * o_corr);
                        tmem_st16(o_addr + (unsigned)c, v);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
                return true;
            };
            while (ok && j < my_nb) {
                uneven = false;
                for (; j < my_nb; ++j) {
                    ok = mbar_wait_warp(bar(B_SFULL + t), (unsigned)(done + j) & 1u, err, 169);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    unsigned s[4][32];
                    tmem_ld32(s_addr, s[0]);
                    tmem_ld32(s_addr + 32, s[1]);
                    tmem_ld32(s_addr + 64, s[2]);
                    tmem_ld32(s_addr + 96, s[3]);
                    const int2* e = exps + ((it + j) % EXPS) * 4;
                    float f[4], ev[4];                           // 32 keys' factor to log2 units, their values' power of two
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int2 x = e[c];
                        f[c] = scale_log2 * pow2f(max(-126, min(120, ex + x.x)));
                        ev[c] = __int_as_float(x.y);
                        uneven = uneven || x.y == UNEVEN || f[c] > FAR;
                    }
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (__any_sync(0xffffffffu, uneven)) break;
                    free_scores();
                    const int key0 = (sg->kb + j) * BKV;
                    // warp-uniform: some row of the half does not see the whole block
                    if (key0 + BKV - 1 > sg->first[t] || (window > 0 && key0 <= sg->past[t] - window)) {
                        const int past = pos - key0 + 1, from = window > 0 ? past - window : 0;
#pragma unroll
                        for (int c = 0; c < 4; ++c)
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (32 * c + i >= past || 32 * c + i < from) s[c][i] = 0xff800000u;
                    }
                    float mx = -INFINITY, top[4];                // top: of 32 keys
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        float a[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int i = 0; i < 32; i += 2) a[(i >> 1) & 3] = max3(a[(i >> 1) & 3], __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
                        top[c] = max3(a[0], a[1], fmaxf(a[2], a[3])) * f[c];
                        mx = fmaxf(mx, top[c]);
                    }
                    const float m_old = m, ref = follow(mx);
                    float most = -INFINITY;
#pragma unroll
                    for (int c = 0; c < 4; ++c) most = fmaxf(most, top[c] - ref + ev[c]);
                    const float o_corr = measure(most, m_old);
                    // exponent of 32 keys' weights less that of their scores, and what brings their sum back to 2^m
                    float lift[4], back[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        lift[c] = fmaxf(ev[c] - rel + WEIGHT_ROOM, -60.f);
                        back[c] = ex2(-lift[c]);
                    }
                    if (!(ok = make_room(o_corr))) break;
                    // weights relative to the accumulator's unit, eight at a time (b); their sums relative to 2^m
                    auto raise = [&](int b) {
                        const int c = b >> 2;
                        const float from = lift[c] - ref;
#pragma unroll
                        for (int i = 8 * (b & 3); i < 8 * (b & 3) + 8; i += 2) {
                            const float2 x = fma2(make_float2(__uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1])), make_float2(f[c], f[c]), make_float2(from, from));
                            s[c][i] = __float_as_uint(ex2(x.x));
                            s[c][i + 1] = __float_as_uint(ex2(x.y));
                        }
                    };
                    float2 sum = make_float2(0.f, 0.f);
                    auto put = [&](int b) {
                        const int c = b >> 2, q4 = b & 3;
                        unsigned w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float2 p = make_float2(__uint_as_float(s[c][8 * q4 + 2 * i]), __uint_as_float(s[c][8 * q4 + 2 * i + 1]));
                            sum = i + q4 ? add2(sum, p) : p;
                            const __half2 v = __floats2half2_rn(p.x, p.y);
                            w[i] = *reinterpret_cast<const unsigned*>(&v);
                        }
                        *reinterpret_cast<uint4*>(p_row + (c >> 1) * (BQ * 128) + (((4 * (c & 1) + q4) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                        if (q4 == 3) l = fmaf(sum.x + sum.y, back[c], l);
                    };
                    // the two warps of a scheduler take turns (a matter of speed only: nothing waits for good)
                    if (t == 0) raising[0][quarter] = 1;
                    for (int k = 0; k < 64 && raising[t ^ 1][quarter]; ++k) ;
                    if (t == 1) raising[1][quarter] = 1;
                    __syncwarp();
                    constexpr int AHEAD = 3;                          // (the unit's latency: 207 us with 1, 204 with 3)
#pragma unroll
                    for (int b = 0; b < AHEAD; ++b) raise(b);
#pragma unroll
                    for (int b = 0; b < 16; ++b) {
                        if (b + AHEAD < 16) raise(b + AHEAD);
                        if (b + AHEAD == 12) raising[t][quarter] = 0;  // (its last ones are under way when the other comes)
                        put(b);
                    }
                    hand_over();
                }
                if (!__any_sync(0xffffffffu, ok && uneven)) break;
                // Every key has powers of two of its own: its score is taken by itself, and its weight and its values' size are added up apart.  (A
                // path of its own, outside of the loop, which reads the scores from tensor memory again.  400 and 700 tokens behind 6,000 and 12,000, which
                // never come here, take 163 us so, 214 us where the scores are held in registers through it, and 161 us without it.  A block that
                // comes here takes some four times as long.)
                const int past = pos - (sg->kb + j) * BKV + 1, from = window > 0 ? past - window : 0;
                auto each = [&](auto use) {                      // use(32 keys, i, score in log2 units, its values' power of two)
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        unsigned x[32];
                        tmem_ld32(s_addr + 32u * (unsigned)c, x);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                        const int2 shared = exps[((it + j) % EXPS) * 4 + c];
                        const int* own_of = own + ((it + j) % EXPS) * BKV + 32 * c;
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const int k = own_of[i], ek = shared.y == UNEVEN ? (int)(short)k : shared.x;
                            const float v = shared.y == UNEVEN ? (float)(k >> 16) : __int_as_float(shared.y);
                            const bool seen = 32 * c + i < past && 32 * c + i >= from;
                            use(c, i, seen ? __fmul_rn(__uint_as_float(x[i]), scale_log2 * pow2f(max(-126, min(120, ex + ek)))) : -INFINITY, v);
                        }
                    }
                };
                float mx = -INFINITY, most = -INFINITY, sum = 0.f;
                each([&](int, int, float x, float) { mx = fmaxf(mx, x); });
                const float m_old = m, ref = follow(mx);
                each([&](int, int, float x, float v) {
                    sum += ex2(x - ref);
                    most = fmaxf(most, x - ref + v);
                });
                l += sum;
                if (!(ok = make_room(measure(most, m_old)))) break;
                unsigned w[4];
                float first = 0.f;
                each([&](int c, int i, float x, float v) {
                    const float p = ex2(x - ref + (v - rel + WEIGHT_ROOM));
                    if (i & 1) {
                        const __half2 h = __floats2half2_rn(first, p);
                        w[(i >> 1) & 3] = *reinterpret_cast<const unsigned*>(&h);
                    }
                    first = p;
                    if ((i & 7) == 7) *reinterpret_cast<uint4*>(p_row + (c >> 1) * (BQ * 128) + (((4 * (c & 1) + (i >> 3)) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                });
                free_scores();
                hand_over();
                ++j;
            }
            if (ok && my_nb > 0) ok = mbar_wait_warp(bar(B_PVDONE + t), (unsigned)(done + my_nb - 1) & 1u, err, 171);
            if (ok && my_nb > 0) asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (!ok) break;
            // ---- the rows out, by the queries' place in shared memory (a warp's own rows: whole lines leave), or a part of them
            const bool read = ok && my_nb > 0;
            // (in two factors: the unit may lie beyond the floats where the result does not.  A part is divided by its sum, too: it may pass them before.)
            const float up0 = ex2(0.5f * (rel - WEIGHT_ROOM)), up1 = l == 0.f ? 0.f : up0 / l;
            // a block has two parts at most: of a tile that it begins, and of one that another block began
            const int slot = 2 * blockIdx.x + (sg->c1 == (int)blockIdx.x ? 1 : 0);
            float4* mine = reinterpret_cast<float4*>(part_o) + (size_t)slot * (ROWS * HD / 4) + t * BQ + r;
            if (my_nb > 0 || parts > 1) {
#pragma unroll
                for (int c = 0; c < HD; c += 32) {
                    unsigned v[32];
                    if (read) {
                        tmem_ld32(o_addr + (unsigned)c, v);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = 0u;
                    }
#pragma unroll
                    for (int d = 0; d < 32; d += 8) {            // stored as 0, 4, 1, 5, 2, 6, 3, 7
                        float x[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(v[d + i]) * up0 * up1;
                        if (parts == 1) {
                            const uint4 w = make_uint4(bits(__floats2bfloat162_rn(x[0], x[2])), bits(__floats2bfloat162_rn(x[4], x[6])),
                                                       bits(__floats2bfloat162_rn(x[1], x[3])), bits(__floats2bfloat162_rn(x[5], x[7])));
                            *reinterpret_cast<uint4*>(q_rows + r * 128 + ((((c + d) >> 3) ^ (r & 7)) << 4)) = w;
                        } else if (live) {
                            mine[(size_t)((c + d) >> 2) * ROWS] = make_float4(x[0], x[2], x[4], x[6]);
                            mine[(size_t)(((c + d) >> 2) + 1) * ROWS] = make_float4(x[1], x[3], x[5], x[7]);
                        }
                    }
                }
            }
            auto rows_out = [&]() {                              // a warp's 32 rows from shared memory, four at a time
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int rr = 4 * i + (lane >> 3), row = __shfl_sync(0xffffffffu, row_at, rr), c = lane & 7;
                    const uint4 w = *reinterpret_cast<const uint4*>(q_rows + (quarter * 32 + rr) * 128 + ((c ^ (rr & 7)) << 4));
                    if (row >= 0 && (EXACT || 8 * c < hd)) *reinterpret_cast<uint4*>(o + (size_t)row * hd + 8 * c) = w;
                }
                __syncwarp();
            };
            if (parts == 1) {
                if (my_nb > 0) rows_out();
            } else {
                if (live) *reinterpret_cast<float2*>(part_ml + ((size_t)slot * ROWS + t * BQ + r) * 2) = make_float2(m, l);
                // (is_last changes when all eight warps have come here again, so after they have read it)
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_PARTS));
                if (warp == 4) {
                    if (!mbar_wait_warp(bar(B_PARTS), (unsigned)merges & 1u, err, 172)) break;
                    if (lane == 0) {
                        __threadfence();
                        is_last = atomicAdd(tickets + sg->unit, 1) == parts - 1;
                        if (is_last) tickets[sg->unit] = 0;
                        __threadfence();
                        mbar_arrive(bar(B_LAST));
                    }
                }
                if (!mbar_wait_warp(bar(B_LAST), (unsigned)merges & 1u, err, 173)) break;
                ++merges;
                const bool last = is_last;
                if (last && t * BQ < sg->nq) {
                    // A part: reference (log2 units), sum, mean of the values.  Where nothing was seen the sum is 0 and the part counts nothing;
                    // where all that was seen is not a number the sum is not one, and stays so.
                    auto weight = [](float mx, float sum, float M) { return mx == -INFINITY ? (sum == 0.f ? 0.f : NAN) : ex2(mx - M); };
                    const int row = t * BQ + r, c1 = sg->c1;
                    auto slot_of = [&](int p) { return p ? 2 * (c1 + p) : 2 * c1 + 1; };
                    float M = -INFINITY, L = 0.f;
                    float4 sum[HD / 4];
#pragma unroll
                    for (int c = 0; c < HD / 4; ++c) sum[c] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (live) {
                        for (int p = 0; p < parts; ++p) M = fmaxf(M, __ldcg(part_ml + ((size_t)slot_of(p) * ROWS + row) * 2));
                        for (int p = 0; p < parts; ++p) {
                            const float2 ml = __ldcg(reinterpret_cast<const float2*>(part_ml + ((size_t)slot_of(p) * ROWS + row) * 2));
                            const float w = ml.y * weight(ml.x, ml.y, M);
                            L += w;
                            const float4* from = reinterpret_cast<const float4*>(part_o) + (size_t)slot_of(p) * (ROWS * HD / 4) + row;
#pragma unroll
                            for (int c = 0; c < HD / 4; ++c) {
                                const float4 x = __ldcg(from + (size_t)c * ROWS);
                                sum[c].x = fmaf(x.x, w, sum[c].x); sum[c].y = fmaf(x.y, w, sum[c].y);
                                sum[c].z = fmaf(x.z, w, sum[c].z); sum[c].w = fmaf(x.w, w, sum[c].w);
                            }
                        }
                    }
                    const float over = 1.0f / L;
#pragma unroll
                    for (int c = 0; c < HD / 8; ++c) {
                        const float4 a = sum[2 * c], b = sum[2 * c + 1];
                        *reinterpret_cast<uint4*>(q_rows + r * 128 + ((c ^ (r & 7)) << 4)) =
                            make_uint4(bits(__floats2bfloat162_rn(a.x * over, a.y * over)), bits(__floats2bfloat162_rn(a.z * over, a.w * over)),
                                       bits(__floats2bfloat162_rn(b.x * over, b.y * over)), bits(__floats2bfloat162_rn(b.z * over, b.w * over)));
                    }
                    rows_out();
                }
            }
            it += sg->n;
            done += my_nb;
        }
    }
    // Only now may the next kernel's blocks be given multiprocessors: signalled earlier, they would take the places of this grid's own
    // later blocks and sit there waiting.
    mv_pdl_launch_dependents();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == MMA_WARP) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
    }
}

}  // namespace

// bfloat16, heads of 8 to 64 in steps of 8.  cu and starts are those of ``n_seqs`` neighbouring sequences (cu counts from q's first row), page_table their rows; at most
// 1,024 sequences of at least one token, and 1,024 tiles of 256 rows (a sequence's tokens times the heads of a kv head).  whole: tiles and
// kv heads are dealt out whole to grid blocks (tiles * nkv at most), back and forth; else grid blocks share all key blocks.  Either way a block a
// multiprocessor at most.  part_o [2 grid, 16, 256, 4],
// part_ml [2 grid, 256, 2] float32 and tickets [tiles * nkv] (zero) are used unless whole.
MV_API int mv_attention_kv4_prefill(const void* q, const void* pool, const int* page_table, int table_stride, int page_size, const int* cu,
                                    const int* starts, void* o, float* part_o, float* part_ml, int* tickets, int n_seqs, int nh, int nkv, int hd,
                                    float scale, int window, int whole, int grid, int* err, cudaStream_t stream) {
    if (n_seqs <= 0 || grid <= 0) return 0;
    if (n_seqs > KQ_MOST || nkv < 1 || hd < 8 || hd > HD || hd % 8 || nh % nkv || page_size < 1 || (page_size & (page_size - 1)) ||
        (((uintptr_t)q | (uintptr_t)pool | (uintptr_t)o) & 15))
        return (int)cudaErrorInvalidValue;
    int page_shift = 0;
    while ((1 << page_shift) < page_size) ++page_shift;
    auto go = [&](auto kernel, cudaError_t e) {
        if (e != cudaSuccess) return (int)e;
        // a plain launch, not a programmatic one (see attention_decode_tc.cu)
        kernel<<<grid, KQ_THREADS, KQ_SMEM, stream>>>((const __nv_bfloat16*)q, (const unsigned char*)pool, page_table, table_stride, page_shift, cu, starts,
                                                      (__nv_bfloat16*)o, part_o, part_ml, tickets, n_seqs, nh, nkv, hd, scale * 1.4426950408889634f,
                                                      window, whole, err);
        return mv_launch_status();
    };
    return hd == HD ? go(attention_kv4_prefill_kernel<true>, mv_allow_smem<attention_kv4_prefill_kernel<true>>(KQ_SMEM))
                    : go(attention_kv4_prefill_kernel<false>, mv_allow_smem<attention_kv4_prefill_kernel<false>>(KQ_SMEM));
}
