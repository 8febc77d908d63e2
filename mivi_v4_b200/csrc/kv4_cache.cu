// The 4-bit cache (kv4.cuh): rows quantised as they are written, rows and pages read back, and attention over it for every head
// size and dtype.
//
// Formulas of the preparation and of attention as in attention.cu and attention_decode.cu (reference:
// crates/mivi-model/src/transformer.rs:81-110, 114-167, 293-298; rotation crates/mivi-core/src/rope.rs:59-61, 219-229).
#include "kv4.cuh"

MV_GUARD_SETTER(kv4_cache)

// ------------------------------------------------- q/k norm, rotation, quantised append
// One warp per token and head: nh query heads, then nkv key heads, then nkv value heads, as they lie in a row of the fused projection.
// A lane holds the neighbouring elements 2i and 2i + 1 with i = lane, lane + 32, ...: one byte of codes.
__global__ void __launch_bounds__(256)
kv4_prepare_kernel(const float* __restrict__ qkv, const float* __restrict__ wq, const float* __restrict__ wk, float eps,
                   const float* __restrict__ inv_freq, int half_split, const int* __restrict__ positions,
                   const int* __restrict__ seq_of, const int* __restrict__ page_table, int table_stride, int page_shift,
                   unsigned char* __restrict__ pool, void* __restrict__ q_out, int q_dtype, int N, int nh, int nkv, int hd) {
    mv_pdl_begin();
    const long long wid = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31, slots = nh + 2 * nkv;
    if (wid >= (long long)N * slots) return;
    const int n = (int)(wid / slots), hs = (int)(wid - (long long)n * slots);
    const bool is_q = hs < nh, is_k = !is_q && hs < nh + nkv;
    const int half = hd >> 1;
    constexpr int MAXJ = KV4_MAX_HEAD_DIM / 64;
    const float* row = qkv + (size_t)wid * hd;
    const int pos = positions[n];
    float2 x[MAXJ];
#pragma unroll
    for (int j = 0; j < MAXJ; ++j) {
        const int i = lane + 32 * j;
        x[j] = i < half ? *reinterpret_cast<const float2*>(row + 2 * i) : make_float2(0.f, 0.f);
    }
    if (is_q || is_k) {
        const float* w = is_q ? wq : wk;
        float scale = 1.f;
        if (w) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < MAXJ; ++j) ss = fmaf(x[j].x, x[j].x, fmaf(x[j].y, x[j].y, ss));
            ss = mv_warp_sum(ss);
            scale = 1.0f / sqrtf(ss / (float)hd + eps);
        }
        // The angle is worked out in 64 bits and brought into one turn: a product of 32 bits is off by 2^-25 of the angle, which at
        // position 32,768 is a thousandth of a turn's radian, more than enough to move a code.
        auto turn = [&](int i, float& c, float& s) {
            const double a = (double)pos * (double)inv_freq[i];
            const double r = fma(rint(a * 0.15915494309189535), -6.283185307179586, a);
            sincosf((float)r, &s, &c);
        };
#pragma unroll
        for (int j = 0; j < MAXJ; ++j) {
            const int i = lane + 32 * j;
            if (i >= half) break;
            float2 y = x[j];
            if (w) {
                const float2 ww = *reinterpret_cast<const float2*>(w + 2 * i);
                y.x = y.x * scale * ww.x;
                y.y = y.y * scale * ww.y;
            }
            if (inv_freq && !half_split) {                       // pairs (2i, 2i + 1)
                float c, s;
                turn(i, c, s);
                y = make_float2(y.x * c - y.y * s, y.x * s + y.y * c);
            } else if (inv_freq) {                               // pairs (i, i + half): the partners are the neighbours 2i -+ half
                const int e = 2 * i, lo = e < half ? e : e - half;
                const int other = e < half ? e + half : e - half;
                float2 z = *reinterpret_cast<const float2*>(row + other);
                if (w) {
                    const float2 ww = *reinterpret_cast<const float2*>(w + other);
                    z.x = z.x * scale * ww.x;
                    z.y = z.y * scale * ww.y;
                }
                float c0, s0, c1, s1;
                turn(lo, c0, s0);
                turn(lo + 1, c1, s1);
                y = e < half ? make_float2(y.x * c0 - z.x * s0, y.y * c1 - z.y * s1) : make_float2(z.x * s0 + y.x * c0, z.y * s1 + y.y * c1);
            }
            x[j] = y;
        }
    }
    if (is_q) {
#pragma unroll
        for (int j = 0; j < MAXJ; ++j) {
            const int i = lane + 32 * j;
            if (i >= half) break;
            const size_t at = ((size_t)n * nh + hs) * hd + 2 * i;
            if (q_dtype == MV_DT_BF16) mv_store2((__nv_bfloat16*)q_out + at, x[j].x, x[j].y);
            else mv_store2((float*)q_out + at, x[j].x, x[j].y);
        }
        return;
    }
    float lo = INFINITY, hi = -INFINITY;
    bool fine = true;
#pragma unroll
    for (int j = 0; j < MAXJ; ++j) {
        if (lane + 32 * j >= half) break;
        lo = fminf(lo, fminf(x[j].x, x[j].y));
        hi = fmaxf(hi, fmaxf(x[j].x, x[j].y));
        fine = fine && fabsf(x[j].x) < INFINITY && fabsf(x[j].y) < INFINITY;
    }
    lo = -mv_warp_max(-lo);
    hi = mv_warp_max(hi);
    fine = __all_sync(0xffffffffu, fine);
    float zero = __bfloat162float(__float2bfloat16_rn(lo));
    // (the lowest floats would round to -infinity)
    zero = fminf(fmaxf(zero, -3.3895313892515355e38f), 3.3895313892515355e38f);
    float step = kv4_step(hi, zero);
    if (!fine) { zero = NAN; step = NAN; }
    const int page = page_table[(size_t)seq_of[n] * table_stride + (pos >> page_shift)];
    if (!mv_page_ok(page)) return;
    const int page_size = 1 << page_shift, at = pos & (page_size - 1);
    const int g = is_k ? hs - nh : hs - nh - nkv;
    unsigned char* base = pool + ((size_t)page * nkv + g) * kv4_head_bytes(page_size, hd);
    unsigned char* codes = base + ((size_t)(is_k ? 0 : page_size) + at) * half;
#pragma unroll
    for (int j = 0; j < MAXJ; ++j) {
        const int i = lane + 32 * j;
        if (i >= half) break;
        codes[i] = fine ? (unsigned char)(kv4_code(x[j].x, zero, step) | kv4_code(x[j].y, zero, step) << 4) : 0;
    }
    if (lane == 0)
        *reinterpret_cast<unsigned*>(base + (size_t)page_size * hd + (size_t)at * 8 + (is_k ? 0 : 4)) = kv4_pack_params(step, zero);
}

// qkv float32 [N, (nh + 2 nkv) * hd]; pool [pages, nkv, page_size * (hd + 8)] bytes.  q_out [N, nh * hd] in q_dtype.
MV_API int mv_kv4_prepare(const float* qkv, const float* wq, const float* wk, float eps, const float* inv_freq, int half_split,
                          const int* positions, const int* seq_of, const int* page_table, int table_stride, int page_size,
                          void* pool, void* q_out, int q_dtype, int N, int nh, int nkv, int hd, cudaStream_t stream) {
    if (N <= 0) return 0;
    if (hd % 8 || hd > KV4_MAX_HEAD_DIM || page_size < 1 || (page_size & (page_size - 1)) || nkv < 1) return (int)cudaErrorInvalidValue;
    int page_shift = 0;
    while ((1 << page_shift) < page_size) ++page_shift;
    const long long warps = (long long)N * (nh + 2 * nkv);
    mv_launch(kv4_prepare_kernel, dim3((unsigned)((warps + 7) / 8)), 256, 0, stream, qkv, wq, wk, eps, inv_freq, half_split, positions,
              seq_of, page_table, table_stride, page_shift, (unsigned char*)pool, q_out, q_dtype, N, nh, nkv, hd);
    return mv_launch_status();
}

// ------------------------------------------------------------------ reading back
// One thread per 8 codes of a row: a word of codes and the row's two numbers in, 8 elements out.
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

MV_API int mv_kv4_read(const void* pool, const int* page_table, int table_stride, int page_size, const int* positions,
                       const int* seq_of, void* k_out, void* v_out, int dtype, int N, int nkv, int hd, cudaStream_t stream) {
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
                kv4_unpack8(kc[w], 1.f, 0.f, c);
#pragma unroll
                for (int h = 0; h < GT; ++h)
#pragma unroll
                    for (int e = 0; e < 8; ++e) dot[h] = fmaf(c[e], qs[h * hd + 8 * w + e], dot[h]);
            }
#pragma unroll
            for (int h = 0; h < GT; ++h) s[h] = fmaf(p.ks, dot[h], p.kz * qsum[h]);
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
MV_API int mv_attention_kv4(const void* q, const void* pool, const int* page_table, int table_stride, int page_size,
                            const int* positions, const int* seq_of, void* o, int dtype, float* part_o, float* part_ml, int* tickets,
                            int N, int nh, int nkv, int hd, float scale, int window, int splits, int gt, int head_tiles,
                            cudaStream_t stream) {
    if (N <= 0) return 0;
    if (hd % 8 || hd > KV4_MAX_HEAD_DIM || nkv < 1 || nh % nkv || page_size < 1 || (page_size & (page_size - 1)) || splits < 1 ||
        gt * head_tiles < nh / nkv || N > 65535 || nkv * head_tiles > 65535)
        return (int)cudaErrorInvalidValue;
    int page_shift = 0;
    while ((1 << page_shift) < page_size) ++page_shift;
    const dim3 grid(splits, nkv * head_tiles, N);
    cudaError_t attr = cudaSuccess;
#define MV_GO(T, GT)                                                                                                              \
    do {                                                                                                                          \
        const size_t smem = sizeof(float) * (5 * GT * hd + 8 * GT);                                                               \
        if (smem > 48 * 1024) attr = mv_allow_smem<attention_kv4_kernel<T, GT>>(sizeof(float) * (5 * GT * KV4_MAX_HEAD_DIM + 8 * GT)); \
        if (attr != cudaSuccess) return (int)attr;                                                                                \
        mv_launch(attention_kv4_kernel<T, GT>, grid, 128, smem, stream, (const T*)q, (const unsigned char*)pool, page_table,       \
                  table_stride, page_shift, positions, seq_of, (T*)o, part_o, part_ml, tickets, nh, nkv, hd, scale, window,        \
                  head_tiles);                                                                                                    \
    } while (0)
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
