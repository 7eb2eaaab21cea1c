// pages_rows.cuh -- rows of a paged Q8_0 cache written straight from a layer's projections, and read back as floats.
#pragma once

#include <cuda_bf16.h>

#include "pages.cuh"
#include "rotary.cuh"

namespace b200 {

// ---- write: norms of queries and keys, their rotation, keys and values quantised into the cache ---------------------------------------------------
//   q, k: x / sqrt(mean x^2 + eps) * w (where there are weights), turned as in rotary.cuh; k and v to Q8_0 as pages_append_kernel stores them
// The mean and its root are formed in 64 bits and rounded once, each product and sum of the rest is one rounded operation: the codes do not depend on the order
// of a sum.
struct PageWrite {
    PageCache C;
    const float *x[3], *w[2];               // q, k, v; weights of the norms, or NULL
    float *q_out;
    int64_t tok_stride[3], head_stride[3];
    const int32_t *pos;                     // or NULL: where the row lies in its sequence
    const double *freq;
    int n_head, n_rot, pairs, layer;
    float amplitude, eps;
};
constexpr int PGW_WARPS = 8;

// A row of a warp, eight values a lane: loaded, normed, turned, and stored.
template <bool VEC>
__device__ __forceinline__ void page_row_load(const float *src, float (&x)[8]) {
    if (VEC) {
        const float4 a = *reinterpret_cast<const float4 *>(src), b = *reinterpret_cast<const float4 *>(src + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = src[i];
    }
}
// Where value a of a row, or angle a of pairs of halves, lies in shared memory: the first four of each eight, then the other four, so that lanes which read eight
// each read 16 bytes side by side.  (In their own order, one value a load, the banks of the 8 x 3 loads took a third of the kernel's time: 2000 tokens 52.9 us, now 33.7.)
template <int N>
__device__ __forceinline__ int page_row_at(int a) {
    return (a >> 2 & 1) * (N / 2) + (a >> 3) * 4 + (a & 3);
}
template <int N>
__device__ __forceinline__ void page_row_lds(const float *at, int a, float (&x)[8]) {
    const float4 u = *reinterpret_cast<const float4 *>(at + (a >> 3) * 4), v = *reinterpret_cast<const float4 *>(at + N / 2 + (a >> 3) * 4);
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
}
struct PageTurn {
    float c[KV_D / 2], s[KV_D / 2];
};
template <bool VEC>
__device__ __forceinline__ void page_row_norm(float (&x)[8], const float *w, float eps, int lane) {
    float wx[8];
    page_row_load<VEC>(w + 8 * lane, wx);
    double ss[4];                           // (four sums and their sum: sums in 64 bits are no more alike for being one chain)
#pragma unroll
    for (int i = 0; i < 4; ++i) ss[i] = __fma_rn((double)x[i + 4], (double)x[i + 4], __dmul_rn((double)x[i], (double)x[i]));
    double all = __dadd_rn(__dadd_rn(ss[0], ss[1]), __dadd_rn(ss[2], ss[3]));
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) all = __dadd_rn(all, __shfl_xor_sync(0xffffffffu, all, o));
    const float sc = __double2float_rn(__ddiv_rn(1.0, __dsqrt_rn(__dadd_rn(__dmul_rn(all, 1.0 / KV_D), (double)eps))));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], sc), wx[i]);
}
__device__ __forceinline__ void page_row_turn(float (&x)[8], const PageTurn &turn, float *row, int n_rot, int pairs, int lane) {
    if (pairs == PAIRS_NEXT) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const int a = 8 * lane + i;
            if (a >= n_rot) break;
            const float2 p = turned_pair(x[i], x[i + 1], make_float2(turn.c[a >> 1], turn.s[a >> 1]));
            x[i] = p.x;
            x[i + 1] = p.y;
        }
        return;
    }
    const int half = n_rot >> 1, a0 = 8 * lane;
    __syncwarp();                           // the row before has been read
    if (a0 < n_rot) {
        *reinterpret_cast<float4 *>(row + 4 * lane) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4 *>(row + KV_D / 2 + 4 * lane) = make_float4(x[4], x[5], x[6], x[7]);
    }
    __syncwarp();
    if (a0 >= n_rot) return;
    if (half % 8 == 0) {                    // a lane's eight are of one half, their partners one lane's
        const bool high = a0 >= half;
        float y[8], c[8], s[8];
        page_row_lds<KV_D>(row, high ? a0 - half : a0 + half, y);
        page_row_lds<KV_D / 2>(turn.c, high ? a0 - half : a0, c);
        page_row_lds<KV_D / 2>(turn.s, high ? a0 - half : a0, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = high ? turned_pair(y[i], x[i], make_float2(c[i], s[i])).y : turned_pair(x[i], y[i], make_float2(c[i], s[i])).x;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int a = a0 + i, j = page_row_at<KV_D / 2>(a < half ? a : a - half);
        if (a >= n_rot) break;
        const float u = row[page_row_at<KV_D>(a < half ? a : a - half)], v = row[page_row_at<KV_D>(a < half ? a + half : a)];
        const float2 p = turned_pair(u, v, make_float2(turn.c[j], turn.s[j]));
        x[i] = a < half ? p.x : p.y;
    }
}
__device__ __forceinline__ void page_row_store(const float (&x)[8], uint8_t *dst, float *row, int lane) {
    const int blk = lane >> 2, sub = lane & 3;
    const float d = __fmul_rn(kv_amax_8(x), PG_SCALE), id = d > 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
    uint32_t w[2];
    kv_words_8(x, id, w);
    __syncwarp();
    uint8_t *bytes = reinterpret_cast<uint8_t *>(row);                      // put together by halfwords, stored by 16-byte words
    unsigned short *p = reinterpret_cast<unsigned short *>(bytes + 34 * blk);
    if (sub == 0) p[0] = (unsigned short)f32_to_f16_bits_ties_away(d);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        p[1 + 4 * sub + 2 * j] = (unsigned short)(w[j] & 0xFFFFu);
        p[2 + 4 * sub + 2 * j] = (unsigned short)(w[j] >> 16);
    }
    __syncwarp();
    if (lane < KV_ROW / 16) reinterpret_cast<uint4 *>(dst)[lane] = reinterpret_cast<const uint4 *>(bytes)[lane];
}

// grid (tokens / TOK, groups of rows).  What bounds it: a token's place and angles, a chain of three loads and sines in 64 bits, then issue slots (half of them)
// and memory (2000 tokens 33.7 us, 0.54 of its rate; a plain copy of as many bytes, timed alike, 25.6).  A CTA finds where its tokens go and forms their angles, then a warp has a row at a time (query heads, then k and v heads of a token; two, so that
// the next one's values are on their way), eight values a lane.  VEC: strides are multiples of 4, pointers (weights' too) 16-byte aligned.
template <bool VEC, int TOK>
__global__ void __launch_bounds__(32 * PGW_WARPS) pages_write_kernel(const __grid_constant__ PageWrite P, int rows_each) {
    __shared__ __align__(16) float rows[PGW_WARPS][KV_D];
    __shared__ __align__(16) PageTurn turn[TOK];
    __shared__ int64_t place[TOK];          // page * 64 + row, -1: nowhere
    const PageCache &C = P.C;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tok0 = (int)blockIdx.x * TOK, toks = min(TOK, C.n_tok - tok0);
    const int all = P.n_head + 2 * C.n_head_kv, first = (int)blockIdx.y * rows_each, each = min(rows_each, all - first), half = P.n_rot >> 1;
    pdl_wait_prior_grid();
    if (TOK == 1) pdl_launch_dependents();
    auto which = [&](int r, int &h) {       // 0 q, 1 k, 2 v
        const int kind = r < P.n_head ? 0 : r < P.n_head + C.n_head_kv ? 1 : 2;
        h = kind == 0 ? r : r - P.n_head - (kind - 1) * C.n_head_kv;
        return kind;
    };
    auto load = [&](int item, float (&x)[8]) {
        const int t = item / each;
        int h;
        const int kind = which(first + item - t * each, h);
        page_row_load<VEC>(P.x[kind] + (int64_t)(tok0 + t) * P.tok_stride[kind] + h * P.head_stride[kind] + 8 * lane, x);
    };
    const int items = toks * each;
    float x[2][8];
    if (warp < items) load(warp, x[0]);
    if (warp + PGW_WARPS < items) load(warp + PGW_WARPS, x[1]);
    if (blockIdx.x == 0 && blockIdx.y == 0) report_ranges(C.start, C.n_seq, C.n_tok);
    for (int t = warp; t < toks; t += PGW_WARPS) {
        const int tok = tok0 + t, s = seq_of_row(C.start, C.n_seq, tok, lane);
        int64_t to = -1;
        int pos = 0;
        if (s < C.n_seq) {                  // (rows behind the last sequence are nobody's)
            const SeqRange range = seq_range(C.start, s, C.n_tok);
            const int64_t at = (int64_t)C.len[s] - range.n + (tok - range.begin);
            int page = -1;
            if (range.n > 0 && tok >= range.begin && at >= 0 && at / PG_POS < C.table_stride) page = C.table[(size_t)s * C.table_stride + at / PG_POS];
            if (page >= 0 && page < C.n_pages) to = (int64_t)page * PG_POS + at % PG_POS;
            else if (lane == 0 && blockIdx.y == 0) bad_sequence();
            pos = P.pos && half ? P.pos[tok] : (int)at;
        }
        if (lane == 0) place[t] = to;
        for (int i = lane; i < half; i += 32) {
            const float2 angle = turn_of(pos, P.freq[i], (double)P.amplitude);
            const int at = P.pairs == PAIRS_NEXT ? i : page_row_at<KV_D / 2>(i);
            turn[t].c[at] = angle.x;
            turn[t].s[at] = angle.y;
        }
    }
    __syncthreads();
    float *row = rows[warp];
    auto finish = [&](int item, float (&v)[8]) {
        const int t = item / each;
        int h;
        const int kind = which(first + item - t * each, h);
        const int64_t to = place[t];
        if (to < 0) return;
        if (kind < 2) {
            if (P.w[kind]) page_row_norm<VEC>(v, P.w[kind], P.eps, lane);
            if (half) page_row_turn(v, turn[t], row, P.n_rot, P.pairs, lane);
        }
        if (kind == 0) {
            float *dst = P.q_out + ((int64_t)(tok0 + t) * P.n_head + h) * KV_D + 8 * lane;
            if (VEC) {
                *reinterpret_cast<float4 *>(dst) = make_float4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<float4 *>(dst + 4) = make_float4(v[4], v[5], v[6], v[7]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) dst[i] = v[i];
            }
        } else {
            page_row_store(v, page_rows(C, (int)(to / PG_POS), P.layer, kind - 1, h) + (size_t)(to % PG_POS) * KV_ROW, row, lane);
        }
    };
#pragma unroll 1
    for (int item = warp; item < items; item += 2 * PGW_WARPS) {
        finish(item, x[0]);
        if (item + 2 * PGW_WARPS < items) load(item + 2 * PGW_WARPS, x[0]);
        if (item + PGW_WARPS < items) finish(item + PGW_WARPS, x[1]);
        if (item + 3 * PGW_WARPS < items) load(item + 3 * PGW_WARPS, x[1]);
    }
}

// ---- read: rows of a layer as floats ---------------------------------------------------------------------------------------------------------------
// What bounds it: memory (35 003 rows of 4 heads to bf16 in 46.7 us, to fp16 46.9, to fp32 75.6: 0.72 and 0.73 of the copy rate; plain copies of as many bytes, timed alike, 40.6 and 61.2).
//   row start[s] + i of the outputs is position first[s] + i of sequence s: code times scale, one product, exact in fp32 and rounded once to fewer bits
enum : int { ROWS_F32 = 0, ROWS_F16 = 1, ROWS_BF16 = 2 };
struct PageRead {
    PageCache C;
    const int32_t *first;                   // or NULL: each sequence's last positions
    void *out[2];                           // K, V; one may be NULL
    int layer;
};
constexpr int PGR_WARPS = 4, PGR_BATCH = 4;

// A warp per token, its rows (K and V of every kv head) PGR_BATCH at a time; a lane has eight values.
template <int TYPE>
__global__ void __launch_bounds__(32 * PGR_WARPS) pages_read_kernel(const __grid_constant__ PageRead P) {
    const PageCache &C = P.C;
    const int lane = threadIdx.x & 31, tok = (int)blockIdx.x * PGR_WARPS + (threadIdx.x >> 5), heads = C.n_head_kv;
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    if (blockIdx.x == 0) report_ranges(C.start, C.n_seq, C.n_tok);
    if (tok >= C.n_tok) return;
    const int s = seq_of_row(C.start, C.n_seq, tok, lane);
    if (s >= C.n_seq) return;               // nobody's
    const SeqRange range = seq_range(C.start, s, C.n_tok);
    const int len = C.len[s];
    const int64_t at = (P.first ? (int64_t)P.first[s] : (int64_t)len - range.n) + (tok - range.begin);
    int page = -1;
    if (range.n > 0 && tok >= range.begin && at >= 0 && at < len && at / PG_POS < C.table_stride) page = C.table[(size_t)s * C.table_stride + at / PG_POS];
    if (page < 0 || page >= C.n_pages) {
        if (lane == 0) bad_sequence();
        return;
    }
    const int blk = lane >> 2, sub = lane & 3, code0 = 34 * blk + 2 + 8 * sub;
    const bool both = P.out[0] && P.out[1];
    const int n = both ? 2 * heads : heads;
    for (int r0 = 0; r0 < n; r0 += PGR_BATCH) {
        uint32_t w[PGR_BATCH][3], d[PGR_BATCH];
#pragma unroll
        for (int e = 0; e < PGR_BATCH; ++e) {
            const int r = min(r0 + e, n - 1), kv = both ? r / heads : P.out[0] ? 0 : 1, h = both ? r - kv * heads : r;
            const uint8_t *row = page_rows(C, page, P.layer, kv, h) + (size_t)(at % PG_POS) * KV_ROW;
            const uint32_t *src = reinterpret_cast<const uint32_t *>(row + (code0 & ~3));
            d[e] = *reinterpret_cast<const uint16_t *>(row + 34 * blk);
            w[e][0] = src[0];
            w[e][1] = src[1];
            w[e][2] = code0 & 2 ? src[2] : 0u;
        }
#pragma unroll
        for (int e = 0; e < PGR_BATCH; ++e) {
            const int r = r0 + e;
            if (r >= n) break;
            const int kv = both ? r / heads : P.out[0] ? 0 : 1, h = both ? r - kv * heads : r;
            const uint32_t a = code0 & 2 ? __byte_perm(w[e][0], w[e][1], 0x5432) : w[e][0], b = code0 & 2 ? __byte_perm(w[e][1], w[e][2], 0x5432) : w[e][1];
            const float sc = f16_bits_to_f32(d[e]);
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __fmul_rn((float)(int8_t)((i < 4 ? a : b) >> (8 * (i & 3)) & 0xFFu), sc);
            const size_t to = ((size_t)tok * heads + h) * KV_D + 8 * lane;
            if (TYPE == ROWS_F32) {
                float4 *dst = reinterpret_cast<float4 *>(static_cast<float *>(P.out[kv]) + to);
                dst[0] = make_float4(x[0], x[1], x[2], x[3]);
                dst[1] = make_float4(x[4], x[5], x[6], x[7]);
            } else {
                uint32_t y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (TYPE == ROWS_F16) {
                        const __half2 v = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                        y[i] = *reinterpret_cast<const uint32_t *>(&v);
                    } else {
                        const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                        y[i] = *reinterpret_cast<const uint32_t *>(&v);
                    }
                }
                *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(P.out[kv]) + to) = make_uint4(y[0], y[1], y[2], y[3]);
            }
        }
    }
}

}  // namespace b200
