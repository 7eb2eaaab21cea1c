// pages_tc.cuh -- attention over a paged cache on the tensor cores (tcgen05.mma.kind::f16), for sequences with many new tokens.
//
// The value is that of pages_attn_kernel.  Operands as in attn_tc.cuh: powers of two times two fp16 planes, high and low -- of a query row or a cache row what Q8_0 stands for, a
// product of 18 bits, exactly; of V's dims a page's values under one power of two -- and three of the four products, sums fp32.
//
// pages_planes_kernel writes the pages of a call's long sequences once as tile images (attn_tc.cuh's, a page a tile).
//
// pages_tc_kernel: CTA = 128 rows (tokens times the heads that share a kv head) and one span of pages.  512 threads, each one row and a quarter of its columns, form weights and add
// outputs; of three warps more one issues the tensor core's instructions, which has a page's scores and the outputs of the page before in flight meanwhile, two copy k and v:
//   tensor core   q . k of page i + 1          | weights x v of page i
//   threads       weights of page i, outputs of page i - 1 added, weights to tensor memory | scores of page i + 1 read
// (Its 19 warps leave a thread 96 registers, of which the 64 sums are most: 260 bytes of stores and 364 of loads spilled a thread.)
// (The issue is a warp's whole time: 2100 cycles for a page's scores, 1100 for its outputs.  By one of the sixteen warps a page took 8000 cycles, with the copies from the issuing
// warp 5850.)
// Tensor memory, all 512 columns: 256 output, 64 scores, 64 weights, 128 q low.  Shared memory: q high, k and v images of one page, 64 KB each.
//
// us with append, planes and join, 24 heads over 4: 512 tokens after 4000 240 (on mma.sync 415), with 48 pages in two rounds of CTAs at about 2.3 each, 20 of a CTA's start and
// end and 25 of the launches around it.  A page's time is the copy of k behind the scores, the scores' products (N = 64: 44 cycles each, 33 were the rows in tensor memory) and the
// softmax's first part, one after the other; the rest runs beside them.  Scores are one sum over 256 dims, small products first: relative error of the outputs 6e-7 there (fp32
// torch 1.3e-6), 4.3e-7 for fresh prompts; six sums as in attn_tc.cuh leave no columns for two pages in flight.
//
// What one plane pair cannot hold beside the largest value (atc_too_wide, of the CTA's rows and pages) is left to pages_redo_kernel, which comes behind and does the CTAs that said
// so.  Sequences with few new tokens are pages_attn_kernel's.
#pragma once

#include "attn_tc.cuh"
#include "pages.cuh"

namespace b200 {

constexpr uint32_t PTC_COL_O = 0, PTC_COL_S = 256, PTC_COL_P = 320, PTC_COL_QL = 384;
constexpr int PTC_THREADS = ATC_THREADS + 96;
constexpr int PTC_SMEM_BYTES = 1024 + 3 * ATC_PLANES + (2 * ATC_KEYS + 2 * ATT_D + 2 * 4 * ATC_M) * 4 + 128;
// Among the threads that have rows.
__device__ __forceinline__ void ptc_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(ATC_THREADS) : "memory"); }
static_assert(PG_POS == ATC_KEYS && KV_D == ATT_D && PTC_ROWS == ATC_M, "");

// grid (sequences on the tensor cores x pages, kv heads, 2): z 0 = k (warp = eight positions, lane = eight dims), z 1 = v (thread = one dim, all 64 positions).
__global__ void __launch_bounds__(ATC_PREP_THREADS) pages_planes_kernel(const __grid_constant__ PageAttn P) {
    __shared__ __align__(16) uint8_t rows[PG_HEAD_BYTES];
    __shared__ uint32_t top[ATC_PREP_THREADS / 32];
    const PageCache &C = P.C;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kvh = blockIdx.y;
    const int page_at = blockIdx.x % P.max_pages;
    int which = blockIdx.x / P.max_pages;               // of the sequences on the tensor cores
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    int seq = -1;
    for (int base = 0; base < C.n_seq; base += 32) {
        const int s = base + lane;
        const unsigned on = __ballot_sync(0xffffffffu, s < C.n_seq && pages_on_tc(P, seq_range(C.start, s, C.n_tok).n, C.len[min(s, C.n_seq - 1)]));
        if (which < __popc(on)) {
            seq = base + __fns(on, 0, which + 1);
            break;
        }
        which -= __popc(on);
    }
    if (seq < 0) return;
    const int n = min(PG_POS, C.len[seq] - page_at * PG_POS);
    if (n <= 0) return;
    const int page = C.table[(size_t)seq * C.table_stride + page_at];
    const bool there = page >= 0 && page < C.n_pages;
    if (!there && threadIdx.x == 0) bad_sequence();
    {
        const uint4 *src = reinterpret_cast<const uint4 *>(page_rows(C, there ? page : 0, P.layer, blockIdx.z, kvh));
        const int words = there ? n * (KV_ROW / 16) : 0;
        for (int i = threadIdx.x; i < PG_HEAD_BYTES / 16; i += ATC_PREP_THREADS) reinterpret_cast<uint4 *>(rows)[i] = i < words ? src[i] : make_uint4(0u, 0u, 0u, 0u);
    }
    __syncthreads();
    uint8_t *img = P.images + ((size_t)blockIdx.x * C.n_head_kv + kvh) * ATC_IMG_BYTES;
    uint32_t *range = reinterpret_cast<uint32_t *>(img + ATC_IMG_RANGE);
    if (blockIdx.z == 0) {
        constexpr int ROWS = ATC_KEYS / (ATC_PREP_THREADS / 32);
        uint32_t seen = 0;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int key = ROWS * warp + r;
            const uint16_t *b = reinterpret_cast<const uint16_t *>(rows + key * KV_ROW + 34 * (lane >> 2));
            const float d = f16_bits_to_f32(b[0]);
            float x[8];
            uint32_t m = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t w = b[1 + 4 * (lane & 3) + e];
                x[2 * e] = __fmul_rn((float)(int8_t)(w & 0xFFu), d);
                x[2 * e + 1] = __fmul_rn((float)(int8_t)(w >> 8), d);
                m = max(m, max(atc_abs_bits(x[2 * e]), atc_abs_bits(x[2 * e + 1])));
            }
            m = __reduce_max_sync(0xffffffffu, m);
            seen = max(seen, m);
            const int s = atc_shift(m, 63);
            uint4 hi, lo;
            atc_split8(x, atc_pow2(s), hi, lo);
            uint8_t *dst = img + (lane >> 3) * ATC_CHUNK + key * 128 + (((lane & 7) ^ (key & 7)) * 16);
            *reinterpret_cast<uint4 *>(dst) = hi;
            *reinterpret_cast<uint4 *>(dst + ATC_KEYS * 128) = lo;
            if (lane == 0) reinterpret_cast<float *>(img + ATC_IMG_KF)[key] = atc_pow2(-s);
        }
        if (lane == 0) top[warp] = seen;
        __syncthreads();
        if (warp == 0) {
            const uint32_t m = __reduce_max_sync(0xffffffffu, top[lane & (ATC_PREP_THREADS / 32 - 1)]);
            if (lane == 0) range[0] = m;
        }
    } else {
        const int d = threadIdx.x;
        float x[ATC_KEYS];
        const uint8_t *b = rows + 34 * (d >> 5);
        uint32_t seen = 0;
#pragma unroll
        for (int e = 0; e < ATC_KEYS; ++e) {
            x[e] = __fmul_rn((float)(int8_t)b[e * KV_ROW + 2 + (d & 31)], f16_bits_to_f32(*reinterpret_cast<const uint16_t *>(b + e * KV_ROW)));
            seen = max(seen, atc_abs_bits(x[e]));
        }
        const int s = atc_shift(seen, 112);
        reinterpret_cast<float *>(img + ATC_IMG_VF)[d] = atc_pow2(-s - 14);          // (and the weights' 2^-14)
#pragma unroll
        for (int g = 0; g < ATC_KEYS / 8; ++g) {
            uint4 hi, lo;
            atc_split8(x + 8 * g, atc_pow2(s), hi, lo);
            uint8_t *dst = img + ATC_PLANES + d * 128 + ((g ^ (d & 7)) * 16);
            *reinterpret_cast<uint4 *>(dst) = hi;
            *reinterpret_cast<uint4 *>(dst + 2 * ATC_CHUNK) = lo;
        }
        // The positions' largest values, by their blocks' scales: 127 of a scale, which the quantiser's blocks reach (others reach less, and their rows stand for less than they say).
        const int tiny = __syncthreads_or(seen > 0u && seen < ATC_TINY ? 1 : 0);
        if (warp == 0) {
            uint32_t most = 0u, least = ATC_NONE;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t own = 0u;
#pragma unroll
                for (int blk = 0; blk < KV_NBLK; ++blk) own = max(own, *reinterpret_cast<const uint16_t *>(rows + (lane + 32 * h) * KV_ROW + 34 * blk) & 0x7FFFu);
                own = atc_abs_bits(__fmul_rn(f16_bits_to_f32(own), 127.0f));
                most = max(most, own);
                least = min(least, own ? own : ATC_NONE);
            }
            most = __reduce_max_sync(0xffffffffu, most);
            least = __reduce_min_sync(0xffffffffu, least);
            if (lane == 0) {
                range[1] = tiny ? ATC_NONE : most;
                range[2] = least;
            }
        }
    }
}

// grid (tiles of 128 rows of all sequences and some that find none, kv heads, splits)
__global__ void __launch_bounds__(PTC_THREADS, 1) pages_tc_kernel(const __grid_constant__ PageAttn P) {
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *qhi = smem + ((1024u - (smem_u32(smem) & 1023u)) & 1023u);
    uint8_t *kpl = qhi + ATC_PLANES, *vpl = kpl + ATC_PLANES;
    float *kf = reinterpret_cast<float *>(vpl + ATC_PLANES);             // [2][64] 2^-s of the page's positions, pages alternate
    float *vf = kf + 2 * ATC_KEYS;                                       // [2][256] 2^-s of the dims (and the weights' 2^-14)
    float *red0 = vf + 2 * ATT_D;                                        // [2][4][128] exchange between the four warps of a row, pages alternate
    // pages alternate between two barriers of the copies: a phase ends when everybody has long waited for the one before
    uint64_t *qk = reinterpret_cast<uint64_t *>(red0 + 2 * 4 * ATC_M), *pv = qk + 1, *scored = qk + 2, *weighed = qk + 3, *kfull = qk + 4, *vfull = qk + 6;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(vfull + 2);
    volatile int *failed = reinterpret_cast<int *>(tmem_slot + 1);

    const PageCache &C = P.C;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int cg = warp >> 2, row = 32 * (warp & 3) + lane;              // a thread's row, and its quarter of the row's columns
    const int kvh = blockIdx.y, split = blockIdx.z;
    pdl_wait_prior_grid();                                               // the images
    pdl_launch_dependents();
    int seq, tile;
    if (!seq_of_item(C.start, C.n_seq, C.n_tok, (int)blockIdx.x, lane, [&](int n) { return ((int64_t)n * P.group + PTC_ROWS - 1) / PTC_ROWS; }, seq, tile)) return;      // CTA-uniform
    const SeqRange range = seq_range(C.start, seq, C.n_tok);
    const int len = C.len[seq];
    if (!pages_on_tc(P, range.n, len)) return;                           // pages_attn_kernel has it (and says what is wrong with it)
    const int n_rows = min(PTC_ROWS, range.n * P.group - tile * PTC_ROWS);
    const int first_tok = tile * PTC_ROWS / P.group, last_tok = (tile * PTC_ROWS + n_rows - 1) / P.group;
    const int before = len - range.n;
    const int seen_pos = min(len, before + last_tok + 1), pages = (max(seen_pos, 0) + PG_POS - 1) / PG_POS;
    const int page0 = split * P.span, page1 = split == P.splits - 1 ? pages : min(page0 + P.span, pages);
    const int ntiles = page1 - page0;
    if (ntiles <= 0 && split > 0) return;
    const int all_see = before + first_tok;
    const int limit = row < n_rows ? before + (tile * PTC_ROWS + row) / P.group : -1;        // the last position that the thread's row sees
    int which = 0;                                                       // of the sequences on the tensor cores
    for (int s = lane; s < seq; s += 32) which += pages_on_tc(P, seq_range(C.start, s, C.n_tok).n, C.len[s]) ? 1 : 0;
    which = __reduce_add_sync(0xffffffffu, which);
    if (which >= P.n_tc) {                                               // (rows that several sequences claim: there is no image for all of them)
        if (threadIdx.x == 0) P.redo[((size_t)blockIdx.x * C.n_head_kv + kvh) * P.splits + split] = 1;
        return;
    }
    const size_t img_stride = (size_t)C.n_head_kv * ATC_IMG_BYTES;
    const uint8_t *img = P.images + (((size_t)which * P.max_pages + page0) * C.n_head_kv + kvh) * ATC_IMG_BYTES;
    auto row_at = [&](int r) {                                           // where a row of the tile lies in q and out
        const int x = tile * PTC_ROWS + r, tok = x / P.group;
        return ((size_t)(range.begin + tok) * P.n_head + kvh * P.group + (x - tok * P.group)) * KV_D;
    };

    if (threadIdx.x == 0) {
        for (int b = 0; b < 8; ++b) mbar_init(qk + b, b == 2 || b == 3 ? ATC_WARPS : 1);
        mbar_fence_init();
        *failed = 0;
    }
    const bool driver = warp >= ATC_WARPS;
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // one thread each: the images of page i of the span
    auto load_k = [&](int i) {
        const uint64_t pol = policy_evict_last_or_default();
        const uint8_t *src = img + (size_t)i * img_stride;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // the factors were read by ordinary loads
        mbar_expect_tx(kfull + (i & 1), ATC_PLANES + ATC_KEYS * 4);
        bulk_g2s(kf + (i & 1) * ATC_KEYS, src + ATC_IMG_KF, ATC_KEYS * 4, kfull + (i & 1), pol);
        bulk_g2s(kpl, src, ATC_PLANES, kfull + (i & 1), pol);
    };
    auto load_v = [&](int i) {
        const uint64_t pol = policy_evict_last_or_default();
        const uint8_t *src = img + (size_t)i * img_stride;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_expect_tx(vfull + (i & 1), ATC_PLANES + ATT_D * 4);
        bulk_g2s(vf + (i & 1) * ATT_D, src + ATC_IMG_VF, ATT_D * 4, vfull + (i & 1), pol);
        bulk_g2s(vpl, src + ATC_PLANES, ATC_PLANES, vfull + (i & 1), pol);
    };

    // ---- q: row of the thread, 64 dims, quantised to Q8_0 (two blocks); high plane to shared memory, low plane to tensor memory.  Queries and outputs pass through shared
    // memory (the planes' of k and v, a warp's 32 rows of 64 values each, 16-byte pieces swizzled), where a row's values become a thread's.
    float4 *box = reinterpret_cast<float4 *>(kpl) + warp * 512;
    const int row0 = 32 * (warp & 3);
    float qf = 0.0f;
    uint32_t seen = 0;                                                   // magnitude bits of the row's largest q
    __syncthreads();                                                     // the barriers, and where tensor memory is
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t tlane = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    // The tensor core's instructions, one elected lane of the driver's warp (the code stays warp-uniform).  Products with a low plane come first: the accumulator is small
    // while they are added.
    auto issue_qk = [&] {
        tc_fence_after();
        constexpr uint32_t LOW = (ATC_KEYS * 128) >> 4;
        const uint32_t a0 = tc16_desc_lo(smem_u32(qhi)), b0 = tc16_desc_lo(smem_u32(kpl)), ql = tmem + PTC_COL_QL, d = tmem + PTC_COL_S;
        auto at = [](int n) { return (uint32_t)((n >> 2) * (ATC_CHUNK >> 4) + 2 * (n & 3)); };
        if (elect_one()) {
            tc_mma_f16_ts<false>(d, ql, b0, atc_idesc(ATC_KEYS));
#pragma unroll
            for (int n = 1; n < 16; ++n) tc_mma_f16_ts<true>(d, ql + (uint32_t)(8 * n), b0 + at(n), atc_idesc(ATC_KEYS));
#pragma unroll
            for (int n = 0; n < 16; ++n) atc_mma_ss<atc_idesc(ATC_KEYS)>(d, a0 + at(n), b0 + LOW + at(n));
#pragma unroll
            for (int n = 0; n < 16; ++n) atc_mma_ss<atc_idesc(ATC_KEYS)>(d, a0 + at(n), b0 + at(n));
            tc_commit(qk);
        }
        __syncwarp();
    };
    auto issue_pv = [&] {
        tc_fence_after();
        const uint32_t b0 = tc16_desc_lo(smem_u32(vpl)), ph = tmem + PTC_COL_P, pl = ph + 32u;
        if (elect_one()) {
#pragma unroll
            for (int n = 0; n < 12; ++n) {
                const uint32_t a = (n < 4 ? pl : ph) + (uint32_t)(8 * (n & 3));
                const uint32_t b = b0 + (uint32_t)((n >= 4 && n < 8 ? (2 * ATC_CHUNK) >> 4 : 0) + 2 * (n & 3));
                if (n == 0) tc_mma_f16_ts<false>(tmem + PTC_COL_O, a, b, atc_idesc(ATT_D));
                else tc_mma_f16_ts<true>(tmem + PTC_COL_O, a, b, atc_idesc(ATT_D));
            }
            tc_commit(pv);
        }
        __syncwarp();
    };
    if (driver) {
        __syncthreads();                                                 // q is in its places
        bool ok = true;                                                  // after a wait that ran out nothing is waited for any more: the CTA comes to its end, and says so
        auto wait = [&](uint64_t *bar, uint32_t parity) { ok = ok && __all_sync(0xffffffffu, mbar_wait_try(bar, parity)); };
        if (warp == ATC_WARPS) {
            for (int i = 0; i <= ntiles && ntiles > 0; ++i) {            // scores of page i, outputs of page i - 1
                if (i < ntiles) {
                    if (i > 0) wait(scored, (uint32_t)((i - 1) & 1));
                    wait(kfull + (i & 1), (uint32_t)((i >> 1) & 1));
                    issue_qk();
                }
                if (i > 0) {
                    wait(weighed, (uint32_t)((i - 1) & 1));
                    wait(vfull + ((i - 1) & 1), (uint32_t)(((i - 1) >> 1) & 1));
                    issue_pv();
                }
            }
        } else if (warp == ATC_WARPS + 1) {
            for (int i = 0; i < ntiles; ++i) {                           // k when the scores of the page before have been read
                if (i > 0) wait(scored, (uint32_t)((i - 1) & 1));
                if (lane == 0) load_k(i);
                __syncwarp();
            }
        } else {
            for (int i = 0; i < ntiles; ++i) {                           // v when the outputs of the page before are there
                if (i > 0) wait(pv, (uint32_t)((i - 1) & 1));
                if (lane == 0) load_v(i);
                __syncwarp();
            }
        }
        if (!ok) *failed = 1;
        __syncthreads();
        return;
    }
    {
        float x[64];
        if ((reinterpret_cast<uintptr_t>(P.q) & 15u) == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = 2 * i + (lane >> 4), c = lane & 15;
                if (row0 + r < n_rows) cp_async16(box + r * 16 + (c ^ (r & 15)), P.q + row_at(row0 + r) + 64 * cg + 4 * c);
            }
            cp_async_commit();
            cp_async_wait<0>();
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 16; ++c) {
                const float4 a = row < n_rows ? box[lane * 16 + (c ^ (lane & 15))] : make_float4(0.f, 0.f, 0.f, 0.f);
                x[4 * c] = a.x; x[4 * c + 1] = a.y; x[4 * c + 2] = a.z; x[4 * c + 3] = a.w;
            }
        } else {
            const float *src = P.q + (row < n_rows ? row_at(row) : 0) + 64 * cg;
#pragma unroll
            for (int e = 0; e < 64; ++e) x[e] = row < n_rows ? src[e] : 0.0f;
        }
        uint32_t m = 0;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            float amax = 0.0f;
#pragma unroll
            for (int e = 0; e < 32; ++e) amax = fmaxf(amax, fabsf(x[32 * b + e]));
            const float d = __fmul_rn(amax, PG_SCALE), id = d > 0.0f ? __fdiv_rn(1.0f, d) : 0.0f, d16 = f16_bits_to_f32(f32_to_f16_bits_ties_away(d));
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                x[32 * b + e] = __fmul_rn((float)max(-127, min(127, round_ties_away(__fmul_rn(x[32 * b + e], id)))), d16);
                m = max(m, atc_abs_bits(x[32 * b + e]));
            }
        }
        uint32_t *redu = reinterpret_cast<uint32_t *>(red0);
        redu[cg * ATC_M + row] = m;
        ptc_barrier();
#pragma unroll
        for (int c = 0; c < 4; ++c) m = max(m, redu[c * ATC_M + row]);
        seen = m;
        const int s = atc_shift(m, 63);
        qf = __fmul_rn(atc_pow2(-s), P.scale);
        uint32_t lo32[32];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint4 hi, lo;
            atc_split8(x + 8 * j, atc_pow2(s), hi, lo);
            *reinterpret_cast<uint4 *>(qhi + cg * ATC_CHUNK + row * 128 + ((j ^ (row & 7)) * 16)) = hi;
            lo32[4 * j] = lo.x; lo32[4 * j + 1] = lo.y; lo32[4 * j + 2] = lo.z; lo32[4 * j + 3] = lo.w;
        }
        tc_st32(tlane + PTC_COL_QL + (uint32_t)(32 * cg), lo32);
        tc_st_wait();
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");        // q high: written here, read by the tensor core
    tc_fence_before();
    __syncthreads();                                                    // (and the box has been read: k and v take its place)
    bool ok = true;
    float acc[64];                                                       // row, dims 64 cg ..
#pragma unroll
    for (int e = 0; e < 64; ++e) acc[e] = 0.0f;
    float m_run = -INFINITY, l_run = 0.0f, alpha = 0.0f;                 // l_run: of the thread's 16 columns of every page
    auto add_page = [&](int par) {
#pragma unroll
        for (int h = 0; h < 8; ++h) {
            int o[8];
            tc_ld8(tlane + PTC_COL_O + (uint32_t)(64 * cg + 8 * h), o);
            tc_ld_wait();
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const float4 f = *reinterpret_cast<const float4 *>(vf + par * ATT_D + 64 * cg + 8 * h + e);
                float *a = acc + 8 * h + e;
                a[0] = __fmaf_rn(__int_as_float(o[e]), f.x, __fmul_rn(a[0], alpha));
                a[1] = __fmaf_rn(__int_as_float(o[e + 1]), f.y, __fmul_rn(a[1], alpha));
                a[2] = __fmaf_rn(__int_as_float(o[e + 2]), f.z, __fmul_rn(a[2], alpha));
                a[3] = __fmaf_rn(__int_as_float(o[e + 3]), f.w, __fmul_rn(a[3], alpha));
            }
        }
    };
    for (int i = 0; i < ntiles; ++i) {
        const int p0 = (page0 + i) * PG_POS;
        const uint32_t par = (uint32_t)(i & 1);
        float *red = red0 + par * 4 * ATC_M;
        float s[16], mx = -INFINITY;
        ok = ok && mbar_wait_both(kfull + par, (uint32_t)((i >> 1) & 1), qk, par);       // (the first is long complete; it makes the copied factors visible)
        tc_fence_after();
        {
            int a[16];
            tc_ld16(tlane + PTC_COL_S + (uint32_t)(16 * cg), a);
            tc_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = __fmul_rn(__int_as_float(a[e]), __fmul_rn(qf, kf[par * ATC_KEYS + 16 * cg + e]));
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(scored);
        if (p0 + PG_POS - 1 > all_see) {                                 // some row does not see some position (one behind the last is behind every row's)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (p0 + 16 * cg + e > limit) s[e] = -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[e]);
        red[cg * ATC_M + row] = mx;
        ptc_barrier();
        float m_new = m_run;
#pragma unroll
        for (int c = 0; c < 4; ++c) m_new = fmaxf(m_new, red[c * ATC_M + row]);
        const float base = m_new == -INFINITY ? 0.0f : m_new, alpha_new = expf(__fsub_rn(m_run, base));
        m_run = m_new;
        uint32_t hi[8], lo[8];
        {
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const float x = expf(__fsub_rn(s[e], base)), y = expf(__fsub_rn(s[e + 1], base));
                sum = __fadd_rn(sum, __fadd_rn(x, y));
                split_f16x2(__fmul_rn(x, 16384.0f), __fmul_rn(y, 16384.0f), hi[e >> 1], lo[e >> 1]);
            }
            l_run = __fadd_rn(__fmul_rn(l_run, alpha_new), sum);
        }
        if (i > 0) {                                                     // the outputs of the page before; its weights have been read
            ok = ok && mbar_wait_both(vfull + (par ^ 1u), (uint32_t)(((i - 1) >> 1) & 1), pv, par ^ 1u);
            tc_fence_after();
        }
        tc_st8(tlane + PTC_COL_P + (uint32_t)(8 * cg), hi);
        tc_st8(tlane + PTC_COL_P + (uint32_t)(32 + 8 * cg), lo);
        if (i > 0) add_page((int)par ^ 1);
        alpha = alpha_new;
        tc_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(weighed);
    }
    if (ntiles > 0) {
        ok = ok && mbar_wait_both(vfull + ((ntiles - 1) & 1), (uint32_t)(((ntiles - 1) >> 1) & 1), pv, (uint32_t)((ntiles - 1) & 1));
        tc_fence_after();
        add_page((ntiles - 1) & 1);
    }
    if (!ok) *failed = 1;
    tc_fence_before();
    __syncthreads();
    float *red = red0;
    red[cg * ATC_M + row] = l_run;
    uint32_t k_most = 0, v_most = 0, v_least = ATC_NONE;
    for (int t = threadIdx.x; t < ntiles; t += ATC_THREADS) {
        const uint32_t *r = reinterpret_cast<const uint32_t *>(img + (size_t)t * img_stride + ATC_IMG_RANGE);
        k_most = max(k_most, r[0]);
        v_most = max(v_most, r[1]);
        v_least = min(v_least, r[2]);
    }
    uint4 *ranges = reinterpret_cast<uint4 *>(kf);                       // a warp each; every page's factors have been read
    seen = __reduce_max_sync(0xffffffffu, seen);
    k_most = __reduce_max_sync(0xffffffffu, k_most);
    v_most = __reduce_max_sync(0xffffffffu, v_most);
    v_least = __reduce_min_sync(0xffffffffu, v_least);
    if (lane == 0) ranges[warp] = make_uint4(seen, k_most, v_most, v_least);
    ptc_barrier();
    const bool all_ok = *failed == 0;
    const uint4 r = ranges[lane & (ATC_WARPS - 1)];
    const uint32_t q_most = __reduce_max_sync(0xffffffffu, r.x);
    const bool redo = q_most >= ATC_HUGE || atc_too_wide(__float_as_uint(fabsf(__fmul_rn(__uint_as_float(q_most), P.scale))), __reduce_max_sync(0xffffffffu, r.y),
                                                       __reduce_max_sync(0xffffffffu, r.z), __reduce_min_sync(0xffffffffu, r.w));
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
    if (threadIdx.x == 0) P.redo[((size_t)blockIdx.x * C.n_head_kv + kvh) * P.splits + split] = redo && all_ok ? 1 : 0;
    if (redo || !all_ok) return;
    const float l = __fadd_rn(__fadd_rn(red[row], red[ATC_M + row]), __fadd_rn(red[2 * ATC_M + row], red[3 * ATC_M + row]));
    const float inv = P.tc_acc != nullptr ? 1.0f : l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);             // a row that sees nothing is zeros
    float *dst = P.tc_acc != nullptr ? P.tc_acc + (size_t)split * C.n_tok * P.n_head * KV_D : P.out;
    if (P.tc_acc != nullptr && cg == 0 && row < n_rows) P.tc_ml[(size_t)split * C.n_tok * P.n_head + row_at(row) / KV_D] = make_float2(m_run, l);
    if ((reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
#pragma unroll
        for (int c = 0; c < 16; ++c)
            box[lane * 16 + (c ^ (lane & 15))] = make_float4(__fmul_rn(acc[4 * c], inv), __fmul_rn(acc[4 * c + 1], inv), __fmul_rn(acc[4 * c + 2], inv), __fmul_rn(acc[4 * c + 3], inv));
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int x = 2 * i + (lane >> 4), c = lane & 15;
            if (row0 + x < n_rows) *reinterpret_cast<float4 *>(dst + row_at(row0 + x) + 64 * cg + 4 * c) = box[x * 16 + (c ^ (x & 15))];
        }
    } else if (row < n_rows) {
        dst += row_at(row) + 64 * cg;
#pragma unroll
        for (int e = 0; e < 64; ++e) dst[e] = __fmul_rn(acc[e], inv);
    }
}

}  // namespace b200
