// pages_shared_tc.cuh -- pages_shared.cuh's attention for entities of many rows (a long prompt's questions, hundreds of answers): 128 rows a tile, rows as the rows of both products.
//
// pages_shared_kernel turns the cache's codes into planes for 48 rows at a time; with that many rows the planes are worth writing down.  pages_shared_planes_kernel writes each page of
// these entities once, as a tile image (attn_tc.cuh's: planes split, swizzled, v transposed), and pages_shared_tc_kernel multiplies: 512 threads, each a row and a quarter of its columns,
// form weights and add outputs; a warp issues the products of scores, one those of outputs, so that the next page's scores and this page's outputs are in flight together; two warps copy
// images, 64 dims of k and 128 of v at a time, each part as soon as its products are done.  Tensor memory: 256 outputs, 64 scores, 64 weights, 128 q low; shared memory: q high, k and v
// of one page.
//
// What bounds it: a chain.  A page takes about 4450 cycles, of which the products of its outputs 1700 (three of four products of planes, 128 x 256 x 64), and adding them and writing the
// next weights 1430: there is one buffer of outputs, since tensor memory has no room for two.  With k, v and both products' waits in one warp it was 6700.  Writing the images takes a
// seventh of a call (53 us for 1000 of them, 131 MB; with conversions by fp32 it took 12 more); beyond 126 MB they also come back from memory.  Its warps' code in 96 registers spills 112 bytes of
// stores a thread.
#pragma once

#include "pages_shared.cuh"

namespace b200 {

constexpr uint32_t PST_COL_O = 0, PST_COL_S = 256, PST_COL_P = 320, PST_COL_QL = 384;
// a fragment: pages of one tile and kv head
struct PstFragment {
    long long part;                     // the first row's place among the parts
    const uint8_t *img;                 // its first page's image
    int begin, row0, n_rows, kvh;       // first token of the entity; of its rows the tile's first, and how many
    int ntiles, pos0;                   // pages (0: no more fragments), first position
    int before, end, all_see;           // row r sees up to before + r / group (INT32_MAX: end - 1); every row sees up to all_see
};
constexpr int PST_THREADS = ATC_THREADS + 128, PST_SCORE_WARP = ATC_WARPS, PST_V_WARP = ATC_WARPS + 2, PST_OUT_WARP = ATC_WARPS + 3;      // (and k's pages)
constexpr int PST_REGS_ROWS = 104, PST_REGS_REST = 64;           // 4 x 104 + 64 = 5 x 96, what the launch has
constexpr int PST_REGS = 32 * (ATC_WARPS * PST_REGS_ROWS + 4 * PST_REGS_REST);
constexpr int PST_BARS = 22;
constexpr int PST_SMEM_BYTES = 1024 + 3 * ATC_PLANES + (2 * ATC_KEYS + 2 * ATT_D + 2 * 4 * ATC_M) * 4 + 8 * PST_BARS + 16 + 2 * (int)sizeof(PstFragment) + 8;
constexpr int PST_IMG_BAD = ATC_IMG_RANGE + 16;                  // 8 bytes of an image: positions whose v is no number
static_assert(PST_IMG_BAD + 8 <= ATC_IMG_BYTES && PST_ROWS == ATC_M && PG_POS == ATC_KEYS && KV_D == ATT_D, "");
__device__ __forceinline__ void pst_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(ATC_THREADS) : "memory"); }        // among the threads that have rows

// Images of the pages of the entities of many rows: image E.image + i is page page0 + i, [kv head] beside each other.  z 0 = k (warp = eight positions, lane = eight dims), z 1 = v
// (thread = one dim, all 64 positions).  Six CTAs of 40 registers fit an SM, and a launch has as many.
__global__ void __launch_bounds__(ATC_PREP_THREADS) pages_shared_planes_kernel(const __grid_constant__ PageShared P) {
    __shared__ __align__(16) uint8_t rows[PG_HEAD_BYTES];
    __shared__ uint32_t odd[2][KV_NBLK];
    __shared__ __align__(16) uint16_t scales[KV_NBLK][ATC_KEYS];
    const PageCache &C = P.C;
    const PshPlan &plan = *P.plan;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, entities = P.n_groups + C.n_seq;
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    const int images = plan.images;
    int e = 0;
#pragma unroll 1
    for (int item = blockIdx.x; item < images * C.n_head_kv; item += gridDim.x) {
        const int image = item / C.n_head_kv, kvh = item - image * C.n_head_kv;
        // whose: the last entity whose images begin at or in front of it
        for (int at = -1; at < 0; e += 32) {
            const bool mine = e + lane < entities && plan.entity[e + lane].image >= 0 && plan.entity[e + lane].image <= image &&
                              image < plan.entity[e + lane].image + (plan.entity[e + lane].end + PG_POS - 1) / PG_POS - plan.entity[e + lane].page0;
            const unsigned found = __ballot_sync(0xffffffffu, mine);
            if (found || e >= entities) {
                at = found ? e + __ffs(found) - 1 : entities;
                e = min(at, entities) - 32;              // (the loop adds them again)
            }
        }
        if (e >= entities) return;
        const PshEntity E = plan.entity[e];
        const int page_at = E.page0 + image - E.image, n = min(PG_POS, E.end - page_at * PG_POS);
        const int page = E.seq >= 0 ? C.table[(size_t)E.seq * C.table_stride + page_at] : -1;
        const bool there = page >= 0 && page < C.n_pages;
        if (!there && threadIdx.x == 0) bad_sequence();
        {
            const uint4 *src = reinterpret_cast<const uint4 *>(page_rows(C, there ? page : 0, P.layer, blockIdx.z, kvh));
            const int words = there ? n * (KV_ROW / 16) : 0;
            for (int i = threadIdx.x; i < PG_HEAD_BYTES / 16; i += ATC_PREP_THREADS) reinterpret_cast<uint4 *>(rows)[i] = i < words ? src[i] : make_uint4(0u, 0u, 0u, 0u);
        }
        __syncthreads();
        uint8_t *img = P.images + (size_t)item * ATC_IMG_BYTES;
        uint32_t hi[4], lo[4];
        if (blockIdx.z == 0) {                           // a row's scales under one power of two, as pages_shared_kernel has them
            constexpr int ROWS = ATC_KEYS / (ATC_PREP_THREADS / 32);
#pragma unroll 2
            for (int r = 0; r < ROWS; ++r) {
                const int key = ROWS * warp + r;
                const uint16_t *b = reinterpret_cast<const uint16_t *>(rows + key * KV_ROW + 34 * (lane >> 2));
                const int s = psh_shift(__reduce_max_sync(0xffffffffu, (uint32_t)b[0] & 0x7FFFu));
                const uint32_t d = psh_scale(b[0], atc_pow2(s));
#pragma unroll
                for (int i = 0; i < 4; ++i) psh_planes(psh_pair((uint32_t)b[1 + 4 * (lane & 3) + i] ^ 0x8080u, false), d, hi[i], lo[i]);
                uint8_t *dst = img + (lane >> 3) * ATC_CHUNK + key * 128 + (((lane & 7) ^ (key & 7)) * 16);
                *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4 *>(dst + ATC_KEYS * 128) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                if (lane == 0) reinterpret_cast<float *>(img + ATC_IMG_KF)[key] = atc_pow2(-s);
            }
        } else {                                         // a warp has a block of 32 dims: its scales under one power of two, those that are no numbers zero
            const int dim = threadIdx.x;
            uint32_t d[2], m = 0;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                d[j] = *reinterpret_cast<const uint16_t *>(rows + (32 * j + lane) * KV_ROW + 34 * warp);
                const bool bad = (d[j] & 0x7FFFu) >= 0x7C00u;
                const uint32_t mask = __ballot_sync(0xffffffffu, bad);       // (its rows are told apart by who has weights for them)
                if (lane == 0) odd[j][warp] = mask;
                if (bad) d[j] = 0;
                m = max(m, d[j] & 0x7FFFu);
            }
            const int s = psh_shift(__reduce_max_sync(0xffffffffu, m));
#pragma unroll
            for (int j = 0; j < 2; ++j) scales[warp][32 * j + lane] = (uint16_t)psh_scale(d[j], atc_pow2(s));
            __syncwarp();
            reinterpret_cast<float *>(img + ATC_IMG_VF)[dim] = atc_pow2(-s - 14);        // (and the weights' 2^-14)
            const int byte = 34 * warp + 2 + lane;
            const uint32_t pick = (uint32_t)(byte & 3) | ((uint32_t)(byte & 3) + 4u) << 8;
            const uint32_t *src = reinterpret_cast<const uint32_t *>(rows + (byte & ~3));
#pragma unroll 2
            for (int g = 0; g < ATC_KEYS / 8; ++g) {
                const uint4 d4 = *reinterpret_cast<const uint4 *>(&scales[warp][8 * g]);
                const uint32_t dd[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t *x = src + (8 * g + 2 * e) * (KV_ROW / 4);
                    psh_planes(psh_codes(x[0], x[KV_ROW / 4], pick), dd[e], hi[e], lo[e]);
                }
                uint8_t *dst = img + ATC_PLANES + dim * 128 + ((g ^ (dim & 7)) * 16);
                *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4 *>(dst + 2 * ATC_CHUNK) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
            __syncthreads();
            if (dim < 2) {
                uint32_t all = 0;
#pragma unroll
                for (int b = 0; b < KV_NBLK; ++b) all |= odd[dim][b];
                reinterpret_cast<uint32_t *>(img + PST_IMG_BAD)[dim] = all;
            }
        }
        __syncthreads();                                 // the next item's rows take the place of these
    }
}

// The warps without rows: one issues the products of scores, one says what the fragments are and issues those of outputs, two copy images.
__device__ __forceinline__ void pst_drivers(const PageShared &P, PstFragment *desc, uint8_t *qhi, uint8_t *kpl, uint8_t *vpl, float *kf, float *vf, uint64_t *qk, unsigned long long *bad,
                                            volatile int *failed, uint32_t tmem) {
    uint64_t *pv = qk + 1, *scored = qk + 2, *weighed = qk + 3, *vfull = qk + 4, *kfull = qk + 6, *kfree = qk + 10, *ffull = qk + 14, *vfree = qk + 16, *gfull = qk + 18, *done = qk + 20;
    const PshPlan &plan = *P.plan;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, heads = P.C.n_head_kv, entities = P.n_groups + P.C.n_seq;
    const size_t img_stride = (size_t)heads * ATC_IMG_BYTES;
    // After a wait that ran out a warp waits for nothing more, copies nothing and issues nothing.  What it has begun ends before the CTA does: tensor memory is given back then, and shared
    // memory becomes another CTA's.
    bool ok = true;
    auto wait = [&](uint64_t *bar, uint32_t parity) { ok = ok && __all_sync(0xffffffffu, psh_wait<true>(bar, parity)); };
    auto copies_end = [&](int begun, uint64_t *full, int parts, uint64_t *factors) {
#pragma unroll 1
        for (int c = 0; c < parts; ++c)
            if (begun > c) psh_wait<true>(full + c, (uint32_t)((in_turn(begun, parts, c) - 1) & 1));
        const int pages = in_turn(begun, parts, 0);
#pragma unroll 1
        for (int c = 0; c < 2; ++c)
            if (pages > c) psh_wait<true>(factors + c, (uint32_t)((in_turn(pages, 2, c) - 1) & 1));
    };
    auto products_end = [&](uint64_t *bar) {
        if (elect_one()) tc_commit(bar);
        __syncwarp();
        psh_wait<true>(bar, 0);
    };
    // 64 dims of k, 128 of v give their place to the next page's when they are done.  (Waits between the products cost 250 cycles each, and nothing is multiplied meanwhile.)
    auto issue_qk = [&](int it) {
        constexpr uint32_t LOW = (ATC_KEYS * 128) >> 4;
        const uint32_t a0 = tc16_desc_lo(smem_u32(qhi)), b0 = tc16_desc_lo(smem_u32(kpl)), d = tmem + PST_COL_S;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) wait(kfull + c, (uint32_t)(it & 1));
        if (!ok) return;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {                // products with a low plane first
                const uint32_t a = a0 + (uint32_t)(c * (ATC_CHUNK >> 4)), b = b0 + (uint32_t)(c * (ATC_CHUNK >> 4)), ql = tmem + PST_COL_QL + (uint32_t)(32 * c);
                if (c == 0) tc_mma_f16_ts<false>(d, ql, b, atc_idesc(ATC_KEYS));
                else tc_mma_f16_ts<true>(d, ql, b, atc_idesc(ATC_KEYS));
#pragma unroll
                for (int n = 1; n < 4; ++n) tc_mma_f16_ts<true>(d, ql + (uint32_t)(8 * n), b + (uint32_t)(2 * n), atc_idesc(ATC_KEYS));
#pragma unroll
                for (int n = 0; n < 4; ++n) atc_mma_ss<atc_idesc(ATC_KEYS)>(d, a + (uint32_t)(2 * n), b + LOW + (uint32_t)(2 * n));
#pragma unroll
                for (int n = 0; n < 4; ++n) atc_mma_ss<atc_idesc(ATC_KEYS)>(d, a + (uint32_t)(2 * n), b + (uint32_t)(2 * n));
                tc_commit(kfree + c);
            }
            tc_commit(qk);
        }
        __syncwarp();
    };
    auto issue_pv = [&](int it) {
        const uint32_t b0 = tc16_desc_lo(smem_u32(vpl)), ph = tmem + PST_COL_P, pl = ph + 32u;
        wait(vfull, (uint32_t)(it & 1));
        wait(vfull + 1, (uint32_t)(it & 1));
        if (!ok) return;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const uint32_t d = tmem + PST_COL_O + (uint32_t)(128 * c), b1 = b0 + (uint32_t)(c * (ATC_CHUNK >> 4));
#pragma unroll
                for (int n = 0; n < 12; ++n) {
                    const uint32_t a = (n < 4 ? pl : ph) + (uint32_t)(8 * (n & 3));
                    const uint32_t b = b1 + (uint32_t)((n >= 4 && n < 8 ? (2 * ATC_CHUNK) >> 4 : 0) + 2 * (n & 3));
                    if (n == 0) tc_mma_f16_ts<false>(d, a, b, atc_idesc(ATT_D / 2));
                    else tc_mma_f16_ts<true>(d, a, b, atc_idesc(ATT_D / 2));
                }
                tc_commit(vfree + c);
            }
            tc_commit(pv);
        }
        __syncwarp();
    };
    // the next fragment of the CTA's line
    const long long per = plan.tc_per, last = min(per * (blockIdx.x + 1), plan.tc_total);
    long long at = per * blockIdx.x;
    int e = plan.tc_first[blockIdx.x];
    auto next = [&](PstFragment &F) {
        F.ntiles = 0;
        while (at < last && e < entities) {
            const PshEntity E = plan.entity[e];
            const int size = E.steps + PST_START, rows = E.tokens * P.group;
            const long long tiles = (rows + PST_ROWS - 1) / PST_ROWS, pair = E.unit < 0 || E.image < 0 ? tiles * heads : (at - E.unit) / size;
            if (pair >= tiles * heads) {
                ++e;
                continue;
            }
            const long long begin = E.unit + pair * size;
            const int tile = (int)(pair / heads), page0 = (int)max(0ll, at - begin - PST_START);
            F.kvh = (int)(pair - (long long)tile * heads);
            F.row0 = tile * PST_ROWS;
            F.n_rows = min(PST_ROWS, rows - F.row0);
            F.end = psh_tile_end(P.group, E, F.row0, PST_ROWS);
            F.ntiles = max(0, min((int)min(last - begin, (long long)size) - PST_START, (F.end + PG_POS - 1) / PG_POS - E.page0) - page0);
            F.begin = E.begin;
            F.before = E.before;
            F.pos0 = (E.page0 + page0) * PG_POS;
            F.all_see = E.before == INT32_MAX ? F.end - 1 : E.before + F.row0 / P.group;
            F.img = P.images + ((size_t)(E.image + page0) * heads + F.kvh) * ATC_IMG_BYTES;
            F.part = plan.tc_row + E.row + (long long)F.row0 * heads + (long long)F.kvh * F.n_rows + (long long)blockIdx.x * PST_ROWS;
            at = begin + size;
            if (F.ntiles > 0) return;
        }
    };
    if (warp == PST_OUT_WARP) {
        PstFragment F;
        int it = 0;
        next(F);
        if (lane == 0) desc[0] = F;
        for (int f = 0;; ++f) {
            __syncthreads();
            const int ntiles = F.ntiles;
            if (ntiles == 0 || *failed) break;
            next(F);                                     // (its place is the last one's, which everybody has left)
            if (lane == 0) desc[(f + 1) & 1] = F;
            __syncthreads();
#pragma unroll 1
            for (int i = 0; i < ntiles && ok; ++i, ++it) {         // outputs
                wait(weighed, (uint32_t)(it & 1));
                issue_pv(it);
            }
            if (!ok) *failed = 1;
            __syncthreads();
            __syncthreads();
        }
        products_end(done);
        return;
    }
    // the fragments one after the other: a warp's part of n pages, their images from img on
    auto fragments = [&](auto part) {
        for (int f = 0;; ++f) {
            __syncthreads();
            const int ntiles = desc[f & 1].ntiles;
            const uint8_t *img = desc[f & 1].img;
            if (ntiles == 0 || *failed) break;
            __syncthreads();
            part(ntiles, img);
            if (!ok) *failed = 1;
            __syncthreads();
            __syncthreads();
        }
    };
    if (warp == PST_SCORE_WARP) {
        int it = 0;
        fragments([&](int n, const uint8_t *) {
#pragma unroll 1
            for (int i = 0; i < n && ok; ++i, ++it) {    // scores
                if (it > 0) wait(scored, (uint32_t)((it - 1) & 1));
                issue_qk(it);
            }
        });
        products_end(done + 1);
    } else if (warp == PST_V_WARP) {
        const uint64_t pol = policy_evict_last_or_default();
        int begun = 0;                                   // parts of pages
        fragments([&](int n, const uint8_t *img) {
#pragma unroll 1
            for (int i = 0; i < 2 * n; ++i, ++begun) {
                const int it = begun >> 1, c = begun & 1;
                if (it > 0) wait(vfree + c, (uint32_t)((it - 1) & 1));
                if (!ok) break;
                if (lane == 0) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");         // the factors were read by ordinary loads
                    if (c == 0) {                        // (their place is the page's before the last: its outputs were added in front of the weights that page `it - 1` waited for)
                        bad[it & 1] = *reinterpret_cast<const unsigned long long *>(img + PST_IMG_BAD);
                        mbar_expect_tx(gfull + (it & 1), ATT_D * 4);
                        bulk_g2s(vf + (it & 1) * ATT_D, img + ATC_IMG_VF, ATT_D * 4, gfull + (it & 1), pol);
                    }
                    mbar_expect_tx(vfull + c, 2 * ATC_CHUNK);
                    bulk_g2s(vpl + c * ATC_CHUNK, img + ATC_PLANES + c * ATC_CHUNK, ATC_CHUNK, vfull + c, pol);
                    bulk_g2s(vpl + (2 + c) * ATC_CHUNK, img + ATC_PLANES + (2 + c) * ATC_CHUNK, ATC_CHUNK, vfull + c, pol);
                }
                __syncwarp();
                if (c == 1) img += img_stride;
            }
        });
        copies_end(begun, vfull, 2, gfull);
    } else {
        const uint64_t pol = policy_evict_last_or_default();
        int begun = 0;
        fragments([&](int n, const uint8_t *img) {
#pragma unroll 1
            for (int i = 0; i < 4 * n; ++i, ++begun) {
                const int it = begun >> 2, c = begun & 3;
                if (it > 0) wait(kfree + c, (uint32_t)((it - 1) & 1));
                if (!ok) break;
                if (lane == 0) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    if (c == 0) {
                        mbar_expect_tx(ffull + (it & 1), ATC_KEYS * 4);
                        bulk_g2s(kf + (it & 1) * ATC_KEYS, img + ATC_IMG_KF, ATC_KEYS * 4, ffull + (it & 1), pol);
                    }
                    mbar_expect_tx(kfull + c, ATC_CHUNK);
                    bulk_g2s(kpl + c * ATC_CHUNK, img + c * ATC_CHUNK, ATC_CHUNK, kfull + c, pol);
                }
                __syncwarp();
                if (c == 3) img += img_stride;
            }
        });
        copies_end(begun, kfull, 4, ffull);
    }
}
// The warps with rows.
__device__ __forceinline__ void pst_rows(const PageShared &P, const PstFragment *desc, uint8_t *qhi, uint8_t *kpl, float *kf, float *vf, float *red0, uint64_t *qk, unsigned long long *bad,
                                         volatile int *failed, uint32_t tmem) {
    uint64_t *pv = qk + 1, *scored = qk + 2, *weighed = qk + 3, *ffull = qk + 14, *gfull = qk + 18;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, cg = warp >> 2, row = 32 * (warp & 3) + lane;         // a thread's row, and its quarter of the row's columns
    const uint32_t tlane = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    int it0 = 0;                                         // pages of the fragments before
    bool ok = true;
#pragma unroll 1
    for (int f = 0;; ++f) {
            __syncthreads();
            const PstFragment &F = desc[f & 1];
            const int ntiles = F.ntiles, n_rows = F.n_rows;
            if (ntiles == 0 || *failed) return;
            // the last position that the thread's row sees
            const int limit = F.before == INT32_MAX ? F.end - 1 : row < n_rows ? F.before + (F.row0 + row) / P.group : -1, all_see = F.all_see, pos0 = F.pos0;
            auto row_at = [&](int r) {                   // where a row of the tile lies in q
                const int x = F.row0 + r, tok = x / P.group;
                return ((size_t)(F.begin + tok) * P.n_head + F.kvh * P.group + (x - tok * P.group)) * KV_D;
            };
            // ---- q: row of the thread, 64 dims, quantised to Q8_0 (two blocks); high plane to shared memory, low plane to tensor memory, through shared memory (the planes' of k and
            // v, a warp's 32 rows of 64 values each, 16-byte pieces swizzled)
            float4 *box = reinterpret_cast<float4 *>(kpl) + warp * 512;
            const int box0 = 32 * (warp & 3);
            float qf = 0.0f;
            {
                float x[64];
                if ((reinterpret_cast<uintptr_t>(P.q) & 15u) == 0) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int r = 2 * i + (lane >> 4), c = lane & 15;
                        if (box0 + r < n_rows) cp_async16(box + r * 16 + (c ^ (r & 15)), P.q + row_at(box0 + r) + 64 * cg + 4 * c);
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
                    for (int i = 0; i < 64; ++i) x[i] = row < n_rows ? src[i] : 0.0f;
                }
                uint32_t m = 0;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    float amax = 0.0f;
#pragma unroll
                    for (int i = 0; i < 32; ++i) amax = fmaxf(amax, fabsf(x[32 * b + i]));
                    const float d = __fmul_rn(amax, PG_SCALE), id = d > 0.0f ? __fdiv_rn(1.0f, d) : 0.0f, d16 = f16_bits_to_f32(f32_to_f16_bits_ties_away(d));
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        x[32 * b + i] = __fmul_rn((float)max(-127, min(127, round_ties_away(__fmul_rn(x[32 * b + i], id)))), d16);
                        m = max(m, atc_abs_bits(x[32 * b + i]));
                    }
                }
                uint32_t *redu = reinterpret_cast<uint32_t *>(red0);
                redu[cg * ATC_M + row] = m;
                pst_barrier();
#pragma unroll
                for (int c = 0; c < 4; ++c) m = max(m, redu[c * ATC_M + row]);
                const int s = atc_shift(min(m, 0x7F7FFFFFu), 63);
                qf = __fmul_rn(atc_pow2(-s), __fmul_rn(__fmul_rn(P.scale, 1.44269504088896340736f), PSH_LIFT));        // scores as powers of two
                uint32_t lo32[32];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    uint4 hi, lo;
                    atc_split8(x + 8 * j, atc_pow2(s), hi, lo);
                    *reinterpret_cast<uint4 *>(qhi + cg * ATC_CHUNK + row * 128 + ((j ^ (row & 7)) * 16)) = hi;
                    lo32[4 * j] = lo.x; lo32[4 * j + 1] = lo.y; lo32[4 * j + 2] = lo.z; lo32[4 * j + 3] = lo.w;
                }
                tc_st32(tlane + PST_COL_QL + (uint32_t)(32 * cg), lo32);
                tc_st_wait();
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");        // q high: written here, read by the tensor core
            tc_fence_before();
            __syncthreads();                                            // (and the box has been read: k and v take its place)
            float2 acc[32];                                             // row, dims 64 cg ..
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[i] = make_float2(0.0f, 0.0f);
            float m_run = -INFINITY, l_run = 0.0f, alpha = 1.0f;        // l_run: of the thread's 16 columns of every page
            auto add_page = [&](int par) {
                if (__any_sync(0xffffffffu, alpha != 1.0f))
#pragma unroll
                    for (int i = 0; i < 32; ++i) acc[i] = mul2(acc[i], make_float2(alpha, alpha));
#pragma unroll
                for (int h = 0; h < 8; ++h) {
                    int o[8];
                    tc_ld8(tlane + PST_COL_O + (uint32_t)(64 * cg + 8 * h), o);
                    tc_ld_wait();
#pragma unroll
                    for (int i = 0; i < 8; i += 4) {
                        const float4 f = *reinterpret_cast<const float4 *>(vf + par * ATT_D + 64 * cg + 8 * h + i);
                        float2 *a = acc + 4 * h + (i >> 1);
                        a[0] = fma2(make_float2(__int_as_float(o[i]), __int_as_float(o[i + 1])), make_float2(f.x, f.y), a[0]);
                        a[1] = fma2(make_float2(__int_as_float(o[i + 2]), __int_as_float(o[i + 3])), make_float2(f.z, f.w), a[1]);
                    }
                }
            };
            // rows that see a position whose v is no number are no numbers
            auto poison = [&](int par, int p0) {
                const unsigned long long who = bad[par];
                if (who && (limit - p0 >= 63 ? true : limit >= p0 && (who & ((2ull << (limit - p0)) - 1)))) l_run = __int_as_float(0x7FC00000);
            };
#pragma unroll 1
            for (int i = 0; i <= ntiles; ++i) {
                const int it = it0 + i, p0 = pos0 + i * PG_POS;
                const uint32_t par = (uint32_t)(it & 1);
                uint32_t hi[8], lo[8];
                float alpha_new = 1.0f;
                if (i < ntiles) {
                    float *red = red0 + par * 4 * ATC_M;
                    float s[16], mx = -INFINITY;
                    ok = ok && psh_wait<true>(ffull + par, (uint32_t)((it >> 1) & 1)) && psh_wait<true>(qk, par);        // (the first is long complete; it makes the copied factors visible)
                    tc_fence_after();
                    tc_ld16(tlane + PST_COL_S + (uint32_t)(16 * cg), reinterpret_cast<int (&)[16]>(s));
                    tc_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const float4 f = *reinterpret_cast<const float4 *>(kf + par * ATC_KEYS + 16 * cg + j);
                        const float2 a = mul2(make_float2(s[j], s[j + 1]), mul2(make_float2(qf, qf), make_float2(f.x, f.y)));
                        const float2 b = mul2(make_float2(s[j + 2], s[j + 3]), mul2(make_float2(qf, qf), make_float2(f.z, f.w)));
                        s[j] = a.x; s[j + 1] = a.y; s[j + 2] = b.x; s[j + 3] = b.y;
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(scored);
                    if (p0 + PG_POS - 1 > all_see) {                    // some row does not see some position (one behind the last is behind every row's)
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (p0 + 16 * cg + j > limit) s[j] = -INFINITY;
                    }
#pragma unroll
                    for (int j = 0; j < 16; j += 2) mx = fmaxf(mx, fmaxf(s[j], s[j + 1]));
                    red[cg * ATC_M + row] = mx;
                    pst_barrier();
                    float m_new = m_run;
#pragma unroll
                    for (int c = 0; c < 4; ++c) m_new = fmaxf(m_new, red[c * ATC_M + row]);
                    const float base = m_new == -INFINITY ? 0.0f : m_new;
                    alpha_new = m_new == m_run ? 1.0f : psh_exp2(__fsub_rn(m_run, base));
                    m_run = m_new;
                    const float less = __fsub_rn(14.0f, base);          // (weights come as 2^14 of themselves)
                    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const float2 t = add2(make_float2(s[j], s[j + 1]), make_float2(less, less)), w = make_float2(psh_exp2(t.x), psh_exp2(t.y));
                        sum = add2(sum, w);
                        const __half2 h = __floats2half2_rn(w.x, w.y);
                        const float2 rest = fma2(__half22float2(h), make_float2(-1.0f, -1.0f), w);       // exact
                        const __half2 r = __floats2half2_rn(rest.x, rest.y);
                        hi[j >> 1] = *reinterpret_cast<const uint32_t *>(&h);
                        lo[j >> 1] = *reinterpret_cast<const uint32_t *>(&r);
                    }
                    l_run = __fmaf_rn(l_run, alpha_new, __fadd_rn(sum.x, sum.y));
                }
                if (i > 0) {                                            // the outputs of the page before; its weights have been read
                    const uint32_t was = par ^ 1u;
                    ok = ok && psh_wait<true>(pv, was) && psh_wait<true>(gfull + was, (uint32_t)(((it - 1) >> 1) & 1));
                    tc_fence_after();
                }
                if (i < ntiles) {
                    tc_st8(tlane + PST_COL_P + (uint32_t)(8 * cg), hi);
                    tc_st8(tlane + PST_COL_P + (uint32_t)(32 + 8 * cg), lo);
                }
                if (i > 0) {
                    add_page((int)par ^ 1);
                    poison((int)par ^ 1, p0 - PG_POS);
                }
                alpha = alpha_new;
                tc_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0 && i < ntiles) mbar_arrive(weighed);
            }
            it0 += ntiles;
            if (!ok) *failed = 1;
            tc_fence_before();
            __syncthreads();
            ok = *failed == 0;
            float *red = red0;
            red[cg * ATC_M + row] = l_run;
            pst_barrier();
            const size_t part = (size_t)F.part;
            if (ok) {
                if (cg == 0 && row < n_rows) {
                    const float l = __fadd_rn(__fadd_rn(red[row], red[ATC_M + row]), __fadd_rn(red[2 * ATC_M + row], red[3 * ATC_M + row]));
                    P.part_ml[part + row] = make_float2(m_run, __fmul_rn(l, 0x1p-14f));
                }
                float *dst = P.part + part * KV_D;
#pragma unroll
                for (int c = 0; c < 16; ++c) box[lane * 16 + (c ^ (lane & 15))] = make_float4(acc[2 * c].x, acc[2 * c].y, acc[2 * c + 1].x, acc[2 * c + 1].y);
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int x = 2 * i + (lane >> 4), c = lane & 15;
                    if (box0 + x < n_rows) *reinterpret_cast<float4 *>(dst + (size_t)(box0 + x) * KV_D + 64 * cg + 4 * c) = box[x * 16 + (c ^ (x & 15))];
                }
            }
            __syncthreads();
    }
}

__global__ void __launch_bounds__(PST_THREADS, 1) pages_shared_tc_kernel(const __grid_constant__ PageShared P) {
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *qhi = smem + ((1024u - (smem_u32(smem) & 1023u)) & 1023u);
    uint8_t *kpl = qhi + ATC_PLANES, *vpl = kpl + ATC_PLANES;
    float *kf = reinterpret_cast<float *>(vpl + ATC_PLANES);             // [2][64] 2^-s of the page's positions, pages alternate
    float *vf = kf + 2 * ATC_KEYS;                                       // [2][256] 2^-s of the dims (and the weights' 2^-14)
    float *red0 = vf + 2 * ATT_D;                                        // [2][4][128] exchange between the four warps of a row, pages alternate
    uint64_t *qk = reinterpret_cast<uint64_t *>(red0 + 2 * 4 * ATC_M);               // scores there, outputs there, scores read, weights there; k and v, by 64 and 128 dims, there and free; factors; all products done
    unsigned long long *bad = reinterpret_cast<unsigned long long *>(qk + PST_BARS);        // [2] positions of the page whose v is no number
    PstFragment *desc = reinterpret_cast<PstFragment *>(bad + 2);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(desc + 2);
    volatile int *failed = reinterpret_cast<int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (int b = 0; b < PST_BARS; ++b) mbar_init(qk + b, b == 2 || b == 3 ? ATC_WARPS : 1);
        mbar_fence_init();
        *failed = 0;
    }
    pdl_wait_prior_grid();                                               // the plan and the images
    pdl_launch_dependents();
    if (P.plan->tc_per * blockIdx.x >= P.plan->tc_total) return;         // CTA-uniform
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    __syncthreads();                                                     // the barriers, and where tensor memory is
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // Every warp is at four barriers of the CTA for a fragment: (1) it is known, (2) q is in its places, (3) its pages are done, (4) its sums are out.
    if (warp >= ATC_WARPS) {
        psh_set_registers<PST_REGS_REST>(false);
        pst_drivers(P, desc, qhi, kpl, vpl, kf, vf, qk, bad, failed, tmem);
    } else {
        psh_set_registers<PST_REGS_ROWS>(true);
        pst_rows(P, desc, qhi, kpl, kf, vf, red0, qk, bad, failed, tmem);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

}  // namespace b200
