// pages.cuh -- a Q8_0 K/V cache in pages of 64 positions: append, attention of several sequences' new tokens over it, copies.
//
// Layout: pool[page][layer][K | V][kv head][64 positions][272 bytes]; a row is the row of kv.cuh (8 blocks of 34 bytes), so the rows of a page for one
// layer and kv head are ONE span of 17408 bytes.  Position p of sequence s lies in page table[s][p / 64], row p % 64.
#pragma once

#include "common.cuh"
#include "kv.cuh"
#include "seqs.cuh"

namespace b200 {

constexpr int PG_POS = 64, PG_HEAD_BYTES = PG_POS * KV_ROW;
static_assert(PG_POS == KV_TILE, "");
constexpr int PG_MAX_PAGES = 1 << 24;                            // of a sequence: its positions are counted in 32 bits

struct PageCache {
    uint8_t *pool;
    const int32_t *table, *len, *start;
    int n_pages, n_layers, n_head_kv, n_seq, table_stride, n_tok;
};

__device__ __forceinline__ uint8_t *page_rows(const PageCache &C, int page, int layer, int kv, int head) {
    return C.pool + ((((size_t)page * C.n_layers + layer) * 2 + kv) * C.n_head_kv + head) * PG_HEAD_BYTES;
}

// ---- append -----------------------------------------------------------------------------------------------------------------------------------
// One warp per (token, kv head) row of K and of V, as kv_append_kernel.  A block's scale is its largest magnitude times 1 / 127, one rounded product where that kernel
// divides: the fp32 scales differ in the last bit for one magnitude in 21, the fp16 ones that are stored for none (all 2^23 mantissas at every exponent looked at), and a code whose
// quotient lies beside a half is the neighbouring one in one value of 10^7.
constexpr float PG_SCALE = 1.0f / 127.0f;
template <bool VEC>
__global__ void __launch_bounds__(32 * KV_APPEND_WARPS) pages_append_kernel(const __grid_constant__ PageCache C, const float *ksrc, const float *vsrc, int layer) {
    __shared__ __align__(16) uint8_t rows[KV_APPEND_WARPS][2][KV_ROW];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = (int64_t)blockIdx.x * KV_APPEND_WARPS + warp;          // token * n_head_kv + head
    if (row >= (int64_t)C.n_tok * C.n_head_kv) return;
    const int tok = (int)(row / C.n_head_kv), h = (int)(row - (int64_t)tok * C.n_head_kv);
    const int blk = lane >> 2, sub = lane & 3;
    const float *kr = ksrc + row * KV_D + blk * 32 + sub * 8;
    const float *vr = vsrc + row * KV_D + blk * 32 + sub * 8;
    float kx[8], vx[8];
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    if (blockIdx.x == 0) report_ranges(C.start, C.n_seq, C.n_tok);
    const int s = seq_of_row(C.start, C.n_seq, tok, lane);
    if (VEC) {
        const float4 a = *reinterpret_cast<const float4 *>(kr), b = *reinterpret_cast<const float4 *>(kr + 4);
        const float4 c = *reinterpret_cast<const float4 *>(vr), e = *reinterpret_cast<const float4 *>(vr + 4);
        kx[0] = a.x; kx[1] = a.y; kx[2] = a.z; kx[3] = a.w; kx[4] = b.x; kx[5] = b.y; kx[6] = b.z; kx[7] = b.w;
        vx[0] = c.x; vx[1] = c.y; vx[2] = c.z; vx[3] = c.w; vx[4] = e.x; vx[5] = e.y; vx[6] = e.z; vx[7] = e.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) { kx[i] = kr[i]; vx[i] = vr[i]; }
    }
    if (s >= C.n_seq) return;                                   // rows behind the last sequence
    const SeqRange r = seq_range(C.start, s, C.n_tok);
    const int64_t pos = (int64_t)C.len[s] - r.n + (tok - r.begin);
    int page = -1;
    if (r.n > 0 && tok >= r.begin && pos >= 0 && pos / PG_POS < C.table_stride) page = C.table[(size_t)s * C.table_stride + pos / PG_POS];
    if (page < 0 || page >= C.n_pages) {
        if (lane == 0) bad_sequence();
        return;
    }
    const size_t at = (size_t)(pos % PG_POS) * KV_ROW;
    // the reciprocals of K by the even lanes of the four, of V by the odd ones
    const float kmax = kv_amax_8(kx), vmax = kv_amax_8(vx), d = __fmul_rn(sub & 1 ? vmax : kmax, PG_SCALE), id = d > 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
    const uint32_t d16 = f32_to_f16_bits_ties_away(d);
    uint32_t kw[2], vw[2];
    kv_words_8(kx, __shfl_sync(0xffffffffu, id, lane & ~3), kw);
    kv_words_8(vx, __shfl_sync(0xffffffffu, id, lane | 1), vw);
    uint8_t *kb = rows[warp][0], *vb = rows[warp][1];           // put together by halfwords, stored by 16-byte words
    unsigned short *kp = reinterpret_cast<unsigned short *>(kb + 34 * blk), *vp = reinterpret_cast<unsigned short *>(vb + 34 * blk);
    if (sub < 2) (sub ? vp : kp)[0] = (unsigned short)d16;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        kp[1 + 4 * sub + 2 * j] = (unsigned short)(kw[j] & 0xFFFFu); kp[2 + 4 * sub + 2 * j] = (unsigned short)(kw[j] >> 16);
        vp[1 + 4 * sub + 2 * j] = (unsigned short)(vw[j] & 0xFFFFu); vp[2 + 4 * sub + 2 * j] = (unsigned short)(vw[j] >> 16);
    }
    __syncwarp();
    if (lane < KV_ROW / 16) {
        reinterpret_cast<uint4 *>(page_rows(C, page, layer, 0, h) + at)[lane] = reinterpret_cast<const uint4 *>(kb)[lane];
        reinterpret_cast<uint4 *>(page_rows(C, page, layer, 1, h) + at)[lane] = reinterpret_cast<const uint4 *>(vb)[lane];
    }
}

// ---- copies -----------------------------------------------------------------------------------------------------------------------------------
constexpr int PG_COPY_PAIRS = 480, PG_COPY_THREADS = 256, PG_COPY_WORDS = 8;            // 16-byte words a thread holds
struct PagePairs { int32_t src[PG_COPY_PAIRS], dst[PG_COPY_PAIRS]; };
// No page is written twice or both read and written (the host has looked), so the order does not matter.  Bound by memory: 300 pages of 2.2 MB, 1.34 GB read and written, 212 us
// (6.3 TB/s); four pages 5.5 us, of which the launch is half.  The pairs are launch parameters: 480 are what fits beside the rest, more are more launches.
__global__ void __launch_bounds__(PG_COPY_THREADS) pages_copy_kernel(const __grid_constant__ PagePairs L, uint8_t *pool, int64_t page_words, int64_t parts, int64_t items) {
    constexpr int PART = PG_COPY_THREADS * PG_COPY_WORDS;
    pdl_wait_prior_grid();
    for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
        const int64_t pair = i / parts, w0 = (i - pair * parts) * PART + threadIdx.x;
        const uint4 *src = reinterpret_cast<const uint4 *>(pool) + L.src[pair] * page_words;
        uint4 *dst = reinterpret_cast<uint4 *>(pool) + L.dst[pair] * page_words;
        uint4 x[PG_COPY_WORDS];
#pragma unroll
        for (int j = 0; j < PG_COPY_WORDS; ++j)
            if (w0 + j * PG_COPY_THREADS < page_words) x[j] = src[w0 + j * PG_COPY_THREADS];
#pragma unroll
        for (int j = 0; j < PG_COPY_WORDS; ++j)
            if (w0 + j * PG_COPY_THREADS < page_words) dst[w0 + j * PG_COPY_THREADS] = x[j];
    }
}

// ---- attention --------------------------------------------------------------------------------------------------------------------------------
// The value is that of kv_attn_kernel for each new token by itself: its queries are quantised to Q8_0 and see the positions up to their own.
//   score    scale * sum over the blocks of dq dk (q8 . k8)              int8 products on mma.sync (m16n8k32), int32 sums, scaled per block in fp32
//   output   sum of p dv v8 / sum of p, p = e^(score - maximum)          p dv in two fp16 planes, v8 as fp16 (exact), fp32 sums
//
// Rows: a token's query heads that share a kv head are rows of one matrix: row r of a sequence is head r % group of new token r / group.  A CTA
// takes 16 ROWT rows (ROWT = 0: 8) of one kv head and one span of the sequence's pages, a page at a time:
//   scales   the page's fp16 scales as floats, the V ones of a block under a power of two of their own
//   scores   a warp has 16 rows and 8, 16 or all 64 positions (ROWT up to 1, 2, 4); weights in fp32 to shared memory
//   outputs  a warp has all rows and 32 dims, a block (ROWT = 4: 64 dims); eight rows' high and low planes are the 16 rows of one product: V's bytes become fp16 once for all rows.  A page's sums are fresh ones, added to the fp32 output by
//            rounded operations (the tensor core cuts the last bits of a sum off)
// K and V rows come by one bulk copy each for a page; a page's room is given to the next but one when every warp has left it.
// Few rows have eight warps: what bounds them is a page's chain of latencies (mma.sync sums, conversions, three barriers; issue slots half full with 16 warps per SM), which is
// shorter for a warp with one block of dims.  us with append and join: 16 sequences of one token, 28 000 positions in all, 39; 5 tokens at 32700 57 (one page takes a
// CTA 4 - 4.5 us, its start 5, its end 2.5).  Unrolling the loops over the blocks' pairs or over the steps of 16 positions further is no faster: the code no longer fits the
// instruction cache beside itself (all unrolled: 512 tokens after 4000 700 us instead of 415).  Planes of dv v8 and of p instead of p dv and v8 (three products for two, a
// third of the conversions): the same time to 1 % for 16 to 64 rows.
constexpr int PGA_BUFS = 2;
constexpr int pga_warps(int rowt) { return rowt == 4 ? 4 : 8; }       // (ROWT = 0: eight rows)
constexpr int PGA_Q_STRIDE = 64 + 4;                            // words of a quantised row: 4 g + t are 32 different banks
constexpr int PGA_W_STRIDE = PG_POS + 8;                        // weights of a row: pairs at 8 g + 2 t, of four rows, are 32 different banks
constexpr int PGA_NUMBER_AT = 120;                               // (bytes: behind the barriers and flags)
constexpr int PGA_RING_BYTES = PGA_BUFS * 2 * PG_HEAD_BYTES;
static_assert(64 * KV_D * 4 <= PGA_RING_BYTES, "the outputs reuse the ring");
constexpr int pga_smem_bytes(int rowt) {
    const int rows = rowt ? 16 * rowt : 8, keyw = pga_warps(rowt) / (rowt ? rowt : 1), q_rows = rowt ? rows : 16;
    return 128 + PGA_RING_BYTES + 3 * 8 * PG_POS * 4 + 16 * 4 + q_rows * (PGA_Q_STRIDE + 8) * 4 + rows * PGA_W_STRIDE * 4 + rows * (2 + 2 * keyw) * 4;
}

struct PageAttn {
    PageCache C;
    const float *q;
    float *out;
    // Where a tile's pages are shared by several CTAs: a CTA's sums [256] of each row, and their maximum and sum of weights.  A tile of one CTA writes the outputs.
    float *tc_acc;              // [splits][token * n_head + head], with more than one split: the sequences on the tensor cores
    float2 *tc_ml;
    float *part_acc[2];         // [part_items][rows of a tile], of each class below
    float2 *part_ml[2];
    int *spans;                 // [2] pages of a CTA, of each class below: what pages_attn_kernel found, for the join
    int layer, n_head, group;
    int span, splits;           // of the sequences on the tensor cores: pages of a CTA, CTAs of a tile
    // of the others, in one class or two by their rows, a launch each: rows of a sequence at most, rows of a tile (as a power of two); CTAs of a tile at most
    int most_rows[2], row_shift[2], most_splits;
    uint32_t most_items, part_items[2];         // that a launch of theirs can have, and how many of them share a tile: more are rows that several sequences claim, and not served
    float scale;
    // the call's long sequences on the tensor cores (pages_tc.cuh): images [sequence][page][kv head], whether a CTA is to be done again [tile][kv head][split]
    uint8_t *images;
    int *redo;
    int max_pages, n_tc;        // pages of a sequence that there are images for, 0: none; sequences
};
constexpr int PTC_ROWS = 128;
// Whether a sequence is on the tensor cores.
__device__ __forceinline__ bool pages_on_tc(const PageAttn &P, int n, int len) {
    return P.max_pages > 0 && n > 0 && (int64_t)n * P.group >= PTC_ROWS && len >= 0 && len <= (int64_t)P.max_pages * PG_POS && len <= (int64_t)P.C.table_stride * PG_POS;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t"
        ".reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\t"
        "mov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 d, a, b;\n\t"
        "mov.b64 {%0, %1}, d;\n\t"
        "}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// int8 products of one 32-value block on top of the bits of 12582912: read as floats they are 12582912 + the sum, exactly (|sum| < 2^20)
__device__ __forceinline__ void pga_mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0x4B400000));
}
// bytes (lo, hi halves: of two positions) of the signed words a, b -> fp16 pairs, exactly: 1024 + (byte ^ 128) - 1152
__device__ __forceinline__ void pga_halves(uint32_t a, uint32_t b, uint32_t (&out)[4]) {
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    const uint32_t lo = __byte_perm(a, b, 0x5140), hi = __byte_perm(a, b, 0x7362);      // a0 b0 a1 b1 | a2 b2 a3 b3
    const __half2 off = __half2half2(__ushort_as_half((unsigned short)0x6480));       // 1152
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = __byte_perm(i < 2 ? lo : hi, 0x64646464u, (i & 1) ? 0x4342 : 0x4140);
        const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&w), off);
        out[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
}

// ---- how the sequences with few rows are divided: by what they hold, which the device knows.  Every CTA finds the same.
struct SeqWork { int tiles, pages; };       // no tiles: not one of them
__device__ __forceinline__ int pages_class(const PageAttn &P, int n) { return (int64_t)n * P.group <= P.most_rows[0] ? 0 : 1; }
__device__ __forceinline__ SeqWork pages_work(const PageAttn &P, int s, int cls) {
    if (s >= P.C.n_seq) return {0, 0};
    const int n = seq_range(P.C.start, s, P.C.n_tok).n, len = P.C.len[s];
    if (n <= 0 || pages_on_tc(P, n, len) || pages_class(P, n) != cls) return {0, 0};
    if (len < 0 || len > (int64_t)P.C.table_stride * PG_POS) return {1, 0};                 // one CTA says so
    return {(n * P.group + (1 << P.row_shift[cls]) - 1) >> P.row_shift[cls], (len + PG_POS - 1) / PG_POS};
}
__device__ __forceinline__ int pages_splits(const PageAttn &P, int pages, int span) { return max(1, min(P.most_splits, (pages + span - 1) / span)); }
// Pages of a CTA such that one round of CTAs (two per SM) takes all of them.  Where T tiles have N pages between them, span >= N heads / slots: their items are at most
// slots + T heads, and those of tiles with several CTAs (more pages than a span, so fewer than twice as many CTAs as spans) at most 2 slots.
__device__ __noinline__ int pages_span(const PageAttn &P, int cls, int lane, int slots) {
    int64_t total = 0;
    for (int base = 0; base < P.C.n_seq; base += 32) {
        const SeqWork w = pages_work(P, base + lane, cls);
        total += (int64_t)w.tiles * w.pages;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    int span = (int)max((int64_t)2, min((int64_t)(1 << 26), (total * P.C.n_head_kv + slots - 1) / slots));           // (no sequence has 2^26 pages)
    if (P.C.n_seq > 128) return span;
    for (int step = 0; step < 8; ++step) {              // (a sequence's last CTA has less: some more pages for each, until they fit)
        int items = 0;
        for (int base = 0; base < P.C.n_seq; base += 32) {
            const SeqWork w = pages_work(P, base + lane, cls);
            items += w.tiles ? min(w.tiles, 1 << 12) * pages_splits(P, w.pages, span) : 0;           // (2^12 tiles are more than there are slots)
        }
        items = __reduce_add_sync(0xffffffffu, items);
        if ((int64_t)items * P.C.n_head_kv <= slots) break;
        span += max(1, span / 8);
    }
    return span;
}
// Items of a sequence whose sums are left for the join: all of them or none.  (No more than one too many, so that sums over any sequences stay small.)
__device__ __forceinline__ uint32_t pages_parts(const PageAttn &P, const SeqWork &w, int cls, int splits) {
    const uint32_t most = P.part_items[cls] + 1u;       // (below 2^10, and splits times heads below 2^17: most_splits is the slots over the heads)
    return splits > 1 ? min(min((uint32_t)w.tiles, most) * (uint32_t)(splits * P.C.n_head_kv), most) : 0u;
}

// One item: rows `tile` of a sequence, one kv head, pages page0 .. page1 - 1 of those that the tile sees.
template <int ROWT>
struct PageItem {
    int seq, tile, kvh, split, page0, page1;            // page1 < 0: to the last
    bool whole;                                         // nobody else has the tile: the outputs are written
};

template <int ROWT, bool TC = false>
__device__ __forceinline__ bool pages_attn_item(const PageAttn &P, const PageItem<ROWT> &I, uint8_t *smem, int &turn, int cls = 0) {
    constexpr int WARPS = pga_warps(ROWT), THREADS = 32 * WARPS, NB = 8 / WARPS;          // NB: blocks of dims of a warp
    constexpr bool EIGHT = ROWT == 0;
    constexpr int MT = EIGHT ? 1 : ROWT, HR = EIGHT ? 1 : 2;              // row tiles; rows of a thread in each
    constexpr int KEYW = WARPS / MT;                    // warps that share the scores of a row tile
    constexpr int KEYS = PG_POS / KEYW, NT = KEYS / 8, ROWS = EIGHT ? 8 : 16 * ROWT, QROWS = EIGHT ? 16 : ROWS;
    uint64_t *kfull = reinterpret_cast<uint64_t *>(smem), *vfull = kfull + PGA_BUFS;
    int *held = reinterpret_cast<int *>(vfull + PGA_BUFS);                       // [PGA_BUFS] positions of the page that there are
    int *wide0 = held + PGA_BUFS;                                                // [2][8] the block's scales of V are too far apart for one pair of planes
    static_assert(2 * PGA_BUFS * 8 + PGA_BUFS * 4 + 16 * 4 <= PGA_NUMBER_AT, "");
    const uint32_t *number = reinterpret_cast<const uint32_t *>(smem + PGA_NUMBER_AT);      // among the items that leave parts: written by a warp in front of the first barrier here
    uint8_t *ring = smem + 128;
    float *ks = reinterpret_cast<float *>(ring + PGA_RING_BYTES);                // [8 blocks][64 positions]
    float *vs0 = ks + 8 * PG_POS;                                                // the same of V times 2^(13 - e), e the exponent of the block's largest; pages alternate
    float *vfac0 = vs0 + 2 * 8 * PG_POS;                                         // [2][8] 2^(e - 13), negative: the block is to be looked at closely
    uint32_t *q8 = reinterpret_cast<uint32_t *>(vfac0 + 16);                     // [QROWS][PGA_Q_STRIDE]
    float *qd = reinterpret_cast<float *>(q8 + QROWS * PGA_Q_STRIDE);            // [QROWS][8] scales of the queries, times the softmax scale
    float *wt = qd + QROWS * 8;                                                  // [ROWS][PGA_W_STRIDE] weights
    float *alphas = wt + ROWS * PGA_W_STRIDE, *sums = alphas + ROWS;             // [ROWS] each: e^(old maximum - new), sum of weights
    float *most = sums + ROWS, *part = most + KEYW * ROWS;                       // [KEYW][ROWS] each: a warp's maxima, its sums

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int rt = warp / KEYW, kw = warp % KEYW;
    const int seq = I.seq, tile = I.tile, kvh = I.kvh, split = I.split;
    const PageCache &C = P.C;
    const SeqRange range = seq_range(C.start, seq, C.n_tok);
    const int32_t *table = C.table + (size_t)seq * C.table_stride;
    const int ahead[2] = {I.page0 < C.table_stride ? table[I.page0] : -1, I.page0 + 1 < C.table_stride ? table[I.page0 + 1] : -1};         // asked for beside the length
    const int len = C.len[seq];
    if (len < 0 || len > (int64_t)C.table_stride * PG_POS) {
        if (tid == 0) bad_sequence();
        return true;
    }
    const int n_rows = min(ROWS, range.n * P.group - tile * ROWS);                      // of this tile
    const int first_tok = tile * ROWS / P.group, last_tok = (tile * ROWS + n_rows - 1) / P.group;
    const int before = len - range.n;                                                   // positions in front of the new tokens
    // positions that any row of the tile sees, in pages; this item's
    const int seen = min(len, before + last_tok + 1);
    const int pages = (max(seen, 0) + PG_POS - 1) / PG_POS;
    const int page0 = I.page0, page1 = I.page1 < 0 ? pages : min(I.page1, pages);
    const int ntiles = page1 - page0;
    if (ntiles <= 0 && split > 0) return true;          // (the first split writes the rows that see nothing)

    auto issue = [&](int i) {                           // one thread
        const int b = (turn + i) % PGA_BUFS, page = i < 2 ? ahead[i] : table[page0 + i];
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if (page < 0 || page >= C.n_pages) {
            bad_sequence();
            held[b] = 0;
            mbar_arrive(&kfull[b]);
            mbar_arrive(&vfull[b]);
            return;
        }
        const uint64_t pol = policy_evict_normal();
        const int n = min(PG_POS, seen - (page0 + i) * PG_POS);
        const uint32_t bytes = (uint32_t)n * KV_ROW;
        uint8_t *dst = ring + (size_t)b * 2 * PG_HEAD_BYTES;
        held[b] = n;
        mbar_expect_tx(&kfull[b], bytes);
        bulk_g2s(dst, page_rows(C, page, P.layer, 0, kvh), bytes, &kfull[b], pol);
        mbar_expect_tx(&vfull[b], bytes);
        bulk_g2s(dst + PG_HEAD_BYTES, page_rows(C, page, P.layer, 1, kvh), bytes, &vfull[b], pol);
    };
    if (tid == THREADS - 32)
        for (int i = 0; i < min(ntiles, PGA_BUFS); ++i) issue(i);
    // the rows' queries, quantised as the cache rows are
    {
        const int blk = lane >> 2, sub = lane & 3;
        const bool vec = (reinterpret_cast<uintptr_t>(P.q) & 15u) == 0;
        constexpr int BATCH = ROWS / WARPS < 4 ? ROWS / WARPS : 4;               // rows of a warp whose loads are on their way together
        static_assert(ROWS % (WARPS * BATCH) == 0, "");
        if (EIGHT)                                      // the products' other eight rows are zeros
            for (int i = tid; i < 8 * PGA_Q_STRIDE; i += THREADS) q8[8 * PGA_Q_STRIDE + i] = 0u;
#pragma unroll 1
        for (int r0 = warp * BATCH; r0 < ROWS; r0 += WARPS * BATCH) {
            float x[BATCH][8];
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                const int r = r0 + e, row = tile * ROWS + (r < n_rows ? r : 0), tok = row / P.group, h = row - tok * P.group;
                const float *qr = P.q + ((size_t)(range.begin + tok) * P.n_head + kvh * P.group + h) * KV_D + blk * 32 + sub * 8;
                if (vec) {
                    const float4 a = *reinterpret_cast<const float4 *>(qr), c = *reinterpret_cast<const float4 *>(qr + 4);
                    x[e][0] = a.x; x[e][1] = a.y; x[e][2] = a.z; x[e][3] = a.w; x[e][4] = c.x; x[e][5] = c.y; x[e][6] = c.z; x[e][7] = c.w;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[e][i] = qr[i];
                }
            }
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                const int r = r0 + e;
                if (r >= n_rows)
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[e][i] = 0.0f;
                const float d = __fmul_rn(kv_amax_8(x[e]), PG_SCALE), id = d > 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
                uint32_t w[2];
                kv_words_8(x[e], id, w);
                // in the order in which the K rows are read: of an even block slot 0 = values 0, 1, 30, 31, slot i = values 4 i - 2 .. 4 i + 1
                const uint32_t below = __shfl_up_sync(0xffffffffu, w[1], 1), last = __shfl_sync(0xffffffffu, w[1], lane | 3);
                uint32_t s0 = w[0], s1 = w[1];
                if (!(blk & 1)) {
                    s0 = sub ? __byte_perm(below, w[0], 0x5432) : __byte_perm(w[0], last, 0x7610);
                    s1 = __byte_perm(w[0], w[1], 0x5432);
                }
                *reinterpret_cast<uint2 *>(q8 + r * PGA_Q_STRIDE + blk * 8 + 2 * sub) = make_uint2(s0, s1);
                if (sub == 0) qd[r * 8 + blk] = __fmul_rn(f16_bits_to_f32(f32_to_f16_bits_ties_away(d)), P.scale);
            }
        }
    }
    float acc[MT][NB][4][2 * HR];                       // row tile, the warp's block, byte of the slot; (row g | g + 8, slot 2 t | 2 t + 1)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 2 * HR; ++i) acc[m][b][j][i] = 0.0f;
    float m_run[HR], l_run[HR];                         // rows 16 rt + g, + 8; l of this thread's columns
    // the last position that they see
    int limit[HR];
#pragma unroll
    for (int i = 0; i < HR; ++i) {
        const int r = 16 * rt + g + 8 * i;
        m_run[i] = -INFINITY;
        l_run[i] = 0.0f;
        limit[i] = r < n_rows ? before + (tile * ROWS + r) / P.group : -1;
    }
    const int all_see = before + first_tok;             // every row of the tile sees the positions up to this one
    bool ok = true;
    for (int i = 0; i < ntiles; ++i) {
        const int b = (turn + i) % PGA_BUFS, p0 = (page0 + i) * PG_POS;
        const uint32_t par = (uint32_t)(((turn + i) / PGA_BUFS) & 1);
        const uint8_t *kt = ring + (size_t)b * 2 * PG_HEAD_BYTES, *vt = kt + PG_HEAD_BYTES;
        float *vs = vs0 + (i & 1) * 8 * PG_POS, *vfac = vfac0 + (i & 1) * 8;
        ok = mbar_wait_hot(&kfull[b], par) && ok;
        ok = mbar_wait_hot(&vfull[b], par) && ok;
        const int n = held[b];
        // ---- scales; those behind the last position are zeros
#pragma unroll
        for (int blk = NB * warp; blk < NB * warp + NB; ++blk) {                 // a warp's blocks, lane = position
            const int off = 34 * blk;
            float x[2];
            uint32_t top = 0, low = 0x7FFFu;
            bool odd = false;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int k = lane + 32 * e;
                const uint32_t hk = k < n ? *reinterpret_cast<const unsigned short *>(kt + k * KV_ROW + off) : 0u;
                const uint32_t hv = k < n ? *reinterpret_cast<const unsigned short *>(vt + k * KV_ROW + off) : 0u;
                ks[blk * PG_POS + k] = f16_bits_to_f32(hk);
                x[e] = f16_bits_to_f32(hv);
                const uint32_t mag = hv & 0x7FFFu;
                if (mag < 0x7C00u) top = max(top, mag);
                else odd = true;
                if (mag) low = min(low, mag);
            }
            top = __reduce_max_sync(0xffffffffu, top);
            low = __reduce_min_sync(0xffffffffu, low);
            odd = __any_sync(0xffffffffu, odd);
            const int e = max((int)(top >> 10), 1);                              // biased fp16 exponent
            const float up = __uint_as_float((uint32_t)(127 + 28 - e) << 23), down = __uint_as_float((uint32_t)(127 - 28 + e) << 23);       // 2^(13 - (e - 15))
#pragma unroll
            for (int j = 0; j < 2; ++j) vs[blk * PG_POS + lane + 32 * j] = __fmul_rn(x[j], up);
            if (lane == 0) {
                const bool wide = top && e - max((int)(low >> 10), 1) > KV_V_RANGE;
                vfac[blk] = odd || wide ? -down : down;
                wide0[(i & 1) * 8 + blk] = wide;
            }
        }
        if (!__syncthreads_and(ok ? 1 : 0)) break;      // (a wait ran out: the CTA leaves as a whole)
        if (tid == THREADS - 32 && i > 0 && i - 1 + PGA_BUFS < ntiles) issue(i - 1 + PGA_BUFS);      // every warp is behind the page before
        // ---- scores: rows 16 rt .., positions KEYS kw ..
        float s[NT][2 * HR];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2 * HR; ++e) s[nt][e] = 0.0f;
        {
            const uint32_t *qa = q8 + (16 * rt + g) * PGA_Q_STRIDE + t;
            const float *qs = qd + (16 * rt + g) * 8, *kd = ks + KEYS * kw + 2 * t;
            const uint32_t *kr = reinterpret_cast<const uint32_t *>(kt) + (size_t)(KEYS * kw + g) * (KV_ROW / 4);
            const float2 low = make_float2(-12582912.0f, -12582912.0f);
#pragma unroll(ROWT >= 2 ? 1 : 2)
            for (int pair = 0; pair < 4; ++pair, qa += 16, qs += 2, kd += 2 * PG_POS, kr += 17) {
#pragma unroll
                for (int odd = 0; odd < 2; ++odd) {
                    const uint32_t a0 = qa[8 * odd], a1 = qa[8 * odd + 8 * PGA_Q_STRIDE], a2 = qa[8 * odd + 4], a3 = qa[8 * odd + 4 + 8 * PGA_Q_STRIDE];
                    const float dq0 = qs[odd], dq1 = EIGHT ? 0.0f : qs[64 + odd];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const uint32_t *u = kr + nt * 8 * (KV_ROW / 4);
                        uint32_t b0, b1;
                        if (odd) {
                            b0 = u[9 + t];
                            b1 = u[13 + t];
                        } else {
                            b0 = u[t];
                            b1 = u[4 + t];
                            if (t == 0) b0 = __byte_perm(b0, u[8], 0x5432);
                        }
                        int d[4];
                        pga_mma_s8(d, a0, a1, a2, a3, b0, b1);
                        const float2 dk = *reinterpret_cast<const float2 *>(kd + odd * PG_POS + 8 * nt);
                        const float2 x0 = mul2(add2(make_float2(__int_as_float(d[0]), __int_as_float(d[1])), low), dk);
                        const float2 y0 = fma2(x0, make_float2(dq0, dq0), make_float2(s[nt][0], s[nt][1]));
                        s[nt][0] = y0.x; s[nt][1] = y0.y;
                        if (!EIGHT) {
                            const float2 x1 = mul2(add2(make_float2(__int_as_float(d[2]), __int_as_float(d[3])), low), dk);
                            const float2 y1 = fma2(x1, make_float2(dq1, dq1), make_float2(s[nt][2 * HR - 2], s[nt][2 * HR - 1]));
                            s[nt][2 * HR - 2] = y1.x; s[nt][2 * HR - 1] = y1.y;
                        }
                    }
                }
            }
        }
        // ---- softmax step
        if (p0 + PG_POS - 1 > all_see || n < PG_POS) {  // some row does not see some position
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2 * HR; ++e) {
                    const int k = KEYS * kw + 8 * nt + 2 * t + (e & 1);
                    if (p0 + k > limit[e >> 1] || k >= n) s[nt][e] = -INFINITY;
                }
        }
        float mx[HR];
#pragma unroll
        for (int h = 0; h < HR; ++h) {
            mx[h] = s[0][2 * h];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mx[h] = fmaxf(mx[h], fmaxf(s[nt][2 * h], s[nt][2 * h + 1]));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
        }
        if (KEYW > 1) {
            if (t == 0)
#pragma unroll
                for (int h = 0; h < HR; ++h) most[kw * ROWS + 16 * rt + g + 8 * h] = mx[h];
            __syncthreads();
#pragma unroll
            for (int h = 0; h < HR; ++h)
#pragma unroll
                for (int w = 0; w < KEYW; ++w) mx[h] = fmaxf(mx[h], most[w * ROWS + 16 * rt + g + 8 * h]);
        }
#pragma unroll
        for (int h = 0; h < HR; ++h) {
            const int r = 16 * rt + g + 8 * h;
            const float m_new = fmaxf(m_run[h], mx[h]), base = m_new == -INFINITY ? 0.0f : m_new;
            const float alpha = expf(__fsub_rn(m_run[h], base));
            float sum = 0.0f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float x = expf(__fsub_rn(s[nt][2 * h], base)), y = expf(__fsub_rn(s[nt][2 * h + 1], base));
                sum = __fadd_rn(sum, __fadd_rn(x, y));
                *reinterpret_cast<float2 *>(wt + r * PGA_W_STRIDE + KEYS * kw + 8 * nt + 2 * t) = make_float2(x, y);
            }
            l_run[h] = __fadd_rn(__fmul_rn(l_run[h], alpha), sum);
            m_run[h] = m_new;
            if (kw == 0 && t == 0) alphas[r] = alpha;
        }
        __syncthreads();
        // ---- outputs: blocks NB warp ..
        const uint32_t *vr0 = reinterpret_cast<const uint32_t *>(vt) + (size_t)(2 * t) * (KV_ROW / 4) + 17 * (NB * warp / 2);
#pragma unroll
        for (int bl = 0; bl < NB; ++bl) {
            const bool second = NB == 2 ? bl : (warp & 1);                       // of a pair of blocks
            const float *dv0 = vs + (NB * warp + bl) * PG_POS + 2 * t;
            const float fac = vfac[NB * warp + bl];
            float o[MT][4][4];                          // EIGHT: rows g of the high plane, rows g of the low one
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[m][j][e] = 0.0f;
            // CAREFUL: a position without weight adds nothing, whatever it holds; REST: what one pair of planes leaves, times 2^24
            auto pass = [&](auto carefulc, auto restc) {
                constexpr bool CAREFUL = decltype(carefulc)::value, REST = decltype(restc)::value;
#pragma unroll(CAREFUL || ROWT == 4 ? 1 : 2)
                for (int k = 0; k < PG_POS / 16; ++k) {
                    uint32_t w[4], b0[4], b1[4];
                    const uint32_t *u = vr0 + (size_t)(16 * k) * (KV_ROW / 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t *x = u + ((e & 1) + 8 * (e >> 1)) * (KV_ROW / 4);
                        if (second) {
                            w[e] = x[9 + g];
                        } else {
                            w[e] = x[g];
                            if (g == 0) w[e] = __byte_perm(w[e], x[8], 0x5432);
                        }
                    }
                    pga_halves(w[0], w[1], b0);
                    pga_halves(w[2], w[3], b1);
                    const float2 dv[2] = {*reinterpret_cast<const float2 *>(dv0 + 16 * k), *reinterpret_cast<const float2 *>(dv0 + 16 * k + 8)};
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        uint32_t ah[4], al[4];
#pragma unroll
                        for (int e = 0; e < 4; e += EIGHT ? 2 : 1) {             // rows g, g + 8 of positions 2 t, then of 2 t + 8
                            const float2 p = *reinterpret_cast<const float2 *>(wt + (16 * m + g + 8 * (e & 1)) * PGA_W_STRIDE + 16 * k + 8 * (e >> 1) + 2 * t);
                            float2 x = mul2(p, dv[e >> 1]);
                            if (CAREFUL) {
                                if (p.x == 0.0f) x.x = 0.0f;
                                if (p.y == 0.0f) x.y = 0.0f;
                            }
                            split_f16x2(x.x, x.y, ah[e], al[e]);
                            if (REST) split_rest_f16x2(x.x, x.y, ah[e], al[e]);
                        }
                        if (EIGHT) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) mma_f16_16816(o[m][j], ah[0], al[0], ah[2], al[2], b0[j], b1[j]);
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j) mma_f16_16816(o[m][j], al[0], al[1], al[2], al[3], b0[j], b1[j]);
#pragma unroll
                            for (int j = 0; j < 4; ++j) mma_f16_16816(o[m][j], ah[0], ah[1], ah[2], ah[3], b0[j], b1[j]);
                        }
                    }
                }
            };
            if (fac > 0.0f) {
                pass(std::false_type{}, std::false_type{});
            } else {
                if (wide0[(i & 1) * 8 + NB * warp + bl]) {
                    pass(std::true_type{}, std::true_type{});
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[m][j][e] = __fmul_rn(o[m][j][e], 0x1p-24f);
                }
                pass(std::true_type{}, std::false_type{});
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
#pragma unroll
                for (int h = 0; h < HR; ++h) {
                    const float al = alphas[16 * m + g + 8 * h];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float x = EIGHT ? __fadd_rn(o[m][j][e], o[m][j][2 + e]) : o[m][j][2 * h + e];
                            acc[m][bl][j][2 * h + e] = __fmaf_rn(x, fabsf(fac), __fmul_rn(acc[m][bl][j][2 * h + e], al));
                        }
                }
            }
        }
    }
    // ---- the sums leave by whole lines
#pragma unroll
    for (int h = 0; h < HR; ++h) {
        float l = __fadd_rn(l_run[h], __shfl_xor_sync(0xffffffffu, l_run[h], 1));
        l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, 2));
        if (t == 0) part[kw * ROWS + 16 * rt + g + 8 * h] = l, most[kw * ROWS + 16 * rt + g + 8 * h] = m_run[h];
    }
    turn += max(ntiles, 0);
    if (!__syncthreads_and(ok ? 1 : 0)) return false;   // (and every warp has left the last page)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int bl = 0; bl < NB; ++bl)
#pragma unroll
            for (int h = 0; h < HR; ++h) {
                const bool second = NB == 2 ? bl : (warp & 1);
                float *dst = reinterpret_cast<float *>(ring) + (size_t)(16 * m + g + 8 * h) * KV_D + 32 * (NB * warp + bl);
#pragma unroll
                for (int c = 0; c < 2; ++c) {           // slot 2 t + c of the block: four values from dim 4 slot (odd block) or 4 slot - 2 (even, round the end)
                    const int slot = 2 * t + c;
                    float *d0 = dst + (second ? 4 * slot : (slot ? 4 * slot - 2 : 0)), *d1 = dst + (second ? 4 * slot + 2 : (slot ? 4 * slot : 30));
                    *reinterpret_cast<float2 *>(d0) = make_float2(acc[m][bl][0][2 * h + c], acc[m][bl][1][2 * h + c]);
                    *reinterpret_cast<float2 *>(d1) = make_float2(acc[m][bl][2][2 * h + c], acc[m][bl][3][2 * h + c]);
                }
            }
    if (tid < ROWS) {
        float l = part[tid];
#pragma unroll
        for (int w = 1; w < KEYW; ++w) l = __fadd_rn(l, part[w * ROWS + tid]);
        sums[tid] = l;
    }
    __syncthreads();
    if (!TC && !I.whole && *number >= P.part_items[cls]) return true;              // (rows that several sequences claim)
    float *const acc_at = TC ? P.tc_acc : P.part_acc[cls];
    float2 *const ml_at = TC ? P.tc_ml : P.part_ml[cls];
    const size_t part0 = I.whole ? 0 : TC ? (size_t)split * C.n_tok * P.n_head : (size_t)*number * ROWS;
    for (int i = tid; i < n_rows * (KV_D / 4); i += THREADS) {
        const int r = i / (KV_D / 4), c = i % (KV_D / 4);
        float4 x = reinterpret_cast<const float4 *>(ring)[(size_t)r * (KV_D / 4) + c];
        const float l = sums[r];
        const int row = tile * ROWS + r, tok = row / P.group;
        const size_t at = (size_t)(range.begin + tok) * P.n_head + kvh * P.group + (row - tok * P.group);
        if (I.whole) {
            const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);             // a row that sees nothing is zeros
            x = make_float4(__fmul_rn(x.x, inv), __fmul_rn(x.y, inv), __fmul_rn(x.z, inv), __fmul_rn(x.w, inv));
            float *o = P.out + at * KV_D + 4 * c;
            if ((reinterpret_cast<uintptr_t>(P.out) & 15u) == 0) {
                *reinterpret_cast<float4 *>(o) = x;
            } else {
                o[0] = x.x; o[1] = x.y; o[2] = x.z; o[3] = x.w;
            }
        } else {
            const size_t at2 = part0 + (TC ? at : (size_t)r);
            reinterpret_cast<float4 *>(acc_at)[at2 * (KV_D / 4) + c] = x;
            if (c == 0) ml_at[at2] = make_float2(most[r], l);
        }
    }
    return true;
}

// The sequences with few rows (pages_on_tc has the others).  grid: two CTAs per SM, which take items until there are none.
template <int ROWT>
__global__ void __launch_bounds__(32 * pga_warps(ROWT), 2) pages_attn_kernel(const __grid_constant__ PageAttn P, int cls) {
    extern __shared__ __align__(128) uint8_t smem[];
    uint64_t *kfull = reinterpret_cast<uint64_t *>(smem), *vfull = kfull + PGA_BUFS;
    const int lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int b = 0; b < PGA_BUFS; ++b) mbar_init(&kfull[b], 1), mbar_init(&vfull[b], 1);
        mbar_fence_init();
    }
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    const int span = pages_span(P, cls, lane, gridDim.x);
    if (P.spans && blockIdx.x == 0 && threadIdx.x == 0) P.spans[cls] = span;
    if (cls == 0 && blockIdx.x == gridDim.x - 1) report_ranges(P.C.start, P.C.n_seq, P.C.n_tok);
    const int heads = P.C.n_head_kv;
    __syncthreads();
    int turn = 0;
    for (uint32_t item = blockIdx.x; item < P.most_items; item += gridDim.x) {
        // whose: the sequences' items one after the other, every warp for itself (a sequence has most_items at most, below 2^31; where several claim rows, sums stop there)
        uint32_t before = 0, parts = 0;
        PageItem<ROWT> I = {-1, 0, 0, 0, 0, 0, true};
        for (int base = 0; base < P.C.n_seq && I.seq < 0; base += 32) {
            const SeqWork w = pages_work(P, base + lane, cls);
            const int splits = pages_splits(P, w.pages, span);
            uint32_t sum = (uint32_t)(w.tiles * splits * heads);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t x = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum = min(sum + x, (uint32_t)INT32_MAX);
            }
            const unsigned past = __ballot_sync(0xffffffffu, before + sum > item);
            const uint32_t front = __shfl_up_sync(0xffffffffu, sum, 1);
            if (threadIdx.x < 32) {                     // (by a warp that does not issue copies: nobody needs it before the item's end)
                const uint32_t own = lane < (past ? __ffs(past) - 1 : 32) ? pages_parts(P, w, cls, splits) : 0u;
                parts = min(parts + __reduce_add_sync(0xffffffffu, own), 1u << 30);
            }
            if (past) {
                const int at = __ffs(past) - 1, rest = (int)(item - before - __shfl_sync(0xffffffffu, lane ? front : 0u, at)), n = __shfl_sync(0xffffffffu, splits, at);
                const int pair = rest / heads;
                I.seq = base + at;
                I.kvh = rest - pair * heads;
                I.tile = pair / n;
                I.split = pair - I.tile * n;
                I.page0 = I.split * span;
                I.page1 = I.split == n - 1 ? -1 : I.page0 + span;
                I.whole = n == 1;
                if (threadIdx.x == 0) *reinterpret_cast<uint32_t *>(smem + PGA_NUMBER_AT) = parts + (uint32_t)rest;
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (I.seq < 0) return;                          // CTA-uniform
        if (!pages_attn_item<ROWT>(P, I, smem, turn, cls)) return;        // (a wait ran out: the CTA leaves as a whole)
        __syncthreads();
    }
}

// Behind pages_tc_kernel, two CTAs for each of its tiles: what it could not hold.
__global__ void __launch_bounds__(32 * pga_warps(4), 2) pages_redo_kernel(const __grid_constant__ PageAttn P) {
    extern __shared__ __align__(128) uint8_t smem[];
    uint64_t *kfull = reinterpret_cast<uint64_t *>(smem), *vfull = kfull + PGA_BUFS;
    const int lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int b = 0; b < PGA_BUFS; ++b) mbar_init(&kfull[b], 1), mbar_init(&vfull[b], 1);
        mbar_fence_init();
    }
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    PageItem<4> I;
    if (!seq_of_item(P.C.start, P.C.n_seq, P.C.n_tok, (int)(blockIdx.x / 2), lane, [&](int n) { return ((int64_t)n * P.group + PTC_ROWS - 1) / PTC_ROWS; }, I.seq, I.tile)) return;
    const int n = seq_range(P.C.start, I.seq, P.C.n_tok).n;
    if (!pages_on_tc(P, n, P.C.len[I.seq])) return;
    if (!P.redo[((size_t)(blockIdx.x / 2) * P.C.n_head_kv + blockIdx.y) * P.splits + blockIdx.z]) return;
    I.tile = 2 * I.tile + (int)(blockIdx.x & 1);
    if (I.tile * (PTC_ROWS / 2) >= n * P.group) return;
    I.kvh = blockIdx.y;
    I.split = blockIdx.z;
    I.page0 = I.split * P.span;
    I.page1 = I.split == P.splits - 1 ? -1 : I.page0 + P.span;
    I.whole = P.tc_acc == nullptr;
    __syncthreads();
    int turn = 0;
    pages_attn_item<4, true>(P, I, smem, turn);
}

// The splits of a row added up: ROWW warps per row (token, head), four dims and four more a lane.  A row's splits are those that its own positions reach.
constexpr int PGJ_WARPS = 8;
template <int ROWW>
__global__ void __launch_bounds__(32 * PGJ_WARPS) pages_join_kernel(const __grid_constant__ PageAttn P) {
    __shared__ float4 sums[PGJ_WARPS][2][32];
    __shared__ float2 ml[PGJ_WARPS];
    const PageCache &C = P.C;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = warp % ROWW;
    const int64_t rows = (int64_t)C.n_tok * P.n_head, row = (int64_t)blockIdx.x * (PGJ_WARPS / ROWW) + warp / ROWW;
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    int n = 0;                                          // 0: not a row of a sequence that was served, or its outputs are there
    const float *acc = nullptr;                         // its first part; the others lie `step` rows behind each other
    const float2 *pml = nullptr;
    int64_t step = rows;
    if (row < rows) {
        const int tok = (int)(row / P.n_head);
        const int s = seq_of_row(C.start, C.n_seq, tok, lane);
        if (s < C.n_seq) {
            const SeqRange r = seq_range(C.start, s, C.n_tok);
            const int len = C.len[s];
            if (r.n > 0 && tok >= r.begin && len >= 0 && len <= (int64_t)C.table_stride * PG_POS) {
                const int seen = len - r.n + (tok - r.begin) + 1;
                const int pages = (max(seen, 0) + PG_POS - 1) / PG_POS;
                if (pages_on_tc(P, r.n, len)) {
                    if (P.tc_acc) {
                        n = max(1, min(P.splits, (pages + P.span - 1) / P.span));
                        acc = P.tc_acc + row * KV_D;
                        pml = P.tc_ml + row;
                    }
                } else {
                    const int cls = pages_class(P, r.n), span = P.spans[cls];
                    const int splits = pages_splits(P, (len + PG_POS - 1) / PG_POS, span);
                    if (splits > 1) {
                        uint32_t parts = 0;             // of the sequences in front
                        for (int i = lane; i < s; i += 32) {
                            const SeqWork x = pages_work(P, i, cls);
                            parts = min(parts + pages_parts(P, x, cls, pages_splits(P, x.pages, span)), 1u << 20);
                        }
                        const int h = (int)(row - (int64_t)tok * P.n_head), kvh = h / P.group, at = (tok - r.begin) * P.group + (h - kvh * P.group), shift = P.row_shift[cls], tile = at >> shift;
                        n = max(1, min(splits, (pages + span - 1) / span));
                        const size_t first = (size_t)__reduce_add_sync(0xffffffffu, parts) + (size_t)tile * splits * C.n_head_kv + kvh;
                        if (first + (size_t)(n - 1) * C.n_head_kv >= P.part_items[cls]) n = 0;
                        const size_t from = (first << shift) + (at & ((1 << shift) - 1));
                        step = (int64_t)C.n_head_kv << shift;
                        acc = P.part_acc[cls] + from * KV_D;
                        pml = P.part_ml[cls] + from;
                    }
                }
            }
        }
    }
    float m = -INFINITY, l = 0.0f;
    for (int i = lane; i < n; i += 32) m = fmaxf(m, pml[i * step].x);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    for (int i0 = mine; i0 < n; i0 += 4 * ROWW) {      // four splits' loads at once
        float2 x[4];
        float4 c[4], d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t at = (int64_t)min(i0 + e * ROWW, n - 1) * step;
            const float4 *src = reinterpret_cast<const float4 *>(acc) + at * (KV_D / 4) + lane;
            x[e] = pml[at];
            c[e] = src[0];
            d[e] = src[32];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (i0 + e * ROWW >= n) break;
            const float w = x[e].x == m ? 1.0f : expf(__fsub_rn(x[e].x, m));
            l = __fmaf_rn(x[e].y, w, l);
            a = make_float4(__fmaf_rn(c[e].x, w, a.x), __fmaf_rn(c[e].y, w, a.y), __fmaf_rn(c[e].z, w, a.z), __fmaf_rn(c[e].w, w, a.w));
            b = make_float4(__fmaf_rn(d[e].x, w, b.x), __fmaf_rn(d[e].y, w, b.y), __fmaf_rn(d[e].z, w, b.z), __fmaf_rn(d[e].w, w, b.w));
        }
    }
    if (ROWW > 1) {
        sums[warp][0][lane] = a;
        sums[warp][1][lane] = b;
        if (lane == 0) ml[warp] = make_float2(0.0f, l);
        __syncthreads();
        if (mine) return;
#pragma unroll
        for (int w = 1; w < ROWW; ++w) {
            const float4 c = sums[warp + w][0][lane], d = sums[warp + w][1][lane];
            l = __fadd_rn(l, ml[warp + w].y);
            a = make_float4(__fadd_rn(a.x, c.x), __fadd_rn(a.y, c.y), __fadd_rn(a.z, c.z), __fadd_rn(a.w, c.w));
            b = make_float4(__fadd_rn(b.x, d.x), __fadd_rn(b.y, d.y), __fadd_rn(b.z, d.z), __fadd_rn(b.w, d.w));
        }
    }
    if (n == 0) return;
    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
    float *o = P.out + row * KV_D + 4 * lane;
    const float x[8] = {__fmul_rn(a.x, inv), __fmul_rn(a.y, inv), __fmul_rn(a.z, inv), __fmul_rn(a.w, inv),
                        __fmul_rn(b.x, inv), __fmul_rn(b.y, inv), __fmul_rn(b.z, inv), __fmul_rn(b.w, inv)};
    if ((reinterpret_cast<uintptr_t>(P.out) & 15u) == 0) {
        *reinterpret_cast<float4 *>(o) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4 *>(o + 128) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = x[e], o[128 + e] = x[4 + e];
    }
}

}  // namespace b200
