// pages_shared.cuh -- attention over a paged Q8_0 cache for groups of sequences that begin with the same pages: each group's queries together over what
// it shares, each sequence's over its own, joined by their maxima and sums.
//
//   score    s = scale * q8 . k8 (codes times fp16 scales, exact 18-bit products), o = sum of e^(s - m) v8 / sum of e^(s - m)
//
// Work: an entity is a group over its shared pages or a sequence over its own positions.  Its rows (tokens times the query heads of a kv head) are cut
// into tiles of PSH_ROWS, its positions into steps of 128.  All (tile, kv head, step) lie on one line, which is cut into equal pieces, one per CTA: a CTA has
// fragments, steps of one tile and kv head that follow each other, and leaves each one's maximum, sum and weighted values for the join.
//
// A fragment on the tensor cores (tcgen05.mma.kind::f16), positions as the rows of both products:
//   S^T [128 positions x rows] = K Q^T        K as A from tensor memory, Q as B from shared memory, both as two fp16 planes
//   O^T [256 dims x rows]     = V^T P         V as A from tensor memory, the weights P as B from shared memory, two planes each
// three of the four products of planes.  A product's time goes with its rows in steps of 16, so a tile of one token's six heads costs a third of a full one.
//
// Warps: 0 - 7 weights and outputs (a thread has a position of S^T, or two dims of O^T, and half of the columns), 8 - 15 V (a dim a thread), 16 - 19 K (a position a
// thread), 20 says what the fragments are and copies pages of V, 21 copies those of K, 22 and 23 issue the products of scores and of outputs.
//
// What bounds it: chains of latencies, that of K's planes first.  A step takes about 8000 cycles.  K's four warps take as long: 1100 for its page and scales, and for each 64 dims 450 to load codes,
// 350 to see that their place is free, 850 for 32 pairs (byte permute, subtraction, product, remainder) and their way to tensor memory.  V's eight take 6500, the products of 48 rows 3900,
// the step's bytes 3000.  (4 x 5 tokens over 32000 positions: 114 us.  Tried when it was 122: planes of zeros for K, V and both 108, 112 and 99; eight warps for K, 48 registers each, 136.  The
// warps' code in 80 registers spills 84 bytes of stores a thread.)  48 rows a tile: planes,
// scores and two buffers of outputs then fill tensor memory.  Positions as rows keep the matrix instructions' 128 rows full whatever the number of tokens (tokens as rows: 6 of 128
// used by one token).
#pragma once

#include "attn_tc.cuh"
#include "pages.cuh"

namespace b200 {

constexpr int PSH_ROWS = 48, PSH_STEP = 2 * PG_POS, PSH_STAGE = 32, PSH_CHUNK = 64, PSH_DESCS = 4;
constexpr int PSH_KSLOTS = 4, PSH_VSLOTS = 3;                    // pages of K and of V in shared memory
constexpr int PSH_KRING = 2, PSH_VRING = 2;                      // in tensor memory: 64 dims of a step's K, 32 positions of V
constexpr int PSH_START = 2;                                     // what a fragment's begin is worth, in steps (1, 2 and 4, us: 4 x 5 tokens 125, 114 and 117, ragged batch 138, 129 and 133, 64 chats 105, 108 and 114)
constexpr int PSH_THREADS = 768, PSH_SUM_WARPS = 8, PSH_V_WARP = 8, PSH_K_WARP = 16, PSH_PLAN_WARP = 20, PSH_LOAD_WARP = 21, PSH_SCORE_WARP = 22, PSH_OUT_WARP = 23;
// registers a thread: 2 x 136 + 2 x 48 + 64 + 48 = 6 x 80, what the launch has
constexpr int PSH_REGS_SUM = 136, PSH_REGS_V = 48, PSH_REGS_K = 64, PSH_REGS_REST = 48;
constexpr int PSH_REGS = 32 * (8 * PSH_REGS_SUM + 8 * PSH_REGS_V + 4 * PSH_REGS_K + 4 * PSH_REGS_REST);
constexpr int PSH_Q_CHUNK = PSH_ROWS * 128, PSH_Q_PLANE = 4 * PSH_Q_CHUNK;              // 64 dims of the rows; a plane of them
constexpr int PSH_P_GROUP = PSH_ROWS / 8 * 128, PSH_P_PLANE = PSH_STEP / 8 * PSH_P_GROUP, PSH_P_BUF = 2 * PSH_P_PLANE;       // 8 positions of the rows
constexpr int PSH_AT_P = 2 * PSH_Q_PLANE, PSH_AT_RAWK = PSH_AT_P + 2 * PSH_P_BUF, PSH_AT_RAWV = PSH_AT_RAWK + PSH_KSLOTS * PG_HEAD_BYTES,
              PSH_AT_D = PSH_AT_RAWV + PSH_VSLOTS * PG_HEAD_BYTES, PSH_AT_SMALL = PSH_AT_D + KV_NBLK * PSH_STEP * 2;
// tensor memory, all 512 columns: K (64 dims: high, low), V (two halves of the dims x high, low), scores, two buffers of outputs
constexpr uint32_t PSH_COL_K = 0, PSH_COL_V = PSH_KRING * 64, PSH_COL_S = PSH_COL_V + PSH_VRING * 64, PSH_COL_O = PSH_COL_S + PSH_ROWS, PSH_O_BUF = 2 * PSH_ROWS;
static_assert(PSH_COL_O + 2 * PSH_O_BUF <= 512 && (PSH_VRING & (PSH_VRING - 1)) == 0, "");
static_assert(PSH_ROWS * KV_D * 4 <= 2 * PSH_P_BUF, "a fragment's queries come by the weights' place");

struct PshFragment {
    int begin, row0, n_rows;            // first token of the entity; of its rows the tile's first, and how many
    int kvh, pos0, steps, end;          // first position; steps (negative: no more fragments); positions that any row sees end here
    int before;                         // the last position that row r sees is before + r / group; INT32_MAX: all up to end
    int seq;                            // whose table
    long long part;                     // the first row's place among the parts
};
struct alignas(16) PshSmall {
    int8_t ks[4][PSH_STEP];             // powers of two of the steps' K rows
    // 2^-s of the step's V blocks, whether scales are no numbers, and at which positions.  Of eight steps: V is at most two stages ahead of the products, and who adds the outputs
    // a step behind
    float vf[8][KV_NBLK];
    uint8_t v_odd[8][KV_NBLK];
    uint32_t v_bad[8][4][KV_NBLK];
    float qf[PSH_ROWS];                 // 2^-s of the query rows times scale and log2 e
    int limit[PSH_ROWS];                // the last position that a row sees
    float less[PSH_ROWS], change[PSH_ROWS], red[4][PSH_ROWS];        // less: a row's reference, negative
    uint8_t none[PSH_ROWS];             // a row has seen a V that is no number
    PshFragment desc[PSH_DESCS];
    uint64_t dfull[PSH_DESCS], dempty[PSH_DESCS], rkfull[PSH_KSLOTS], rkempty[PSH_KSLOTS], rvfull[PSH_VSLOTS], rvempty[PSH_VSLOTS], kready[PSH_KRING], kempty[PSH_KRING],
        vready[PSH_VRING], vempty[PSH_VRING];
    uint64_t qready, qkdone, sempty, pready[2], pvdone[2], oempty[2], done[2];
    int held_k[PSH_KSLOTS], held_v[PSH_VSLOTS];          // rows of a page that there are
    uint32_t tmem;
    int failed;
};
constexpr int PSH_SMEM_BYTES = 1024 + PSH_AT_SMALL + (int)sizeof(PshSmall);
static_assert(PSH_SMEM_BYTES <= 227 * 1024, "");

// Entities of many rows are pages_shared_tc_kernel's (pages_shared_tc.cuh): tiles of 128 rows, steps of a page, a line of their own.  Two launches more cost 10 to 20 us, and what images save
// goes with the rows and pages of all kv heads.  Measured, whole calls in us, as 48 rows a tile against as images (one new token a sequence behind a common prefix):
//   4 kv heads of 6   642 rows over 16, 32, 64, 256 pages 80 / 81, 92 / 91, 119 / 110, 261 / 255; 384 rows 60 / 70, 69 / 76, 83 / 90, 166 / 183; 1200 rows 124 / 115, 146 / 126, 191 / 156, 444 / 347
//   8 of 4            644 rows over 32, 64, 256 pages 186 / 157, 237 / 205, 521 / 516; 384 rows 125 / 123, 157 / 159, 320 / 337        8 of 8    648 rows 138 / 129, 189 / 177, 472 / 487
//   3 of 4            700 rows over 32, 64, 128 pages 94 / 93, 113 / 108, 154 / 144
//   2 of 8            704 rows over 32, 128, 256 pages 61 / 74, 98 / 104, 147 / 152; 1040 rows over 32, 64, 128, 256 pages 74 / 78, 94 / 91, 130 / 119, 207 / 177; 1504 rows over 32, 64 95 / 94, 124 / 108
//   1 of 8            1800 rows over 32, 64, 128, 256 pages 71 / 77, 86 / 86, 117 / 104, 181 / 142; 3000 rows 96 / 95, 128 / 109, 177 / 139, 286 / 190
//   1 of 6            642 rows over 64, 256 pages 55 / 68, 92 / 96; 900 rows 63 / 77, 109 / 114; 1200 rows 71 / 81, 137 / 122; 2400 rows 113 / 101, 243 / 169
//   1 of 24           two sequences: 2064 rows over 32, 64 pages 60 / 73, 76 / 84; 3000 rows 69 / 80, 101 / 94
// With three kv heads and more the first two numbers decide.
constexpr int PST_ROWS = 128, PST_MIN_ROWS = 640, PST_MIN_PAGES = 32, PST_ALL_ROWS = 1024, PST_ALL_WORK = 95000;
__host__ __device__ __forceinline__ bool pst_rows_many(int64_t rows, int n_head_kv) { return rows > PST_MIN_ROWS && rows * n_head_kv > PST_ALL_ROWS; }
__device__ __forceinline__ bool pst_many(int64_t rows, int pages, int n_head_kv) {
    return pst_rows_many(rows, n_head_kv) && pages >= PST_MIN_PAGES && (float)rows * (float)n_head_kv * ((float)pages * (float)n_head_kv) >= (float)PST_ALL_WORK;
}
constexpr int PST_START = 8;                                     // what a fragment's begin is worth, in pages (2, 8 and 20, us: 200 answers 383, 371 and 381, 12 questions 370, 372 and 370)
// The tensor core drops what a sum has behind its 24 bits: sums come out low by about 2^-24 for each of the twelve or so that a score is made of.  Scores are lifted by the mean of that
// (root mean square of the outputs' error 3.4e-6 without, 1.3e-6 with it).  A score of few large products is cut less and lifted all the same.  What that can do is bounded: scores times
// 1 + L move an output by L times the covariance of scores and values under the weights, which is at most the largest |v| times sqrt(ln(n)^2 / 4 + 1) of n positions, the largest standard
// deviation that scores have under their own weights: 3.0e-6 of it at 4000 positions, 3.8e-6 at 32 000.
constexpr float PSH_LIFT = 1.0f + 6 * 0x1p-23f;

// What there is to do, found by pages_shared_plan_kernel: a group over its shared pages, or a sequence over its own positions.
struct alignas(16) PshEntity {
    int begin, tokens;                  // rows of tokens
    int page0, end;                     // first page, end of its positions
    int before;                         // the last position that token i sees is before + i; INT32_MAX: all up to end
    int steps;                          // (pages, of an entity of many rows) 0: nothing; -1: numbers that do not fit
    int seq, group;                     // whose table; the group that a sequence shares page0 pages with
    int image;                          // of an entity of many rows: its first page's image; others -1
    long long unit, row;                // units and rows of parts in front, on its line (unit negative: not served)
};
constexpr int PSH_CTAS = 160;                                    // most CTAs of a launch
struct PshPlan {
    long long total, per;               // units; of a CTA
    long long tc_total, tc_per, tc_row; // the same of the other line, and where its parts begin
    int images, first[PSH_CTAS], tc_first[PSH_CTAS];             // images; the entity that a CTA's units begin in
    PshEntity entity[1];                // groups, then sequences
};
constexpr int64_t psh_plan_bytes(int64_t entities) { return (int64_t)sizeof(PshPlan) + entities * (int64_t)sizeof(PshEntity); }
struct PageShared {
    PageCache C;
    const float *q;
    float *out, *part;                  // [part_rows][256]
    float2 *part_ml;                    // maximum (as a power of two's exponent) and sum of a part's rows
    PshPlan *plan;
    uint8_t *images;                    // [image_room][kv head]
    const int32_t *group_first, *group_pages;
    long long part_rows;                // of entities; CTAs' own come beside them
    int n_groups, layer, n_head, group, ctas, image_room;
    float scale;
};

// ---- what there is to do ------------------------------------------------------------------------------------------------------------------------
struct PshGroup { int first, last, begin, end, pages; };         // sequences, rows of tokens, pages in common (negative: numbers that do not fit)
__device__ __forceinline__ PshGroup psh_group(const PageShared &P, int g) {
    const PageCache &C = P.C;
    PshGroup G = {P.group_first[g], P.group_first[g + 1], 0, 0, -1};
    const int pages = P.group_pages[g];
    if (G.first < 0 || G.last < G.first || G.last > C.n_seq || pages < 0 || pages > C.table_stride) return G;
    G.begin = C.start[G.first];
    G.end = C.start[G.last];
    // (one sequence has nobody to share with; rows that are not the call's are some sequence's own trouble: the others of the group go by themselves)
    G.pages = G.last - G.first < 2 || G.begin < 0 || G.end < G.begin || G.end > C.n_tok ? 0 : pages;
    return G;
}
// The group that sequence s belongs to, n_groups: none.
__device__ __forceinline__ int psh_group_of(const PageShared &P, int s) {
    int lo = 0, hi = P.n_groups;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (P.group_first[mid + 1] <= s) lo = mid + 1;
        else hi = mid;
    }
    return lo < P.n_groups && P.group_first[lo] <= s ? lo : P.n_groups;
}
__device__ __forceinline__ int psh_steps(int positions) { return (positions + PSH_STEP - 1) / PSH_STEP; }
__device__ __forceinline__ PshEntity psh_entity(const PageShared &P, int e) {
    const PageCache &C = P.C;
    PshEntity E = {0, 0, 0, 0, INT32_MAX, 0, -1, 0, -1, 0, 0};
    if (e < P.n_groups) {
        const PshGroup G = psh_group(P, e);
        E.begin = G.begin;
        E.tokens = G.end - G.begin;
        E.end = max(G.pages, 0) * PG_POS;
        if (E.tokens > 0) E.steps = psh_steps(E.end);
        return E;
    }
    const int s = e - P.n_groups, len = C.len[s];
    const SeqRange r = seq_range(C.start, s, C.n_tok);
    E.begin = r.begin;
    E.tokens = max(r.n, 0);
    E.seq = s;
    E.group = psh_group_of(P, s);
    if (r.n < 0) E.steps = -1;
    if (r.n <= 0) return E;
    bool fits = len >= 0 && len <= (int64_t)C.table_stride * PG_POS;
    if (E.group < P.n_groups) {
        const PshGroup G = psh_group(P, E.group);
        E.page0 = max(G.pages, 0);
        // (its new tokens lie behind what it shares)
        fits = fits && G.pages >= 0 && (G.pages == 0 || (r.begin >= G.begin && r.begin + r.n <= G.end && (int64_t)len - r.n >= (int64_t)G.pages * PG_POS));
    }
    E.end = len;
    E.before = len - r.n;
    E.steps = fits ? psh_steps(len - E.page0 * PG_POS) : -1;
    return E;
}
// Where what a tile sees ends: with its last row.
__device__ __forceinline__ int psh_tile_end(int group, const PshEntity &E, int row0, int rows) {
    if (E.before == INT32_MAX) return E.end;
    const int last = min(row0 + rows, E.tokens * group) - 1;
    return max(E.page0 * PG_POS, min(E.end, E.before + last / group + 1));
}

__device__ __forceinline__ long long psh_scan(long long x, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    return x;
}

// One CTA.  The work of every entity, and what lies in front of it.  (Each CTA of the attention finding that by itself took it 9 us, most of them instructions that are not in the cache
// yet; here they are few, and the attention's CTAs start meanwhile.)
constexpr int PSP_THREADS = 512;
__global__ void __launch_bounds__(PSP_THREADS) pages_shared_plan_kernel(const __grid_constant__ PageShared P) {
    __shared__ long long sums[PSP_THREADS / 32];
    __shared__ int place[PSP_THREADS], taken;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, entities = P.n_groups + P.C.n_seq;
    PshPlan &plan = *P.plan;
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    // what lies in front of a thread's x, and of the next 512 threads' (front)
    auto in_front = [&](long long x, long long &front) {
        long long y = psh_scan(x, lane);
        if (lane == 31) sums[warp] = y;
        __syncthreads();
        long long all = 0;
        for (int w = 0; w < PSP_THREADS / 32; ++w) {
            if (w == warp) y += all;
            all += sums[w];
        }
        __syncthreads();
        y += front - x;
        front += all;
        return y;
    };
    auto tiles = [&](const PshEntity &E) { return (long long)((E.tokens * P.group + (E.image < 0 ? PSH_ROWS : PST_ROWS) - 1) / (E.image < 0 ? PSH_ROWS : PST_ROWS)) * P.C.n_head_kv; };
    auto units = [&](const PshEntity &E) { return tiles(E) * (E.steps + (E.image < 0 ? PSH_START : PST_START)); };        // (rows of a call are below 2^30)
    long long rows0 = 0, images0 = 0, unit0 = 0, row0 = 0, tc_unit0 = 0, tc_row0 = 0;
#pragma unroll 1
    for (int base = 0; base < entities; base += PSP_THREADS) {
        const int e = base + tid;
        PshEntity E = {0, 0, 0, 0, 0, 0, -1, 0, -1, 0, 0};
        if (e < entities) E = psh_entity(P, e);
        if (E.steps < 0) bad_sequence();
        long long rows = E.steps > 0 ? (long long)E.tokens * P.n_head : 0;
        if (in_front(rows, rows0) + rows > P.part_rows && rows) {        // rows that several sequences claim
            bad_sequence();
            rows = 0;
        }
        const int pages = (E.end + PG_POS - 1) / PG_POS - E.page0;
        const int images = rows && pst_many((int64_t)E.tokens * P.group, pages, P.C.n_head_kv) && pages <= P.image_room ? pages : 0;
        const long long before = images0;
        long long image = in_front(images, images0);
        if (images0 > P.image_room) {        // there is no room for all of them: each in its turn that finds some (the same for all threads)
            place[tid] = images;
            __syncthreads();
            if (tid == 0) {
                int at = (int)before;
                for (int i = 0; i < PSP_THREADS; ++i) {
                    const int n = place[i];
                    if (n == 0) continue;
                    place[i] = n <= P.image_room - at ? at : -1;
                    at += place[i] < 0 ? 0 : n;
                }
                taken = at;
            }
            __syncthreads();
            image = place[tid];
            images0 = taken;
        }
        const bool many = images && image >= 0;
        if (many) E.image = (int)image, E.steps = pages;
        const long long own = rows ? units(E) : 0;
        const long long a = in_front(many ? 0 : own, unit0), b = in_front(many ? own : 0, tc_unit0), c = in_front(many ? 0 : rows, row0), d = in_front(many ? rows : 0, tc_row0);
        E.unit = !rows ? -1 : many ? b : a;
        E.row = many ? d : c;
        if (e < entities) plan.entity[e] = E;
    }
    const long long per = (unit0 + P.ctas - 1) / P.ctas, tc_per = (tc_unit0 + P.ctas - 1) / P.ctas;
    if (tid < PSH_CTAS) plan.first[tid] = plan.tc_first[tid] = entities;
    if (tid == 0) {
        plan.total = unit0;
        plan.per = per;
        plan.tc_total = tc_unit0;
        plan.tc_per = tc_per;
        plan.tc_row = row0 + (long long)P.ctas * PSH_ROWS;
        plan.images = (int)images0;
    }
    __syncthreads();
#pragma unroll 1
    for (int e = tid; e < entities; e += PSP_THREADS) {          // (its own entities)
        PshEntity &E = plan.entity[e];
        if (E.unit < 0) continue;
        const long long end = E.unit + units(E), own = E.image < 0 ? per : tc_per;
        int *const first = E.image < 0 ? plan.first : plan.tc_first;
        for (long long c = (E.unit + own - 1) / own; c * own < end; ++c) first[c] = e;
        // the table of a group: of its first sequence that has the pages in common
        if (e < P.n_groups)
            for (int s = P.group_first[e]; s < P.group_first[e + 1] && E.seq < 0; ++s)
                if (plan.entity[P.n_groups + s].steps > 0) E.seq = s;
    }
}

// ---- small pieces -------------------------------------------------------------------------------------------------------------------------------
// A from tensor memory, B the weights: 8 rows x 8 positions a piece of 128 bytes, rows side by side.
template <bool ADD>
__device__ __forceinline__ void psh_mma_weights(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        ".reg .b64 db;\n\t"
        "mov.b64 db, {%2, %4};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t"
        "}\n"
        ::"r"(d), "r"(a), "r"(b_lo), "r"(idesc), "r"((uint32_t)(128 >> 4) | (1u << 14)), "n"(ADD ? 1 : 0)
        : "memory");
}
__device__ __forceinline__ float psh_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));        // 2^-22 of the value
    return y;
}
// Eight of a warp's columns (all lanes the same), at this place in the code: a thread has no registers to have them early.
template <typename T>
__device__ __forceinline__ void psh_lds8(const T *p, T (&x)[8]) {
    uint32_t (&y)[8] = reinterpret_cast<uint32_t (&)[8]>(x);
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(y[0]), "=r"(y[1]), "=r"(y[2]), "=r"(y[3]) : "r"(smem_u32(p)) : "memory");
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(y[4]), "=r"(y[5]), "=r"(y[6]), "=r"(y[7]) : "r"(smem_u32(p) + 16u) : "memory");
}
// Barriers of some warps: 1 and 2 of the four of a half of the columns, 3 of both halves.
template <int THREADS>
__device__ __forceinline__ void psh_barrier(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(THREADS) : "memory"); }
template <int THREADS>
__device__ __forceinline__ bool psh_any(int id, bool x) {
    uint32_t y;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(y) : "r"(x ? 1u : 0u), "r"(id), "n"(THREADS) : "memory");
    return y != 0;
}
// A pair of codes (bytes 0 and 1, or 2 and 3, of w) as fp16, exactly: 1024 + (byte ^ 128) - 1152; w comes with its bytes' signs turned.
__device__ __forceinline__ uint32_t psh_pair(uint32_t w, bool upper) {
    uint32_t y;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(__byte_perm(w, 0x64646464u, upper ? 0x4342 : 0x4140)), "r"(0x64806480u));
    return y;
}
// The same of one byte of each of two words: pick says which byte of x comes first, and which of y third.
__device__ __forceinline__ uint32_t psh_codes(uint32_t x, uint32_t y, uint32_t pick) {
    uint32_t c;
    asm("lop3.b32 %0, %1, 0x00FF00FF, 0x64806480, 0x6A;" : "=r"(c) : "r"(__byte_perm(x, y, pick)));                   // (both & mask) ^ 1024 + 128
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(c) : "r"(0x64806480u));
    return c;
}
// Codes times a scale of two fp16 planes: the rounded product and, exactly, what it leaves.
__device__ __forceinline__ void psh_planes(uint32_t codes, uint32_t d, uint32_t &hi, uint32_t &lo) {
    asm("{\n\t.reg .b32 n;\n\tmul.rn.f16x2 %0, %2, %3;\n\tneg.f16x2 n, %0;\n\tfma.rn.f16x2 %1, %2, %3, n;\n\t}" : "=&r"(hi), "=r"(lo) : "r"(codes), "r"(d));
}
// s with 2^7 <= d 2^s < 2^8 for the largest scale d of those under one power of two (magnitude bits of an fp16; no number, zero: 0)
__device__ __forceinline__ int psh_shift(uint32_t mag) { return mag == 0 || mag >= 0x7C00u ? 0 : 134 - (int)(__float_as_uint(f16_bits_to_f32(mag)) >> 23); }
__device__ __forceinline__ uint32_t psh_scale(uint32_t d16, float up) {
    const uint32_t d = __half_as_ushort(__float2half_rn(__fmul_rn(f16_bits_to_f32(d16), up)));
    return d | (d << 16);
}
template <int N>
__device__ __forceinline__ void psh_set_registers(bool more) {
    if (more) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

struct PshStep { int valid, pages, stages; };                    // of a step: positions, pages and stages of V that there are
__device__ __forceinline__ PshStep psh_step(const PshFragment &F, int i) {
    const int valid = min(PSH_STEP, F.end - F.pos0 - i * PSH_STEP);
    return {valid, valid > PG_POS ? 2 : 1, (valid + PSH_STAGE - 1) / PSH_STAGE};
}

// ---- the warps ----------------------------------------------------------------------------------------------------------------------------------
// A wait that runs out (2^18 looks, each of which the unit holds for as long as it sees fit; not a time that is known): nothing is waited for any more, the CTA comes to its end and leaves its
// parts unfinished.  One that waits for it runs out behind it.  (One loop for a wait: what bounds this kernel next to the tensor core is instructions that are not in the cache.)
// TEST: a look without a wait in front of it.  pages_shared_tc_kernel, whose waits are mostly over: 200 answers 371 us with it and 377 without.  In this kernel 4 x 5 tokens would take 113 of
// 114 us, but the code then spills more than its 84 bytes a thread.
template <bool TEST = false>
__device__ __forceinline__ bool psh_wait(uint64_t *bar, uint32_t parity) {
    if (TEST) {
        uint32_t over;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(over) : "r"(smem_u32(bar)), "r"(parity) : "memory");
        if (over) return true;
    }
    uint32_t left;
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "mov.u32 %0, 0x40000;\n\t"
        "PSH_LOOP:\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "@p bra PSH_DONE;\n\t"
        "sub.u32 %0, %0, 1;\n\t"
        "setp.ne.u32 p, %0, 0;\n\t"
        "@p bra PSH_LOOP;\n\t"
        "PSH_DONE:\n\t"
        "}"
        : "=&r"(left)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (left == 0) atomicExch(&g_device_status, STATUS_MBARRIER_TIMEOUT);
    return left != 0;
}
struct PshWait {
    PshSmall &S;
    bool ok = true;
    __device__ __forceinline__ PshWait(PshSmall &s) : S(s) {}
    __device__ __forceinline__ void operator()(uint64_t *bar, uint32_t parity) {
        if (!ok) return;
        ok = __all_sync(0xffffffffu, psh_wait(bar, parity));
        if (!ok) *(volatile int *)&S.failed = 1;
    }
};
// The next fragment, as every warp but the one that says it sees it.
struct PshReader {
    PshSmall &S;
    PshWait &wait;
    int n = 0;
    __device__ __forceinline__ bool next(PshFragment &F) {
        wait(&S.dfull[n % PSH_DESCS], (uint32_t)((n / PSH_DESCS) & 1));
        F = S.desc[n % PSH_DESCS];
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&S.dempty[n % PSH_DESCS]);
        ++n;
        return wait.ok && F.steps > 0;
    }
};

// Pages to shared memory, KV 0: K, 1: V.
template <int KV>
struct PshLoader {
    static constexpr int SLOTS = KV ? PSH_VSLOTS : PSH_KSLOTS;
    const PageShared &P;
    PshSmall &S;
    PshWait &wait;
    uint8_t *raw;
    int n = 0;
    __device__ __forceinline__ PshLoader(const PageShared &p, PshSmall &s, PshWait &w, uint8_t *smem) : P(p), S(s), wait(w), raw(smem + (KV ? PSH_AT_RAWV : PSH_AT_RAWK)) {}
    __device__ __forceinline__ void load(const PshFragment &F) {
        const PageCache &C = P.C;
        uint64_t *const fulls = KV ? S.rvfull : S.rkfull, *const empties = KV ? S.rvempty : S.rkempty;
        int *const helds = KV ? S.held_v : S.held_k;
        const int lane = threadIdx.x & 31;
        const int32_t *table = C.table + (size_t)max(F.seq, 0) * C.table_stride + F.pos0 / PG_POS;
        const int pages = (min(F.end, F.pos0 + F.steps * PSH_STEP) - F.pos0 + PG_POS - 1) / PG_POS;
        int own = -1;                                    // 32 pages, a lane each
#pragma unroll 1
        for (int p = 0; p < pages && wait.ok; ++p, ++n) {
            if ((p & 31) == 0) own = F.seq >= 0 && p + lane < pages ? table[p + lane] : -1;
            const int page = __shfl_sync(0xffffffffu, own, p & 31), rows = min(PG_POS, F.end - F.pos0 - p * PG_POS), j = n % SLOTS;
            const bool there = page >= 0 && page < C.n_pages;
            if (!there && lane == 0) bad_sequence();
            if (n >= SLOTS) wait(&empties[j], (uint32_t)((n / SLOTS - 1) & 1));
            if (!wait.ok) break;                         // (the slot's last copy may be in flight: nothing is counted on its barrier then)
            if (lane == 0) {
                helds[j] = there ? rows : 0;
                if (there) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    mbar_expect_tx(&fulls[j], (uint32_t)rows * KV_ROW);
                    bulk_g2s(raw + j * PG_HEAD_BYTES, page_rows(C, page, P.layer, KV, F.kvh), (uint32_t)rows * KV_ROW, &fulls[j], policy_evict_normal());
                } else {
                    mbar_arrive(&fulls[j]);
                }
            }
            __syncwarp();
        }
    }
    __device__ __forceinline__ void end() {              // no copy outlives the CTA
        uint64_t *const fulls = KV ? S.rvfull : S.rkfull;
        for (int k = max(0, n - SLOTS); k < n; ++k) psh_wait(&fulls[k % SLOTS], (uint32_t)((k / SLOTS) & 1));
    }
};
__device__ __forceinline__ void psh_load_k_warp(const PageShared &P, PshSmall &S, uint8_t *smem) {
    PshWait wait(S);
    PshReader frags{S, wait};
    PshLoader<0> loader(P, S, wait, smem);
    PshFragment F;
    while (frags.next(F)) loader.load(F);
    loader.end();
}
// Says what the CTA's fragments are, and copies their pages of V.
__device__ __forceinline__ void psh_plan_warp(const PageShared &P, PshSmall &S, uint8_t *smem) {
    const int lane = threadIdx.x & 31, entities = P.n_groups + P.C.n_seq, heads = P.C.n_head_kv;
    const PshPlan &plan = *P.plan;
    PshWait wait(S);
    PshLoader<1> loader(P, S, wait, smem);
    const long long per = plan.per, last = min(per * (blockIdx.x + 1), plan.total);
    long long at = per * blockIdx.x;
    int said = 0;
    auto say = [&](const PshFragment &F) {
        if (said >= PSH_DESCS) wait(&S.dempty[said % PSH_DESCS], (uint32_t)((said / PSH_DESCS - 1) & 1));
        if (!wait.ok) return;                            // (somebody may be reading what lies there; who waits for the next one gives up as well)
        if (lane == 0) {
            S.desc[said % PSH_DESCS] = F;
            mbar_arrive(&S.dfull[said % PSH_DESCS]);
        }
        __syncwarp();
        ++said;
        if (F.steps > 0) loader.load(F);
    };
    PshFragment F = {};
    F.steps = -1;
#pragma unroll 1
    for (int e = plan.first[blockIdx.x]; e < entities && at < last && wait.ok; ++e) {
        const PshEntity E = plan.entity[e];
        if (E.unit < 0 || E.image >= 0) continue;
        const int size = E.steps + PSH_START, rows = E.tokens * P.group, pairs = (rows + PSH_ROWS - 1) / PSH_ROWS * heads;
        // the tile and kv head that the next unit lies in
        int pair = (int)((at - E.unit) / size);
#pragma unroll 1
        for (long long begin = E.unit + (long long)pair * size; pair < pairs && begin < last && wait.ok; ++pair, begin += size) {
            const int tile = pair / heads;
            F.kvh = pair - tile * heads;
            F.begin = E.begin;
            F.row0 = tile * PSH_ROWS;
            F.n_rows = min(PSH_ROWS, rows - F.row0);
            F.end = psh_tile_end(P.group, E, F.row0, PSH_ROWS);
            F.before = E.before;
            F.seq = E.seq;
            F.part = E.row + (long long)F.row0 * heads + F.kvh * F.n_rows + (long long)blockIdx.x * PSH_ROWS;
            const int s0 = (int)max(0ll, at - begin - PSH_START), s1 = min((int)min(last - begin, (long long)size) - PSH_START, psh_steps(F.end - E.page0 * PG_POS));
            F.pos0 = E.page0 * PG_POS + s0 * PSH_STEP;
            F.steps = s1 - s0;
            if (F.steps > 0) say(F);
            at = begin + size;
        }
    }
    F.steps = -1;
    say(F);
    loader.end();
}

// 64 dims of a row (words w: a scale's halfword, 32 codes, again) to planes.
__device__ __forceinline__ void psh_k_chunk(const uint32_t *w, uint32_t none, float up, uint32_t to) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int s = 17 * b;                            // the block's first halfword
        const uint32_t d = psh_scale((s & 1 ? w[s >> 1] >> 16 : w[s >> 1] & 0xFFFFu) & none, up);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int half = s + 1 + 8 * k + e;
                psh_planes(psh_pair(w[half >> 1] ^ 0x80808080u, half & 1), d, hi[e], lo[e]);
            }
            tc_st8(to + (uint32_t)(16 * b + 8 * k), hi);
            tc_st8(to + (uint32_t)(32 + 16 * b + 8 * k), lo);
        }
    }
}
// K rows to planes in tensor memory: a position a thread, 64 dims at a time.
__device__ __forceinline__ void psh_k_warps(const PageShared &P, PshSmall &S, uint8_t *smem, uint32_t tmem) {
    const int lane = threadIdx.x & 31, quarter = (threadIdx.x >> 5) & 3, pos = 32 * quarter + lane;
    const uint32_t lanes = tmem + PSH_COL_K + ((uint32_t)(32 * quarter) << 16);
    PshWait wait(S);
    PshReader frags{S, wait};
    PshFragment F;
    int it = 0, n = 0, chunk = 0, slot = 0;              // steps, pages; 64 dims: how many, and where in tensor memory
    while (frags.next(F)) {
#pragma unroll 1
        for (int i = 0; i < F.steps && wait.ok; ++i, ++it) {
            const PshStep T = psh_step(F, i);
            const bool mine = T.pages > quarter >> 1;
            const int page = (n + (quarter >> 1)) % PSH_KSLOTS;
            const uint8_t *row = smem + PSH_AT_RAWK + page * PG_HEAD_BYTES + (pos & (PG_POS - 1)) * KV_ROW;
            uint32_t w[18], none = 0u;
            float up = 1.0f;
            if (mine) {
                wait(&S.rkfull[page], (uint32_t)(((n + (quarter >> 1)) / PSH_KSLOTS) & 1));
                none = (pos & (PG_POS - 1)) < S.held_k[page] ? 0xFFFFFFFFu : 0u;
                uint32_t top = 0;
#pragma unroll
                for (int b = 0; b < KV_NBLK; ++b) top = max(top, (uint32_t)*reinterpret_cast<const uint16_t *>(row + 34 * b) & 0x7FFFu);
                const int s = psh_shift(top & none);
                up = atc_pow2(s);
                S.ks[it & 3][pos] = (int8_t)s;
            }
#pragma unroll 1
            for (int c = 0; c < 4; ++c, ++chunk) {
                if (mine) {                              // (words of an odd chunk begin in the middle of eight bytes: one that is there already, and eight pairs)
                    const uint8_t *src = row + 136 * (c >> 1);
                    if (c & 1) {
                        w[0] = w[17];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint2 x = *reinterpret_cast<const uint2 *>(src + 72 + 8 * j);
                            w[1 + 2 * j] = x.x;
                            w[2 + 2 * j] = x.y;
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 9; ++j) {
                            const uint2 x = *reinterpret_cast<const uint2 *>(src + 8 * j);
                            w[2 * j] = x.x;
                            w[2 * j + 1] = x.y;
                        }
                    }
                }
                if (chunk >= PSH_KRING) wait(&S.kempty[slot], (uint32_t)((chunk / PSH_KRING - 1) & 1));
                tc_fence_after();
                if (mine) {
                    psh_k_chunk(w, none, up, lanes + (uint32_t)(64 * slot));
                    tc_st_wait();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&S.kready[slot]);
                    if (mine && c == 3) mbar_arrive(&S.rkempty[page]);
                }
                slot = slot == PSH_KRING - 1 ? 0 : slot + 1;
            }
            n += T.pages;
        }
    }
}

// V to planes in tensor memory, 32 positions at a time: a dim a thread, a block of 32 dims a warp, so that a position has one scale.
__device__ __forceinline__ void psh_v_warps(const PageShared &P, PshSmall &S, uint8_t *smem, uint32_t tmem) {
    const int lane = threadIdx.x & 31, block = (threadIdx.x >> 5) - PSH_V_WARP;
    const uint32_t lanes = tmem + PSH_COL_V + (uint32_t)(32 * (block >> 2)) + ((uint32_t)(32 * (block & 3)) << 16);
    // the dim's byte in a row: which word, which of its bytes (of two rows' words)
    const int byte = 34 * block + 2 + lane;
    const uint32_t pick2 = (uint32_t)(byte & 3) | ((uint32_t)(byte & 3) + 4u) << 8;        // byte 0 and byte 2 of the result
    PshWait wait(S);
    PshReader frags{S, wait};
    PshFragment F;
    uint16_t *const scales = reinterpret_cast<uint16_t *>(smem + PSH_AT_D) + block * PSH_STEP;
    int it = 0, nv = 0, stage = 0;
    while (frags.next(F)) {
#pragma unroll 1
        for (int i = 0; i < F.steps && wait.ok; ++i, ++it) {
            const PshStep T = psh_step(F, i);
            // the block's scales of the step, under one power of two; a lane has a position of each stage
            const int slot0 = nv % PSH_VSLOTS, slot1 = slot0 == PSH_VSLOTS - 1 ? 0 : slot0 + 1;
            wait(&S.rvfull[slot0], (uint32_t)((nv / PSH_VSLOTS) & 1));
            if (T.pages > 1) wait(&S.rvfull[slot1], (uint32_t)(((nv + 1) / PSH_VSLOTS) & 1));
            {
                const int held0 = S.held_v[slot0], held1 = T.pages > 1 ? S.held_v[slot1] : 0;
                const uint8_t *own = smem + PSH_AT_RAWV + lane * KV_ROW + 34 * block;
                uint32_t d[4], top = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    d[j] = *reinterpret_cast<const uint16_t *>(own + (j >> 1 ? slot1 : slot0) * PG_HEAD_BYTES + 32 * (j & 1) * KV_ROW);
                    if (32 * (j & 1) + lane >= (j >> 1 ? held1 : held0)) d[j] = 0;
                    top = max(top, d[j] & 0x7FFFu);
                }
                const bool odd = __any_sync(0xffffffffu, top >= 0x7C00u);
                if (odd) {                               // scales that are no numbers
                    top = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const bool bad = (d[j] & 0x7FFFu) >= 0x7C00u;
                        const uint32_t mask = __ballot_sync(0xffffffffu, bad);
                        if (lane == 0) S.v_bad[it & 7][j][block] = mask;
                        if (bad) d[j] = 0;
                        top = max(top, d[j] & 0x7FFFu);
                    }
                }
                const int s = psh_shift(__reduce_max_sync(0xffffffffu, top));
                if (lane == 0) {
                    S.vf[it & 7][block] = atc_pow2(-s);
                    S.v_odd[it & 7][block] = odd;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) scales[32 * j + lane] = (uint16_t)psh_scale(d[j], atc_pow2(s));
                __syncwarp();
            }
            const uint8_t *src = smem + PSH_AT_RAWV + slot0 * PG_HEAD_BYTES + (byte & ~3);
            const uint4 *ds = reinterpret_cast<const uint4 *>(scales);
#pragma unroll 1
            for (int j = 0; j < T.stages && wait.ok; ++j, ++stage) {
                const int at = stage & (PSH_VRING - 1);
                const uint32_t to = lanes + (uint32_t)(64 * at);
                if (j == 2) src += (slot1 - slot0) * PG_HEAD_BYTES - 64 * KV_ROW;
                if (stage >= PSH_VRING) wait(&S.vempty[at], (uint32_t)((stage / PSH_VRING - 1) & 1));
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < 2; ++k) {            // 16 positions
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint4 d4 = ds[2 * k + h];
                        const uint32_t d[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t *x = reinterpret_cast<const uint32_t *>(src + (16 * k + 8 * h + 2 * e) * KV_ROW);
                            psh_planes(psh_codes(x[0], x[KV_ROW / 4], pick2), d[e], hi[4 * h + e], lo[4 * h + e]);
                        }
                    }
                    tc_st8(to + (uint32_t)(8 * k), hi);
                    tc_st8(to + (uint32_t)(16 + 8 * k), lo);
                }
                tc_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&S.vready[at]);
                    if ((j & 1) || j == T.stages - 1) mbar_arrive(&S.rvempty[j >> 1 ? slot1 : slot0]);
                }
                src += 32 * KV_ROW;
                ds += 4;
            }
            nv += T.pages;
            __syncwarp();                                // (the scales have been read)
        }
    }
}

__device__ __forceinline__ void psh_score_warp(const PageShared &P, PshSmall &S, uint8_t *smem, uint32_t tmem) {
    PshWait wait(S);
    PshReader frags{S, wait};
    PshFragment F;
    int it = 0, frag = 0, chunk = 0, slot = 0;
    const uint32_t q0 = tc16_desc_lo(smem_u32(smem));
    while (frags.next(F)) {
        const uint32_t idesc = atc_idesc((F.n_rows + 15) / 16 * 16);
        wait(&S.qready, (uint32_t)(frag & 1));
#pragma unroll 1
        for (int i = 0; i < F.steps && wait.ok; ++i, ++it) {
            if (it > 0) wait(&S.sempty, (uint32_t)((it - 1) & 1));
            const uint32_t d = tmem + PSH_COL_S;
#pragma unroll 1
            for (int c = 0; c < 4; ++c, ++chunk) {       // 64 dims: low K, low queries, both high
                wait(&S.kready[slot], (uint32_t)((chunk / PSH_KRING) & 1));
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t a = tmem + PSH_COL_K + (uint32_t)(64 * slot), b = q0 + (uint32_t)(c * (PSH_Q_CHUNK >> 4));
                    if (c == 0) tc_mma_f16_ts<false>(d, a + 32u, b, idesc);
                    else tc_mma_f16_ts<true>(d, a + 32u, b, idesc);
#pragma unroll
                    for (int k = 1; k < 4; ++k) tc_mma_f16_ts<true>(d, a + 32u + (uint32_t)(8 * k), b + (uint32_t)(2 * k), idesc);
#pragma unroll
                    for (int k = 0; k < 4; ++k) tc_mma_f16_ts<true>(d, a + (uint32_t)(8 * k), b + (uint32_t)(PSH_Q_PLANE >> 4) + (uint32_t)(2 * k), idesc);
#pragma unroll
                    for (int k = 0; k < 4; ++k) tc_mma_f16_ts<true>(d, a + (uint32_t)(8 * k), b + (uint32_t)(2 * k), idesc);
                    tc_commit(&S.kempty[slot]);
                    if (c == 3) tc_commit(&S.qkdone);
                }
                __syncwarp();
                slot = slot == PSH_KRING - 1 ? 0 : slot + 1;
            }
        }
        ++frag;
    }
    if (elect_one()) tc_commit(&S.done[0]);              // everything that was issued
    __syncwarp();
    psh_wait(&S.done[0], 0);
}
__device__ __forceinline__ void psh_out_warp(const PageShared &P, PshSmall &S, uint8_t *smem, uint32_t tmem) {
    PshWait wait(S);
    PshReader frags{S, wait};
    PshFragment F;
    int it = 0, stage = 0;
    const uint32_t p0 = ((smem_u32(smem + PSH_AT_P) >> 4) & 0x3FFFu) | ((uint32_t)(PSH_P_GROUP >> 4) << 16);
    while (frags.next(F)) {
        const uint32_t idesc = atc_idesc((F.n_rows + 15) / 16 * 16) | (1u << 16);        // (weights: rows side by side)
#pragma unroll 1
        for (int i = 0; i < F.steps && wait.ok; ++i, ++it) {
            const PshStep T = psh_step(F, i);
            wait(&S.pready[it & 1], (uint32_t)((it >> 1) & 1));
            if (it > 1) wait(&S.oempty[it & 1], (uint32_t)(((it - 2) >> 1) & 1));
#pragma unroll 1
            for (int j = 0; j < T.stages; ++j, ++stage) {
                wait(&S.vready[stage % PSH_VRING], (uint32_t)((stage / PSH_VRING) & 1));
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t v = tmem + PSH_COL_V + (uint32_t)(64 * (stage % PSH_VRING)), o = tmem + PSH_COL_O + (uint32_t)((it & 1) * PSH_O_BUF);
                    const uint32_t b = p0 + (uint32_t)((it & 1) * (PSH_P_BUF >> 4) + j * (PSH_STAGE / 8) * (PSH_P_GROUP >> 4));
                    constexpr uint32_t LOW = PSH_P_PLANE >> 4, K16 = 2 * PSH_P_GROUP >> 4;
#pragma unroll
                    for (int m = 0; m < 2; ++m) {        // low V, low weights, both high
                        const uint32_t a = v + (uint32_t)(32 * m), d = o + (uint32_t)(m * PSH_ROWS);
                        if (j == 0) psh_mma_weights<false>(d, a + 16u, b, idesc);
                        else psh_mma_weights<true>(d, a + 16u, b, idesc);
                        psh_mma_weights<true>(d, a + 24u, b + K16, idesc);
                        psh_mma_weights<true>(d, a, b + LOW, idesc);
                        psh_mma_weights<true>(d, a + 8u, b + LOW + K16, idesc);
                        psh_mma_weights<true>(d, a, b, idesc);
                        psh_mma_weights<true>(d, a + 8u, b + K16, idesc);
                    }
                    tc_commit(&S.vempty[stage % PSH_VRING]);
                    if (j == T.stages - 1) tc_commit(&S.pvdone[it & 1]);
                }
                __syncwarp();
            }
        }
    }
    if (elect_one()) tc_commit(&S.done[1]);              // everything that was issued
    __syncwarp();
    psh_wait(&S.done[1], 0);
}

// A fragment's queries, quantised as the cache rows are, to planes: a row a warp.  They come by the place of the weights, which nobody reads now.
__device__ __forceinline__ void psh_queries(const PageShared &P, PshSmall &S, uint8_t *smem, const PshFragment &F, int n) {
    constexpr float LOG2E = 1.44269504088896340736f;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint8_t *box = smem + PSH_AT_P + 32 * lane;
#pragma unroll 1
    for (int r = warp; r < F.n_rows; r += PSH_SUM_WARPS) {
        const int row = F.row0 + r, tok = row / P.group;
        const float *src = P.q + ((size_t)(F.begin + tok) * P.n_head + F.kvh * P.group + (row - tok * P.group)) * KV_D + 8 * lane;
        const uint32_t dst = smem_u32(box + r * (KV_D * 4));
        if ((reinterpret_cast<uintptr_t>(P.q) & 15u) == 0) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + 16u), "l"(src + 4) : "memory");
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + 4u * e), "l"(src + e) : "memory");
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");     // (a lane reads what it has copied itself)
#pragma unroll 1
    for (int r = warp; r < n; r += PSH_SUM_WARPS) {
        float x[8];
        const float4 a = *reinterpret_cast<const float4 *>(box + r * (KV_D * 4)), b = *reinterpret_cast<const float4 *>(box + r * (KV_D * 4) + 16);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
        const float d = __fmul_rn(kv_amax_8(x), PG_SCALE), id = d > 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
        const uint32_t d16 = r < F.n_rows ? f32_to_f16_bits_ties_away(d) : 0u;           // (rows behind the last: zeros)
        const int s = psh_shift(__reduce_max_sync(0xffffffffu, d16));
        const uint32_t sc = psh_scale(d16, atc_pow2(s));
        uint32_t w[2], hi[4], lo[4];
        kv_words_8(x, id, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) psh_planes(psh_pair(w[j >> 1] ^ 0x80808080u, j & 1), sc, hi[j], lo[j]);
        uint8_t *dst = smem + (lane >> 3) * PSH_Q_CHUNK + r * 128 + (((lane & 7) ^ (r & 7)) << 4);
        *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4 *>(dst + PSH_Q_PLANE) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        if (lane == 0) {
            S.qf[r] = __fmul_rn(__fmul_rn(__fmul_rn(P.scale, LOG2E), PSH_LIFT), atc_pow2(-s));
            S.limit[r] = F.before == INT32_MAX ? F.end - 1 : F.before + (F.row0 + min(r, F.n_rows - 1)) / P.group;
            S.less[r] = 1e30f;
            S.none[r] = 0;
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    psh_barrier<256>(3);                                 // every row's numbers
    if (lane == 0) mbar_arrive(&S.qready);
}

// Eight values reduced over a warp: value psh_of_lane(lane) at each lane.
template <typename F>
__device__ __forceinline__ float psh_over8(const float2 (&v)[4], int lane, F op) {
    float x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float a = k & 1 ? v[k >> 1].y : v[k >> 1].x, b = k & 1 ? v[2 + (k >> 1)].y : v[2 + (k >> 1)].x;
        x[k] = op(lane & 16 ? b : a, __shfl_xor_sync(0xffffffffu, lane & 16 ? a : b, 16));
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) x[k] = op(lane & 8 ? x[k + 2] : x[k], __shfl_xor_sync(0xffffffffu, lane & 8 ? x[k] : x[k + 2], 8));
    x[0] = op(lane & 4 ? x[1] : x[0], __shfl_xor_sync(0xffffffffu, lane & 4 ? x[0] : x[1], 4));
    x[0] = op(x[0], __shfl_xor_sync(0xffffffffu, x[0], 2));
    return op(x[0], __shfl_xor_sync(0xffffffffu, x[0], 1));
}
__device__ __forceinline__ int psh_of_lane(int lane) { return (lane >> 2) & 7; }
__device__ __forceinline__ void psh_sum_warps(const PageShared &P, PshSmall &S, uint8_t *smem, uint32_t tmem) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quarter = warp & 3, half = warp >> 2, pos = 32 * quarter + lane;
    const uint32_t tlane = tmem + ((uint32_t)(32 * quarter) << 16);
    constexpr float BASE = 7.0f, MOST = 15.0f;           // a weight is 2^7 at its row's reference and 2^15 at most
    PshWait wait(S);
    PshReader frags{S, wait};
    PshFragment F;
    int it = 0;
    while (true) {
        // (the eight warps go on, and leave, together: they meet at barriers)
        if (psh_any<256>(3, !frags.next(F))) break;
        const int n = (F.n_rows + 15) / 16 * 16;
        psh_queries(P, S, smem, F, n);
        const int all_see = F.before == INT32_MAX ? F.end - 1 : F.before + F.row0 / P.group;
        const int groups = (n - 8 * half + 15) / 16;     // of eight columns: 16 c + 8 half ..
        float2 acc[2][3][4], l[3][4];
#pragma unroll
        for (int c = 0; c < 3; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[0][c][e] = acc[1][c][e] = l[c][e] = make_float2(0.0f, 0.0f);
        bool dead = false;
#pragma unroll 1
        for (int i = 0; i <= F.steps; ++i, ++it) {
            const int p0 = F.pos0 + i * PSH_STEP;
            bool changed = false;
            if (i < F.steps) {
                const bool hidden = p0 + PSH_STEP - 1 > all_see;         // some row does not see some position
                wait(&S.qkdone, (uint32_t)(it & 1));
                tc_fence_after();
                const float kf = atc_pow2(-(int)S.ks[it & 3][pos]);
                float s[3][8];                           // scores in powers of two, less the rows' references
#pragma unroll 1
                for (int turn = 0; turn < 2; ++turn) {
#pragma unroll
                    for (int c = 0; c < 3; ++c)
                        if (c < groups) tc_ld8(tlane + PSH_COL_S + (uint32_t)(16 * c + 8 * half), reinterpret_cast<int (&)[8]>(s[c]));
                    tc_ld_wait();
                    float most = wait.ok ? -INFINITY : INFINITY;
#pragma unroll
                    for (int c = 0; c < 3; ++c)
                        if (c < groups) {
                            float f[8], r[8];
                            psh_lds8(S.qf + 16 * c + 8 * half, f);
                            psh_lds8(S.less + 16 * c + 8 * half, r);
#pragma unroll
                            for (int e = 0; e < 8; e += 2) {
                                const float2 y = fma2(mul2(make_float2(s[c][e], s[c][e + 1]), make_float2(kf, kf)), make_float2(f[e], f[e + 1]), make_float2(r[e], r[e + 1]));
                                s[c][e] = y.x;
                                s[c][e + 1] = y.y;
                            }
                            if (hidden) {
                                int limit[8];
                                psh_lds8(S.limit + 16 * c + 8 * half, limit);
#pragma unroll
                                for (int e = 0; e < 8; ++e)
                                    if (p0 + pos > limit[e]) s[c][e] = -INFINITY;
                            }
#pragma unroll
                            for (int e = 0; e < 8; e += 2) most = fmaxf(most, fmaxf(s[c][e], s[c][e + 1]));
                        }
                    if (turn || !psh_any<128>(1 + half, most > MOST)) break;
                    // a row's first step, then where its scores grow by much: the references move
                    dead = psh_any<128>(1 + half, !wait.ok);
                    if (dead) break;
#pragma unroll 1
                    for (int c = 0; c < groups; ++c) {
                        const int col = 16 * c + 8 * half;
                        float x[8], f[8];
                        int limit[8];
                        tc_ld8(tlane + PSH_COL_S + (uint32_t)col, reinterpret_cast<int (&)[8]>(x));
                        psh_lds8(S.qf + col, f);
                        psh_lds8(S.limit + col, limit);
                        tc_ld_wait();
                        float2 y[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            y[e] = make_float2(p0 + pos > limit[2 * e] ? -INFINITY : __fmul_rn(__fmul_rn(x[2 * e], kf), f[2 * e]),
                                               p0 + pos > limit[2 * e + 1] ? -INFINITY : __fmul_rn(__fmul_rn(x[2 * e + 1], kf), f[2 * e + 1]));
                        const float m = psh_over8(y, lane, [](float a, float b) { return fmaxf(a, b); });
                        if ((lane & 3) == 0) S.red[quarter][col + psh_of_lane(lane)] = m;
                    }
                    psh_barrier<128>(1 + half);
                    if (quarter == 0 && lane < 8 * groups) {
                        const int col = 16 * (lane >> 3) + 8 * half + (lane & 7);
                        const float was = -S.less[col];
                        float m = S.red[0][col];
#pragma unroll
                        for (int w = 1; w < 4; ++w) m = S.red[w][col] > m || S.red[w][col] != S.red[w][col] ? S.red[w][col] : m;
                        m = __fsub_rn(m, BASE);
                        const float now = m > was || m != m ? m : was;
                        S.less[col] = -now;
                        S.change[col] = psh_exp2(__fsub_rn(was, now));
                    }
                    psh_barrier<128>(1 + half);
                    changed = i > 0;
#pragma unroll
                    for (int c = 0; c < 3; ++c)
                        if (c < groups) {
                            float f[8];
                            psh_lds8(S.change + 16 * c + 8 * half, f);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float2 g = make_float2(f[2 * e], f[2 * e + 1]);
                                l[c][e] = mul2(l[c][e], g);
                                acc[0][c][e] = mul2(acc[0][c][e], g);
                                acc[1][c][e] = mul2(acc[1][c][e], g);
                            }
                        }
                }
                if (dead) break;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.sempty);
                uint8_t *dst = smem + PSH_AT_P + (it & 1) * PSH_P_BUF + (pos >> 3) * PSH_P_GROUP + half * 128 + (pos & 7) * 16;
#pragma unroll
                for (int c = 0; c < 3; ++c)
                    if (c < groups) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 a = make_float2(psh_exp2(s[c][2 * e]), psh_exp2(s[c][2 * e + 1]));
                            l[c][e] = add2(l[c][e], a);
                            const __half2 h = __floats2half2_rn(a.x, a.y);
                            const float2 rest = fma2(__half22float2(h), make_float2(-1.0f, -1.0f), a);       // exact
                            const __half2 r = __floats2half2_rn(rest.x, rest.y);
                            hi[e] = *reinterpret_cast<const uint32_t *>(&h);
                            lo[e] = *reinterpret_cast<const uint32_t *>(&r);
                        }
                        *reinterpret_cast<uint4 *>(dst + 256 * c) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        *reinterpret_cast<uint4 *>(dst + 256 * c + PSH_P_PLANE) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.pready[it & 1]);
            }
            if (i == 0) continue;
            // ---- outputs of the step before
            const int o = it - 1;
            wait(&S.pvdone[o & 1], (uint32_t)((o >> 1) & 1));
            tc_fence_after();
            const uint32_t from = tlane + PSH_COL_O + (uint32_t)((o & 1) * PSH_O_BUF + 8 * half);
            const float *vf = S.vf[o & 7] + quarter;
            const float f0 = *(volatile const float *)vf, f1 = *(volatile const float *)(vf + 4);
#pragma unroll
            for (int c = 0; c < 3; ++c) {
                if (c >= groups) break;
                int x[2][8];
                tc_ld8(from + (uint32_t)(16 * c), x[0]);
                tc_ld8(from + (uint32_t)(PSH_ROWS + 16 * c), x[1]);
                tc_ld_wait();
                if (changed) {
                    float g[8];
                    psh_lds8(S.change + 16 * c + 8 * half, g);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        x[0][e] = __float_as_int(__fmul_rn(__int_as_float(x[0][e]), g[e]));
                        x[1][e] = __float_as_int(__fmul_rn(__int_as_float(x[1][e]), g[e]));
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    acc[0][c][e] = fma2(make_float2(__int_as_float(x[0][2 * e]), __int_as_float(x[0][2 * e + 1])), make_float2(f0, f0), acc[0][c][e]);
                    acc[1][c][e] = fma2(make_float2(__int_as_float(x[1][2 * e]), __int_as_float(x[1][2 * e + 1])), make_float2(f1, f1), acc[1][c][e]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.oempty[o & 1]);
            // rows that see a position whose V is no number are no numbers
            if (*reinterpret_cast<const volatile unsigned long long *>(S.v_odd[o & 7])) {
                bool bad = false;
#pragma unroll 1
                for (int b = 0; b < KV_NBLK; ++b) bad = bad || (S.v_odd[o & 7][b] && (S.v_bad[o & 7][quarter][b] >> lane & 1u));
#pragma unroll 1
                for (int r = 0; bad && r < F.n_rows; ++r)
                    if (p0 - PSH_STEP + pos <= S.limit[r]) S.none[r] = 1;
            }
        }
        --it;                                            // (the last turn had outputs only)
        // ---- the fragment's sums
        const bool good = *(volatile int *)&S.failed == 0;
        float *dst = P.part + (F.part + 8 * half) * KV_D + pos;
#pragma unroll
        for (int c = 0; c < 3; ++c)
            if (c < groups) {
                const float x = psh_over8(l[c], lane, [](float a, float b) { return __fadd_rn(a, b); });
                if ((lane & 3) == 0) S.red[quarter][16 * c + 8 * half + psh_of_lane(lane)] = x;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (16 * c + 8 * half + e < F.n_rows && good) {
                        dst[(16 * c + e) * KV_D] = e & 1 ? acc[0][c][e >> 1].y : acc[0][c][e >> 1].x;
                        dst[(16 * c + e) * KV_D + 128] = e & 1 ? acc[1][c][e >> 1].y : acc[1][c][e >> 1].x;
                    }
            }
        psh_barrier<256>(3);                             // (rows that have seen no number are said by both halves)
        if (quarter == 0 && lane < 8 * groups) {
            const int col = 16 * (lane >> 3) + 8 * half + (lane & 7);
            if (col < F.n_rows && good)
                P.part_ml[F.part + col] = make_float2(-S.less[col], S.none[col] ? __int_as_float(0x7FC00000) : __fadd_rn(__fadd_rn(S.red[0][col], S.red[1][col]), __fadd_rn(S.red[2][col], S.red[3][col])));
        }
    }
}

__global__ void __launch_bounds__(PSH_THREADS, 1) pages_shared_kernel(const __grid_constant__ PageShared P) {
    extern __shared__ __align__(128) uint8_t raw[];
    uint8_t *smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    PshSmall &S = *reinterpret_cast<PshSmall *>(smem + PSH_AT_SMALL);
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (int i = 0; i < PSH_DESCS; ++i) mbar_init(&S.dfull[i], 1), mbar_init(&S.dempty[i], PSH_THREADS / 32 - 1);
        for (int i = 0; i < PSH_KSLOTS; ++i) mbar_init(&S.rkfull[i], 1), mbar_init(&S.rkempty[i], 2);
        for (int i = 0; i < PSH_VSLOTS; ++i) mbar_init(&S.rvfull[i], 1), mbar_init(&S.rvempty[i], 8);
        for (int i = 0; i < PSH_KRING; ++i) mbar_init(&S.kready[i], 4), mbar_init(&S.kempty[i], 1);
        for (int i = 0; i < PSH_VRING; ++i) mbar_init(&S.vready[i], 8), mbar_init(&S.vempty[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&S.pready[i], PSH_SUM_WARPS), mbar_init(&S.pvdone[i], 1), mbar_init(&S.oempty[i], PSH_SUM_WARPS);
        mbar_init(&S.qready, PSH_SUM_WARPS);
        mbar_init(&S.qkdone, 1);
        mbar_init(&S.sempty, PSH_SUM_WARPS);
        mbar_init(&S.done[0], 1);
        mbar_init(&S.done[1], 1);
        mbar_fence_init();
        S.failed = 0;
    }
    pdl_wait_prior_grid();                               // (the plan)
    pdl_launch_dependents();
    if (warp == PSH_OUT_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&S.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = S.tmem;
    if (warp < PSH_SUM_WARPS) {
        psh_set_registers<PSH_REGS_SUM>(true);
        psh_sum_warps(P, S, smem, tmem);
    } else if (warp < PSH_K_WARP) {
        psh_set_registers<PSH_REGS_V>(false);
        psh_v_warps(P, S, smem, tmem);
    } else if (warp < PSH_PLAN_WARP) {
        psh_set_registers<PSH_REGS_K>(false);
        psh_k_warps(P, S, smem, tmem);
    } else {
        psh_set_registers<PSH_REGS_REST>(false);
        if (warp == PSH_PLAN_WARP) psh_plan_warp(P, S, smem);
        else if (warp == PSH_LOAD_WARP) psh_load_k_warp(P, S, smem);
        else if (warp == PSH_SCORE_WARP) psh_score_warp(P, S, smem, tmem);
        else psh_out_warp(P, S, smem, tmem);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == PSH_OUT_WARP) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// A row's parts added up: ROWW warps per row (token, head), four dims and four more a lane.
constexpr int PSJ_WARPS = 8;
template <int ROWW>
__global__ void __launch_bounds__(32 * PSJ_WARPS) pages_shared_join_kernel(const __grid_constant__ PageShared P) {
    __shared__ float4 sums[PSJ_WARPS][2][32];
    __shared__ float lsum[PSJ_WARPS];
    const PageCache &C = P.C;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = warp % ROWW, heads = C.n_head_kv;
    const int64_t row = (int64_t)blockIdx.x * (PSJ_WARPS / ROWW) + warp / ROWW;
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    const float *acc[2] = {nullptr, nullptr};
    const float2 *ml[2] = {nullptr, nullptr};
    int n[2] = {0, 0}, gap[2] = {0, 0};                  // a row's parts, and how far apart they are
    bool served = false;
    const int tok = (int)(row / P.n_head), h = (int)(row - (int64_t)tok * P.n_head), kvh = h / P.group;
    const int s = row < (int64_t)C.n_tok * P.n_head ? seq_of_row(C.start, C.n_seq, tok, lane) : C.n_seq;
    if (s < C.n_seq) {                                   // (a row behind the last sequence is nobody's)
        const PshPlan &plan = *P.plan;
        const PshEntity own = plan.entity[P.n_groups + s];
        served = own.steps >= 0 && tok >= own.begin && tok < own.begin + own.tokens;
#pragma unroll
        for (int i = 0; i < 2; ++i) {                    // its own positions; what it shares
            if (!served || (i == 1 && own.page0 == 0)) break;
            const PshEntity E = i ? plan.entity[own.group] : own;
            if (E.steps <= 0) continue;
            if (E.unit < 0) {
                served = false;
                break;
            }
            const bool many = E.image >= 0;
            const int size = many ? PST_ROWS : PSH_ROWS, start = many ? PST_START : PSH_START;
            const int at = (tok - E.begin) * P.group + (h - kvh * P.group), tile = at / size, row0 = tile * size, end = psh_tile_end(P.group, E, row0, size);
            const int steps = many ? (end + PG_POS - 1) / PG_POS - E.page0 : psh_steps(end - E.page0 * PG_POS);
            if (steps <= 0) continue;
            const long long per = many ? plan.tc_per : plan.per, begin = E.unit + (long long)(tile * heads + kvh) * (E.steps + start) + start;
            const long long c0 = begin / per, c1 = (begin + steps - 1) / per;
            const long long first = (many ? plan.tc_row : 0) + E.row + (long long)row0 * heads + kvh * min(size, E.tokens * P.group - row0) + c0 * size + (at - row0);
            n[i] = (int)(c1 - c0 + 1);
            gap[i] = size;
            acc[i] = P.part + first * KV_D;
            ml[i] = P.part_ml + first;
        }
    }
    const int all = served ? n[0] + n[1] : 0;
    float m = -INFINITY, l = 0.0f;
    for (int i = lane; i < all; i += 32) m = fmaxf(m, i < n[0] ? ml[0][(size_t)i * gap[0]].x : ml[1][(size_t)(i - n[0]) * gap[1]].x);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    for (int i0 = mine; i0 < all; i0 += 4 * ROWW) {      // four parts' loads at once
        float2 x[4];
        float4 c[4], d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = min(i0 + e * ROWW, all - 1);
            const size_t step = i < n[0] ? (size_t)i * gap[0] : (size_t)(i - n[0]) * gap[1];
            const float4 *src = reinterpret_cast<const float4 *>((i < n[0] ? acc[0] : acc[1]) + step * KV_D) + lane;
            x[e] = (i < n[0] ? ml[0] : ml[1])[step];
            c[e] = src[0];
            d[e] = src[32];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (i0 + e * ROWW >= all) break;
            const float w = x[e].x == m ? 1.0f : psh_exp2(__fsub_rn(x[e].x, m));
            l = __fmaf_rn(x[e].y, w, l);
            a = make_float4(__fmaf_rn(c[e].x, w, a.x), __fmaf_rn(c[e].y, w, a.y), __fmaf_rn(c[e].z, w, a.z), __fmaf_rn(c[e].w, w, a.w));
            b = make_float4(__fmaf_rn(d[e].x, w, b.x), __fmaf_rn(d[e].y, w, b.y), __fmaf_rn(d[e].z, w, b.z), __fmaf_rn(d[e].w, w, b.w));
        }
    }
    if (ROWW > 1) {
        sums[warp][0][lane] = a;
        sums[warp][1][lane] = b;
        if (lane == 0) lsum[warp] = l;
        __syncthreads();
        if (mine) return;
#pragma unroll
        for (int w = 1; w < ROWW; ++w) {
            const float4 c = sums[warp + w][0][lane], d = sums[warp + w][1][lane];
            l = __fadd_rn(l, lsum[warp + w]);
            a = make_float4(__fadd_rn(a.x, c.x), __fadd_rn(a.y, c.y), __fadd_rn(a.z, c.z), __fadd_rn(a.w, c.w));
            b = make_float4(__fadd_rn(b.x, d.x), __fadd_rn(b.y, d.y), __fadd_rn(b.z, d.z), __fadd_rn(b.w, d.w));
        }
    }
    if (!served) return;
    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);     // a row that sees nothing is zeros
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
