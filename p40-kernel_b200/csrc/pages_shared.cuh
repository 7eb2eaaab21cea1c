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
//   O^T [256 dims x rows]     = V^T P         V as A and the weights P as B from shared memory, two planes each
// three of the four products of planes.  A product's time goes with its rows in steps of 16, so a tile of one token's six heads costs a third of a full one.
//
// Warps: 0 - 7 weights and outputs (a thread has a position of S^T, or two dims of O^T, and half of the columns), 8 - 11 K (a position a thread), 12 - 15 V (a
// position and two of eight blocks a thread), 16 says what the fragments are, 17 copies pages, 18 issues the products.
#pragma once

#include "attn_tc.cuh"
#include "pages.cuh"

namespace b200 {

constexpr int PSH_ROWS = 48, PSH_STEP = 2 * PG_POS, PSH_STAGE = 32, PSH_STAGES = 2, PSH_VSLOTS = 3, PSH_DESCS = 4;
constexpr int PSH_START = 1;                                     // what a fragment's begin is worth, in steps
constexpr int PSH_THREADS = 640, PSH_SUM_WARPS = 8, PSH_K_WARP = 8, PSH_V_WARP = 12, PSH_PLAN_WARP = 16, PSH_LOAD_WARP = 17, PSH_MMA_WARP = 18;
// registers a thread: 2 x 136 + 2 x 80 + 48 = 5 x 96, what the launch has
constexpr int PSH_REGS_SUM = 136, PSH_REGS_PLANES = 80, PSH_REGS_REST = 48;
constexpr int PSH_REGS = 32 * (PSH_SUM_WARPS * PSH_REGS_SUM + 8 * PSH_REGS_PLANES + 4 * PSH_REGS_REST);
constexpr int PSH_Q_CHUNK = PSH_ROWS * 128, PSH_Q_PLANE = 4 * PSH_Q_CHUNK;              // 64 dims of the rows; a plane of them
constexpr int PSH_V_PLANE = PSH_STAGE * KV_D * 2, PSH_V_STAGE = 2 * PSH_V_PLANE;
constexpr int PSH_P_GROUP = PSH_ROWS / 8 * 128, PSH_P_PLANE = PSH_STEP / 8 * PSH_P_GROUP;       // 8 positions of the rows
constexpr int PSH_AT_V = 2 * PSH_Q_PLANE, PSH_AT_P = PSH_AT_V + PSH_STAGES * PSH_V_STAGE, PSH_AT_RAWK = PSH_AT_P + 2 * PSH_P_PLANE,
              PSH_AT_RAWV = PSH_AT_RAWK + 2 * PG_HEAD_BYTES, PSH_AT_SMALL = PSH_AT_RAWV + PSH_VSLOTS * PG_HEAD_BYTES;
constexpr uint32_t PSH_COL_K = 0, PSH_COL_S = 256, PSH_COL_O = 320, PSH_O_BUF = 2 * PSH_ROWS;   // tensor memory: K planes, scores, two buffers of outputs
static_assert(PSH_COL_S + PSH_ROWS <= PSH_COL_O && PSH_COL_O + 2 * PSH_O_BUF <= 512, "");

struct PshFragment {
    int begin, row0, n_rows;            // first token of the entity; of its rows the tile's first, and how many
    int kvh, pos0, steps, end;          // first position; steps (negative: no more fragments); positions that any row sees end here
    int before;                         // the last position that row r sees is before + r / group; INT32_MAX: all up to end
    int group, seq;                     // whose table: of a group's sequences the first that has it (seq < 0), or the sequence's
    long long part;                     // the first row's place among the parts
};
struct PshSmall {
    float kf[2][PSH_STEP];              // 2^-s of the step's K rows; steps alternate
    float vf[4][KV_NBLK];               // 2^-s of the step's V blocks; of four steps: V is at most three ahead of who adds the outputs
    uint32_t v_bad[4][4][4];            // positions whose V is no number, by warp
    float qf[PSH_ROWS];                 // 2^-s of the query rows times scale and log2 e
    int limit[PSH_ROWS];                // the last position that a row sees
    float ref[PSH_ROWS], change[PSH_ROWS], red[4][PSH_ROWS];
    PshFragment desc[PSH_DESCS];
    uint64_t dfull[PSH_DESCS], dempty[PSH_DESCS], rkfull[2], rkempty[2], rvfull[PSH_VSLOTS], rvempty[PSH_VSLOTS], vready[PSH_STAGES], vempty[PSH_STAGES];
    uint64_t qready, kready, qkdone, sempty, pready, pvdone, done;
    int held_k[2], held_v[PSH_VSLOTS];  // rows of a page that there are
    uint32_t tmem;
    int failed;
    // the division
    long long warp_sum[2][PSH_THREADS / 32], found[2], total;
    int found_at;
};
constexpr int PSH_SMEM_BYTES = 1024 + PSH_AT_SMALL + (int)sizeof(PshSmall);
static_assert(PSH_SMEM_BYTES <= 227 * 1024, "");

struct PshPlan { long long unit, row; };                         // of an entity: units and rows of parts in front
struct PageShared {
    PageCache C;
    const float *q;
    float *out, *part;                  // [part_rows][256]
    float2 *part_ml;                    // maximum (as a power of two's exponent) and sum of a part's rows
    PshPlan *plan;                      // [1 + entities]; the first says how many units a CTA has
    const int32_t *group_first, *group_pages;
    long long part_rows;                // of entities; CTAs' own come beside them
    int n_groups, layer, n_head, group;
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
struct PshWork {
    int begin, tokens, page0, end, before, steps;                // steps 0: nothing; -1: numbers that do not fit
};
__device__ __forceinline__ PshWork psh_sequence(const PageShared &P, int s) {
    const PageCache &C = P.C;
    const SeqRange r = seq_range(C.start, s, C.n_tok);
    PshWork W = {r.begin, r.n, 0, 0, 0, 0};
    if (r.n <= 0) {
        if (r.n < 0) W.steps = -1;
        return W;
    }
    const int len = C.len[s], g = psh_group_of(P, s);
    if (len < 0 || len > (int64_t)C.table_stride * PG_POS) {
        W.steps = -1;
        return W;
    }
    if (g < P.n_groups) {
        const PshGroup G = psh_group(P, g);
        // (its new tokens lie behind what it shares)
        if (G.pages < 0 || (G.pages > 0 && (r.begin < G.begin || r.begin + r.n > G.end || (int64_t)len - r.n < (int64_t)G.pages * PG_POS))) {
            W.steps = -1;
            return W;
        }
        W.page0 = G.pages;
    }
    W.end = len;
    W.before = len - r.n;
    W.steps = (len - W.page0 * PG_POS + PSH_STEP - 1) / PSH_STEP;
    return W;
}
__device__ __forceinline__ PshWork psh_work(const PageShared &P, int e) {
    if (e >= P.n_groups) return psh_sequence(P, e - P.n_groups);
    const PshGroup G = psh_group(P, e);
    PshWork W = {G.begin, G.end - G.begin, 0, max(G.pages, 0) * PG_POS, INT32_MAX, 0};
    if (W.tokens > 0) W.steps = (W.end + PSH_STEP - 1) / PSH_STEP;
    return W;
}
__device__ __forceinline__ long long psh_rows(const PageShared &P, const PshWork &W) { return W.steps > 0 ? (long long)W.tokens * P.n_head : 0; }
__device__ __forceinline__ long long psh_units(const PageShared &P, const PshWork &W) {
    return W.steps > 0 ? ((long long)W.tokens * P.group + PSH_ROWS - 1) / PSH_ROWS * P.C.n_head_kv * (W.steps + PSH_START) : 0;
}
// Steps of a tile: those that its last row sees.
__device__ __forceinline__ int psh_tile_end(const PageShared &P, const PshWork &W, long long row0) {
    if (W.before == INT32_MAX) return W.end;
    const long long last = min(row0 + PSH_ROWS, (long long)W.tokens * P.group) - 1;
    return max(W.page0 * PG_POS, min(W.end, W.before + (int)(last / P.group) + 1));
}
__device__ __forceinline__ int psh_tile_steps(const PshWork &W, int end) { return (end - W.page0 * PG_POS + PSH_STEP - 1) / PSH_STEP; }

__device__ __forceinline__ long long psh_scan(long long x, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    return x;
}

// Units of a CTA, and where this one's begin: entity small.found_at, which has found[0] units and found[1] rows in front.  By the whole CTA; the last one leaves the
// plan for the join, and says what does not fit.
__device__ __forceinline__ long long psh_divide(const PageShared &P, PshSmall &S) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, entities = P.n_groups + P.C.n_seq;
    const bool writer = blockIdx.x == gridDim.x - 1;
    long long unit0 = 0, row0 = 0, per = 0;
    long long units = 0, rows = 0, unit_end = 0, row_end = 0;
    for (int pass = 0; pass < 2; ++pass) {               // how many; whose the CTA's first is
        unit0 = row0 = 0;
        for (int base = 0; base < entities; base += PSH_THREADS) {
            const int e = base + tid;
            if (pass == 0 || entities > PSH_THREADS) {
                PshWork W = {0, 0, 0, 0, 0, 0};
                if (e < entities) W = psh_work(P, e);
                if (pass == 0 && writer && W.steps < 0) bad_sequence();
                units = psh_units(P, W);
                rows = psh_rows(P, W);
                row_end = psh_scan(rows, lane);
                if (lane == 31) S.warp_sum[1][warp] = row_end;
                __syncthreads();
                for (int w = 0; w < warp; ++w) row_end += S.warp_sum[1][w];
                row_end += row0;
                if (row_end > P.part_rows) {             // rows that several sequences claim
                    if (pass == 0 && writer && rows) bad_sequence();
                    units = 0;
                }
                unit_end = psh_scan(units, lane);
                if (lane == 31) S.warp_sum[0][warp] = unit_end;
                __syncthreads();
                long long all = 0, all_rows = 0;
                for (int w = 0; w < PSH_THREADS / 32; ++w) {
                    if (w == warp) unit_end += all;
                    all += S.warp_sum[0][w];
                    all_rows += S.warp_sum[1][w];
                }
                unit_end += unit0;
                unit0 += all;
                row0 += all_rows;
                __syncthreads();
            }
            if (pass == 1) {
                const long long first = per * blockIdx.x;
                if (units && unit_end - units <= first && first < unit_end) {
                    S.found_at = e;
                    S.found[0] = unit_end - units;
                    S.found[1] = row_end - rows;
                }
                if (writer && e < entities) P.plan[1 + e] = {units ? unit_end - units : -1, row_end - rows};
            }
        }
        if (pass == 0) per = (unit0 + gridDim.x - 1) / gridDim.x;
        if (pass == 0 && tid == 0) {
            S.total = unit0;
            S.found_at = entities;
            if (writer) P.plan[0] = {per, unit0};
        }
        __syncthreads();
    }
    return per;
}

// ---- small pieces -------------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void psh_mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, bool add) {
    // A: V planes, dims by 64 side by side (128-byte swizzle, 8 positions a kilobyte); B: weights, 8 rows x 8 positions a piece of 128 bytes
    constexpr uint32_t A_HI = (uint32_t)(1024 >> 4) | (1u << 14) | (2u << 29), B_HI = (uint32_t)(128 >> 4) | (1u << 14);
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        ".reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %4};\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t"
        "}\n"
        ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(A_HI), "r"(B_HI), "r"(add ? 1u : 0u)
        : "memory");
}
__device__ __forceinline__ float psh_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));        // 2^-22 of the value
    return y;
}
// Among the four warps of a half of the columns.
__device__ __forceinline__ void psh_half_barrier(int half) { asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory"); }
__device__ __forceinline__ bool psh_half_any(int half, bool x) {
    uint32_t y;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(y) : "r"(x ? 1u : 0u), "r"(1 + half) : "memory");
    return y != 0;
}
// A pair of codes (bytes 0 and 1, or 2 and 3, of w) as fp16, exactly: 1024 + (byte ^ 128) - 1152; w comes with its bytes' signs turned.
__device__ __forceinline__ __half2 psh_pair(uint32_t w, bool upper) {
    const uint32_t x = __byte_perm(w, 0x64646464u, upper ? 0x4342 : 0x4140);
    return __hsub2_rn(*reinterpret_cast<const __half2 *>(&x), __half2half2(__ushort_as_half((unsigned short)0x6480)));
}
// Codes times a scale of two fp16 planes: the rounded product and, exactly, what it leaves.
__device__ __forceinline__ void psh_planes(__half2 codes, __half2 d, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __hmul2_rn(codes, d), l = __hfma2(codes, d, __hneg2(h));
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}
// s with 2^7 <= d 2^s < 2^8 for the largest scale d of those under one power of two (magnitude bits of an fp16; no number, zero: 0)
__device__ __forceinline__ int psh_shift(uint32_t mag) { return mag == 0 || mag >= 0x7C00u ? 0 : 134 - (int)(__float_as_uint(f16_bits_to_f32(mag)) >> 23); }
__device__ __forceinline__ __half2 psh_scale(uint32_t d16, float up) { return __half2half2(__float2half_rn(__fmul_rn(f16_bits_to_f32(d16), up))); }
__device__ __forceinline__ int psh_key(float x) {                // ordered as the floats are
    const int b = __float_as_int(x);
    return b ^ ((b >> 31) & 0x7FFFFFFF);
}
__device__ __forceinline__ float psh_from_key(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7FFFFFFF)); }
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
// A wait that runs out: nothing is waited for any more, the CTA comes to its end and leaves its parts unfinished.
struct PshWait {
    PshSmall &S;
    bool ok = true;
    __device__ __forceinline__ PshWait(PshSmall &s) : S(s) {}
    __device__ __forceinline__ void operator()(uint64_t *bar, uint32_t parity) {
        if (!ok) return;
        ok = __all_sync(0xffffffffu, mbar_wait_try(bar, parity));
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

__device__ __forceinline__ void psh_plan_warp(const PageShared &P, PshSmall &S, long long per) {
    const int lane = threadIdx.x & 31, entities = P.n_groups + P.C.n_seq, heads = P.C.n_head_kv;
    PshWait wait(S);
    long long at = per * blockIdx.x;
    const long long last = min(at + per, S.total);
    int n = 0;
    auto say = [&](const PshFragment &F) {
        if (n >= PSH_DESCS) wait(&S.dempty[n % PSH_DESCS], (uint32_t)((n / PSH_DESCS - 1) & 1));
        if (lane == 0) {
            S.desc[n % PSH_DESCS] = F;
            mbar_arrive(&S.dfull[n % PSH_DESCS]);
        }
        __syncwarp();
        ++n;
    };
    long long unit0 = S.found[0], row0 = S.found[1];
    for (int base = S.found_at; base < entities && at < last && wait.ok; base += 32) {
        PshWork W = {0, 0, 0, 0, 0, 0};
        if (base + lane < entities) W = psh_work(P, base + lane);
        const long long rows = psh_rows(P, W), row_end = row0 + psh_scan(rows, lane);
        const long long units = row_end > P.part_rows ? 0 : psh_units(P, W), unit_end = unit0 + psh_scan(units, lane);
        for (int l = 0; l < 32 && at < last && wait.ok; ++l) {
            const long long e_end = __shfl_sync(0xffffffffu, unit_end, l), e_units = __shfl_sync(0xffffffffu, units, l);
            if (e_units == 0 || e_end <= at) continue;
            PshWork X;
            X.begin = __shfl_sync(0xffffffffu, W.begin, l);
            X.tokens = __shfl_sync(0xffffffffu, W.tokens, l);
            X.page0 = __shfl_sync(0xffffffffu, W.page0, l);
            X.end = __shfl_sync(0xffffffffu, W.end, l);
            X.before = __shfl_sync(0xffffffffu, W.before, l);
            X.steps = __shfl_sync(0xffffffffu, W.steps, l);
            const long long e_row = __shfl_sync(0xffffffffu, row_end - rows, l);
            const int e = base + l, size = X.steps + PSH_START;
            const long long unit = e_end - e_units;
            while (at < e_end && at < last && wait.ok) {
                const long long pair = (at - unit) / size, tile = pair / heads, begin = unit + pair * size;      // the tile and kv head that the next unit lies in
                PshFragment F;
                F.kvh = (int)(pair - tile * heads);
                F.begin = X.begin;
                F.row0 = (int)(tile * PSH_ROWS);
                F.n_rows = (int)min((long long)PSH_ROWS, (long long)X.tokens * P.group - F.row0);
                F.end = psh_tile_end(P, X, F.row0);
                F.before = X.before;
                F.group = e < P.n_groups ? e : -1;
                F.seq = e < P.n_groups ? -1 : e - P.n_groups;
                F.part = e_row + tile * PSH_ROWS * heads + (long long)F.kvh * F.n_rows + (long long)blockIdx.x * PSH_ROWS;
                const long long stop = min(last, begin + size);
                const int s0 = (int)max(0ll, at - begin - PSH_START), s1 = (int)min(stop - begin - PSH_START, (long long)psh_tile_steps(X, F.end));
                F.pos0 = X.page0 * PG_POS + s0 * PSH_STEP;
                F.steps = s1 - s0;
                if (F.steps > 0) say(F);
                at = stop;
            }
        }
        unit0 = __shfl_sync(0xffffffffu, unit_end, 31);
        row0 = __shfl_sync(0xffffffffu, row_end, 31);
    }
    PshFragment F = {};
    F.steps = -1;
    say(F);
}

__device__ __forceinline__ void psh_load_warp(const PageShared &P, PshSmall &S, uint8_t *smem) {
    const PageCache &C = P.C;
    const int lane = threadIdx.x & 31;
    PshWait wait(S);
    PshReader frags{S, wait};
    PshFragment F;
    int nk[2] = {0, 0}, nv = 0;
    while (frags.next(F)) {
        int seq = F.seq;
        if (seq < 0) {                                   // the first sequence of the group that has the pages in common: one with new tokens behind them
            const int first = P.group_first[F.group], last = P.group_first[F.group + 1];
            for (int base = first; base < last && seq < 0; base += 32) {
                bool has = false;
                if (base + lane < last) {
                    const PshWork W = psh_sequence(P, base + lane);
                    has = W.steps > 0;
                }
                const unsigned found = __ballot_sync(0xffffffffu, has);
                if (found) seq = base + __ffs(found) - 1;
            }
        }
        const int32_t *table = C.table + (size_t)max(seq, 0) * C.table_stride;
        const int page0 = F.pos0 / PG_POS, pages = (F.end - F.pos0 + PG_POS - 1) / PG_POS;
        const uint64_t pol = policy_evict_normal();
        for (int i = 0; i < F.steps && wait.ok; ++i) {
            const PshStep T = psh_step(F, i);
            int own = -1;
            if (lane < T.pages && seq >= 0 && 2 * i + lane < pages) own = table[page0 + 2 * i + lane];
            for (int j = 0; j < T.pages; ++j) {
                int page = __shfl_sync(0xffffffffu, own, j);
                const bool there = page >= 0 && page < C.n_pages;
                if (!there && lane == 0) bad_sequence();
                const int n = min(PG_POS, T.valid - j * PG_POS);
                const uint32_t bytes = (uint32_t)n * KV_ROW;
                auto copy = [&](int kv, uint8_t *dst, uint64_t *full, int *held) {
                    if (lane) return;
                    *held = there ? n : 0;
                    if (there) {
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        mbar_expect_tx(full, bytes);
                        bulk_g2s(dst, page_rows(C, page, P.layer, kv, F.kvh), bytes, full, pol);
                    } else {
                        mbar_arrive(full);
                    }
                };
                if (nk[j] > 0) wait(&S.rkempty[j], (uint32_t)((nk[j] - 1) & 1));
                if (!wait.ok) break;
                copy(0, smem + PSH_AT_RAWK + j * PG_HEAD_BYTES, &S.rkfull[j], &S.held_k[j]);
                ++nk[j];
                __syncwarp();
            }
            for (int j = 0; j < T.pages && wait.ok; ++j) {
                int page = __shfl_sync(0xffffffffu, own, j);
                const bool there = page >= 0 && page < C.n_pages;
                const int n = min(PG_POS, T.valid - j * PG_POS), slot = nv % PSH_VSLOTS;
                const uint32_t bytes = (uint32_t)n * KV_ROW;
                if (nv >= PSH_VSLOTS) wait(&S.rvempty[slot], (uint32_t)((nv / PSH_VSLOTS - 1) & 1));
                if (!wait.ok) break;
                if (lane == 0) {
                    S.held_v[slot] = there ? n : 0;
                    if (there) {
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        mbar_expect_tx(&S.rvfull[slot], bytes);
                        bulk_g2s(smem + PSH_AT_RAWV + slot * PG_HEAD_BYTES, page_rows(C, page, P.layer, 1, F.kvh), bytes, &S.rvfull[slot], pol);
                    } else {
                        mbar_arrive(&S.rvfull[slot]);
                    }
                }
                ++nv;
                __syncwarp();
            }
        }
    }
    // no copy outlives the CTA
    for (int j = 0; j < 2; ++j)
        if (nk[j]) mbar_wait_try(&S.rkfull[j], (uint32_t)((nk[j] - 1) & 1));
    for (int k = max(0, nv - PSH_VSLOTS); k < nv; ++k) mbar_wait_try(&S.rvfull[k % PSH_VSLOTS], (uint32_t)((k / PSH_VSLOTS) & 1));
}

// K rows to planes in tensor memory: a position a thread.
__device__ __forceinline__ void psh_k_warps(const PageShared &P, PshSmall &S, uint8_t *smem, uint32_t tmem) {
    const int lane = threadIdx.x & 31, quarter = (threadIdx.x >> 5) & 3, pos = 32 * quarter + lane, slot = quarter >> 1;
    const uint32_t to = tmem + PSH_COL_K + ((uint32_t)(32 * quarter) << 16);
    const uint8_t *row = smem + PSH_AT_RAWK + slot * PG_HEAD_BYTES + (pos & (PG_POS - 1)) * KV_ROW;
    PshWait wait(S);
    PshReader frags{S, wait};
    PshFragment F;
    int it = 0, n = 0;                                   // steps; pages of the slot
    while (frags.next(F)) {
        for (int i = 0; i < F.steps && wait.ok; ++i, ++it) {
            const PshStep T = psh_step(F, i);
            const bool mine = T.pages > slot;
            if (it > 0) wait(&S.qkdone, (uint32_t)((it - 1) & 1));                // the planes have been read
            tc_fence_after();
            if (mine) {
                wait(&S.rkfull[slot], (uint32_t)(n & 1));
                ++n;
                const bool there = (pos & (PG_POS - 1)) < S.held_k[slot];
                uint32_t top = 0;
#pragma unroll
                for (int b = 0; b < KV_NBLK; ++b) top = max(top, (uint32_t)*reinterpret_cast<const uint16_t *>(row + 34 * b) & 0x7FFFu);
                const int s = there ? psh_shift(top) : 0;
                const float up = atc_pow2(s);
                S.kf[it & 1][pos] = atc_pow2(-s);
#pragma unroll
                for (int h = 0; h < 2; ++h) {            // blocks 4 h ..: bytes 0 .. 143, 128 .. 271
                    uint32_t w[36];
#pragma unroll
                    for (int j = 0; j < 9; ++j) {
                        const uint4 x = *reinterpret_cast<const uint4 *>(row + 128 * h + 16 * j);
                        w[4 * j] = x.x; w[4 * j + 1] = x.y; w[4 * j + 2] = x.z; w[4 * j + 3] = x.w;
                    }
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const int byte = 34 * (4 * h + b) - 128 * h, at = byte >> 2;              // of the block, in w
                        const bool odd = byte & 2;
                        const uint32_t d16 = odd ? w[at] >> 16 : w[at] & 0xFFFFu;
                        const __half2 d = psh_scale(there ? d16 : 0u, up);
                        uint32_t hi[16], lo[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {   // halfword 1 + e of the block
                            const int half = (byte >> 1) + 1 + e;
                            psh_planes(psh_pair(w[half >> 1] ^ 0x80808080u, half & 1), d, hi[e], lo[e]);
                        }
                        tc_st16(to + (uint32_t)(16 * (4 * h + b)), hi);
                        tc_st16(to + (uint32_t)(128 + 16 * (4 * h + b)), lo);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.rkempty[slot]);
                tc_st_wait();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.kready);
        }
    }
}

// V rows to planes in shared memory, 32 positions a stage: a warp has two of the eight blocks, under one power of two each for a step.
template <int W>
__device__ __forceinline__ void psh_v_rows(const uint8_t *row, const float (&up)[2], bool there, uint8_t *dst, uint32_t lane) {
    uint32_t w[20];
#pragma unroll
    for (int j = 0; j < 5; ++j) {
        const uint4 x = *reinterpret_cast<const uint4 *>(row + 64 * W + 16 * j);
        w[4 * j] = x.x; w[4 * j + 1] = x.y; w[4 * j + 2] = x.z; w[4 * j + 3] = x.w;
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int byte = 4 * W + 34 * b;
        const uint32_t d16 = b ? w[byte >> 2] >> 16 : w[byte >> 2] & 0xFFFFu;
        const bool number = (d16 & 0x7FFFu) < 0x7C00u;
        const __half2 d = psh_scale(there && number ? d16 : 0u, up[b]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int half = (byte >> 1) + 1 + 4 * j + e;
                psh_planes(psh_pair(w[half >> 1] ^ 0x80808080u, half & 1), d, hi[e], lo[e]);
            }
            uint8_t *to = dst + (((uint32_t)(4 * b + j) ^ (lane & 7u)) << 4);
            *reinterpret_cast<uint4 *>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4 *>(to + PSH_V_PLANE) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
    }
}
__device__ __forceinline__ void psh_v_warps(const PageShared &P, PshSmall &S, uint8_t *smem) {
    const uint32_t lane = threadIdx.x & 31, quarter = (threadIdx.x >> 5) & 3;
    PshWait wait(S);
    PshReader frags{S, wait};
    PshFragment F;
    int it = 0, nv = 0, stage = 0;
    while (frags.next(F)) {
        for (int i = 0; i < F.steps && wait.ok; ++i, ++it) {
            const PshStep T = psh_step(F, i);
            const uint8_t *page[2] = {nullptr, nullptr};
            int held[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (j >= T.pages) break;
                const int slot = (nv + j) % PSH_VSLOTS;
                wait(&S.rvfull[slot], (uint32_t)(((nv + j) / PSH_VSLOTS) & 1));
                page[j] = smem + PSH_AT_RAWV + slot * PG_HEAD_BYTES;
                held[j] = S.held_v[slot];
            }
            uint32_t top[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 4; ++j) {                // a lane's position of each stage
                const int at = 32 * (j & 1) + (int)lane;
                bool bad = false;
                if (j < T.stages && at < held[j >> 1]) {
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const uint32_t mag = *reinterpret_cast<const uint16_t *>(page[j >> 1] + at * KV_ROW + 34 * (2 * quarter + b)) & 0x7FFFu;
                        if (mag < 0x7C00u) top[b] = max(top[b], mag);
                        else bad = true;
                    }
                }
                const uint32_t mask = __ballot_sync(0xffffffffu, bad);
                if (lane == 0) S.v_bad[it & 3][quarter][j] = mask;
            }
            float up[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int s = psh_shift(__reduce_max_sync(0xffffffffu, top[b]));
                up[b] = atc_pow2(s);
                if (lane == 0) S.vf[it & 3][2 * quarter + b] = atc_pow2(-s);
            }
            for (int j = 0; j < T.stages && wait.ok; ++j, ++stage) {
                if (stage >= PSH_STAGES) wait(&S.vempty[stage % PSH_STAGES], (uint32_t)((stage / PSH_STAGES - 1) & 1));
                const int at = 32 * (j & 1) + (int)lane;
                const uint8_t *row = (j >> 1 ? page[1] : page[0]) + at * KV_ROW;
                const bool there = at < (j >> 1 ? held[1] : held[0]);
                uint8_t *dst = smem + PSH_AT_V + (stage % PSH_STAGES) * PSH_V_STAGE + quarter * (PSH_STAGE * 128) + lane * 128;
                if (quarter == 0) psh_v_rows<0>(row, up, there, dst, lane);
                else if (quarter == 1) psh_v_rows<1>(row, up, there, dst, lane);
                else if (quarter == 2) psh_v_rows<2>(row, up, there, dst, lane);
                else psh_v_rows<3>(row, up, there, dst, lane);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&S.vready[stage % PSH_STAGES]);
                    if ((j & 1) || j == T.stages - 1) mbar_arrive(&S.rvempty[(nv + (j >> 1)) % PSH_VSLOTS]);
                }
            }
            nv += T.pages;
        }
    }
}

__device__ __forceinline__ void psh_mma_warp(const PageShared &P, PshSmall &S, uint8_t *smem, uint32_t tmem) {
    constexpr uint32_t MAJOR_MN = (1u << 15) | (1u << 16);
    PshWait wait(S);
    PshReader frags{S, wait};
    PshFragment F;
    int it = 0, stage = 0, frag = 0;
    const uint32_t q0 = tc16_desc_lo(smem_u32(smem));
    const uint32_t v0 = ((smem_u32(smem + PSH_AT_V) >> 4) & 0x3FFFu) | ((uint32_t)(PSH_STAGE * 128 >> 4) << 16);
    const uint32_t p0 = ((smem_u32(smem + PSH_AT_P) >> 4) & 0x3FFFu) | ((uint32_t)(PSH_P_GROUP >> 4) << 16);
    while (frags.next(F)) {
        const int n = (F.n_rows + 15) / 16 * 16;
        const uint32_t idesc = atc_idesc(n);
        for (int i = 0; i <= F.steps && wait.ok; ++i) {
            if (i < F.steps) {                           // scores of step i
                if (i == 0) wait(&S.qready, (uint32_t)(frag & 1));
                wait(&S.kready, (uint32_t)(it & 1));
                if (it > 0) wait(&S.sempty, (uint32_t)((it - 1) & 1));
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t k = tmem + PSH_COL_K, d = tmem + PSH_COL_S;
                    auto at = [](int c) { return (uint32_t)((c >> 2) * (PSH_Q_CHUNK >> 4) + 2 * (c & 3)); };
                    tc_mma_f16_ts<false>(d, k + 128u, q0, idesc);
#pragma unroll
                    for (int c = 1; c < 16; ++c) tc_mma_f16_ts<true>(d, k + 128u + (uint32_t)(8 * c), q0 + at(c), idesc);
#pragma unroll
                    for (int c = 0; c < 16; ++c) tc_mma_f16_ts<true>(d, k + (uint32_t)(8 * c), q0 + (uint32_t)(PSH_Q_PLANE >> 4) + at(c), idesc);
#pragma unroll
                    for (int c = 0; c < 16; ++c) tc_mma_f16_ts<true>(d, k + (uint32_t)(8 * c), q0 + at(c), idesc);
                    tc_commit(&S.qkdone);
                }
                __syncwarp();
            }
            if (i > 0) {                                 // outputs of step i - 1, whose number is pv
                const int pv = it - 1;
                const PshStep T = psh_step(F, i - 1);
                wait(&S.pready, (uint32_t)(pv & 1));
                for (int j = 0; j < T.stages; ++j, ++stage) {
                    wait(&S.vready[stage % PSH_STAGES], (uint32_t)((stage / PSH_STAGES) & 1));
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t va = v0 + (uint32_t)((stage % PSH_STAGES) * (PSH_V_STAGE >> 4)), pb = p0 + (uint32_t)(j * (PSH_STAGE / 8) * (PSH_P_GROUP >> 4));
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            const uint32_t d = tmem + PSH_COL_O + (uint32_t)((pv & 1) * PSH_O_BUF + m * PSH_ROWS);
                            const uint32_t a = va + (uint32_t)(m * (2 * PSH_STAGE * 128 >> 4));
#pragma unroll
                            for (int pr = 0; pr < 3; ++pr)               // low V, low weights, both high
#pragma unroll
                                for (int c = 0; c < 2; ++c)
                                    psh_mma_ss(d, a + (uint32_t)((pr == 0 ? PSH_V_PLANE : 0) >> 4) + (uint32_t)(c * (2048 >> 4)),
                                               pb + (uint32_t)((pr == 1 ? PSH_P_PLANE : 0) >> 4) + (uint32_t)(2 * c * (PSH_P_GROUP >> 4)), idesc | MAJOR_MN, j + pr + c > 0);
                        }
                        tc_commit(&S.vempty[stage % PSH_STAGES]);
                        if (j == T.stages - 1) tc_commit(&S.pvdone);
                    }
                    __syncwarp();
                }
            }
            if (i < F.steps) ++it;
        }
        ++frag;
    }
    if (elect_one()) tc_commit(&S.done);                 // everything that was issued
    __syncwarp();
    mbar_wait_try(&S.done, 0);
}

__device__ __forceinline__ void psh_sum_warps(const PageShared &P, PshSmall &S, uint8_t *smem, uint32_t tmem) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quarter = warp & 3, half = warp >> 2, pos = 32 * quarter + lane;
    const uint32_t tlane = tmem + ((uint32_t)(32 * quarter) << 16);
    constexpr float LOG2E = 1.44269504088896340736f;
    constexpr float BASE = 7.0f, MOST = 15.0f;           // a weight is 2^7 at its row's reference and 2^15 at most
    PshWait wait(S);
    PshReader frags{S, wait};
    PshFragment F;
    int it = 0;
    while (true) {
        // (the eight warps go on, and leave, together: they meet at barriers)
        const bool more = frags.next(F);
        uint32_t all;
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, 3, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(all) : "r"(more ? 1u : 0u) : "memory");
        if (!all) break;
        // ---- queries, quantised as the cache rows are, to planes
        const int n = (F.n_rows + 15) / 16 * 16;
        {
            const bool vec = (reinterpret_cast<uintptr_t>(P.q) & 15u) == 0;
            float x[PSH_ROWS / PSH_SUM_WARPS][8];
#pragma unroll
            for (int e = 0; e < PSH_ROWS / PSH_SUM_WARPS; ++e) {
                const int r = warp + PSH_SUM_WARPS * e;
                if (r >= n) break;
                const int row = F.row0 + min(r, F.n_rows - 1), tok = row / P.group;
                const float *src = P.q + ((size_t)(F.begin + tok) * P.n_head + F.kvh * P.group + (row - tok * P.group)) * KV_D + 8 * lane;
                if (vec) {
                    const float4 a = *reinterpret_cast<const float4 *>(src), b = *reinterpret_cast<const float4 *>(src + 4);
                    x[e][0] = a.x; x[e][1] = a.y; x[e][2] = a.z; x[e][3] = a.w; x[e][4] = b.x; x[e][5] = b.y; x[e][6] = b.z; x[e][7] = b.w;
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[e][j] = src[j];
                }
            }
#pragma unroll
            for (int e = 0; e < PSH_ROWS / PSH_SUM_WARPS; ++e) {
                const int r = warp + PSH_SUM_WARPS * e;
                if (r >= n) break;
                const float d = __fmul_rn(kv_amax_8(x[e]), PG_SCALE), id = d > 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
                const uint32_t d16 = r < F.n_rows ? f32_to_f16_bits_ties_away(d) : 0u;
                const int s = psh_shift(__reduce_max_sync(0xffffffffu, d16));
                const __half2 sc = psh_scale(d16, atc_pow2(s));
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int a = max(-127, min(127, round_ties_away(__fmul_rn(x[e][2 * j], id)))), b = max(-127, min(127, round_ties_away(__fmul_rn(x[e][2 * j + 1], id))));
                    psh_planes(__halves2half2(__int2half_rn(a), __int2half_rn(b)), sc, hi[j], lo[j]);
                }
                uint8_t *dst = smem + (lane >> 3) * PSH_Q_CHUNK + r * 128 + (((lane & 7) ^ (r & 7)) << 4);
                *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4 *>(dst + PSH_Q_PLANE) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                if (lane == 0) {
                    S.qf[r] = __fmul_rn(__fmul_rn(P.scale, LOG2E), atc_pow2(-s));
                    S.limit[r] = r >= F.n_rows ? -1 : F.before == INT32_MAX ? F.end - 1 : F.before + (F.row0 + r) / P.group;
                    S.ref[r] = -1e30f;
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            asm volatile("bar.sync 3, 256;" ::: "memory");               // every row's numbers
            if (lane == 0) mbar_arrive(&S.qready);
        }
        const int all_see = F.before == INT32_MAX ? F.end - 1 : F.before + F.row0 / P.group;
        const int groups = (n - 8 * half + 15) / 16;     // of eight columns: 16 c + 8 half ..
        float acc[2][3][8], l[3][8];
#pragma unroll
        for (int c = 0; c < 3; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[0][c][e] = acc[1][c][e] = l[c][e] = 0.0f;
        bool changed = false;
        const int first = it;
        auto drain = [&](int i) {                        // outputs of step i
            const uint32_t from = tlane + PSH_COL_O + (uint32_t)((i & 1) * PSH_O_BUF + 8 * half);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const float f = S.vf[i & 3][4 * m + quarter];
#pragma unroll
                for (int c = 0; c < 3; ++c) {
                    if (c >= groups) break;
                    int o[8];
                    tc_ld8(from + (uint32_t)(m * PSH_ROWS + 16 * c), o);
                    tc_ld_wait();
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float g = changed ? __fmul_rn(f, S.change[16 * c + 8 * half + e]) : f;
                        acc[m][c][e] = __fmaf_rn(__int_as_float(o[e]), g, acc[m][c][e]);
                    }
                }
            }
            tc_fence_before();
        };
        // rows that see a position whose V is no number are no numbers
        auto poison = [&](int i, int p0) {
            const uint32_t (*bad)[4] = S.v_bad[i & 3];
            if ((bad[0][quarter] | bad[1][quarter] | bad[2][quarter] | bad[3][quarter]) >> lane & 1u)
#pragma unroll
                for (int c = 0; c < 3; ++c)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (c < groups && p0 + pos <= S.limit[16 * c + 8 * half + e]) l[c][e] = __int_as_float(0x7FC00000);
        };
        for (int i = 0; i < F.steps; ++i, ++it) {
            const int p0 = F.pos0 + i * PSH_STEP;
            wait(&S.qkdone, (uint32_t)(it & 1));
            tc_fence_after();
            float s[3][8];
            {
                int x[3][8];
#pragma unroll
                for (int c = 0; c < 3; ++c)
                    if (c < groups) tc_ld8(tlane + PSH_COL_S + (uint32_t)(16 * c + 8 * half), x[c]);
                tc_ld_wait();
                const float kf = S.kf[it & 1][pos];
#pragma unroll
                for (int c = 0; c < 3; ++c)
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[c][e] = c < groups ? __fmul_rn(__int_as_float(x[c][e]), __fmul_rn(kf, S.qf[16 * c + 8 * half + e])) : 0.0f;
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.sempty);
            if (p0 + PSH_STEP - 1 > all_see) {           // some row does not see some position
#pragma unroll
                for (int c = 0; c < 3; ++c)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (c < groups && p0 + pos > S.limit[16 * c + 8 * half + e]) s[c][e] = -INFINITY;
            }
            bool above = !wait.ok;
#pragma unroll
            for (int c = 0; c < 3; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c < groups) above = above || s[c][e] > __fadd_rn(S.ref[16 * c + 8 * half + e], MOST);
            if (psh_half_any(half, above)) {             // (a row's first step, then where its scores grow by much: the references move)
                if (psh_half_any(half, !wait.ok)) break;
#pragma unroll
                for (int c = 0; c < 3; ++c)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (c < groups) {
                            const float m = psh_from_key(__reduce_max_sync(0xffffffffu, psh_key(s[c][e])));
                            if (lane == 0) S.red[quarter][16 * c + 8 * half + e] = m;
                        }
                psh_half_barrier(half);
                if (quarter == 0 && lane < 8 * groups) {
                    const int col = 16 * (lane >> 3) + 8 * half + (lane & 7);
                    const float was = S.ref[col];
                    float m = S.red[0][col];
#pragma unroll
                    for (int w = 1; w < 4; ++w) m = S.red[w][col] > m || S.red[w][col] != S.red[w][col] ? S.red[w][col] : m;
                    m = __fsub_rn(m, BASE);
                    const float now = m > was || m != m ? m : was;
                    S.ref[col] = now;
                    S.change[col] = psh_exp2(__fsub_rn(was, now));
                }
                psh_half_barrier(half);
                changed = it > first;
#pragma unroll
                for (int c = 0; c < 3; ++c)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (c < groups) {
                            const float f = S.change[16 * c + 8 * half + e];
                            l[c][e] = __fmul_rn(l[c][e], f);
                            acc[0][c][e] = __fmul_rn(acc[0][c][e], f);
                            acc[1][c][e] = __fmul_rn(acc[1][c][e], f);
                        }
            }
            uint32_t hi[3][4], lo[3][4];
#pragma unroll
            for (int c = 0; c < 3; ++c)
#pragma unroll
                for (int e = 0; e < 8; e += 2)
                    if (c < groups) {
                        const float a = psh_exp2(__fsub_rn(s[c][e], S.ref[16 * c + 8 * half + e])), b = psh_exp2(__fsub_rn(s[c][e + 1], S.ref[16 * c + 8 * half + e + 1]));
                        l[c][e] = __fadd_rn(l[c][e], a);
                        l[c][e + 1] = __fadd_rn(l[c][e + 1], b);
                        split_f16x2(a, b, hi[c][e >> 1], lo[c][e >> 1]);
                    }
            if (it > first) {
                wait(&S.pvdone, (uint32_t)((it - 1) & 1));               // the weights before have been read
                tc_fence_after();
            }
            uint8_t *dst = smem + PSH_AT_P + (pos >> 3) * PSH_P_GROUP + half * 128 + (pos & 7) * 16;
#pragma unroll
            for (int c = 0; c < 3; ++c)
                if (c < groups) {
                    *reinterpret_cast<uint4 *>(dst + 256 * c) = make_uint4(hi[c][0], hi[c][1], hi[c][2], hi[c][3]);
                    *reinterpret_cast<uint4 *>(dst + 256 * c + PSH_P_PLANE) = make_uint4(lo[c][0], lo[c][1], lo[c][2], lo[c][3]);
                }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.pready);
            if (it > first) {
                drain(it - 1);
                poison(it - 1, p0 - PSH_STEP);
            }
            changed = false;
        }
        wait(&S.pvdone, (uint32_t)((it - 1) & 1));
        tc_fence_after();
        drain(it - 1);
        poison(it - 1, F.pos0 + (F.steps - 1) * PSH_STEP);
        // ---- the fragment's sums
        const bool good = *(volatile int *)&S.failed == 0;
#pragma unroll
        for (int c = 0; c < 3; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c < groups) {
                    float x = l[c][e];
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) x = __fadd_rn(x, __shfl_xor_sync(0xffffffffu, x, o));
                    const int col = 16 * c + 8 * half + e;
                    if (lane == 0) S.red[quarter][col] = x;
                    if (col < F.n_rows && good) {
                        float *dst = P.part + (F.part + col) * KV_D + pos;
                        dst[0] = acc[0][c][e];
                        dst[128] = acc[1][c][e];
                    }
                }
        psh_half_barrier(half);
        if (quarter == 0 && lane < 8 * groups) {
            const int col = 16 * (lane >> 3) + 8 * half + (lane & 7);
            if (col < F.n_rows && good)
                P.part_ml[F.part + col] = make_float2(S.ref[col], __fadd_rn(__fadd_rn(S.red[0][col], S.red[1][col]), __fadd_rn(S.red[2][col], S.red[3][col])));
        }
    }
}

__global__ void __launch_bounds__(PSH_THREADS, 1) pages_shared_kernel(const __grid_constant__ PageShared P) {
    extern __shared__ __align__(128) uint8_t raw[];
    uint8_t *smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    PshSmall &S = *reinterpret_cast<PshSmall *>(smem + PSH_AT_SMALL);
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (int i = 0; i < PSH_DESCS; ++i) mbar_init(&S.dfull[i], 1), mbar_init(&S.dempty[i], PSH_SUM_WARPS + 10);
        for (int i = 0; i < 2; ++i) mbar_init(&S.rkfull[i], 1), mbar_init(&S.rkempty[i], 2);
        for (int i = 0; i < PSH_VSLOTS; ++i) mbar_init(&S.rvfull[i], 1), mbar_init(&S.rvempty[i], 4);
        for (int i = 0; i < PSH_STAGES; ++i) mbar_init(&S.vready[i], 4), mbar_init(&S.vempty[i], 1);
        mbar_init(&S.qready, PSH_SUM_WARPS);
        mbar_init(&S.kready, 4);
        mbar_init(&S.qkdone, 1);
        mbar_init(&S.sempty, PSH_SUM_WARPS);
        mbar_init(&S.pready, PSH_SUM_WARPS);
        mbar_init(&S.pvdone, 1);
        mbar_init(&S.done, 1);
        mbar_fence_init();
        S.failed = 0;
    }
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    if (warp == PSH_MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&S.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const long long per = psh_divide(P, S);              // (and its barriers: the ones above are there)
    tc_fence_after();
    const uint32_t tmem = S.tmem;
    if (warp < PSH_SUM_WARPS) {
        psh_set_registers<PSH_REGS_SUM>(true);
        psh_sum_warps(P, S, smem, tmem);
    } else if (warp < PSH_V_WARP) {
        psh_set_registers<PSH_REGS_PLANES>(false);
        psh_k_warps(P, S, smem, tmem);
    } else if (warp < PSH_PLAN_WARP) {
        psh_set_registers<PSH_REGS_PLANES>(false);
        psh_v_warps(P, S, smem);
    } else {
        psh_set_registers<PSH_REGS_REST>(false);
        if (warp == PSH_PLAN_WARP) psh_plan_warp(P, S, per);
        else if (warp == PSH_LOAD_WARP) psh_load_warp(P, S, smem);
        else if (warp == PSH_MMA_WARP) psh_mma_warp(P, S, smem, tmem);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == PSH_MMA_WARP) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// A row's parts added up: a warp per row (token, head), eight dims a lane.
constexpr int PSJ_WARPS = 8;
__global__ void __launch_bounds__(32 * PSJ_WARPS) pages_shared_join_kernel(const __grid_constant__ PageShared P) {
    const PageCache &C = P.C;
    const int lane = threadIdx.x & 31, heads = C.n_head_kv;
    const int64_t row = (int64_t)blockIdx.x * PSJ_WARPS + (threadIdx.x >> 5);
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    if (row >= (int64_t)C.n_tok * P.n_head) return;
    const int tok = (int)(row / P.n_head), h = (int)(row - (int64_t)tok * P.n_head), kvh = h / P.group;
    const int s = seq_of_row(C.start, C.n_seq, tok, lane);
    if (s >= C.n_seq) return;                            // nobody's
    const PshWork own = psh_sequence(P, s);
    if (own.steps < 0 || tok < own.begin || tok >= own.begin + own.tokens) return;
    const long long per = P.plan[0].unit;
    const float *acc[2] = {nullptr, nullptr};
    const float2 *ml[2] = {nullptr, nullptr};
    int n[2] = {0, 0};
    bool served = true;
#pragma unroll
    for (int i = 0; i < 2; ++i) {                        // its own positions; what it shares
        PshWork W = own;
        int e = P.n_groups + s;
        if (i == 1) {
            if (own.page0 == 0) break;
            e = psh_group_of(P, s);
            W = psh_work(P, e);
        }
        if (W.steps <= 0) continue;
        const PshPlan plan = P.plan[1 + e];
        if (plan.unit < 0) {
            served = false;
            break;
        }
        const long long at = (long long)(tok - W.begin) * P.group + (h - kvh * P.group), tile = at / PSH_ROWS;
        const long long begin = plan.unit + (tile * heads + kvh) * (W.steps + PSH_START) + PSH_START;
        const int steps = psh_tile_steps(W, psh_tile_end(P, W, tile * PSH_ROWS));
        if (steps <= 0) continue;
        const long long c0 = begin / per, c1 = (begin + steps - 1) / per;
        const long long tile_rows = min((long long)PSH_ROWS, (long long)W.tokens * P.group - tile * PSH_ROWS);
        const long long first = plan.row + tile * PSH_ROWS * heads + kvh * tile_rows + c0 * PSH_ROWS + (at - tile * PSH_ROWS);
        n[i] = (int)(c1 - c0 + 1);
        acc[i] = P.part + first * KV_D;
        ml[i] = P.part_ml + first;
    }
    if (!served) return;
    const int all = n[0] + n[1];
    float m = -INFINITY, l = 0.0f;
    for (int i = lane; i < all; i += 32) m = fmaxf(m, i < n[0] ? ml[0][(size_t)i * PSH_ROWS].x : ml[1][(size_t)(i - n[0]) * PSH_ROWS].x);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    for (int i0 = 0; i0 < all; i0 += 4) {                // four parts' loads at once
        float2 x[4];
        float4 c[4], d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = min(i0 + e, all - 1);
            const float2 *pml = i < n[0] ? ml[0] + (size_t)i * PSH_ROWS : ml[1] + (size_t)(i - n[0]) * PSH_ROWS;
            const float4 *src = reinterpret_cast<const float4 *>(i < n[0] ? acc[0] + (size_t)i * PSH_ROWS * KV_D : acc[1] + (size_t)(i - n[0]) * PSH_ROWS * KV_D) + lane;
            x[e] = *pml;
            c[e] = src[0];
            d[e] = src[32];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (i0 + e >= all) break;
            const float w = x[e].x == m ? 1.0f : psh_exp2(__fsub_rn(x[e].x, m));
            l = __fmaf_rn(x[e].y, w, l);
            a = make_float4(__fmaf_rn(c[e].x, w, a.x), __fmaf_rn(c[e].y, w, a.y), __fmaf_rn(c[e].z, w, a.z), __fmaf_rn(c[e].w, w, a.w));
            b = make_float4(__fmaf_rn(d[e].x, w, b.x), __fmaf_rn(d[e].y, w, b.y), __fmaf_rn(d[e].z, w, b.z), __fmaf_rn(d[e].w, w, b.w));
        }
    }
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
