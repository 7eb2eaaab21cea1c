// gdn_seqs.cuh -- the gated delta rule over the tokens of several sequences: S <- e^g S, d = beta (v - k S), S <- S + k d, o = q S for each token in turn (gdn_step_kernel's step).
// Sequences of up to GDC_STEP_MOST tokens go token by token, longer ones in chunks of 64 (K = V = 128; other shapes go token by token whatever their length).
#pragma once

#include "attn_tc.cuh"
#include "common.cuh"
#include "kv.cuh"
#include "ops.cuh"
#include "seqs.cuh"

namespace b200 {

struct GdnSeqs {
    float *state;
    const float *q, *k, *v, *g, *beta;
    float *out;
    const int32_t *start, *slot;
    int n_seq, n_slots, n_tok, n_k_heads, n_v_heads, K, V;
};

// Where sequence s keeps its state: its slot, or s itself.  -1 (every thread of the CTA): the slot is not one of the pool's, or another sequence with new
// tokens names it too (one without them does nothing with its state: a captured call's spare sequences may name any slot).
__device__ __forceinline__ int gdn_slot_of(const GdnSeqs &P, int s) {
    const int mine = P.slot ? P.slot[s] : s;
    int bad = mine < 0 || mine >= P.n_slots;
    if (P.slot)
        for (int i = threadIdx.x; i < P.n_seq; i += blockDim.x) bad |= i != s && P.slot[i] == mine && seq_range(P.start, i, P.n_tok).n > 0;
    return __syncthreads_or(bad) ? -1 : mine;
}

// ---- token by token: the form for few tokens --------------------------------------------------------------------------------------------
// As gdn_step_kernel: one CTA per (sequence, value head, 32 PER columns of the state), eight warps, lane = PER columns, warp w holds rows w, w + 8, ... in registers over all of
// the sequence's tokens: the state is read once and written once.  Sequences of more than `most` tokens are not its own.
// Bound by memory for many sequences (16 of one token: 101 MB in 23 us; of 32 columns a CTA 28.7, where a state's tile is 16 KB), for few tokens of one by latency: 4.3 us for
// one token of 48 heads, about 1.0 for each one more (two sums over eight warps and three barriers).  gdn_step_kernel, which asks L2 for its state and inputs in front of the wait, takes 2.7.
template <int PER>
struct GdnCols { float x[PER]; };
template <int PER>
__device__ __forceinline__ GdnCols<PER> gdn_load_cols(const float *p) {
    GdnCols<PER> c;
    if constexpr (PER == 4) {
        const float4 v = *reinterpret_cast<const float4 *>(p);
        c.x[0] = v.x; c.x[1] = v.y; c.x[2] = v.z; c.x[3] = v.w;
    } else {
        c.x[0] = p[0];
    }
    return c;
}
template <int PER>
__device__ __forceinline__ void gdn_store_cols(float *p, const GdnCols<PER> &c) {
    if constexpr (PER == 4) *reinterpret_cast<float4 *>(p) = make_float4(c.x[0], c.x[1], c.x[2], c.x[3]);
    else p[0] = c.x[0];
}
template <int PER>
__global__ void __launch_bounds__(GDN_WARPS * 32) gdn_seqs_step_kernel(const __grid_constant__ GdnSeqs P, int most) {
    __shared__ float ks[2][GDN_KMAX], qs[2][GDN_KMAX];
    __shared__ __align__(16) float part[2][GDN_WARPS][32 * PER];
    using Cols = GdnCols<PER>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tiles = P.V / (32 * PER), s = blockIdx.y;
    const int vh = blockIdx.x / tiles, vt = blockIdx.x - vh * tiles;
    const int j = (vt * 32 + lane) * PER;
    const int kh = vh / (P.n_v_heads / P.n_k_heads);
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    // the state and the first token are asked for beside each other, before the slot is known to be the sequence's own
    const int mine = P.slot ? P.slot[s] : s;
    const SeqRange r = seq_range(P.start, s, P.n_tok);
    if (r.n <= 0 || r.n > most) {
        if (r.n < 0 && threadIdx.x == 0) bad_sequence();
        return;
    }
    const bool there = mine >= 0 && mine < P.n_slots;
    float *Sg = P.state + ((size_t)(there ? mine : 0) * P.n_v_heads + vh) * P.K * P.V + j;
    Cols col[GDN_RPW];
#pragma unroll
    for (int i = 0; i < GDN_RPW; ++i) {
        const int row = warp + GDN_WARPS * i;
        if (there && row < P.K) col[i] = gdn_load_cols<PER>(Sg + (size_t)row * P.V);
        else
#pragma unroll
            for (int c = 0; c < PER; ++c) col[i].x[c] = 0.0f;
    }
    // a token's scalars and this thread's values of k or q (K <= 128: threads 0 .. 127 have k, the others q)
    const int kq_at = threadIdx.x & (GDN_KMAX - 1);
    const float *kq_src = threadIdx.x < GDN_KMAX ? P.k : P.q;
    float b, gt, kq;
    Cols vj;
    auto fetch = [&](int t) {
        const size_t tok = (size_t)(r.begin + t);
        b = P.beta[tok * P.n_v_heads + vh];
        vj = gdn_load_cols<PER>(P.v + (tok * P.n_v_heads + vh) * P.V + j);
        gt = P.g[tok * P.n_v_heads + vh];
        kq = kq_at < P.K ? kq_src[(tok * P.n_k_heads + kh) * P.K + kq_at] : 0.0f;
    };
    // (sums over the warps' rows, in ascending order of the warps)
    auto joined = [&](const float (*p)[32 * PER]) {
        Cols sum = gdn_load_cols<PER>(&p[0][lane * PER]);
#pragma unroll
        for (int w = 1; w < GDN_WARPS; ++w) {
            const Cols x = gdn_load_cols<PER>(&p[w][lane * PER]);
#pragma unroll
            for (int c = 0; c < PER; ++c) sum.x[c] = __fadd_rn(sum.x[c], x.x[c]);
        }
        return sum;
    };
    fetch(0);
    if (gdn_slot_of(P, s) < 0) {
        if (threadIdx.x == 0) bad_sequence();
        return;
    }
    for (int t = 0; t < r.n; ++t) {
        const int b2 = t & 1;
        const size_t tok = (size_t)(r.begin + t);
        const float beta = b, decay = expf(gt);
        const Cols value = vj;
        (threadIdx.x < GDN_KMAX ? ks : qs)[b2][kq_at] = kq;
        if (t + 1 < r.n) fetch(t + 1);                      // the next token's are on their way
        __syncthreads();
        Cols kv, o;
#pragma unroll
        for (int c = 0; c < PER; ++c) kv.x[c] = o.x[c] = 0.0f;
#pragma unroll
        for (int i = 0; i < GDN_RPW; ++i) {
            const int row = warp + GDN_WARPS * i;
            if (row < P.K) {
                const float k = ks[b2][row];
#pragma unroll
                for (int c = 0; c < PER; ++c) {
                    col[i].x[c] = __fmul_rn(col[i].x[c], decay);
                    kv.x[c] = __fadd_rn(kv.x[c], __fmul_rn(k, col[i].x[c]));
                }
            }
        }
        gdn_store_cols<PER>(&part[0][warp][lane * PER], kv);
        __syncthreads();
        kv = joined(part[0]);
        Cols d;
#pragma unroll
        for (int c = 0; c < PER; ++c) d.x[c] = __fsub_rn(value.x[c], kv.x[c]);
#pragma unroll
        for (int i = 0; i < GDN_RPW; ++i) {
            const int row = warp + GDN_WARPS * i;
            if (row < P.K) {
                const float k = __fmul_rn(beta, ks[b2][row]), q = qs[b2][row];
#pragma unroll
                for (int c = 0; c < PER; ++c) {
                    col[i].x[c] = __fadd_rn(col[i].x[c], __fmul_rn(k, d.x[c]));
                    o.x[c] = __fadd_rn(o.x[c], __fmul_rn(q, col[i].x[c]));
                }
            }
        }
        gdn_store_cols<PER>(&part[1][warp][lane * PER], o);
        __syncthreads();
        if (warp == 0) gdn_store_cols<PER>(P.out + (tok * P.n_v_heads + vh) * P.V + j, joined(part[1]));
    }
#pragma unroll
    for (int i = 0; i < GDN_RPW; ++i) {
        const int row = warp + GDN_WARPS * i;
        if (row < P.K) gdn_store_cols<PER>(Sg + (size_t)row * P.V, col[i]);
    }
}

// ---- in chunks of 64 tokens: the form for many -----------------------------------------------------------------------------------------------
// With G_i the sum of g from the chunk's begin to token i, S the state in front of the chunk and u_i what token i adds along its key,
//   u_i = beta_i (v_i - e^G_i k_i S - sum over j < i of e^(G_i - G_j) (k_i . k_j) u_j)                U = Tb (V - e^G K S), Tb = (1 + A)^-1 diag(beta)
//   o_i = e^G_i q_i S + sum over j <= i of e^(G_i - G_j) (q_i . k_j) u_j                              O = e^G Q S + P U
//   S' = e^G_63 S + sum of k_j e^(G_63 - G_j) u_j                                                     S' = e^G_63 S + K^T (e^(G_63 - G) U)
// with A_ij = beta_i e^(G_i - G_j) (k_i . k_j), j < i.  gdn_planes_kernel and gdn_chunk_kernel form the planes of K and Q, and Tb and P, of every chunk at once; gdn_scan_kernel carries the state through
// the chunks of a sequence, a CTA per value head and 48 or 40 columns of it (the columns do not know of each other).
//
// Products are fp32 to about 2^-22: each operand is two fp16 planes, high and low, of its values times a power of two -- K, Q, Tb and P a row, S, V - e^G K S and U eight columns
// -- of which a plane pair holds 2^-38 of the largest; three of the four products on mma.sync (m16n8k16), sums fp32.  (Two TF32 parts, which need no powers of
// two, are four times the instructions for the same: the tensor core's 554 TFLOP/s of fp16 are 278 of TF32, and the parts were made anew by every warp.)
// What eight columns of V - e^G K S hold less than 2^-20 of the largest (a token behind one that was 2^20 times as large and is forgotten, a column beside one that is: planes have
// 18 bits left for it at most) would be lost to the state for good: such a chunk goes token by token, as one with values past 2^60 does.  It is looked for by pairs of neighbouring columns,
// which of ordinary values are both that small once in 10^12.
// The tensor core cuts the last bits of a sum off instead of rounding it, so a sum is of one step of 16 values, small products first, and rounded additions join the
// steps.  (One sum over all steps, the state's own among them: error of 2048 tokens' outputs against 64 bits 1.6e-6, now 2.3e-7.)
constexpr int GDC_T = 64, GDC_D = 128;
constexpr int GDC_PREP_THREADS = 128, GDC_THREADS = 256;
constexpr int GDC_COLS = 48, GDC_NT = GDC_COLS / 8, GDC_SLICES = 3;
// row strides in bytes of planes in shared memory: 16-byte pieces of eight rows lie in different banks
constexpr int GDC_KB = GDC_D * 2 + 16, GDC_TB = GDC_T * 2 + 16, GDC_CB = GDC_COLS * 2 + 16;
constexpr int GDC_KP = GDC_T * GDC_KB, GDC_TP = GDC_T * GDC_TB, GDC_SP = GDC_D * GDC_CB, GDC_UP = GDC_T * GDC_CB;        // a plane of K or Q, Tb or P, S, U
constexpr int GDC_VS = GDC_COLS + 8;                                  // floats: a row of V
constexpr int GDC_TS = GDC_T + 4;                                     // floats: a row of A and of its inverse
constexpr int GDC_STEP_MOST = 24;                                     // tokens of a sequence that go one by one (us, one by one / in chunks: 16 19 / 28, 24 25 / 28, 48 45 / 28.6)
// What the first two kernels leave, in bytes, planes with the row strides of shared memory so that one bulk copy fetches them: of a chunk and key head the planes of K and Q and
// the exponents s of their rows' powers of two; of a chunk and value head the planes of Tb and P, then floats: per row e^G 2^-s of K, e^G 2^-s of Q, e^(G_63 - G) 2^(s_min - s) of K,
// 2^-s of Tb, 2^-s of P; then e^G_63, 2^-s_min, whether the chunk is to go token by token.
constexpr int GDC_KQ_REC = 4 * GDC_KP + 2 * GDC_T * 4, GDC_TP_PLANES = 4 * GDC_TP, GDC_VEC = 5 * GDC_T + 4, GDC_TP_REC = GDC_TP_PLANES + GDC_VEC * 4;
constexpr int GDC_QB = 16 * GDC_KB;                                    // 16 rows of a plane of Q
constexpr uint32_t GDC_FAR = 20;                                       // (powers of two)
constexpr int gdc_prep_smem() { return 2 * GDC_KP + 4 * GDC_QB + GDC_T * 8 + 3 * GDC_T * 4 + 32; }
constexpr int gdc_scan_smem() { return 6 * GDC_KP + 4 * GDC_TP + GDC_T * GDC_VS * 4 + 2 * GDC_SP + 6 * GDC_UP + GDC_VEC * 4 + 5 * 8 * 4 + 4 * 8; }
static_assert(gdc_scan_smem() <= 227 * 1024 && 4 * gdc_prep_smem() <= 224 * 1024 && GDC_D * GDC_CB * 2 >= GDC_D * GDC_COLS * 4 && 2 * GDC_T * GDC_TS * 4 <= 2 * GDC_KP, "");

__device__ __forceinline__ int gdc_chunks(int n) { return n > GDC_STEP_MOST ? (n + GDC_T - 1) / GDC_T : 0; }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm2_t(uint32_t (&r)[4], uint32_t addr) {       // (into the first two)
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
}
// The products have no other effect than their sums, so that the compiler may put them where it likes.
__device__ __forceinline__ void gdc_mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void gdc_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// c[m] = A[m] B over 16 STEPS values, each A 16 rows, B 8 NT columns.  a[m], b: the lane's addresses of the high planes, the low ones a_low and b_low behind, a step a_step and
// b_step behind the one before; of a pair of column tiles b_pair.  AT: A lies by columns; BT: B lies by rows.
template <int MT, int NT, int STEPS, bool AT, bool BT>
__device__ __forceinline__ void gdc_product(float (&c)[MT][NT][4], const uint32_t (&a)[MT], uint32_t a_low, uint32_t a_step, uint32_t b, uint32_t b_low, uint32_t b_step, uint32_t b_pair,
                                            int steps = STEPS) {
    constexpr int PAIRS = (NT + 1) / 2;
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
        if (k >= steps) break;
        uint32_t ah[MT][4], al[MT][4], bh[PAIRS][4], bl[PAIRS][4];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            if (AT) ldsm4_t(ah[m], a[m] + k * a_step), ldsm4_t(al[m], a[m] + k * a_step + a_low);
            else ldsm4(ah[m], a[m] + k * a_step), ldsm4(al[m], a[m] + k * a_step + a_low);
        }
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) {
            const uint32_t at = b + k * b_step + j * b_pair;
            if (2 * j + 1 == NT) ldsm2_t(bh[j], at), ldsm2_t(bl[j], at + b_low);
            else if (BT) ldsm4_t(bh[j], at), ldsm4_t(bl[j], at + b_low);
            else ldsm4(bh[j], at), ldsm4(bl[j], at + b_low);
        }
        float sum[MT][NT][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j) gdc_mma_first(sum[m][j], al[m], bh[j >> 1][2 * (j & 1)], bh[j >> 1][2 * (j & 1) + 1]);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j) gdc_mma(sum[m][j], ah[m], bl[j >> 1][2 * (j & 1)], bl[j >> 1][2 * (j & 1) + 1]);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j) gdc_mma(sum[m][j], ah[m], bh[j >> 1][2 * (j & 1)], bh[j >> 1][2 * (j & 1) + 1]);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) c[m][j][e] = k == 0 ? sum[m][j][e] : __fadd_rn(c[m][j][e], sum[m][j][e]);
    }
}
// Lane's place in a matrix of rows of `stride` bytes: (rows, values) of A by rows; of B by rows (k) and of A by columns; of B by columns (n).
__device__ __forceinline__ uint32_t gdc_at_rows(int lane, int stride) { return (lane & 15) * stride + (lane >> 4) * 16; }
__device__ __forceinline__ uint32_t gdc_at_turned(int lane, int stride) { return ((lane & 7) + 8 * (lane >> 4)) * stride + ((lane >> 3) & 1) * 16; }

// grid (chunks of all sequences and some that find none, key heads): planes of K and Q, a warp per row, lane = four values.
__global__ void __launch_bounds__(GDC_THREADS) gdn_planes_kernel(const __grid_constant__ GdnSeqs P, uint8_t *kq_recs) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kh = blockIdx.y;
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    int seq, chunk;
    if (!seq_of_item(P.start, P.n_seq, P.n_tok, (int)blockIdx.x, lane, [](int n) { return gdc_chunks(n); }, seq, chunk)) return;
    const SeqRange range = seq_range(P.start, seq, P.n_tok);
    const int n = min(GDC_T, range.n - chunk * GDC_T);
    const size_t tok = (size_t)range.begin + chunk * GDC_T;
    uint8_t *rec = kq_recs + ((size_t)blockIdx.x * P.n_k_heads + kh) * GDC_KQ_REC;
    const bool vec = ((reinterpret_cast<uintptr_t>(P.k) | reinterpret_cast<uintptr_t>(P.q)) & 15u) == 0;
    constexpr int ROWS = 2 * GDC_T / (GDC_THREADS / 32);
    float4 x[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = ROWS * warp + i, row = r & (GDC_T - 1);
        const float *src = (r < GDC_T ? P.k : P.q) + ((tok + row) * P.n_k_heads + kh) * GDC_D + 4 * lane;
        x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row < n) x[i] = vec ? *reinterpret_cast<const float4 *>(src) : make_float4(src[0], src[1], src[2], src[3]);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = ROWS * warp + i, row = r & (GDC_T - 1);
        const uint32_t m = __reduce_max_sync(0xffffffffu, max(max(atc_abs_bits(x[i].x), atc_abs_bits(x[i].y)), max(atc_abs_bits(x[i].z), atc_abs_bits(x[i].w))));
        const int s = atc_shift(m, 63);
        const float f = atc_pow2(s);
        uint2 hi, lo;
        split_f16x2(__fmul_rn(x[i].x, f), __fmul_rn(x[i].y, f), hi.x, lo.x);
        split_f16x2(__fmul_rn(x[i].z, f), __fmul_rn(x[i].w, f), hi.y, lo.y);
        uint8_t *out = rec + (r < GDC_T ? 0 : 2 * GDC_KP) + row * GDC_KB + 8 * lane;
        *reinterpret_cast<uint2 *>(out) = hi;
        *reinterpret_cast<uint2 *>(out + GDC_KP) = lo;
        if (lane == 0) reinterpret_cast<int *>(rec + 4 * GDC_KP)[r] = s;
    }
}

// grid (the same chunks, value heads): Tb and P.  Bound by issue and latency: 59 us for 2048 tokens and 48 heads, four CTAs per SM (128 registers, 48 bytes spilled a thread), whose rounds are three (with all of Q in
// shared memory and P passing through it, three CTAs, four rounds, 75 us).  About 3900 instructions a warp, half of them the inverse.
__global__ void __launch_bounds__(GDC_PREP_THREADS, 4) gdn_chunk_kernel(const __grid_constant__ GdnSeqs P, const uint8_t *kq_recs, uint8_t *tp_recs) {
    extern __shared__ __align__(16) uint8_t gdc_smem[];
    uint8_t *kp = gdc_smem, *qp = kp + 2 * GDC_KP;                           // Q: 16 rows of both planes of each of two warps
    float *at = reinterpret_cast<float *>(kp), *tt = at + GDC_T * GDC_TS;    // when the planes of K have been read
    double *gs = reinterpret_cast<double *>(qp + 4 * GDC_QB);
    float *bs = reinterpret_cast<float *>(gs + GDC_T);
    int *shift = reinterpret_cast<int *>(bs + GDC_T);                        // [2][64] of K, of Q
    uint64_t *full = reinterpret_cast<uint64_t *>(shift + 2 * GDC_T);       // K and its Q; the other 16 rows of Q of each of the two warps
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    constexpr int WARPS = GDC_PREP_THREADS / 32;
    const int vh = blockIdx.y, share = P.n_v_heads / P.n_k_heads, kh = vh / share;
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    int seq, chunk;
    if (!seq_of_item(P.start, P.n_seq, P.n_tok, (int)blockIdx.x, lane, [](int n) { return gdc_chunks(n); }, seq, chunk)) return;
    const SeqRange range = seq_range(P.start, seq, P.n_tok);
    const int n = min(GDC_T, range.n - chunk * GDC_T);
    const size_t tok = (size_t)range.begin + chunk * GDC_T;
    const uint8_t *kq = kq_recs + ((size_t)blockIdx.x * P.n_k_heads + kh) * GDC_KQ_REC;
    uint8_t *rec = tp_recs + ((size_t)blockIdx.x * P.n_v_heads + vh) * GDC_TP_REC;
    float *vec = reinterpret_cast<float *>(rec + GDC_TP_PLANES);
    bool odd = false;                           // something that sums may not hold: the chunk goes token by token
    const uint64_t pol = policy_evict_normal();
    const bool of_q = warp >= 2;
    const int top = warp & 1;
    auto load_q = [&](int w, int m, uint64_t *bar) {
        for (int p = 0; p < 2; ++p) bulk_g2s(qp + (2 * w + p) * GDC_QB, kq + (2 + p) * GDC_KP + m * GDC_QB, GDC_QB, bar, pol);
    };
    if (tid == 0) {
        for (int b = 0; b < 3; ++b) mbar_init(full + b, 1);
        mbar_fence_init();
        mbar_expect_tx(full, 2 * GDC_KP + 2 * GDC_T * 4 + 4 * GDC_QB);
        bulk_g2s(kp, kq, 2 * GDC_KP, full, pol);
        bulk_g2s(shift, kq + 4 * GDC_KP, 2 * GDC_T * 4, full, pol);
        load_q(0, 0, full);
        load_q(1, 1, full);
    }
    if (warp == 0) {
        // a decay below e^-1000 is none; sums in 64 bits: of two that are far from zero the difference matters
        double x[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = 2 * lane + h;
            const float gi = i < n ? P.g[(tok + i) * P.n_v_heads + vh] : 0.0f, bi = i < n ? P.beta[(tok + i) * P.n_v_heads + vh] : 0.0f;
            odd = odd || !(gi < 1e30f) || !(fabsf(bi) < 1e30f);
            x[h] = (double)fmaxf(gi, -1000.0f);
            bs[i] = bi;
        }
        x[1] += x[0];
        double sum = x[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += y;
        }
        gs[2 * lane] = sum - x[1] + x[0];
        gs[2 * lane + 1] = sum;
    }
    __syncthreads();
    if (!__syncthreads_and(mbar_wait_hot(full, 0) ? 1 : 0)) return;          // (a wait ran out: the CTA leaves as a whole)
    // ---- K K^T (two warps) and Q K^T, blocks of 16 x 16 on and below the diagonal: a warp has rows of blocks w and 3 - w, five blocks
    float c[5][1][2][4];
    bool ok = true;
    {
        const uint32_t a_k = smem_u32(kp) + gdc_at_rows(lane, GDC_KB), a_q = smem_u32(qp) + 2 * top * GDC_QB + gdc_at_rows(lane, GDC_KB), b0 = smem_u32(kp) + gdc_at_turned(lane, GDC_KB);
#pragma unroll
        for (int i = 0; i < 5; ++i) {
            const int m = i <= top ? top : 3 - top, j = i <= top ? i : i - top - 1;
            if (of_q && i == top + 1) {                                     // the rows of Q of the second row of blocks, in the place of the first's
                __syncwarp();
                if (lane == 0) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    mbar_expect_tx(full + 1 + top, 2 * GDC_QB);
                    load_q(top, m, full + 1 + top);
                }
                ok = mbar_wait_hot(full + 1 + top, 0);
            }
            const uint32_t a[1] = {of_q ? a_q : a_k + 16 * m * GDC_KB};
            gdc_product<1, 2, GDC_D / 16, false, false>(c[i], a, of_q ? GDC_QB : GDC_KP, 32, b0 + 16 * j * GDC_KB, GDC_KP, 32, 0);
        }
    }
    if (!__syncthreads_and(ok ? 1 : 0)) return; // the planes have been read: A and its inverse in fp32 take the place of K's
    if (tid < GDC_T) odd = odd || min(shift[tid], shift[GDC_T + tid]) <= 141 - (int)(ATC_HUGE >> 23);
#pragma unroll
    for (int i = 0; i < 5; ++i) {
        const int m = i <= top ? top : 3 - top, jb = i <= top ? i : i - top - 1;
        double gr[2], gc[4];                    // of the lane's two rows and four columns: sums of g, factors
        float fr[2], fc[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = 16 * m + g + 8 * h;
            gr[h] = gs[row];
            fr[h] = atc_pow2(-shift[(of_q ? GDC_T : 0) + row]);
            if (!of_q) fr[h] = __fmul_rn(fr[h], bs[row]);
            if (row >= n) fr[h] = 0.0f;
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const int col = 16 * jb + 8 * (h >> 1) + 2 * t + (h & 1);
            gc[h] = gs[col];
            fc[h] = atc_pow2(-shift[col]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int h = (e >> 1) & 1, v = 2 * (e >> 2) + (e & 1), row = 16 * m + g + 8 * h, col = 16 * jb + 8 * (e >> 2) + 2 * t + (e & 1);
            float x = __fmul_rn(__fmul_rn(__fmul_rn(c[i][0][e >> 2][e & 3], fr[h]), fc[v]), expf((float)(gr[h] - gc[v])));
            if (col > row || (!of_q && col == row)) x = 0.0f;
            odd = odd || !(fabsf(x) < 1e30f);
            if (of_q) c[i][0][e >> 2][e & 3] = x;
            else at[row * GDC_TS + col] = x;
        }
    }
    if (of_q) {
        // planes of P: a row lies in four lanes.  (Blocks above the diagonal are not read.)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int m = half ? 3 - top : top;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t most = 0u;
#pragma unroll
                for (int i = 0; i < 5; ++i)
                    if ((i > top) == (half != 0))
#pragma unroll
                        for (int v = 0; v < 4; ++v) most = max(most, atc_abs_bits(c[i][0][v >> 1][2 * h + (v & 1)]));
                most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
                odd = odd || most >= ATC_HUGE;
                const int s = atc_shift(most, 63), row = 16 * m + g + 8 * h;
                const float f = atc_pow2(s);
                uint8_t *out = rec + 2 * GDC_TP + row * GDC_TB + 4 * t;
#pragma unroll
                for (int i = 0; i < 5; ++i)
                    if ((i > top) == (half != 0)) {
                        const int jb = i <= top ? i : i - top - 1;
#pragma unroll
                        for (int v = 0; v < 2; ++v) {
                            uint32_t hi, lo;
                            split_f16x2(__fmul_rn(c[i][0][v][2 * h], f), __fmul_rn(c[i][0][v][2 * h + 1], f), hi, lo);
                            *reinterpret_cast<uint32_t *>(out + 32 * jb + 16 * v) = hi;
                            *reinterpret_cast<uint32_t *>(out + 32 * jb + 16 * v + GDC_TP) = lo;
                        }
                    }
                if (t == 0) vec[4 * GDC_T + row] = atc_pow2(-s);
            }
        }
    }
    __syncthreads();
    // ---- (1 + A)^-1: the four 16 x 16 blocks on the diagonal, a warp each, lane = column, from the top row down ...
    if (lane < 16) {
        const int blk = 16 * warp;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float s = i == lane ? 1.0f : 0.0f;
#pragma unroll
            for (int j = 0; j < i; j += 4) {
                const float4 a = *reinterpret_cast<const float4 *>(at + (blk + i) * GDC_TS + blk + j);
                s = __fmaf_rn(-a.x, x[j], s);
                if (j + 1 < i) s = __fmaf_rn(-a.y, x[j + 1], s);
                if (j + 2 < i) s = __fmaf_rn(-a.z, x[j + 2], s);
                if (j + 3 < i) s = __fmaf_rn(-a.w, x[j + 3], s);
            }
            x[i] = s;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) tt[(blk + i) * GDC_TS + blk + lane] = x[i];
    }
    __syncthreads();
    // ... and below it, a row of blocks after the other: T_ij = -T_ii (sum of A_ik T_kj, j <= k < i).  A thread has eight rows of one column.
    for (int i = 1; i < 4; ++i) {
        const int r0 = 16 * i + 8 * (tid & 1), col = tid >> 1;          // 64 columns, of which 16 i have work
        float s[8] = {};
        if (col < 16 * i) {
            for (int k = col & ~15; k < 16 * i; k += 4) {
                const float x0 = tt[k * GDC_TS + col], x1 = tt[(k + 1) * GDC_TS + col], x2 = tt[(k + 2) * GDC_TS + col], x3 = tt[(k + 3) * GDC_TS + col];
#pragma unroll
                for (int h = 0; h < 8; ++h) {
                    const float4 a = *reinterpret_cast<const float4 *>(at + (r0 + h) * GDC_TS + k);
                    s[h] = __fmaf_rn(a.w, x3, __fmaf_rn(a.z, x2, __fmaf_rn(a.y, x1, __fmaf_rn(a.x, x0, s[h]))));
                }
            }
        }
        __syncthreads();
        if (col < 16 * i)
#pragma unroll
            for (int h = 0; h < 8; ++h) at[(r0 + h) * GDC_TS + col] = s[h];          // A's row of blocks has been read
        __syncthreads();
        if (col < 16 * i) {
#pragma unroll
            for (int h = 0; h < 8; ++h) s[h] = 0.0f;
#pragma unroll
            for (int k = 0; k < 16; k += 4) {
                const float *y = at + (16 * i + k) * GDC_TS + col;
                const float x0 = y[0], x1 = y[GDC_TS], x2 = y[2 * GDC_TS], x3 = y[3 * GDC_TS];
#pragma unroll
                for (int h = 0; h < 8; ++h) {
                    const float4 a = *reinterpret_cast<const float4 *>(tt + (r0 + h) * GDC_TS + 16 * i + k);
                    s[h] = __fmaf_rn(a.w, x3, __fmaf_rn(a.z, x2, __fmaf_rn(a.y, x1, __fmaf_rn(a.x, x0, s[h]))));
                }
            }
#pragma unroll
            for (int h = 0; h < 8; ++h) tt[(r0 + h) * GDC_TS + col] = -s[h];
        }
        __syncthreads();
    }
    // ---- planes of Tb: a warp per row, lane = two values
#pragma unroll 4
    for (int row = warp; row < GDC_T; row += WARPS) {
        const int col = 2 * lane;
        float2 x = make_float2(0.0f, 0.0f);
        if ((col >> 4) <= (row >> 4)) {
            x = *reinterpret_cast<const float2 *>(tt + row * GDC_TS + col);
            x = make_float2(__fmul_rn(x.x, bs[col]), __fmul_rn(x.y, bs[col + 1]));
        }
        const uint32_t m = __reduce_max_sync(0xffffffffu, max(atc_abs_bits(x.x), atc_abs_bits(x.y)));
        odd = odd || m >= ATC_HUGE;
        const int s = atc_shift(m, 63);
        const float f = atc_pow2(s);
        uint32_t hi, lo;
        split_f16x2(__fmul_rn(x.x, f), __fmul_rn(x.y, f), hi, lo);
        uint8_t *out = rec + row * GDC_TB + 4 * lane;
        *reinterpret_cast<uint32_t *>(out) = hi;
        *reinterpret_cast<uint32_t *>(out + GDC_TP) = lo;
        if (lane == 0) vec[3 * GDC_T + row] = atc_pow2(-s);
    }
    int least = 63;                             // K's smallest shift
#pragma unroll
    for (int h = 0; h < 2; ++h) least = min(least, shift[lane + 32 * h]);
    least = __reduce_min_sync(0xffffffffu, least);
    if (tid < GDC_T) {
        const float eg = expf((float)gs[tid]);
        vec[tid] = __fmul_rn(eg, atc_pow2(-shift[tid]));
        vec[GDC_T + tid] = __fmul_rn(eg, atc_pow2(-shift[GDC_T + tid]));
        const float left = __fmul_rn(expf((float)(gs[GDC_T - 1] - gs[tid])), atc_pow2(max(least - shift[tid], -126)));
        vec[2 * GDC_T + tid] = left;
        odd = odd || left >= 0x1p60f;
    }
    if (tid == 0) {
        vec[5 * GDC_T] = expf((float)gs[GDC_T - 1]);
        vec[5 * GDC_T + 1] = atc_pow2(-least);
    }
    const int any = __syncthreads_or(odd ? 1 : 0);
    if (tid == 0) vec[5 * GDC_T + 2] = any ? 1.0f : 0.0f;
}

// A chunk is a chain: K S | V - e^G K S scaled | U, and Q S beside it | U scaled | K^T U and P U | S scaled, with a barrier between any two, on eight warps: about 10 800 cycles, of which
// the tensor core's products are 4200; shared memory's pipe is half busy.  What was worth it, in us of the scan over 2048 tokens: products by fp16 planes instead of TF32 parts
// (389 -> 317), powers of two by eight columns instead of one and bulk copies (-> 249), tokens' rows and half of the columns to a warp (-> 216), no blocks above the
// diagonals and rows of V in different banks (-> 209), Q S behind U (-> 204).  What was not: eight more warps for Q S, P U and V's copies beside the chain (they share its pipes: 216 -> 225), the
// next chunk's Tb ahead of time, with a barrier less (204 -> 209).  Three slices of the columns put 144 CTAs on 148 SMs; two would leave a third of them idle, four make the
// fuller SMs do two.
// grid (value heads x 3, sequences): columns 0 .. 47, 48 .. 87, 88 .. 127.  Warp w of eight: 16 of the tokens and half of the columns of all that has a row for each
// token, and rows 16 w .. of the state, which stay in registers in fp32; its planes in shared memory are what the products read.
__global__ void __launch_bounds__(GDC_THREADS, 1) gdn_scan_kernel(const __grid_constant__ GdnSeqs P, const uint8_t *kq_recs, const uint8_t *tp_recs, int n_chunks) {
    extern __shared__ __align__(16) uint8_t gdc_smem[];
    uint8_t *kp0 = gdc_smem, *qp = kp0 + 4 * GDC_KP, *tp = qp + 2 * GDC_KP, *sp = tp + 4 * GDC_TP, *up = sp + 2 * GDC_SP, *rp = up + 4 * GDC_UP;       // K twice; Q; Tb, P; S; U, U times its factors; V - e^G K S
    float *vt = reinterpret_cast<float *>(rp + 2 * GDC_UP), *vec = vt + GDC_T * GDC_VS;
    uint32_t *s_most = reinterpret_cast<uint32_t *>(vec + GDC_VEC), *r_most = s_most + 2 * 8, *u_most = r_most + 8;          // largest magnitudes of eight columns: S's of this chunk and of the next; U's, U's times its factors
    uint64_t *kfull = reinterpret_cast<uint64_t *>(u_most + 2 * 8), *qvfull = kfull + 2, *tpfull = kfull + 3;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int vh = blockIdx.x / GDC_SLICES, slice = blockIdx.x % GDC_SLICES, s = blockIdx.y;
    const int c0 = slice == 0 ? 0 : 48 + 40 * (slice - 1), cols = slice == 0 ? 48 : 40;
    const int kh = vh / (P.n_v_heads / P.n_k_heads), mt = warp < 4 ? warp : 7 - warp;           // (a scheduler's two warps: as many steps of Tb and P as any other's)
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    const SeqRange range = seq_range(P.start, s, P.n_tok);
    const int nchunk = range.n > 0 ? gdc_chunks(range.n) : 0;
    if (nchunk == 0) return;
    const int slot = gdn_slot_of(P, s);
    if (slot < 0) {
        if (tid == 0) bad_sequence();
        return;
    }
    // the chunks of the sequences in front
    int first = 0;
    for (int i = lane; i < s; i += 32) first += gdc_chunks(max(0, seq_range(P.start, i, P.n_tok).n));
    first = __reduce_add_sync(0xffffffffu, first);
    if (first > n_chunks - nchunk) {                            // (rows that several sequences claim: there are not as many records)
        if (tid == 0) bad_sequence();
        return;
    }
    const uint8_t *kq = kq_recs + ((size_t)first * P.n_k_heads + kh) * GDC_KQ_REC, *rec = tp_recs + ((size_t)first * P.n_v_heads + vh) * GDC_TP_REC;
    const size_t kq_stride = (size_t)P.n_k_heads * GDC_KQ_REC, rec_stride = (size_t)P.n_v_heads * GDC_TP_REC;
    const size_t vstride = (size_t)P.n_v_heads * GDC_D;
    const bool vvec = (reinterpret_cast<uintptr_t>(P.v) & 15u) == 0;

    // what a chunk brings, as room for it becomes free: bulk copies by one thread, V's rows by a warp
    const uint64_t pol = policy_evict_normal();
    auto load_k = [&](int c) {
        mbar_expect_tx(kfull + (c & 1), 2 * GDC_KP);
        bulk_g2s(kp0 + (c & 1) * 2 * GDC_KP, kq + c * kq_stride, 2 * GDC_KP, kfull + (c & 1), pol);
    };
    auto load_tp = [&](int c) {
        mbar_expect_tx(tpfull, GDC_TP_REC);
        bulk_g2s(tp, rec + c * rec_stride, GDC_TP_PLANES, tpfull, pol);
        bulk_g2s(vec, rec + c * rec_stride + GDC_TP_PLANES, GDC_VEC * 4, tpfull, pol);
    };
    int v_row[3], v_col[3];                                     // a thread's three pieces of four values
#pragma unroll
    for (int e = 0; e < 3; ++e) v_row[e] = (tid + e * GDC_THREADS) / (GDC_COLS / 4), v_col[e] = 4 * ((tid + e * GDC_THREADS) % (GDC_COLS / 4));
    auto load_qv = [&](int c) {                                 // the whole CTA (V by sixteen bytes each: 64 bulk copies of a row took a warp 3600 cycles)
        const float *src = P.v + (((size_t)range.begin + c * GDC_T) * P.n_v_heads + vh) * GDC_D + c0;
        const int n = min(GDC_T, range.n - c * GDC_T);
        if (tid == 0) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_expect_tx(qvfull, 2 * GDC_KP);
            bulk_g2s(qp, kq + c * kq_stride + 2 * GDC_KP, 2 * GDC_KP, qvfull, pol);
        }
#pragma unroll
        for (int e = 0; e < 3; ++e) {
            float *dst = vt + v_row[e] * GDC_VS + v_col[e];
            const float *x = src + (size_t)v_row[e] * vstride + v_col[e];
            if (v_row[e] >= n || v_col[e] >= cols) *reinterpret_cast<float4 *>(dst) = make_float4(0.f, 0.f, 0.f, 0.f);
            else if (vvec) cp_async16(dst, x);
            else *reinterpret_cast<float4 *>(dst) = make_float4(x[0], x[1], x[2], x[3]);
        }
        cp_async_commit();
    };
    if (tid == 0) {
        for (int b = 0; b < 4; ++b) mbar_init(kfull + b, 1);
        mbar_fence_init();
    }
    if (tid < 5 * 8) s_most[tid] = 0u;
    __syncthreads();
    if (tid == 0) load_k(0);
    load_qv(0);
    float *Sg = P.state + ((size_t)slot * P.n_v_heads + vh) * GDC_D * GDC_D + c0;
    float S[GDC_NT][4];                                         // rows 16 warp + g, + 8; columns 8 nt + 2 t, + 1
#pragma unroll
    for (int j = 0; j < GDC_NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) S[j][e] = 8 * j < cols ? Sg[(size_t)(16 * warp + g + 8 * (e >> 1)) * GDC_D + 8 * j + 2 * t + (e & 1)] : 0.0f;
    // the largest magnitude of each eight columns of a warp's 16 rows, into dst
    auto tiles_most = [&](auto &x, uint32_t *dst) {
        constexpr int N = sizeof(x) / sizeof(x[0]);
        uint32_t mine = 0u;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t m = __reduce_max_sync(0xffffffffu, max(max(atc_abs_bits(x[j][0]), atc_abs_bits(x[j][1])), max(atc_abs_bits(x[j][2]), atc_abs_bits(x[j][3]))));
            if (lane == j) mine = m;
        }
        if (lane < N) atomicMax(dst + lane, mine);
    };
    // planes of two values of a row, times f
    auto store_planes = [&](uint8_t *at, int low, float x, float y, float f) {
        uint32_t hi, lo;
        split_f16x2(__fmul_rn(x, f), __fmul_rn(y, f), hi, lo);
        *reinterpret_cast<uint32_t *>(at) = hi;
        *reinterpret_cast<uint32_t *>(at + low) = lo;
    };
    auto store_s = [&](const uint32_t *most) {
#pragma unroll
        for (int j = 0; j < GDC_NT; ++j) {
            const float f = atc_pow2(atc_shift(most[j], 63));
#pragma unroll
            for (int h = 0; h < 2; ++h) store_planes(sp + (16 * warp + g + 8 * h) * GDC_CB + 16 * j + 4 * t, GDC_SP, S[j][2 * h], S[j][2 * h + 1], f);
        }
    };
    tiles_most(S, s_most);
    __syncthreads();
    store_s(s_most);
    constexpr int NH = GDC_NT / 2;                              // column tiles of a warp that has tokens' rows, from j0 on
    const int j0 = NH * (warp >> 2);
    const uint32_t at_k = gdc_at_rows(lane, GDC_KB), at_t = gdc_at_rows(lane, GDC_TB), at_kt = gdc_at_turned(lane, GDC_KB);
    const uint32_t b_s = smem_u32(sp) + gdc_at_rows(lane, GDC_CB), b_r = smem_u32(rp) + gdc_at_rows(lane, GDC_CB), b_u = smem_u32(up) + gdc_at_rows(lane, GDC_CB);
    bool ok = true;
    for (int c = 0; c < nchunk; ++c) {
        const int n = min(GDC_T, range.n - c * GDC_T);
        const size_t tok = (size_t)range.begin + c * GDC_T;
        const uint32_t kb = smem_u32(kp0) + (c & 1) * 2 * GDC_KP;
        uint32_t *most = s_most + (c & 1) * 8, *next = s_most + ((c & 1) ^ 1) * 8;
        ok = mbar_wait_hot(kfull + (c & 1), (uint32_t)((c >> 1) & 1)) && ok;
        ok = mbar_wait_hot(qvfull, (uint32_t)(c & 1)) && ok;
        cp_async_wait<0>();
        if (!__syncthreads_and(ok ? 1 : 0)) return;             // the chunk's K, Q and V, and the planes of the state (a wait ran out: the CTA leaves as a whole)
        if (tid == 0) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            load_tp(c);
        }
        if (tid == 32 && c + 1 < nchunk) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            load_k(c + 1);
        }
        if (tid < 8) r_most[tid] = u_most[tid] = u_most[tid + 8] = next[tid] = 0u;
        // ---- V - e^G K S
        float r[1][NH][4], y[1][NH][4];
        {
            const uint32_t a[1] = {kb + 16 * mt * GDC_KB + at_k};
            gdc_product<1, NH, GDC_D / 16, false, true>(r, a, GDC_KP, 32, b_s + 16 * j0, GDC_SP, 16 * GDC_CB, 32);
        }
        ok = mbar_wait_hot(tpfull, (uint32_t)(c & 1)) && ok;
        if (!__syncthreads_and(ok ? 1 : 0)) return;             // Tb, P and the factors
        bool odd = vec[5 * GDC_T + 2] != 0.0f;
#pragma unroll
        for (int j = 0; j < NH; ++j) {
            const float fs = atc_pow2(-atc_shift(most[j0 + j], 63));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = 16 * mt + g + 8 * h;
                const float fk = vec[i];
                const float2 v = *reinterpret_cast<const float2 *>(vt + i * GDC_VS + 8 * (j0 + j) + 2 * t);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float &x = r[0][j][2 * h + e];
                    x = __fsub_rn(e ? v.y : v.x, __fmul_rn(__fmul_rn(x, fs), fk));
                    odd = odd || !(fabsf(x) < 0x1p60f);
                }
            }
        }
        tiles_most(r[0], r_most + j0);
        int slow = __syncthreads_or(odd ? 1 : 0);
        bool far = false;                                       // values that the largest of their eight columns leaves fewer than 18 bits
#pragma unroll
        for (int j = 0; j < NH; ++j) {
            const uint32_t largest = r_most[j0 + j];
            const float f = atc_pow2(atc_shift(largest, 63));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t own = max(atc_abs_bits(r[0][j][2 * h]), atc_abs_bits(r[0][j][2 * h + 1]));
                far = far || (own != 0u && own + (GDC_FAR << 23) < largest);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) store_planes(rp + (16 * mt + g + 8 * h) * GDC_CB + 16 * (j0 + j) + 4 * t, GDC_UP, r[0][j][2 * h], r[0][j][2 * h + 1], f);
        }
        __syncthreads();
        // ---- U = Tb (V - e^G K S); x: the same times the factors of the state's update
        {
            float u[1][NH][4], x[NH][4];
            const uint32_t a[1] = {smem_u32(tp) + 16 * mt * GDC_TB + at_t};
            gdc_product<1, NH, GDC_T / 16, false, true>(u, a, GDC_TP, 32, b_r + 16 * j0, GDC_UP, 16 * GDC_CB, 32, mt + 1);
            odd = far;
            // e^G Q S here, between products that the whole chunk waits for: its instructions fill their latencies (2048 tokens: beside K S 277 us, here 272, each without the look for values far apart, 3 us)
            const uint32_t aq[1] = {smem_u32(qp) + 16 * mt * GDC_KB + at_k};
            gdc_product<1, NH, GDC_D / 16, false, true>(y, aq, GDC_KP, 32, b_s + 16 * j0, GDC_SP, 16 * GDC_CB, 32);
#pragma unroll
            for (int j = 0; j < NH; ++j) {
                const float fs = atc_pow2(-atc_shift(most[j0 + j], 63));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    y[0][j][e] = __fmul_rn(__fmul_rn(y[0][j][e], fs), vec[GDC_T + 16 * mt + g + 8 * (e >> 1)]);
                    odd = odd || !(fabsf(y[0][j][e]) < 0x1p60f);
                }
            }
#pragma unroll
            for (int j = 0; j < NH; ++j) {
                const float fr = atc_pow2(-atc_shift(r_most[j0 + j], 63));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 16 * mt + g + 8 * (e >> 1);
                    u[0][j][e] = __fmul_rn(__fmul_rn(u[0][j][e], fr), vec[3 * GDC_T + i]);
                    x[j][e] = __fmul_rn(u[0][j][e], vec[2 * GDC_T + i]);
                    odd = odd || !(fabsf(u[0][j][e]) < 0x1p60f) || !(fabsf(x[j][e]) < 0x1p60f);
                }
            }
            tiles_most(u[0], u_most + j0);
            tiles_most(x, u_most + 8 + j0);
            slow |= __syncthreads_or(odd ? 1 : 0);              // (Q and V - e^G K S have been read)
#pragma unroll
            for (int j = 0; j < NH; ++j) {
                const float fu = atc_pow2(atc_shift(u_most[j0 + j], 63)), fx = atc_pow2(atc_shift(u_most[8 + j0 + j], 63));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint8_t *dst = up + (16 * mt + g + 8 * h) * GDC_CB + 16 * (j0 + j) + 4 * t;
                    store_planes(dst, GDC_UP, u[0][j][2 * h], u[0][j][2 * h + 1], fu);
                    store_planes(dst + 2 * GDC_UP, GDC_UP, x[j][2 * h], x[j][2 * h + 1], fx);
                }
            }
        }
        __syncthreads();
        if (!slow) {
            if (c + 1 < nchunk) load_qv(c + 1);
            // ---- S = e^G_63 S + K^T (e^(G_63 - G) U), O = e^G Q S + P U
            float o[1][NH][4];
            {
                float d[1][GDC_NT][4];
                const uint32_t a[1] = {kb + 32 * warp + at_kt}, ap[1] = {smem_u32(tp) + 2 * GDC_TP + 16 * mt * GDC_TB + at_t};
                gdc_product<1, GDC_NT, GDC_T / 16, true, true>(d, a, GDC_KP, 16 * GDC_KB, b_u + 2 * GDC_UP, GDC_UP, 16 * GDC_CB, 32);
                gdc_product<1, NH, GDC_T / 16, false, true>(o, ap, GDC_TP, 32, b_u + 16 * j0, GDC_UP, 16 * GDC_CB, 32, mt + 1);
                const float decay = vec[5 * GDC_T], kf = vec[5 * GDC_T + 1];
#pragma unroll
                for (int j = 0; j < GDC_NT; ++j) {
                    const float f = __fmul_rn(kf, atc_pow2(-atc_shift(u_most[8 + j], 63)));
#pragma unroll
                    for (int e = 0; e < 4; ++e) S[j][e] = __fmaf_rn(S[j][e], decay, __fmul_rn(d[0][j][e], f));
                }
            }
            tiles_most(S, next);
            {
#pragma unroll
                for (int j = 0; j < NH; ++j) {
                    const float fu = atc_pow2(-atc_shift(u_most[j0 + j], 63));
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int i = 16 * mt + g + 8 * h;
                        const float f = vec[4 * GDC_T + i];
                        if (i < n && 8 * (j0 + j) < cols) {
                            float *dst = P.out + ((tok + i) * P.n_v_heads + vh) * GDC_D + c0 + 8 * (j0 + j) + 2 * t;
                            dst[0] = __fmaf_rn(__fmul_rn(o[0][j][2 * h], f), fu, y[0][j][2 * h]);
                            dst[1] = __fmaf_rn(__fmul_rn(o[0][j][2 * h + 1], f), fu, y[0][j][2 * h + 1]);
                        }
                    }
                }
            }
        } else {
            // ---- a value that sums may not hold: token by token, as the definition has it.  Thread = a column and every fifth row; the state in the place of its planes.
            float *st = reinterpret_cast<float *>(sp), *x1 = reinterpret_cast<float *>(up), *x2 = x1 + 5 * GDC_COLS;
#pragma unroll
            for (int j = 0; j < GDC_NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) st[(16 * warp + g + 8 * (e >> 1)) * GDC_COLS + 8 * j + 2 * t + (e & 1)] = S[j][e];
            __syncthreads();
            const int col = tid % GDC_COLS, part = tid / GDC_COLS;
            for (int i = 0; i < n; ++i) {
                const float decay = expf(P.g[(tok + i) * P.n_v_heads + vh]), beta = P.beta[(tok + i) * P.n_v_heads + vh];
                const float *k = P.k + ((tok + i) * P.n_k_heads + kh) * GDC_D, *q = P.q + ((tok + i) * P.n_k_heads + kh) * GDC_D;
                if (part < 5) {
                    float x = 0.0f;
                    for (int r = part; r < GDC_D; r += 5) {
                        const float y = __fmul_rn(st[r * GDC_COLS + col], decay);
                        st[r * GDC_COLS + col] = y;
                        x = __fadd_rn(x, __fmul_rn(k[r], y));
                    }
                    x1[part * GDC_COLS + col] = x;
                }
                __syncthreads();
                if (part < 5) {
                    float x = 0.0f;
                    for (int p = 0; p < 5; ++p) x = __fadd_rn(x, x1[p * GDC_COLS + col]);
                    const float d = __fsub_rn(vt[i * GDC_VS + col], x);
                    x = 0.0f;
                    for (int r = part; r < GDC_D; r += 5) {
                        const float y = __fadd_rn(st[r * GDC_COLS + col], __fmul_rn(__fmul_rn(beta, k[r]), d));
                        st[r * GDC_COLS + col] = y;
                        x = __fadd_rn(x, __fmul_rn(q[r], y));
                    }
                    x2[part * GDC_COLS + col] = x;
                }
                __syncthreads();
                if (part == 0 && col < cols) {
                    float x = 0.0f;
                    for (int p = 0; p < 5; ++p) x = __fadd_rn(x, x2[p * GDC_COLS + col]);
                    P.out[((tok + i) * P.n_v_heads + vh) * GDC_D + c0 + col] = x;
                }
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < GDC_NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) S[j][e] = st[(16 * warp + g + 8 * (e >> 1)) * GDC_COLS + 8 * j + 2 * t + (e & 1)];
            if (c + 1 < nchunk) load_qv(c + 1);
            tiles_most(S, next);
        }
        __syncthreads();                                        // the maxima; S's planes have long been read
        store_s(next);
    }
#pragma unroll
    for (int j = 0; j < GDC_NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (8 * j < cols) Sg[(size_t)(16 * warp + g + 8 * (e >> 1)) * GDC_D + 8 * j + 2 * t + (e & 1)] = S[j][e];
}

}  // namespace b200
