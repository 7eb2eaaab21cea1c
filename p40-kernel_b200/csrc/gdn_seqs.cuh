// gdn_seqs.cuh -- the gated delta rule over the tokens of several sequences.
#pragma once

#include "common.cuh"
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

// Where sequence s keeps its state: its slot, or s itself.  -1 (every thread of the CTA): the slot is not one of the pool's, or another sequence names it too.
__device__ __forceinline__ int gdn_slot_of(const GdnSeqs &P, int s) {
    const int mine = P.slot ? P.slot[s] : s;
    int bad = mine < 0 || mine >= P.n_slots;
    if (P.slot)
        for (int i = threadIdx.x; i < P.n_seq; i += blockDim.x) bad |= i != s && P.slot[i] == mine;
    return __syncthreads_or(bad) ? -1 : mine;
}

// ---- token by token: the form for few tokens --------------------------------------------------------------------------------------------
// As gdn_step_kernel: one CTA per (sequence, value head, 32 columns of the state), eight warps, lane = column, warp w holds rows w, w + 8, ... in
// registers over all of the sequence's tokens: the state is read once and written once.  Sequences of more than `most` tokens are not its own.
__global__ void __launch_bounds__(GDN_WARPS * 32) gdn_seqs_step_kernel(const __grid_constant__ GdnSeqs P, int most) {
    __shared__ float ks[2][GDN_KMAX], qs[2][GDN_KMAX];
    __shared__ float part[2][GDN_WARPS][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tiles = P.V / 32, s = blockIdx.y;
    const int vh = blockIdx.x / tiles, vt = blockIdx.x - vh * tiles;
    const int j = vt * 32 + lane;
    const int kh = vh / (P.n_v_heads / P.n_k_heads);
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    const SeqRange r = seq_range(P.start, s, P.n_tok);
    if (r.n <= 0 || r.n > most) {
        if (r.n < 0 && threadIdx.x == 0) bad_sequence();
        return;
    }
    const int slot = gdn_slot_of(P, s);
    if (slot < 0) {
        if (threadIdx.x == 0) bad_sequence();
        return;
    }
    float *Sg = P.state + ((size_t)slot * P.n_v_heads + vh) * P.K * P.V + j;
    float col[GDN_RPW];
#pragma unroll
    for (int i = 0; i < GDN_RPW; ++i) {
        const int row = warp + GDN_WARPS * i;
        col[i] = row < P.K ? Sg[(size_t)row * P.V] : 0.0f;
    }
    for (int t = 0; t < r.n; ++t) {
        const int b2 = t & 1;
        const size_t tok = (size_t)(r.begin + t);
        const float b = P.beta[tok * P.n_v_heads + vh], vj = P.v[(tok * P.n_v_heads + vh) * P.V + j], decay = expf(P.g[tok * P.n_v_heads + vh]);
        for (int i = threadIdx.x; i < P.K; i += blockDim.x) {
            ks[b2][i] = P.k[(tok * P.n_k_heads + kh) * P.K + i];
            qs[b2][i] = P.q[(tok * P.n_k_heads + kh) * P.K + i];
        }
        __syncthreads();
        float kv = 0.0f;
#pragma unroll
        for (int i = 0; i < GDN_RPW; ++i) {
            const int row = warp + GDN_WARPS * i;
            if (row < P.K) {
                col[i] = __fmul_rn(col[i], decay);
                kv = __fadd_rn(kv, __fmul_rn(ks[b2][row], col[i]));
            }
        }
        part[0][warp][lane] = kv;
        __syncthreads();
        kv = 0.0f;
#pragma unroll
        for (int w = 0; w < GDN_WARPS; ++w) kv = __fadd_rn(kv, part[0][w][lane]);
        const float d = __fsub_rn(vj, kv);
        float o = 0.0f;
#pragma unroll
        for (int i = 0; i < GDN_RPW; ++i) {
            const int row = warp + GDN_WARPS * i;
            if (row < P.K) {
                col[i] = __fadd_rn(col[i], __fmul_rn(__fmul_rn(b, ks[b2][row]), d));
                o = __fadd_rn(o, __fmul_rn(qs[b2][row], col[i]));
            }
        }
        part[1][warp][lane] = o;
        __syncthreads();
        if (warp == 0) {
            o = 0.0f;
#pragma unroll
            for (int w = 0; w < GDN_WARPS; ++w) o = __fadd_rn(o, part[1][w][lane]);
            P.out[(tok * P.n_v_heads + vh) * P.V + j] = o;
        }
    }
#pragma unroll
    for (int i = 0; i < GDN_RPW; ++i) {
        const int row = warp + GDN_WARPS * i;
        if (row < P.K) Sg[(size_t)row * P.V] = col[i];
    }
}

// ---- in chunks of 64 tokens: the form for many -----------------------------------------------------------------------------------------------
// With G_i the sum of g from the chunk's begin to token i, S the state in front of the chunk and u_i what token i adds along its key,
//   u_i = beta_i (v_i - e^G_i k_i S - sum over j < i of e^(G_i - G_j) (k_i . k_j) u_j)                U = Tb (V - e^G K S), Tb = (1 + A)^-1 diag(beta)
//   o_i = e^G_i q_i S + sum over j <= i of e^(G_i - G_j) (q_i . k_j) u_j                              O = e^G Q S + P U
//   S' = e^G_63 S + sum of k_j e^(G_63 - G_j) u_j                                                     S' = e^G_63 S + K^T (e^(G_63 - G) U)
// with A_ij = beta_i e^(G_i - G_j) (k_i . k_j), j < i.  gdn_chunk_kernel forms Tb and P of every chunk at once; gdn_scan_kernel carries the state through
// the chunks of a sequence, a CTA per value head and 48 or 40 columns of it (the columns do not know of each other).
//
// Products are fp32 to 2^-22: each operand is split into two TF32 parts (11 bits each, any exponent), three of the four products on mma.sync (m16n8k8), sums fp32.
constexpr int GDC_T = 64, GDC_D = 128, GDC_THREADS = 256;
constexpr int GDC_KS = GDC_D + 4, GDC_TS = GDC_T + 4;                 // row strides: 4 g + t are 32 different banks
constexpr int GDC_COLS = 48, GDC_CS = GDC_COLS + 8, GDC_NT = GDC_COLS / 8, GDC_SLICES = 3;       // 24 t + g are 32 different banks
constexpr int GDC_STEP_MOST = 16;                                     // tokens of a sequence that go one by one
// What the first kernel leaves of a chunk and value head: Tb, P [64][64], e^G, e^(G_63 - G) [64], and whether the chunk is to go token by token
constexpr int GDC_REC = 2 * GDC_T * GDC_T + 2 * GDC_T + 4;            // floats, 16-byte aligned
constexpr int gdc_chunk_smem() { return (2 * GDC_T * GDC_KS + 4 * GDC_T * GDC_TS) * 4 + GDC_T * 8 + GDC_T * 4; }
constexpr int gdc_scan_smem() { return (3 * GDC_T * GDC_KS + 3 * GDC_T * GDC_TS + GDC_T * GDC_COLS + (GDC_D + 2 * GDC_T) * GDC_CS + 4 * GDC_T + 8) * 4; }

__device__ __forceinline__ int gdc_chunks(int n) { return n > GDC_STEP_MOST ? (n + GDC_T - 1) / GDC_T : 0; }

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// x = hi + lo: hi rounded to 11 bits, lo to the 11 behind them
__device__ __forceinline__ uint32_t tf32_of(float x) { return (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u; }
__device__ __forceinline__ void tf32_split(float x, uint32_t &hi, uint32_t &lo) {
    hi = tf32_of(x);
    lo = tf32_of(__fsub_rn(x, __uint_as_float(hi)));
}
// c += A B over 8 `steps` values, an even number of steps: A 16 rows, element (i, k) at a[i * as + k * ak], B 8 NT columns, (k, j) at b[k * bs + j * bj]; a and b point at the lane's own
// corner, (g, t) and (t, g).  A's value k is multiplied by the lane's factor(k) first.
// The tensor core cuts the last bits of a sum off instead of rounding it: a sum is of two steps of 8, small products first, and rounded additions join them.  (One sum over all
// steps, the state's own among them: error of 2048 tokens' outputs against 64 bits 1.6e-6.)
template <int NT, typename F>
__device__ __forceinline__ void gdc_product(float (&c)[NT][4], const float *a, int as, int ak, const float *b, int bs, int bj, int steps, F factor) {
#pragma unroll 1
    for (int s = 0; s < steps; s += 2, a += 16 * ak, b += 16 * bs) {
        float sum[NT][4];
        uint32_t ah[2][4], al[2][4], bh[2][NT][2], bl[2][NT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float f0 = factor(8 * (s + h)), f1 = factor(8 * (s + h) + 4);
            const float *x = a + 8 * h * ak, *y = b + 8 * h * bs;
            tf32_split(__fmul_rn(x[0], f0), ah[h][0], al[h][0]);
            tf32_split(__fmul_rn(x[8 * as], f0), ah[h][1], al[h][1]);
            tf32_split(__fmul_rn(x[4 * ak], f1), ah[h][2], al[h][2]);
            tf32_split(__fmul_rn(x[8 * as + 4 * ak], f1), ah[h][3], al[h][3]);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                tf32_split(y[8 * j * bj], bh[h][j][0], bl[h][j][0]);
                tf32_split(y[8 * j * bj + 4 * bs], bh[h][j][1], bl[h][j][1]);
            }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) sum[j][0] = sum[j][1] = sum[j][2] = sum[j][3] = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < NT; ++j) mma_tf32(sum[j], al[h], bh[h][j]);
#pragma unroll
            for (int j = 0; j < NT; ++j) mma_tf32(sum[j], ah[h], bl[h][j]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < NT; ++j) mma_tf32(sum[j], ah[h], bh[h][j]);
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) c[j][e] = __fadd_rn(c[j][e], sum[j][e]);
    }
}
template <int NT>
__device__ __forceinline__ void gdc_product(float (&c)[NT][4], const float *a, int as, int ak, const float *b, int bs, int bj, int steps) {
    gdc_product<NT>(c, a, as, ak, b, bs, bj, steps, [](int) { return 1.0f; });
}
__device__ __forceinline__ void cp_async4(void *dst, const void *src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory"); }
// `rows` rows of COLS floats (row stride `from` in memory, `to` in shared memory) by the whole CTA, asynchronously; rows up to 64 are filled up with zeros.
template <int COLS>
__device__ __forceinline__ void gdc_load(float *dst, int to, const float *src, size_t from, int rows, bool vec, int cols = COLS) {
    if (vec) {
        for (int i = threadIdx.x; i < GDC_T * (COLS / 4); i += GDC_THREADS) {
            const int r = i / (COLS / 4), c = 4 * (i % (COLS / 4));
            if (c >= cols) continue;
            if (r < rows) cp_async16(dst + r * to + c, src + r * from + c);
            else *reinterpret_cast<float4 *>(dst + r * to + c) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    } else {
        for (int i = threadIdx.x; i < GDC_T * COLS; i += GDC_THREADS) {
            const int r = i / COLS, c = i % COLS;
            if (c >= cols) continue;
            if (r < rows) cp_async4(dst + r * to + c, src + r * from + c);
            else dst[r * to + c] = 0.0f;
        }
    }
}

// grid (chunks of all sequences and some that find none, key heads): K K^T and Q K^T once, then Tb and P for each value head of the key head.
__global__ void __launch_bounds__(GDC_THREADS, 1) gdn_chunk_kernel(const __grid_constant__ GdnSeqs P, float *recs) {
    extern __shared__ __align__(16) float gdc_smem[];
    float *kt = gdc_smem, *qt = kt + GDC_T * GDC_KS, *kk = qt + GDC_T * GDC_KS, *qk = kk + GDC_T * GDC_TS, *at = qk + GDC_T * GDC_TS, *tt = at + GDC_T * GDC_TS;
    double *gs = reinterpret_cast<double *>(tt + GDC_T * GDC_TS);
    float *bs = reinterpret_cast<float *>(gs + GDC_T);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int kh = blockIdx.y;
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    int seq, chunk;
    if (!seq_of_item(P.start, P.n_seq, P.n_tok, (int)blockIdx.x, lane, [](int n) { return gdc_chunks(n); }, seq, chunk)) return;
    const SeqRange range = seq_range(P.start, seq, P.n_tok);
    const int n = min(GDC_T, range.n - chunk * GDC_T);
    const size_t tok = (size_t)range.begin + chunk * GDC_T;
    const size_t stride = (size_t)P.n_k_heads * GDC_D;
    const bool vec = ((reinterpret_cast<uintptr_t>(P.k) | reinterpret_cast<uintptr_t>(P.q)) & 15u) == 0;
    gdc_load<GDC_D>(kt, GDC_KS, P.k + (tok * P.n_k_heads + kh) * GDC_D, stride, n, vec);
    gdc_load<GDC_D>(qt, GDC_KS, P.q + (tok * P.n_k_heads + kh) * GDC_D, stride, n, vec);
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();
    {   // of rows 16 m .. the columns up to 16 m + 15; a sub-core's two warps take rows that add up to the same number of columns
        const bool of_q = warp >= 4;
        const int m = of_q ? 7 - warp : warp;
        const float *a = (of_q ? qt : kt) + (16 * m + g) * GDC_KS + t;
        float *dst = (of_q ? qk : kk) + (16 * m + g) * GDC_TS + 2 * t;
        for (int j = 0; j <= m; ++j) {
            float c[2][4] = {};
            gdc_product<2>(c, a, GDC_KS, 1, kt + (16 * j + g) * GDC_KS + t, 1, GDC_KS, GDC_D / 8);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                *reinterpret_cast<float2 *>(dst + 16 * j + 8 * h) = make_float2(c[h][0], c[h][1]);
                *reinterpret_cast<float2 *>(dst + 16 * j + 8 * h + 8 * GDC_TS) = make_float2(c[h][2], c[h][3]);
            }
        }
    }
    const int share = P.n_v_heads / P.n_k_heads;
    for (int sub = 0; sub < share; ++sub) {
        const int vh = kh * share + sub;
        float *rec = recs + ((size_t)blockIdx.x * P.n_v_heads + vh) * GDC_REC;
        bool odd = false;                       // something that sums may not hold: the chunk goes token by token
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
            const double before = sum - x[1], last = __shfl_sync(0xffffffffu, sum, 31);
            gs[2 * lane] = before + x[0];
            gs[2 * lane + 1] = sum;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const double gi = h ? sum : before + x[0];
                rec[2 * GDC_T * GDC_T + 2 * lane + h] = expf((float)gi);
                rec[2 * GDC_T * GDC_T + GDC_T + 2 * lane + h] = expf((float)(last - gi));
            }
        }
        __syncthreads();
        for (int e = tid; e < GDC_T * GDC_T; e += GDC_THREADS) {
            const int i = e / GDC_T, j = e % GDC_T;
            float a = 0.0f, p = 0.0f;
            if (j <= i) {
                const float decay = expf((float)(gs[i] - gs[j]));
                p = i < n ? __fmul_rn(decay, qk[i * GDC_TS + j]) : 0.0f;
                a = j < i ? __fmul_rn(__fmul_rn(bs[i], decay), kk[i * GDC_TS + j]) : 0.0f;
                odd = odd || !(fabsf(p) < 1e30f) || !(fabsf(a) < 1e30f);
            }
            at[i * GDC_TS + j] = a;
            rec[GDC_T * GDC_T + e] = p;
        }
        __syncthreads();
        // inverses of the four 16 x 16 blocks on the diagonal: a half-warp each, lane = column, from the top row down
        if (warp < 2) {
            const int blk = 16 * (2 * warp + (lane >> 4)), c = lane & 15;
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float s = i == c ? 1.0f : 0.0f;
#pragma unroll
                for (int j = 0; j < i; ++j) s = __fmaf_rn(-at[(blk + i) * GDC_TS + blk + j], x[j], s);
                x[i] = s;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) tt[(blk + i) * GDC_TS + blk + c] = x[i];
        }
        __syncthreads();
        // below the diagonal, a row of blocks after the other: T_ij = -T_ii (sum of A_ik T_kj, j <= k < i).  A thread has four rows of one column.
        for (int i = 1; i < 4; ++i) {
            const int r0 = 16 * i + 4 * (tid & 3), col = tid >> 2;              // 64 columns, of which 16 i have work
            float s[4] = {};
            if (col < 16 * i) {
                for (int k = col & ~15; k < 16 * i; ++k) {
                    const float x = tt[k * GDC_TS + col];
#pragma unroll
                    for (int h = 0; h < 4; ++h) s[h] = __fmaf_rn(at[(r0 + h) * GDC_TS + k], x, s[h]);
                }
            }
            __syncthreads();
            if (col < 16 * i)
#pragma unroll
                for (int h = 0; h < 4; ++h) at[(r0 + h) * GDC_TS + col] = s[h];          // A's row of blocks has been read
            __syncthreads();
            if (col < 16 * i) {
#pragma unroll
                for (int h = 0; h < 4; ++h) s[h] = 0.0f;
                for (int k = 0; k < 16; ++k) {
                    const float x = at[(16 * i + k) * GDC_TS + col];
#pragma unroll
                    for (int h = 0; h < 4; ++h) s[h] = __fmaf_rn(tt[(r0 + h) * GDC_TS + 16 * i + k], x, s[h]);
                }
#pragma unroll
                for (int h = 0; h < 4; ++h) tt[(r0 + h) * GDC_TS + col] = -s[h];
            }
            __syncthreads();
        }
        for (int e = tid; e < GDC_T * GDC_T; e += GDC_THREADS) {
            const int i = e / GDC_T, j = e % GDC_T;
            const float x = (j >> 4) <= (i >> 4) ? __fmul_rn(tt[i * GDC_TS + j], bs[j]) : 0.0f;
            odd = odd || !(fabsf(x) < 1e30f);
            rec[e] = x;
        }
        const int any = __syncthreads_or(odd ? 1 : 0);
        if (tid == 0) rec[2 * GDC_T * GDC_T + 2 * GDC_T] = any ? 1.0f : 0.0f;
    }
}

// grid (value heads x 3, sequences): columns 0 .. 47, 48 .. 87, 88 .. 127.  Warp w of eight: rows 16 (w % 4) .. of K S (w < 4) or Q S, and rows 16 w .. of the state, which
// stay in registers; a copy of the state in shared memory is what the products read.
__global__ void __launch_bounds__(GDC_THREADS, 1) gdn_scan_kernel(const __grid_constant__ GdnSeqs P, const float *recs) {
    extern __shared__ __align__(16) float gdc_smem[];
    float *kt0 = gdc_smem, *qt = kt0 + 2 * GDC_T * GDC_KS, *tb = qt + GDC_T * GDC_KS, *pt0 = tb + GDC_T * GDC_TS, *vt = pt0 + 2 * GDC_T * GDC_TS;           // K and P twice
    float *st = vt + GDC_T * GDC_COLS, *rt = st + GDC_D * GDC_CS, *ut = rt + GDC_T * GDC_CS;
    float *since0 = ut + GDC_T * GDC_CS, *flag = since0 + 4 * GDC_T;                   // e^G, behind it e^(G_63 - G), twice; [2]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int vh = blockIdx.x / GDC_SLICES, slice = blockIdx.x % GDC_SLICES, s = blockIdx.y;
    const int c0 = slice == 0 ? 0 : 48 + 40 * (slice - 1), cols = slice == 0 ? 48 : 40;
    const int kh = vh / (P.n_v_heads / P.n_k_heads), mt = warp & 3;
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
    const float *rec0 = recs + ((size_t)first * P.n_v_heads + vh) * GDC_REC;
    const size_t rec_stride = (size_t)P.n_v_heads * GDC_REC;
    const bool vec = ((reinterpret_cast<uintptr_t>(P.k) | reinterpret_cast<uintptr_t>(P.q)) & 15u) == 0, vvec = (reinterpret_cast<uintptr_t>(P.v) & 15u) == 0;
    const size_t kstride = (size_t)P.n_k_heads * GDC_D, vstride = (size_t)P.n_v_heads * GDC_D;

    // what a chunk brings, in the order in which room for it becomes free
    auto load_qv = [&](int c) {
        const size_t tok = (size_t)range.begin + c * GDC_T;
        const int n = min(GDC_T, range.n - c * GDC_T);
        gdc_load<GDC_D>(qt, GDC_KS, P.q + (tok * P.n_k_heads + kh) * GDC_D, kstride, n, vec);
        gdc_load<GDC_COLS>(vt, GDC_COLS, P.v + (tok * P.n_v_heads + vh) * GDC_D + c0, vstride, n, vvec, cols);
    };
    auto load_t = [&](int c) { gdc_load<GDC_T>(tb, GDC_TS, rec0 + c * rec_stride, GDC_T, GDC_T, true); };
    auto load_kp = [&](int c) {
        const size_t tok = (size_t)range.begin + c * GDC_T;
        const int n = min(GDC_T, range.n - c * GDC_T), b = c & 1;
        gdc_load<GDC_D>(kt0 + b * GDC_T * GDC_KS, GDC_KS, P.k + (tok * P.n_k_heads + kh) * GDC_D, kstride, n, vec);
        const float *rec = rec0 + c * rec_stride + GDC_T * GDC_T;
        gdc_load<GDC_T>(pt0 + b * GDC_T * GDC_TS, GDC_TS, rec, GDC_T, GDC_T, true);
        if (tid < 2 * GDC_T / 4) cp_async16(since0 + 2 * GDC_T * b + 4 * tid, rec + GDC_T * GDC_T + 4 * tid);
        if (tid == 2 * GDC_T / 4) cp_async4(flag + b, rec + GDC_T * GDC_T + 2 * GDC_T);
    };
    load_kp(0);
    load_qv(0);
    load_t(0);
    cp_async_commit();
    float *Sg = P.state + ((size_t)slot * P.n_v_heads + vh) * GDC_D * GDC_D + c0;
    float S[GDC_NT][4];                                         // rows 16 warp + g, + 8; columns 8 nt + 2 t, + 1
#pragma unroll
    for (int j = 0; j < GDC_NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) S[j][e] = 8 * j < cols ? Sg[(size_t)(16 * warp + g + 8 * (e >> 1)) * GDC_D + 8 * j + 2 * t + (e & 1)] : 0.0f;
    auto store_s = [&] {
#pragma unroll
        for (int j = 0; j < GDC_NT; ++j) {
            *reinterpret_cast<float2 *>(st + (16 * warp + g) * GDC_CS + 8 * j + 2 * t) = make_float2(S[j][0], S[j][1]);
            *reinterpret_cast<float2 *>(st + (16 * warp + g + 8) * GDC_CS + 8 * j + 2 * t) = make_float2(S[j][2], S[j][3]);
        }
    };
    if (slice)                                                  // columns 40 .. 47 are nobody's: zeros
        for (int i = tid; i < GDC_T * 8; i += GDC_THREADS) vt[(i / 8) * GDC_COLS + 40 + i % 8] = 0.0f;
    store_s();
    for (int c = 0; c < nchunk; ++c) {
        const int b = c & 1, n = min(GDC_T, range.n - c * GDC_T);
        const size_t tok = (size_t)range.begin + c * GDC_T;
        cp_async_wait<0>();
        __syncthreads();                                        // the chunk, and the state of the one before
        if (c + 1 < nchunk) load_kp(c + 1);
        const float *kt = kt0 + b * GDC_T * GDC_KS, *pt = pt0 + b * GDC_T * GDC_TS, *eg = since0 + 2 * GDC_T * b, *left = eg + GDC_T;
        // ---- K S (then R = V - e^G K S) and Q S
        float acc[GDC_NT][4];
#pragma unroll
        for (int j = 0; j < GDC_NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][e] = 0.0f;
        gdc_product<GDC_NT>(acc, (warp < 4 ? kt : qt) + (16 * mt + g) * GDC_KS + t, GDC_KS, 1, st + t * GDC_CS + g, GDC_CS, 1, GDC_D / 8);
        bool odd = flag[b] != 0.0f;
#pragma unroll
        for (int j = 0; j < GDC_NT; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = 16 * mt + g + 8 * h, col = 8 * j + 2 * t;
                float2 x = make_float2(__fmul_rn(acc[j][2 * h], eg[i]), __fmul_rn(acc[j][2 * h + 1], eg[i]));
                if (warp < 4) {
                    const float2 v = *reinterpret_cast<const float2 *>(vt + i * GDC_COLS + col);
                    x = make_float2(__fsub_rn(v.x, x.x), __fsub_rn(v.y, x.y));
                    *reinterpret_cast<float2 *>(rt + i * GDC_CS + col) = x;
                }
                odd = odd || !(fabsf(x.x) < 1e30f) || !(fabsf(x.y) < 1e30f);
                acc[j][2 * h] = x.x;
                acc[j][2 * h + 1] = x.y;
            }
        int slow = __syncthreads_or(odd ? 1 : 0);
        // ---- U = Tb R, rows 16 mt .., half of the columns
        {
            float u[GDC_NT / 2][4];
#pragma unroll
            for (int j = 0; j < GDC_NT / 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) u[j][e] = 0.0f;
            const int h0 = (warp >> 2) * (GDC_COLS / 2);
            gdc_product<GDC_NT / 2>(u, tb + (16 * mt + g) * GDC_TS + t, GDC_TS, 1, rt + t * GDC_CS + h0 + g, GDC_CS, 1, 2 * (mt + 1));
            odd = false;
#pragma unroll
            for (int j = 0; j < GDC_NT / 2; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    odd = odd || !(fabsf(u[j][2 * h]) < 1e30f) || !(fabsf(u[j][2 * h + 1]) < 1e30f);
                    *reinterpret_cast<float2 *>(ut + (16 * mt + g + 8 * h) * GDC_CS + h0 + 8 * j + 2 * t) = make_float2(u[j][2 * h], u[j][2 * h + 1]);
                }
        }
        slow |= __syncthreads_or(odd ? 1 : 0);
        if (!slow) {
            if (c + 1 < nchunk) {                               // Q, V and Tb have been read
                load_qv(c + 1);
                load_t(c + 1);
            }
            cp_async_commit();
            // ---- S = e^G_63 S + K^T (e^(G_63 - G) U)
            const float decay = eg[GDC_T - 1];
#pragma unroll
            for (int j = 0; j < GDC_NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) S[j][e] = __fmul_rn(S[j][e], decay);
            gdc_product<GDC_NT>(S, kt + t * GDC_KS + 16 * warp + g, 1, GDC_KS, ut + t * GDC_CS + g, GDC_CS, 1, GDC_T / 8, [&](int k) { return left[k + t]; });
            store_s();                                          // (K S and Q S were read in front of two barriers)
            // ---- O = e^G Q S + P U
            if (warp >= 4) {
                gdc_product<GDC_NT>(acc, pt + (16 * mt + g) * GDC_TS + t, GDC_TS, 1, ut + t * GDC_CS + g, GDC_CS, 1, 2 * (mt + 1));
#pragma unroll
                for (int j = 0; j < GDC_NT; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int i = 16 * mt + g + 8 * h;
                        if (i < n && 8 * j < cols) {
                            float *o = P.out + ((tok + i) * P.n_v_heads + vh) * GDC_D + c0 + 8 * j + 2 * t;
                            o[0] = acc[j][2 * h];
                            o[1] = acc[j][2 * h + 1];
                        }
                    }
            }
        } else {
            // ---- a value that sums may not hold: token by token, as the definition has it.  Thread = a column and every fifth row.
            const int col = tid % GDC_COLS, part = tid / GDC_COLS;
            for (int i = 0; i < n; ++i) {
                const float decay = expf(P.g[(tok + i) * P.n_v_heads + vh]), beta = P.beta[(tok + i) * P.n_v_heads + vh];
                const float *k = kt + i * GDC_KS, *q = qt + i * GDC_KS;
                float x = 0.0f;
                if (part < 5)
                    for (int r = part; r < GDC_D; r += 5) {
                        const float y = __fmul_rn(st[r * GDC_CS + col], decay);
                        st[r * GDC_CS + col] = y;
                        x = __fadd_rn(x, __fmul_rn(k[r], y));
                    }
                if (part < 5) rt[part * GDC_CS + col] = x;
                __syncthreads();
                if (part < 5) {
                    x = 0.0f;
                    for (int p = 0; p < 5; ++p) x = __fadd_rn(x, rt[p * GDC_CS + col]);
                    const float d = __fsub_rn(vt[i * GDC_COLS + col], x);
                    x = 0.0f;
                    for (int r = part; r < GDC_D; r += 5) {
                        const float y = __fadd_rn(st[r * GDC_CS + col], __fmul_rn(__fmul_rn(beta, k[r]), d));
                        st[r * GDC_CS + col] = y;
                        x = __fadd_rn(x, __fmul_rn(q[r], y));
                    }
                    ut[part * GDC_CS + col] = x;
                }
                __syncthreads();
                if (part == 0 && col < cols) {
                    x = 0.0f;
                    for (int p = 0; p < 5; ++p) x = __fadd_rn(x, ut[p * GDC_CS + col]);
                    P.out[((tok + i) * P.n_v_heads + vh) * GDC_D + c0 + col] = x;
                }
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < GDC_NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) S[j][e] = st[(16 * warp + g + 8 * (e >> 1)) * GDC_CS + 8 * j + 2 * t + (e & 1)];
            __syncthreads();
            if (c + 1 < nchunk) {
                load_qv(c + 1);
                load_t(c + 1);
            }
            cp_async_commit();
        }
    }
#pragma unroll
    for (int j = 0; j < GDC_NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (8 * j < cols) Sg[(size_t)(16 * warp + g + 8 * (e >> 1)) * GDC_D + 8 * j + 2 * t + (e & 1)] = S[j][e];
}

}  // namespace b200
