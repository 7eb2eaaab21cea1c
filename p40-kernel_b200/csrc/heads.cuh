// heads.cuh -- norms of queries and keys for each head, with the position rotation in the same pass: what an attention layer does
// between its q / k projections and its cache.
//
//   y = x / sqrt(mean(x^2) + eps) * w          over the head_dim values of one head of one token, w shared by the heads
//   y_i, y_(i + n_rot / 2) <- turned by the angle pos * freq_i, i < n_rot / 2; values from n_rot on are not turned
//
// The angle is formed in 64 bits and brought into [-pi, pi] there: at position 262143 an fp32 product is off by 0.016 of a turn's radian.
#pragma once

#include "common.cuh"
#include "ops.cuh"

namespace b200 {

constexpr int QKN_MAX_DIM = 256, QKN_MAX_WARPS = 8;

struct QkNormParams {
    const float *x[2], *w[2];               // q, k
    float *y[2];
    int64_t tok_stride[2], head_stride[2];  // of x, in floats; y is packed
    const int32_t *pos;
    const double *freq;
    int n_head[2], head_dim, n_rot;
    float inv_dim, eps;                     // 1 / head_dim
};

// cos and sin of pos * freq.  Two parts of 2 pi (Cody and Waite's reduction): what is left of the ROUNDED product is exact to 2^-50 for any int32 position and freq <= 1.  The product
// itself is off by 2^-53 of the angle at most (3e-11 at position 262143, 1.2e-7 at 2^31), and the angle that is left is rounded to fp32 (1.2e-7 at most).
__device__ __forceinline__ float2 rotation_of(int pos, double freq) {
    const double a = __dmul_rn((double)pos, freq), turns = rint(__dmul_rn(a, 0.15915494309189535));
    const double r = __fma_rn(-turns, 2.4492935982947064e-16, __fma_rn(-turns, 6.283185307179586, a));
    float s, c;
    sincosf((float)r, &s, &c);
    return make_float2(c, s);
}

// grid (tokens, groups of heads); a warp has up to PER heads.  VEC: head_dim and the strides are multiples of 4, all pointers 16-byte aligned.
// 28 heads of 256 in and out are 57 KB a token, 2000 tokens 115 MB in 25 us (4.5 TB/s).  Bound by latency and issue, not by memory (57 MB read from DRAM and 11 MB written in that time, issue
// slots 0.59): 2000 short CTAs, in each of which loads, angles, a barrier and stores follow one another.  PER = 4 forms a token's angles once for all
// heads (a head a warp: the same time, with four times the 64-bit operations); of few tokens a warp has one head, whose chain is shorter.
template <bool VEC, int PER>
__global__ void __launch_bounds__(32 * QKN_MAX_WARPS) qk_norm_rope_kernel(const __grid_constant__ QkNormParams P) {
    __shared__ __align__(16) float rows[QKN_MAX_WARPS][QKN_MAX_DIM];
    __shared__ float2 turn[QKN_MAX_DIM / 2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (int)blockDim.x >> 5;
    const int64_t tok = blockIdx.x;
    const int heads = P.n_head[0] + P.n_head[1], first = (int)blockIdx.y * warps * PER + warp;
    const int n = P.head_dim, half = P.n_rot >> 1;
    pdl_wait_prior_grid();
    if (PER == 1) pdl_launch_dependents();
    // (q's heads first, then k's)
    const float *x0[2] = {P.x[0] + tok * P.tok_stride[0], P.x[1] + tok * P.tok_stride[1]};
    float *y0[2] = {P.y[0] + tok * P.n_head[0] * n, P.y[1] + tok * P.n_head[1] * n};
    float4 f[PER][2];
#pragma unroll
    for (int r = 0; r < PER; ++r) {
        const int head = first + warps * r;
        if (head < heads) {
            const bool second = head >= P.n_head[0];
            const float *x = second ? x0[1] + (head - P.n_head[0]) * P.head_stride[1] : x0[0] + head * P.head_stride[0];
#pragma unroll
            for (int j = 0; j < 2; ++j) f[r][j] = rms_load<VEC>(x, 128 * j + 4 * lane, n);
        }
    }
    for (int i = threadIdx.x; i < half; i += blockDim.x) turn[i] = rotation_of(P.pos[tok], P.freq[i]);
    __syncthreads();
    float *row = rows[warp];
#pragma unroll
    for (int r = 0; r < PER; ++r) {
        const int head = first + warps * r;
        if (head >= heads) break;
        const int which = head >= P.n_head[0];
        float4 w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) w[j] = rms_load<VEC>(P.w[which], 128 * j + 4 * lane, n);
        float ss = __fadd_rn(lane_sumsq(f[r][0]), lane_sumsq(f[r][1]));          // (past the end there are zeros)
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, o));
        const float sc = rsqrtf(__fmaf_rn(ss, P.inv_dim, P.eps));
        if (r) __syncwarp();                            // the row before has been read
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            f[r][j].x = __fmul_rn(__fmul_rn(f[r][j].x, sc), w[j].x);
            f[r][j].y = __fmul_rn(__fmul_rn(f[r][j].y, sc), w[j].y);
            f[r][j].z = __fmul_rn(__fmul_rn(f[r][j].z, sc), w[j].z);
            f[r][j].w = __fmul_rn(__fmul_rn(f[r][j].w, sc), w[j].w);
            if (128 * j < P.n_rot) reinterpret_cast<float4 *>(row)[32 * j + lane] = f[r][j];
        }
        __syncwarp();
        float *y = y0[which] + (which ? head - P.n_head[0] : head) * n;
        auto turned = [&](int i, float own) {
            if (i >= P.n_rot) return own;
            const bool second = i >= half;
            const float2 t = turn[second ? i - half : i];
            const float other = row[second ? i - half : i + half];
            return second ? __fmaf_rn(own, t.x, __fmul_rn(other, t.y)) : __fmaf_rn(own, t.x, -__fmul_rn(other, t.y));
        };
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = 128 * j + 4 * lane;
            if (i < n) {
                float4 o = f[r][j];
                if (i < P.n_rot) o = make_float4(turned(i, o.x), turned(i + 1, o.y), turned(i + 2, o.z), turned(i + 3, o.w));
                if (VEC) {
                    *reinterpret_cast<float4 *>(y + i) = o;
                } else {
                    y[i] = o.x;
                    if (i + 1 < n) y[i + 1] = o.y;
                    if (i + 2 < n) y[i + 2] = o.z;
                    if (i + 3 < n) y[i + 3] = o.w;
                }
            }
        }
    }
}

}  // namespace b200
