// rotary.cuh -- queries and keys turned by their positions, without norms: pairs of a head's halves or of neighbours, part of the head, an amplitude.
//
//   (x_a, x_b) <- A (x_a cos t - x_b sin t, x_b cos t + x_a sin t),  t = pos * freq_i, i < n_rot / 2
//   halves: a = i, b = i + n_rot / 2;  neighbours: a = 2 i, b = 2 i + 1;  values from n_rot on are not turned
//
// Frequencies and A are the caller's: contexts scaled by whatever rule are a table (bonsai_b200_rope_freq makes the common ones).
#pragma once

#include "common.cuh"

namespace b200 {

enum : int { PAIRS_HALVES = 0, PAIRS_NEXT = 1 };
constexpr int ROPE_MAX_DIM = 256, ROPE_THREADS = 256, ROPE_MAX_ITEMS = 6;

// A cos t and A sin t.  Formed in 64 bits, angle included, and rounded once: the functions' arguments are as large as positions are, and what turns quantised rows has
// to give the same codes wherever it is written down.
__device__ __forceinline__ float2 turn_of(int pos, double freq, double amplitude) {
    double s, c;
    sincos(__dmul_rn((double)pos, freq), &s, &c);
    return make_float2(__double2float_rn(__dmul_rn(c, amplitude)), __double2float_rn(__dmul_rn(s, amplitude)));
}
// Each product rounded, then their sum.
__device__ __forceinline__ float2 turned_pair(float a, float b, float2 t) {
    return make_float2(__fsub_rn(__fmul_rn(a, t.x), __fmul_rn(b, t.y)), __fadd_rn(__fmul_rn(b, t.x), __fmul_rn(a, t.y)));
}

struct RopeParams {
    const float *x[2];                      // q, k
    float *y[2];
    int64_t tok_stride[2], head_stride[2];  // of x, in floats; y is packed
    const int32_t *pos;
    const double *freq;
    int n_head[2], head_dim, n_rot, pairs;
    float amplitude;
};

// What bounds it: memory (2999 tokens of 40 heads of 128, all turned, in 26.6 us, 0.70 of the copy rate; a plain copy of as many bytes, timed alike, 26.1); the angles, in 64 bits, are formed
// once a CTA while its values are on their way.  Of 28 heads of 256 with 64 turned a token is two CTAs of 784 items for 256 threads, a fourth round for sixteen of them: 3000 tokens 40.9 us,
// the copy 32.7 (1000 tokens 15.9 and 15.7).
// grid (tokens, parts of a token's items).  An item is what one thread turns: eight values (four pairs of halves, or two times two of neighbours) or four that are
// not turned.  VEC: head_dim and n_rot are multiples of 8, strides of 4, pointers 16-byte aligned; otherwise an item is a pair or a value.
template <bool VEC>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(const __grid_constant__ RopeParams P, int items, int per) {
    __shared__ float2 turn[ROPE_MAX_DIM / 2];
    const int n = P.head_dim, half = P.n_rot >> 1;
    const int64_t tok = blockIdx.x;
    const int turned = VEC ? half / 4 : half, each = turned + (n - P.n_rot) / (VEC ? 4 : 1);      // items of a head
    const int first = (int)blockIdx.y * per, last = min(first + per, items);
    pdl_wait_prior_grid();
    auto row = [&](int head, const float *&x, float *&y) {
        const bool second = head >= P.n_head[0];
        const int h = second ? head - P.n_head[0] : head;
        x = second ? P.x[1] + tok * P.tok_stride[1] + h * P.head_stride[1] : P.x[0] + tok * P.tok_stride[0] + h * P.head_stride[0];
        y = second ? P.y[1] + (tok * P.n_head[1] + h) * n : P.y[0] + (tok * P.n_head[0] + h) * n;
    };
    // where an item's values lie
    auto place = [&](int i, int &a, int &b) {
        if (i >= turned) a = P.n_rot + (VEC ? 4 : 1) * (i - turned), b = -1;
        else if (P.pairs == PAIRS_NEXT) a = (VEC ? 8 : 2) * i, b = a + (VEC ? 4 : 1);
        else a = (VEC ? 4 : 1) * i, b = a + half;
    };
    if (VEC) {
        float4 u[ROPE_MAX_ITEMS], v[ROPE_MAX_ITEMS];
#pragma unroll
        for (int k = 0; k < ROPE_MAX_ITEMS; ++k) {
            const int item = first + (int)threadIdx.x + k * ROPE_THREADS;
            if (item >= last) break;
            const int head = item / each;
            const float *x;
            float *y;
            int a, b;
            row(head, x, y);
            place(item - head * each, a, b);
            u[k] = *reinterpret_cast<const float4 *>(x + a);
            if (b >= 0) v[k] = *reinterpret_cast<const float4 *>(x + b);
        }
        for (int i = threadIdx.x; i < half; i += ROPE_THREADS) turn[i] = turn_of(P.pos[tok], P.freq[i], (double)P.amplitude);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ROPE_MAX_ITEMS; ++k) {
            const int item = first + (int)threadIdx.x + k * ROPE_THREADS;
            if (item >= last) break;
            const int head = item / each, i = item - head * each;
            const float *x;
            float *y;
            int a, b;
            row(head, x, y);
            place(i, a, b);
            if (b >= 0) {
                const float2 *t = turn + 4 * i;
                if (P.pairs == PAIRS_NEXT) {
                    const float2 p0 = turned_pair(u[k].x, u[k].y, t[0]), p1 = turned_pair(u[k].z, u[k].w, t[1]);
                    const float2 p2 = turned_pair(v[k].x, v[k].y, t[2]), p3 = turned_pair(v[k].z, v[k].w, t[3]);
                    u[k] = make_float4(p0.x, p0.y, p1.x, p1.y);
                    v[k] = make_float4(p2.x, p2.y, p3.x, p3.y);
                } else {
                    const float2 p0 = turned_pair(u[k].x, v[k].x, t[0]), p1 = turned_pair(u[k].y, v[k].y, t[1]);
                    const float2 p2 = turned_pair(u[k].z, v[k].z, t[2]), p3 = turned_pair(u[k].w, v[k].w, t[3]);
                    u[k] = make_float4(p0.x, p1.x, p2.x, p3.x);
                    v[k] = make_float4(p0.y, p1.y, p2.y, p3.y);
                }
                *reinterpret_cast<float4 *>(y + b) = v[k];
            }
            *reinterpret_cast<float4 *>(y + a) = u[k];
        }
    } else {
        for (int i = threadIdx.x; i < half; i += ROPE_THREADS) turn[i] = turn_of(P.pos[tok], P.freq[i], (double)P.amplitude);
        __syncthreads();
        for (int item = first + (int)threadIdx.x; item < last; item += ROPE_THREADS) {
            const int head = item / each, i = item - head * each;
            const float *x;
            float *y;
            int a, b;
            row(head, x, y);
            place(i, a, b);
            if (b >= 0) {
                const float2 p = turned_pair(x[a], x[b], turn[i]);
                y[a] = p.x;
                y[b] = p.y;
            } else {
                y[a] = x[a];
            }
        }
    }
}

}  // namespace b200
