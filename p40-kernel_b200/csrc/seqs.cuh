// seqs.cuh -- several sequences in one call: rows start[s] .. start[s + 1] - 1 of the call's tensors are the new tokens of sequence s.  The numbers are
// the caller's and lie on the device, so a captured call can be replayed with others; the kernels check them before they use them.
#pragma once

#include "common.cuh"

namespace b200 {

enum : int { STATUS_BAD_SEQUENCE = 3 };

// (a wait that ran out is the graver report, and stays)
__device__ __forceinline__ void bad_sequence() { atomicCAS(&g_device_status, 0, STATUS_BAD_SEQUENCE); }

struct SeqRange { int begin, n; };      // n < 0: not rows of the call
__device__ __forceinline__ SeqRange seq_range(const int32_t *start, int s, int n_tok) {
    const int a = start[s], b = start[s + 1];
    return {a, 0 <= a && a <= b && b <= n_tok ? b - a : -1};
}

// A CTA says so where a sequence's numbers are not rows of the call.
__device__ __forceinline__ void report_ranges(const int32_t *start, int n_seq, int n_tok) {
    for (int s = threadIdx.x; s < n_seq; s += blockDim.x)
        if (seq_range(start, s, n_tok).n < 0) bad_sequence();
}

// The first sequence whose rows end behind row `tok`, found by a warp, 32 sequences a step.  n_seq: none, the row is nobody's.
__device__ __forceinline__ int seq_of_row(const int32_t *start, int n_seq, int tok, int lane) {
    for (int base = 0; base < n_seq; base += 32) {
        const unsigned found = __ballot_sync(0xffffffffu, base + lane < n_seq && start[base + lane + 1] > tok);
        if (found) return base + __ffs(found) - 1;
    }
    return n_seq;
}

// Item `item` of the sequences' items, `of(new tokens)` each, one sequence's after the other's: whose it is and which of them.  Found by a warp; false: there are not as many.
template <typename F>
__device__ __forceinline__ bool seq_of_item(const int32_t *start, int n_seq, int n_tok, int item, int lane, F of, int &seq, int &which) {
    int64_t before = 0;
    for (int base = 0; base < n_seq; base += 32) {
        int64_t own = 0;
        if (base + lane < n_seq) own = of(max(0, seq_range(start, base + lane, n_tok).n));
        int64_t sum = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        const unsigned past = __ballot_sync(0xffffffffu, before + sum > (int64_t)item);
        if (past) {
            const int at = __ffs(past) - 1;
            seq = base + at;
            which = (int)((int64_t)item - before - __shfl_sync(0xffffffffu, sum - own, at));
            return true;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return false;
}

}  // namespace b200
