// Stable counting sort of integers by one digit, the base of the sort of tokens and of the experts' order.
//
// A tile of TILE consecutive items belongs to one block. Three steps: every block counts its digits; the counts of a digit are
// added up over the blocks (exclusive), and their total per digit; every block then knows where its items of a digit begin
// and gives each item its rank among the block's items of that digit, in the items' order. Nothing depends on the order in
// which blocks or threads run, so the result is the same every time.
#pragma once
#include "common.cuh"

namespace qmlp {
namespace kernel {
namespace ops {

constexpr int PARTITION_THREADS = 256, PARTITION_WARPS = PARTITION_THREADS / 32;
constexpr int PARTITION_MAX_DIGITS = 1024;

// Ranks of one tile: items `item(i)` -> digit (or -1: no item) for i in [0, ITEMS * 256), in order; warp w holds the items
// [w * ITEMS * 32, (w + 1) * ITEMS * 32). `counts` (warps x digits ints in shared memory) is left with the number of items of
// a digit in the warps before, `rank` with an item's rank within its warp. All threads of the block call it.
template <int ITEMS, class F>
__device__ __forceinline__ void tileRanks(F&& item, int digits, int* counts, int (&digit)[ITEMS], int (&rank)[ITEMS])
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < PARTITION_WARPS * digits; i += PARTITION_THREADS) counts[i] = 0;
    __syncthreads();
    int* mine = counts + warp * digits;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int d = item((warp * ITEMS + k) * 32 + lane);
        const unsigned same = __match_any_sync(0xffffffffu, d);
        const int before = d >= 0 ? mine[d] : 0;
        __syncwarp();
        digit[k] = d;
        rank[k] = before + __popc(same & ((1u << lane) - 1));
        if (d >= 0 && lane == 31 - __clz(same)) mine[d] = before + __popc(same);
        __syncwarp();
    }
    __syncthreads();
}
// counts (warps x digits) -> items of the digit in the warps before; returns the block's count of digit `d`
__device__ __forceinline__ int warpOffsets(int* counts, int digits, int d, int start)
{
    int sum = start;
#pragma unroll
    for (int w = 0; w < PARTITION_WARPS; ++w) {
        const int c = counts[w * digits + d];
        counts[w * digits + d] = sum;
        sum += c;
    }
    return sum - start;
}

// exclusive sums of up to 1024 ints by one block of 256 threads: values in `v` (shared, n ints) are replaced; `warpSums`: 8 ints.
// Returns the total to every thread.
__device__ __forceinline__ int blockExclusive(int* v, int n, int* warpSums)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int own[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = threadIdx.x * 4 + i;
        own[i] = k < n ? v[k] : 0;
        sum += own[i];
    }
    int inclusive = sum;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int up = __shfl_up_sync(0xffffffffu, inclusive, o);
        if (lane >= o) inclusive += up;
    }
    if (lane == 31) warpSums[warp] = inclusive;
    __syncthreads();
    int before = inclusive - sum, total = 0;
#pragma unroll
    for (int w = 0; w < PARTITION_WARPS; ++w) {
        if (w < warp) before += warpSums[w];
        total += warpSums[w];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = threadIdx.x * 4 + i;
        if (k < n) v[k] = before;
        before += own[i];
    }
    __syncthreads();
    return total;
}

// counts[digit * blocks + block] -> exclusive sums over the blocks; totals[digit]. One warp per digit.
static __global__ void __launch_bounds__(PARTITION_THREADS) partition_scan_kernel(int* __restrict__ counts, int* __restrict__ totals, int digits, int blocks)
{
    const int d = blockIdx.x * PARTITION_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (d >= digits) return;
    int* row = counts + static_cast<long long>(d) * blocks;
    int carry = 0;
    for (int b0 = 0; b0 < blocks; b0 += 128) {
        int v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = b0 + i * 32 + lane < blocks ? row[b0 + i * 32 + lane] : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int inclusive = v[i];
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int up = __shfl_up_sync(0xffffffffu, inclusive, o);
                if (lane >= o) inclusive += up;
            }
            if (b0 + i * 32 + lane < blocks) row[b0 + i * 32 + lane] = carry + inclusive - v[i];
            carry += __shfl_sync(0xffffffffu, inclusive, 31);
        }
    }
    if (lane == 0) totals[d] = carry;
}

} // namespace ops
} // namespace kernel
} // namespace qmlp
