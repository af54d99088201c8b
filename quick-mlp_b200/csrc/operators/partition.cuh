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

// lanes whose digit is this lane's (-1: no item), by a vote per bit
__device__ __forceinline__ unsigned sameDigit(int d, int bits)
{
    unsigned same = __ballot_sync(0xffffffffu, d >= 0);
    if (d < 0) same = ~same;
#pragma unroll
    for (int b = 0; b < 10; ++b) {
        if (b >= bits) break;
        const unsigned set = __ballot_sync(0xffffffffu, (d >> b) & 1);
        same &= (d >> b) & 1 ? set : ~set;
    }
    return same;
}

// Ranks of one tile: items `item(i)` -> digit (or -1: no item) for i in [0, ITEMS * 32 * WARPS), in order; warp w holds the items
// [w * ITEMS * 32, (w + 1) * ITEMS * 32). `counts` (WARPS x digits, 16 bits each, in shared memory) is left with the number of items of a digit in
// each warp, `rank` with an item's rank within its warp. All threads of the block call it; it ends in a barrier.
template <int ITEMS, int WARPS, class F>
__device__ __forceinline__ void tileRanks(F&& item, int digits, uint16_t* counts, int (&digit)[ITEMS], int (&rank)[ITEMS])
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) digit[k] = item((warp * ITEMS + k) * 32 + lane);   // (all on their way before the first is used)
    for (int i = threadIdx.x; i < (WARPS * digits + 1) / 2; i += WARPS * 32) reinterpret_cast<uint32_t*>(counts)[i] = 0;
    __syncthreads();
    uint16_t* mine = counts + warp * digits;
    const int bits = 32 - __clz(digits - 1);
    unsigned same[ITEMS];   // (votes of all items first: they do not wait for one another's counters)
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) same[k] = sameDigit(digit[k], bits);
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int d = digit[k];
        const int before = d >= 0 ? mine[d] : 0;
        __syncwarp();
        rank[k] = before + __popc(same[k] & ((1u << lane) - 1));
        if (d >= 0 && lane == 31 - __clz(same[k])) mine[d] = static_cast<uint16_t>(before + __popc(same[k]));
        __syncwarp();
    }
    __syncthreads();
}
// counts (WARPS x digits) of digit `d` -> items of the digit in the warps before; returns the block's count of it
template <int WARPS>
__device__ __forceinline__ int warpOffsets(uint16_t* counts, int digits, int d)
{
    int c[WARPS], sum = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) c[w] = counts[w * digits + d];
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        counts[w * digits + d] = static_cast<uint16_t>(sum);
        sum += c[w];
    }
    return sum;
}

// exclusive sums of up to 1024 ints by one block of at least 256 threads: values in `v` (shared, n ints) are replaced; `warpSums`: an int per warp.
// Returns the total to every thread.
template <int WARPS = PARTITION_WARPS>
__device__ __forceinline__ int blockExclusive(int* v, int n, int* warpSums)
{
    constexpr int EACH = 1024 / (WARPS * 32);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int own[EACH], sum = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int k = threadIdx.x * EACH + i;
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
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += warpSums[w];
        total += warpSums[w];
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int k = threadIdx.x * EACH + i;
        if (k < n) v[k] = before;
        before += own[i];
    }
    __syncthreads();
    return total;
}

// counts[digit * blocks + block] -> exclusive sums over the blocks, before[block * digits + digit]; totals[digit]. One thread block per digit. (Either side reads
// what it needs side by side.)
static __global__ void __launch_bounds__(PARTITION_THREADS)
    partition_scan_kernel(const int* __restrict__ counts, int* __restrict__ before, int* __restrict__ totals, int digits, int blocks)
{
    chained();
    __shared__ int warpSums[PARTITION_WARPS];
    const int d = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int* row = counts + static_cast<long long>(d) * blocks;
    int carry = 0;
    for (int b0 = 0; b0 < blocks; b0 += 4 * PARTITION_THREADS) {
        int v[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int b = b0 + static_cast<int>(threadIdx.x) * 4 + i;
            v[i] = b < blocks ? row[b] : 0;
            sum += v[i];
        }
        int inclusive = sum;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int up = __shfl_up_sync(0xffffffffu, inclusive, o);
            if (lane >= o) inclusive += up;
        }
        if (lane == 31) warpSums[warp] = inclusive;
        __syncthreads();
        int at = carry + inclusive - sum;
#pragma unroll
        for (int w = 0; w < PARTITION_WARPS; ++w) {
            if (w < warp) at += warpSums[w];
            carry += warpSums[w];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int b = b0 + static_cast<int>(threadIdx.x) * 4 + i;
            if (b < blocks) before[static_cast<long long>(b) * digits + d] = at;
            at += v[i];
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) totals[d] = carry;
}

} // namespace ops
} // namespace kernel
} // namespace qmlp
