// Sums of columns over partial sums that CTAs left behind, in a fixed order: the same bits whenever the same call is made.
#pragma once

#include "rowformat.cuh"

namespace ashb {

// out[c] = sum over i < count of partial[i][c], c < n; partial null: nothing to do.
struct Sums {
    const float* partial;
    int64_t count, n;
    void* out;
};

// A column has a thread where there are few terms.  Where there are many, 32 warps share the terms of 32 columns: with 8 of
// them and twice the terms a sum of 1184 x 64 took 15 us, all of it one round trip to memory after another.
constexpr int64_t kFewTerms = 8;
constexpr int kSumThreads = 1024;
inline unsigned sum_blocks(const Sums& s) {
    if (s.partial == nullptr) return 0;
    const int64_t columns = s.count <= kFewTerms ? kSumThreads : 32;
    return (unsigned)((s.n + columns - 1) / columns);
}

// Two sets of sums in one launch: the first first_blocks CTAs take the first.
template <class T>
__global__ void __launch_bounds__(kSumThreads) sums_kernel(const Sums first, const Sums second, unsigned first_blocks) {
    __shared__ float mine[32][33];
    const bool is_first = blockIdx.x < first_blocks;
    const Sums& s = is_first ? first : second;
    const int64_t block = is_first ? blockIdx.x : blockIdx.x - first_blocks;
    T* out = static_cast<T*>(s.out);
    if (s.count <= kFewTerms) {
        const int64_t col = block * kSumThreads + threadIdx.x;
        if (col >= s.n) return;
        float v = 0.0f;
        for (int64_t i = 0; i < s.count; ++i) v += s.partial[i * s.n + col];
        out[col] = from_float<T>(v);
        return;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t col = block * 32 + lane;
    float v = 0.0f;
    if (col < s.n) {
#pragma unroll 16
        for (int64_t i = warp; i < s.count; i += 32) v += s.partial[i * s.n + col];
    }
    mine[warp][lane] = v;
    __syncthreads();
    // warp w joins column w: lane i has the share of warp i
    v = mine[lane][warp];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0 && block * 32 + warp < s.n) out[block * 32 + warp] = from_float<T>(v);
}

template <class T>
void launch_sums(const Sums& first, const Sums& second, cudaStream_t st) {
    const unsigned a = sum_blocks(first), b = sum_blocks(second);
    if (a + b) sums_kernel<T><<<a + b, kSumThreads, 0, st>>>(first, second, a);
}

}  // namespace ashb
