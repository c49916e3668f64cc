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
// Of many columns a lane takes four: 16,384 columns of 148 terms are one round of CTAs instead of four (11 us).
constexpr int64_t kManyColumns = 4096;
__host__ __device__ inline int64_t columns_of(const Sums& s) {
    return s.count <= kFewTerms ? kSumThreads : s.n >= kManyColumns && s.n % 4 == 0 ? 128 : 32;
}
inline unsigned sum_blocks(const Sums& s) { return s.partial ? (unsigned)((s.n + columns_of(s) - 1) / columns_of(s)) : 0u; }

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
    if (columns_of(s) == 128) {
        __shared__ float4 mine4[32][33];
        const int64_t col = block * 128 + 4 * lane;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (col < s.n) {
#pragma unroll 8
            for (int64_t i = warp; i < s.count; i += 32) {
                const float4 p = *reinterpret_cast<const float4*>(s.partial + i * s.n + col);
                v.x += p.x;
                v.y += p.y;
                v.z += p.z;
                v.w += p.w;
            }
        }
        mine4[warp][lane] = v;
        __syncthreads();
        v = mine4[lane][warp];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
            v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
            v.z += __shfl_xor_sync(0xffffffffu, v.z, o);
            v.w += __shfl_xor_sync(0xffffffffu, v.w, o);
        }
        const int64_t at = block * 128 + 4 * warp;
        if (lane == 0 && at < s.n) {
            out[at] = from_float<T>(v.x);
            out[at + 1] = from_float<T>(v.y);
            out[at + 2] = from_float<T>(v.z);
            out[at + 3] = from_float<T>(v.w);
        }
        return;
    }
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
