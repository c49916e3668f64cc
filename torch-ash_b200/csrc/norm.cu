// Root-mean-square norm of rows, with the addition of a residual before it and, for layers served in 8 bits, a
// quantised output after it; and its gradient.
//
//   s = x + r                                   (r optional; s is an output then)
//   y = s rstd w,   rstd = (mean(s^2) + eps)^(-1/2)
//   8 bits: the row's codes and scale by the rules of rowformat.cuh
//   gradient, with g = dy w and n = s rstd:  dx = dr = ds + rstd (g - n mean(g n)),   dw = sum over rows of dy n
// A row that holds an infinity or a NaN is NaN throughout; one whose squares leave float32's range is normed all the same.
//
// Everything is memory traffic: each input is read once and each output written once, the row staying in the
// registers of the lanes that share it between the sum of squares, the largest magnitude and the stores.  Accesses are 16
// bytes.  Rows that are no multiples of that are taken through windows: the row's lanes walk the 16-byte words that hold it,
// whose first and last it shares with its neighbours and stores value by value (12383 rows of 3230 bf16 values with a residual and
// gradients 518 us with accesses of one value, 310 so).  Sums are
// float32; s enters the statistics before it is rounded to its type, the backward pass reads it rounded.  A row has
// 8, 32 or 256 threads by its width; rows wider than 8192 are read again for each of their passes.
// The weight's gradient is summed by a thread over the rows of its CTA, then over the CTAs in their order by a second
// small kernel: the same bits whenever the same call is made.
#include <algorithm>

#include "columnsums.cuh"
#include "rowformat.cuh"

namespace ashb {

struct NormArgs {
    const void *x, *residual, *weight;
    void *y, *sum;
    uint8_t* codes;
    float *scales, *rstd;
    int64_t rows, width, x_stride, residual_stride;
    float eps;
};

struct NormGradArgs {
    const void *dy, *dsum, *s, *weight;
    const float* rstd;
    void* dx;
    float* partial;    // [CTAs][width]
    int64_t rows, width;
    int64_t period;    // rows from one to the next that begins alike in a 16-byte word
};

// Reductions over the TPR threads of a row (a CTA of 256 threads where TPR is 256; `shared` has 2 x 8 words, used in turn).
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* shared) {
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (TPR > 32) {
        if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < TPR / 32; ++w) v += shared[w];
    }
    return v;
}
template <int TPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* shared) {
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) >> 1; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    if constexpr (TPR > 32) {
        if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int w = 0; w < TPR / 32; ++w) v = max(v, shared[w]);
    }
    return v;
}

// Rows whose squares leave the range of float32.  A sum that is not finite, or so small with its eps that squares were lost on
// the way (2^-100 and less, where a square's last place is 2^-149), is formed again of the row times a power of two that brings
// its largest value, or the root of eps if that is larger, to 2^40 (as near as 2^127 does): 2^30 squares are far from 2^128, and
// a value that the factor would make subnormal is 2^-166 of the largest, whose normed value no type holds.
constexpr float kLeastMean = 0x1p-100f;
__device__ __forceinline__ bool out_of_range(float mean) { return !(mean >= kLeastMean && mean <= 3.402823466e38f); }     // of eps and all
__device__ __forceinline__ float row_factor(uint32_t amax, float eps) {
    const uint32_t field = __float_as_uint(fmaxf(__uint_as_float(amax), sqrtf(eps))) >> 23;      // 0: of a row of zeros too
    return __uint_as_float(min(294u - min(field, 254u), 254u) << 23);
}
// 1 / sqrt(mean + eps) of the row times `factor`; a row that holds an infinity or a NaN has none.
__device__ __forceinline__ float factored_rstd(uint32_t amax, float squares, int64_t width, float eps, float factor) {
    return amax >= kInfBits ? __uint_as_float(0x7FC00000u) : 1.0f / sqrtf(squares / (float)width + eps * factor * factor);
}

// VEC values of a row at p from column `col`, which may begin before the row or end behind it (WINDOW): what is not the row's is
// zero.  `whole`: the 16 bytes are the tensor's.
template <bool WINDOW, class T, int VEC>
__device__ __forceinline__ void load_cols(const T* __restrict__ p, int col, int width, bool whole, float (&v)[VEC]) {
    if (!WINDOW || whole) {
        load_n<T, VEC>(p + col, v);
        if (WINDOW) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[k] = (unsigned)(col + k) < (unsigned)width ? v[k] : 0.0f;
        }
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = (unsigned)(col + k) < (unsigned)width ? to_float(p[col + k]) : 0.0f;
    }
}
template <bool WINDOW, class T, int VEC>
__device__ __forceinline__ void store_cols(T* __restrict__ p, int col, int width, const float (&v)[VEC]) {
    if (!WINDOW || (col >= 0 && col + VEC <= width)) {
        store_n<T, VEC>(p + col, v);
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            if ((unsigned)(col + k) < (unsigned)width) p[col + k] = from_float<T>(v[k]);
    }
}
// The weights of columns: through windows they lie askew, and come one by one, from L1.
template <bool WINDOW, class T, int VEC>
__device__ __forceinline__ void load_weights(const T* __restrict__ w, int col, int width, float (&v)[VEC]) {
    if constexpr (!WINDOW) {
        load_n<T, VEC>(w + col, v);
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = (unsigned)(col + k) < (unsigned)width ? to_float(__ldg(w + col + k)) : 0.0f;
    }
}

// VEC values an access (one where rows have strides or buffers are not aligned for more), NV accesses a thread.
// Eight CTAs an SM where registers allow it: 8192 rows of 4096 bf16 values with residual and 8-bit output 43 us (5.5 TB/s), 46 with
// the six that the compiler left room for, 54 with the weights fetched ahead of the sum in registers of their own.
template <class T, int VEC, int TPR, int NV, bool QUANT, bool WINDOW>
__global__ void __launch_bounds__(256, NV * VEC <= 16 && !WINDOW ? 8 : 1) norm_forward_kernel(const NormArgs a) {
    __shared__ float shared[16];
    const int sub = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    const bool live = row < a.rows;
    const T* x = static_cast<const T*>(a.x) + (live ? row * a.x_stride : 0);
    const T* r = a.residual ? static_cast<const T*>(a.residual) + (live ? row * a.residual_stride : 0) : nullptr;
    const T* w = static_cast<const T*>(a.weight);
    const int width = (int)a.width;
    const int64_t at = live ? row * a.width : 0;
    const int skew = WINDOW ? (int)(at % VEC) : 0;                                              // columns before the row in its first word
    const int behind = (int)min(a.rows * a.width - at, (int64_t)1 << 20);                       // first column behind the tensor
    float v[NV][VEC];
    float squares = 0.0f;
    const auto column = [&](int j) { return (j * TPR + sub) * VEC - skew; };
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int col = column(j);
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[j][k] = 0.0f;
        if (live && col < width) load_cols<WINDOW, T, VEC>(x, col, width, col + VEC <= behind, v[j]);
    }
    if (r != nullptr) {
        T* s = static_cast<T*>(a.sum) + at;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = column(j);
            if (live && col < width) {
                float u[VEC];
                load_cols<WINDOW, T, VEC>(r, col, width, col + VEC <= behind, u);
#pragma unroll
                for (int k = 0; k < VEC; ++k) v[j][k] += u[k];
                store_cols<WINDOW, T, VEC>(s, col, width, v[j]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < VEC; ++k) squares = fmaf(v[j][k], v[j][k], squares);
    squares = row_sum<TPR>(squares, shared);
    const float mean = squares / (float)a.width + a.eps;
    float rstd = 1.0f / sqrtf(mean), whole = rstd;      // of the values in registers, and of the row
    uint32_t amax = 0;
    const bool odd = out_of_range(mean);
    if (TPR > 32 ? odd : __any_sync(0xffffffffu, odd)) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < VEC; ++k) amax = max(amax, magnitude_bits(v[j][k]));
        amax = row_max<TPR>(amax, reinterpret_cast<uint32_t*>(shared) + 8);
        const float factor = odd ? row_factor(amax, a.eps) : 1.0f;
        squares = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                v[j][k] *= factor;
                squares = fmaf(v[j][k], v[j][k], squares);
            }
        squares = row_sum<TPR>(squares, shared);
        if (odd) {
            rstd = factored_rstd(amax, squares, a.width, a.eps, factor);
            whole = rstd * factor;
        }
        amax = 0;
    }
    if (a.rstd != nullptr && live && sub == 0) a.rstd[row] = whole;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int col = column(j);
        if (live && col < width) {
            float u[VEC];
            load_weights<WINDOW, T, VEC>(w, col, width, u);
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[j][k] = v[j][k] * rstd * u[k];
            if constexpr (QUANT) {
#pragma unroll
                for (int k = 0; k < VEC; ++k)      // not of columns beside the row: there a rstd of infinity makes NaN of zero
                    if (!WINDOW || (col + k >= 0 && col + k < width)) amax = max(amax, magnitude_bits(v[j][k]));
            } else {
                store_cols<WINDOW, T, VEC>(static_cast<T*>(a.y) + at, col, width, v[j]);
            }
        }
    }
    if constexpr (QUANT) {
        amax = row_max<TPR>(amax, reinterpret_cast<uint32_t*>(shared) + 8);
        if (!live) return;
        const RowScale q(amax, kFormatE4M3);
        if (sub == 0) a.scales[row] = q.scale;
        uint8_t* codes = a.codes + at;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = column(j);
            if (col >= width) continue;
            if constexpr (VEC == 1) {
                const float u[4] = {v[j][0], 0.0f, 0.0f, 0.0f};
                codes[col] = (uint8_t)encode4(u, q.inverse, kFormatE4M3);
            } else {
                uint32_t c[VEC / 4];
#pragma unroll
                for (int h = 0; h < VEC / 4; ++h) {
                    const float u[4] = {v[j][4 * h], v[j][4 * h + 1], v[j][4 * h + 2], v[j][4 * h + 3]};
                    c[h] = encode4(u, q.inverse, kFormatE4M3);
                }
                if (!WINDOW || (col >= 0 && col + VEC <= width)) {
                    if constexpr (VEC == 8) *reinterpret_cast<uint2*>(codes + col) = make_uint2(c[0], c[1]);
                    else *reinterpret_cast<uint32_t*>(codes + col) = c[0];
                } else {
#pragma unroll
                    for (int k = 0; k < VEC; ++k)
                        if (col + k >= 0 && col + k < width) codes[col + k] = (uint8_t)(c[k / 4] >> (8 * (k % 4)));
                }
            }
        }
    }
}

// Rows beyond what registers hold: a CTA a row, x (and the residual) read once a pass.
template <class T, bool QUANT>
__global__ void __launch_bounds__(256) norm_forward_long_kernel(const NormArgs a) {
    __shared__ float shared[16];
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* r = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    const T* w = static_cast<const T*>(a.weight);
    const auto value = [&](int64_t c) { return to_float(x[c]) + (r ? to_float(r[c]) : 0.0f); };
    float squares = 0.0f;
    for (int64_t c = threadIdx.x; c < a.width; c += 256) {
        const float v = value(c);
        squares = fmaf(v, v, squares);
    }
    squares = row_sum<256>(squares, shared);
    const float mean = squares / (float)a.width + a.eps;
    float rstd = 1.0f / sqrtf(mean), factor = 1.0f;
    uint32_t amax = 0;
    if (out_of_range(mean)) {
        for (int64_t c = threadIdx.x; c < a.width; c += 256) amax = max(amax, magnitude_bits(value(c)));
        amax = row_max<256>(amax, reinterpret_cast<uint32_t*>(shared) + 8);
        factor = row_factor(amax, a.eps);
        squares = 0.0f;
        for (int64_t c = threadIdx.x; c < a.width; c += 256) {
            const float v = value(c) * factor;
            squares = fmaf(v, v, squares);
        }
        rstd = factored_rstd(amax, row_sum<256>(squares, shared), a.width, a.eps, factor);
        amax = 0;
    }
    if (a.rstd != nullptr && threadIdx.x == 0) a.rstd[row] = rstd * factor;
    for (int64_t c = threadIdx.x; c < a.width; c += 256) {
        const float v = value(c), y = v * factor * rstd * to_float(w[c]);
        amax = max(amax, magnitude_bits(y));
        if constexpr (!QUANT) {
            static_cast<T*>(a.y)[row * a.width + c] = from_float<T>(y);
            if (r) static_cast<T*>(a.sum)[row * a.width + c] = from_float<T>(v);
        }
    }
    if constexpr (QUANT) {
        amax = row_max<256>(amax, reinterpret_cast<uint32_t*>(shared) + 8);
        const RowScale q(amax, kFormatE4M3);
        if (threadIdx.x == 0) a.scales[row] = q.scale;
        for (int64_t c = threadIdx.x; c < a.width; c += 256) {
            const float v = value(c);
            const float u[4] = {v * factor * rstd * to_float(w[c]), 0.0f, 0.0f, 0.0f};
            a.codes[row * a.width + c] = (uint8_t)encode4(u, q.inverse, kFormatE4M3);
            if (r) static_cast<T*>(a.sum)[row * a.width + c] = from_float<T>(v);
        }
    }
}

// Rows in turn, so that a thread keeps the weight's gradient of its columns in registers.  With 32 columns a thread, and through
// windows with 16, s, g, ds and dw spill (16-bit rows of 513 to 1024 values 200 bytes a thread, as windows 360): fewer columns would
// take a second CTA's or warp's sums per row.  Through windows the columns of a
// thread depend on where its row begins in a 16-byte word: a group takes rows that begin alike, `period` apart.
template <class T, int VEC, int TPR, int NV, bool WINDOW>
__global__ void __launch_bounds__(256, NV * VEC <= 8 ? 4 : NV * VEC <= 16 ? 3 : 2) norm_backward_kernel(const NormGradArgs a) {
    __shared__ float shared[16];
    extern __shared__ float columns[];     // width: the CTA's sums
    constexpr int kGroups = 256 / TPR;
    const int sub = threadIdx.x % TPR, group = threadIdx.x / TPR;
    const T* w = static_cast<const T*>(a.weight);
    const int64_t groups = (int64_t)gridDim.x * kGroups, me = (int64_t)blockIdx.x * kGroups + group;      // a multiple of 8
    const int64_t start = WINDOW ? me % a.period : 0, step = WINDOW ? a.period : 1;
    const int skew = WINDOW ? (int)(start * a.width % VEC) : 0, width = (int)a.width;
    float dw[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < VEC; ++k) dw[j][k] = 0.0f;
    const auto column = [&](int j) { return (j * TPR + sub) * VEC - skew; };
    int turn = 0;
    // as many rounds for every group, that the lanes of a warp and the threads of a CTA stay together
    const int64_t rounds = (a.rows + groups - 1) / groups + (WINDOW ? 1 : 0);
    for (int64_t round = 0; round < rounds; ++round) {
        const int64_t row = start + step * (me / step + round * (groups / step));
        const bool live = row < a.rows;
        const int64_t at = live ? row * a.width : 0;
        const int behind = (int)min(a.rows * a.width - at, (int64_t)1 << 20);
        const float rstd = live ? a.rstd[row] : 0.0f;
        // all that the row needs at once: what is added at the end would be another round trip to memory after the sum
        float s[NV][VEC], g[NV][VEC], ds[NV][VEC];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = column(j);
#pragma unroll
            for (int k = 0; k < VEC; ++k) s[j][k] = g[j][k] = ds[j][k] = 0.0f;
            if (live && col < width) {
                load_cols<WINDOW, T, VEC>(static_cast<const T*>(a.s) + at, col, width, col + VEC <= behind, s[j]);
                load_cols<WINDOW, T, VEC>(static_cast<const T*>(a.dy) + at, col, width, col + VEC <= behind, g[j]);
                if (a.dsum != nullptr)
                    load_cols<WINDOW, T, VEC>(static_cast<const T*>(a.dsum) + at, col, width, col + VEC <= behind, ds[j]);
            }
        }
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = column(j);
            if (col < width) {
                float u[VEC];
                load_weights<WINDOW, T, VEC>(w, col, width, u);
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    s[j][k] *= rstd;      // before it is multiplied: the normed value is in range whatever s is
                    dw[j][k] = fmaf(g[j][k], s[j][k], dw[j][k]);
                    g[j][k] *= u[k];
                    dot = fmaf(g[j][k], s[j][k], dot);
                }
            }
        }
        // the sums of two rows in turn go through different words: no second barrier
        dot = row_sum<TPR>(dot, shared + 8 * turn);
        turn ^= 1;
        const float c = dot / (float)a.width;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = column(j);
            if (live && col < width) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) ds[j][k] += rstd * fmaf(-s[j][k], c, g[j][k]);
                store_cols<WINDOW, T, VEC>(static_cast<T*>(a.dx) + at, col, width, ds[j]);
            }
        }
    }
    // the groups of the CTA add to its sums one after another
    for (int owner = 0; owner < kGroups; ++owner) {
        if (group == owner) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const int col = column(j) + k;
                    if (col >= 0 && col < width) columns[col] = owner == 0 ? dw[j][k] : columns[col] + dw[j][k];
                }
        }
        __syncthreads();
    }
    for (int64_t col = threadIdx.x; col < width; col += 256) a.partial[blockIdx.x * a.width + col] = columns[col];
}

// Rows beyond registers: a CTA a row in turn, the CTA's sums in its row of `partial` from the start.
template <class T>
__global__ void __launch_bounds__(256) norm_backward_long_kernel(const NormGradArgs a) {
    __shared__ float shared[16];
    const T* w = static_cast<const T*>(a.weight);
    float* sums = a.partial + blockIdx.x * a.width;
    for (int64_t c = threadIdx.x; c < a.width; c += 256) sums[c] = 0.0f;
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* s = static_cast<const T*>(a.s) + row * a.width;
        const T* dy = static_cast<const T*>(a.dy) + row * a.width;
        const T* ds = a.dsum ? static_cast<const T*>(a.dsum) + row * a.width : nullptr;
        const float rstd = a.rstd[row];
        float dot = 0.0f;
        for (int64_t c = threadIdx.x; c < a.width; c += 256) {
            const float n = to_float(s[c]) * rstd, dv = to_float(dy[c]);
            sums[c] = fmaf(dv, n, sums[c]);
            dot = fmaf(dv * to_float(w[c]), n, dot);
        }
        dot = row_sum<256>(dot, shared + 8 * turn);
        turn ^= 1;
        const float q = dot / (float)a.width;
        for (int64_t c = threadIdx.x; c < a.width; c += 256) {
            const float d = rstd * fmaf(-to_float(s[c]) * rstd, q, to_float(dy[c]) * to_float(w[c]));
            static_cast<T*>(a.dx)[row * a.width + c] = from_float<T>(ds ? to_float(ds[c]) + d : d);
        }
    }
}

// ---- launches ----------------------------------------------------------------------------------------------------
constexpr int64_t kLongRow = 8192;

// Threads a row and accesses a thread for a width: as few threads as keep 32 values or less each, so that narrow rows
// leave no lane idle; the largest NV of a vector width is 32 / VEC.  A window may be a word longer than its row.
constexpr int64_t kNarrowRow = 64, kWideRow = 1024;      // of eight threads and of a warp at most
static int threads_of(int64_t width, int vec, bool window) {
    const int64_t most = width + (window ? vec - 1 : 0);
    return most <= kNarrowRow ? 8 : most <= kWideRow ? 32 : 256;
}
// Whether rows of any width have TPR threads with NV accesses of VEC values, so that only those are compiled.
constexpr bool is_taken(int vec, int tpr, int nv) {
    const int64_t above = tpr == 8 ? 0 : tpr == 32 ? kNarrowRow : kWideRow, most = tpr == 8 ? kNarrowRow : tpr == 32 ? kWideRow : kLongRow;
    const int64_t covers = (int64_t)nv * vec * tpr;
    return covers > above && (nv == 1 || covers / 2 < most);
}
template <int VEC, int TPR, int NV, class F>
static void by_accesses(int nv, F&& f) {
    if constexpr (is_taken(VEC, TPR, NV))
        if (nv == NV) f(std::integral_constant<int, NV>{});
    if constexpr (NV < 32) by_accesses<VEC, TPR, 2 * NV>(nv, f);
}
template <int VEC, bool WINDOW, class F>
static void by_width(int64_t width, F&& f) {
    const int tpr = threads_of(width, VEC, WINDOW);
    int nv = 1;
    while ((int64_t)nv * VEC * tpr < width + (WINDOW ? VEC - 1 : 0)) nv <<= 1;
    const auto with = [&](auto threads) {
        by_accesses<VEC, decltype(threads)::value, 1>(nv, [&](auto accesses) { f(threads, accesses); });
    };
    if (tpr == 8) with(std::integral_constant<int, 8>{});
    else if (tpr == 32) with(std::integral_constant<int, 32>{});
    else with(std::integral_constant<int, 256>{});
}

template <class T, int VEC, bool QUANT, bool WINDOW>
static void forward_by_width(const NormArgs& a, cudaStream_t st) {
    by_width<VEC, WINDOW>(a.width, [&](auto threads, auto accesses) {
        constexpr int TPR = decltype(threads)::value, NV = decltype(accesses)::value;
        norm_forward_kernel<T, VEC, TPR, NV, QUANT, WINDOW><<<(unsigned)((a.rows + 256 / TPR - 1) / (256 / TPR)), 256, 0, st>>>(a);
    });
}

// Whether every pointer is a multiple of `bytes` (null is).
static bool aligned(uintptr_t bytes, std::initializer_list<const void*> pointers) {
    uintptr_t bits = 0;
    for (const void* p : pointers) bits |= (uintptr_t)p;
    return bits % bytes == 0;
}

template <class T>
static void forward_typed(const NormArgs& a, cudaStream_t st) {
    constexpr int kVec = 16 / sizeof(T);
    const bool based = aligned(16, {a.x, a.residual, a.weight, a.y, a.sum}) && aligned(kVec, {a.codes});
    const bool wide = based && a.width % kVec == 0 && a.x_stride % kVec == 0 && a.residual_stride % kVec == 0;
    const bool window = based && a.width >= kVec && a.width + kVec - 1 <= kLongRow && a.x_stride == a.width &&
                        (!a.residual || a.residual_stride == a.width);
    if (a.width > kLongRow) {
        if (a.codes) norm_forward_long_kernel<T, true><<<(unsigned)a.rows, 256, 0, st>>>(a);
        else norm_forward_long_kernel<T, false><<<(unsigned)a.rows, 256, 0, st>>>(a);
    } else if (wide) {
        if (a.codes) forward_by_width<T, kVec, true, false>(a, st);
        else forward_by_width<T, kVec, false, false>(a, st);
    } else if (window) {
        if (a.codes) forward_by_width<T, kVec, true, true>(a, st);
        else forward_by_width<T, kVec, false, true>(a, st);
    } else {
        if (a.codes) forward_by_width<T, 1, true, false>(a, st);
        else forward_by_width<T, 1, false, false>(a, st);
    }
}

// CTAs of the backward pass: what is resident at once, and no more than there are rows for.
// Whole multiples of eight where a CTA has one row at a time, for windows.
static unsigned backward_ctas(int64_t rows, int64_t width) {
    const int groups = 256 / threads_of(width, 8, true);
    const int64_t ctas = std::max<int64_t>(1, std::min<int64_t>((rows + groups - 1) / groups, (int64_t)sm_count() * 4));
    return (unsigned)(groups == 1 ? (ctas + 7) / 8 * 8 : ctas);
}

template <class T>
static void backward_typed(const NormGradArgs& a, unsigned grid, void* dw, cudaStream_t st) {
    constexpr int kVec = 16 / sizeof(T);
    if (a.width > kLongRow) {
        norm_backward_long_kernel<T><<<grid, 256, 0, st>>>(a);
    } else {
        const bool based = aligned(16, {a.dy, a.dsum, a.s, a.weight, a.dx});
        const auto go = [&](auto vec, auto window) {
            constexpr int VEC = decltype(vec)::value;
            constexpr bool WINDOW = decltype(window)::value;
            by_width<VEC, WINDOW>(a.width, [&](auto threads, auto accesses) {
                norm_backward_kernel<T, VEC, decltype(threads)::value, decltype(accesses)::value, WINDOW>
                        <<<grid, 256, (size_t)a.width * 4, st>>>(a);
            });
        };
        if (based && a.width % kVec == 0) go(std::integral_constant<int, kVec>{}, std::false_type{});
        else if (based && a.width >= kVec && a.width + kVec - 1 <= kLongRow) go(std::integral_constant<int, kVec>{}, std::true_type{});
        else go(std::integral_constant<int, 1>{}, std::false_type{});
    }
    launch_sums<T>(Sums{a.partial, grid, a.width, dw}, Sums{}, st);
}

}  // namespace ashb

using namespace ashb;

extern "C" {

int ashb_rms_norm_forward(int dtype, const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                          const void* weight, int64_t rows, int64_t width, float eps, void* y, uint8_t* codes,
                          float* scales, void* sum, float* rstd, void* stream) {
    ASHB_REQUIRE(is_value_type(dtype), "value type %d", dtype);
    ASHB_REQUIRE(rows >= 0 && rows <= 0x7FFFFFFF && width >= 1 && width <= 1 << 30, "%lld rows of %lld", (long long)rows,
                 (long long)width);
    if (rows == 0) return ASHB_OK;
    ASHB_REQUIRE(x && weight && (y != nullptr) != (codes != nullptr) && (codes == nullptr) == (scales == nullptr) &&
                         (residual == nullptr) == (sum == nullptr),
                 "null buffer, or neither or both kinds of output");
    ASHB_REQUIRE(x_stride >= width || rows == 1, "rows overlap");
    ASHB_REQUIRE(aligned(value_bytes(dtype), {x, residual, weight, y, sum}), "buffers not aligned to their type");
    const NormArgs a{x, residual, weight, y, sum, codes, scales, rstd, rows, width, x_stride, residual ? residual_stride : 0, eps};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == ASHB_F32) forward_typed<float>(a, st);
    else if (dtype == ASHB_F16) forward_typed<__half>(a, st);
    else forward_typed<__nv_bfloat16>(a, st);
    ASHB_LAUNCH_CHECK();
    return ASHB_OK;
}

int64_t ashb_rms_norm_workspace(int64_t rows, int64_t width) {
    if (rows <= 0 || width <= 0) return 0;
    return (int64_t)backward_ctas(rows, width) * width * (int64_t)sizeof(float);
}

int ashb_rms_norm_backward(int dtype, const void* dy, const void* dsum, const void* s, const void* weight, const float* rstd,
                           int64_t rows, int64_t width, void* dx, void* dweight, void* workspace, int64_t workspace_bytes,
                           void* stream) {
    ASHB_REQUIRE(is_value_type(dtype), "value type %d", dtype);
    ASHB_REQUIRE(rows >= 0 && rows <= 0x7FFFFFFF && width >= 1 && width <= 1 << 30, "%lld rows of %lld", (long long)rows,
                 (long long)width);
    ASHB_REQUIRE(dweight != nullptr, "null buffer");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
        ASHB_CUDA_TRY(cudaMemsetAsync(dweight, 0, (size_t)(width * value_bytes(dtype)), st));
        return ASHB_OK;
    }
    ASHB_REQUIRE(dy && s && weight && rstd && dx && workspace, "null buffer");
    ASHB_REQUIRE(workspace_bytes >= ashb_rms_norm_workspace(rows, width) && aligned(16, {workspace}), "small or unaligned workspace");
    ASHB_REQUIRE(aligned(value_bytes(dtype), {dy, dsum, s, weight, dx, dweight}), "buffers not aligned to their type");
    int64_t period = 8;      // of rows that begin alike, whatever the type: eight values are a multiple of 16 bytes
    while (period > 1 && width * (period / 2) % 8 == 0) period /= 2;
    const NormGradArgs a{dy, dsum, s, weight, rstd, dx, static_cast<float*>(workspace), rows, width, period};
    const unsigned grid = backward_ctas(rows, width);
    if (dtype == ASHB_F32) backward_typed<float>(a, grid, dweight, st);
    else if (dtype == ASHB_F16) backward_typed<__half>(a, grid, dweight, st);
    else backward_typed<__nv_bfloat16>(a, grid, dweight, st);
    ASHB_LAUNCH_CHECK();
    return ASHB_OK;
}

}  // extern "C"
