// Dense layers: y = act(x W^T + b) + r and the gradients, in one launch per matrix product.
//
//   z = x W^T + b,  y = act(z) + r                     x (rows, inputs), W (outputs, inputs)
//   dz = dy act'(z);  dx = dz W;  dW = dz^T x;  db = column sums of dz;  dr = dy
//
// One kernel computes all three products (layer_gemm_kernel), each as C[m][n] = sum_k A(m, k) B(n, k) with either
// operand's k along its rows or down them:
//     forward   A = x   (k along rows)   B = W (k along rows)
//     dx        A = dz  (k along rows)   B = W (k down the rows)
//     dW        A = dz  (k down rows)    B = x (k down the rows)
// so nothing is transposed in memory: the tensor cores take shared-memory tiles of either kind.
//
// Types.  f16 and bf16 are multiplied as they are, e4m3 with the scales of its rows applied to the sums.  float32 values
// are split exactly into three bf16 parts, v = hi + mid + lo (8 bits each), and six of the nine products are formed:
// what is left out is below 2^-22 of a term (two products of parts of 2^-7 and 2^-16).  Their sums are kept apart, hi hi in one
// accumulator and the five small ones in another, and both are added to float32 registers, rounded to nearest, every 512 values:
// the tensor cores truncate as they accumulate, which over thousands of steps would be seen in 32 bits.  (An infinity in float32
// operands becomes NaN: its mid part is infinity less infinity.)
//
// Shape of a CTA, one per SM and looping over tiles of 128 x bn: one thread fills a ring of shared-memory stages by tiled bulk
// copies, one warp issues the products, and eight or twelve warps finish the tiles before, whose sums are in tensor memory.
// Rows that bulk copies do not take are copied to ones that they do (pad_kernel); sums along k are split where there are few
// tiles (join_layer_kernel; always in the same order, no atomics).
// A layer's rows are many and few values wide as often as not: then the kernel is bound by memory, and a weight tile that
// serves every tile of a CTA is loaded once (`b_stays`).
//
// Measured (B200, 6547 GB/s and 1657 TFLOP/s bf16 measured; kernels alone, back to back): 8192 x 4096 -> 4096 bf16 with gelu and
// residual 204 us, 81 % of those; e4m3 111 us; a sine layer of 1M float32 rows 64 -> 64 143 us, 3.6 TB/s; without an activation
// 98 us, 5.2 TB/s, bf16 57 us.  Calls that do not follow one another in a burst: 241, 137 and 151 us.
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cstring>

#include "columnsums.cuh"
#include "rowformat.cuh"
#include "tensorcore.cuh"

namespace ashb {

constexpr int kRowBytes = 128;            // of a tile row: 64 values of 16 bits, 128 of 8
constexpr int kTileM = 128;
// Warps, 16 in all (128 registers): one that issues copies, one that issues products, two that idle (of float32 products six
// that split values into parts), and eight or twelve that finish tiles.
constexpr int kGemmThreads = 512, kFirstFinisher = 4, kFirstSplitFinisher = 8;
constexpr int kMaxStages = 8;
constexpr int kMaxSlots = 8;              // tiles whose sums are in tensor memory
constexpr size_t kSharedLimit = 232448;

enum Activation { kNone = ASHB_ACT_NONE, kRelu = ASHB_ACT_RELU, kSilu = ASHB_ACT_SILU, kGelu = ASHB_ACT_GELU, kSin = ASHB_ACT_SIN };

// CTAs in which a wait ran out.  What they had left to write is not written, so the host has to learn of it: by this count, for
// which it waits, and by a word of its own memory, which the next call looks at.
__device__ unsigned int g_layer_timeouts = 0;

__device__ __noinline__ void tell_timeout(unsigned int* told) {
    atomicAdd(&g_layer_timeouts, 1u);
    if (told) *static_cast<volatile unsigned int*>(told) = 1u;
    __threadfence_system();
}

// ---- activations -----------------------------------------------------------------------------------------------------
// Short and without branches, so that a block's 32 values a lane are straight code.  ROUNDED: the results are rounded to 16
// bits, and the hardware's exponential will do: e^x is off by (2 + 1.2 |x|) 2^-23 of itself, which is less than half a step of
// float16 (2^-11) wherever e^x is neither 0 nor infinite.  The quotient of silu is 0 below -87.3, where its value is 2^-119.

// sin(x + turn pi / 2), turn 0 or 1.  Reduction by a multiple k of pi in two parts (W. J. Cody, W. Waite, Software Manual for
// the Elementary Functions, 1980): k times the first part is a multiple of x's last place, so the first step is exact.
// Then an odd polynomial fitted to the sine on 1.01 times (-pi / 2, pi / 2), the largest error made least: of degree 9 it is
// 5.2e-9, of degree 7 (for results rounded to 16 bits) 9.6e-7.  Phases beyond 2^17, where a float32 phase is good to 2^-7 at
// best, take the library's reduction.
constexpr float kLongPhase = 131072.0f;
__device__ __noinline__ float long_phase(float x, int turn) { return turn ? cosf(x) : sinf(x); }

template <int TURN, bool ROUNDED>
__device__ __forceinline__ float short_phase(float x) {
    constexpr float kRound = 12582912.0f;             // 1.5 * 2^23: what is added to it is rounded to a whole number
    // cos x = (-1)^(m+1) sin(x - (m + 1/2) pi)
    const float m = TURN ? __fadd_rn(fmaf(x, 0.318309886f, -0.5f), kRound) : fmaf(x, 0.318309886f, kRound);
    const uint32_t sign = (__float_as_uint(m) << 31) ^ (TURN ? 0x80000000u : 0u);
    const float k = __fadd_rn(m, -kRound) + (TURN ? 0.5f : 0.0f);
    float r = fmaf(-k, 3.14159274f, x);               // pi rounded to float32
    r = fmaf(-k, -8.74227766e-8f, r);                 // and what that leaves
    const float u = r * r;
    float p;
    if (ROUNDED) {
        p = fmaf(u, -0.00018465964f, 0.008311534f);
        p = fmaf(u, p, -0.16665621f);
    } else {
        p = fmaf(u, 2.5970119e-06f, -0.00019805235f);
        p = fmaf(u, p, 0.008332998f);
        p = fmaf(u, p, -0.16666657f);
    }
    return __uint_as_float(__float_as_uint(fmaf(u * r, p, r)) ^ sign);
}

// act(z) and, where SLOPE, act'(z); not of a sine's long phases.
template <int ACT, bool SLOPE, bool ROUNDED>
__device__ __forceinline__ float activate_one(float omega, float z, float& slope) {
    if constexpr (ACT == kRelu) {
        if (SLOPE) slope = z > 0.0f ? 1.0f : 0.0f;
        return z < 0.0f ? 0.0f : z;      // a NaN stays
    } else if constexpr (ACT == kSilu) {
        const float p = __fdividef(1.0f, 1.0f + (ROUNDED ? __expf(-z) : expf(-z)));
        if (SLOPE) slope = p * fmaf(z, 1.0f - p, 1.0f);
        return z * p;
    } else if constexpr (ACT == kGelu) {
        // erfc(x) = t e^(-x^2) p(t), t = 1 / (1 + 0.42 x), p fitted on 0 .. 12 with the largest error made least: of degree 5 3.7e-7
        // of c, and 2^-15 of c in the tail (results rounded to 16 bits); of degree 9 2^-28 of c, to which rounded operations add
        // 6 half steps.  The tail is not made of 1 + erf, which leaves nothing of it; the exponential is the density that the slope
        // wants.
        const float x = fabsf(z) * 0.70710678f, t = __fdividef(1.0f, fmaf(0.42f, x, 1.0f));
        float p;
        if (ROUNDED) {
            p = fmaf(t, -0.16004942f, 0.4657282f);
            p = fmaf(t, p, -0.06626895f);
            p = fmaf(t, p, 0.30008131f);
            p = fmaf(t, p, 0.22261356f);
            p = fmaf(t, p, 0.23789604f);
        } else {
            p = fmaf(t, -0.0411370234f, 0.230703075f);
            p = fmaf(t, p, -0.486637957f);
            p = fmaf(t, p, 0.437143898f);
            p = fmaf(t, p, -0.19732447f);
            p = fmaf(t, p, 0.213731084f);
            p = fmaf(t, p, 0.150041524f);
            p = fmaf(t, p, 0.219894308f);
            p = fmaf(t, p, 0.23661224f);
            p = fmaf(t, p, 0.23697332f);
        }
        const float e = ROUNDED ? __expf(-x * x) : expf(-x * x), tail = 0.5f * p * t * e, c = z < 0.0f ? tail : 1.0f - tail;
        if (SLOPE) slope = fmaf(z * 0.39894228f, e, c);
        return z * c;
    } else if constexpr (ACT == kSin) {
        if (SLOPE) slope = omega * short_phase<1, ROUNDED>(omega * z);
        return short_phase<0, ROUNDED>(omega * z);
    } else {
        if (SLOPE) slope = 1.0f;
        return z;
    }
}

// What a slope is kept as for the backward pass: in float32, so that dz is rounded once (in 16 bits as well the gradients of a
// wide float16 layer are off by 3.7e-4 of their norm, 2.9e-4 so); relu's is one or zero in any type, and read by its sign.
template <class T, int ACT>
using SlopeOf = std::conditional_t<ACT == kRelu, T, float>;

// N values in place and their slopes.  Long phases are looked for once for all of them: a branch per value would keep the
// values from being worked on side by side.
template <int ACT, bool SLOPE, bool ROUNDED, int N>
__device__ __forceinline__ void activate(float omega, float (&z)[N], float (&slope)[N]) {
    if constexpr (ACT == kSin) {
        float most = 0.0f;
#pragma unroll
        for (int k = 0; k < N; ++k) most = fmaxf(most, fabsf(omega * z[k]));     // a NaN takes either way
        if (most > kLongPhase) {
#pragma unroll 1
            for (int k = 0; k < N; ++k) {
                float x = 0.0f;
#pragma unroll
                for (int j = 0; j < N; ++j) x = j == k ? omega * z[j] : x;
                const float s = long_phase(x, 0), c = SLOPE ? omega * long_phase(x, 1) : 0.0f;
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    z[j] = j == k ? s : z[j];
                    if (SLOPE) slope[j] = j == k ? c : slope[j];
                }
            }
            return;
        }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] = activate_one<ACT, SLOPE, ROUNDED>(omega, z[k], slope[k]);
}

// f(std::integral_constant<int, activation>), so that a launch runs the code of one activation: with the choice made
// value by value the sums' way out did not fit the instruction cache (a sine layer 1118 us, 40 % of it waiting for code).
template <class F>
__device__ __forceinline__ void by_activation(int activation, F&& f) {
    switch (activation) {
        case kRelu: f(std::integral_constant<int, kRelu>{}); break;
        case kSilu: f(std::integral_constant<int, kSilu>{}); break;
        case kGelu: f(std::integral_constant<int, kGelu>{}); break;
        case kSin: f(std::integral_constant<int, kSin>{}); break;
        default: f(std::integral_constant<int, kNone>{});
    }
}

// ---- the product kernel ------------------------------------------------------------------------------------------------
enum Kind { kHalf, kSplit, kEight };     // operands: 16 bits, float32 in three parts, e4m3

struct Operand {
    const void* at;
    int64_t stride;      // values between rows
};

struct Finish {          // what becomes of the sums
    const float *a_scales, *b_scales;      // e4m3: of the rows of A and B
    const void *bias, *residual;           // of out's type
    void *out, *slope;                     // slope: SlopeOf
    float* partial;                        // float32 sums instead of out: [splits][m][n]
    int64_t residual_stride;
    int type, activation, wide;            // of out; quadruples are aligned everywhere
    float omega;
};

struct GemmArgs {
    Operand a, b;
    Finish f;
    int64_t m, n, k;
    uint32_t tiles_m, tiles_n, tiles, items;             // tiles = tiles_m * tiles_n, items = tiles * splits
    uint32_t splits, blocks_k, split_blocks, block_k;    // stages along k: all, of a split; values of a stage
    uint32_t desc;
    // groups: of four finishers; places: blocks of a finisher in shared memory; columns: tensor memory to allocate
    int bn, stages, slots, groups, places, b_stays, columns;
    int raws;      // split_gemm_kernel: stages of values as they came
    int bulk_out, bufs;      // finishing by bulk copies, from this many blocks in turn
    int64_t finish_bytes;    // of shared memory, a finisher's
    uint32_t slope_bytes;    // of a block of slopes there
    int polls;               // of a wait
    unsigned int* told;      // the host's word for waits that ran out (may be null)
};

__device__ __forceinline__ void put16(uint32_t at, uint4 w) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
}
// Eight float32 values as a word of each of their three parts.  hi is truncated, so that the largest finite value stays finite; what follows is exact, v = hi + mid + lo.
__device__ __forceinline__ void put_parts(uint32_t at, uint32_t part, const float (&v)[8]) {
    uint32_t h[4], m[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t a = __float_as_uint(v[2 * j]), b = __float_as_uint(v[2 * j + 1]);
        h[j] = __byte_perm(a, b, 0x7632);
        const float ra = v[2 * j] - __uint_as_float(a & 0xFFFF0000u), rb = v[2 * j + 1] - __uint_as_float(b & 0xFFFF0000u);
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(m[j]) : "f"(rb), "f"(ra));
        const float la = ra - __uint_as_float(m[j] << 16), lb = rb - __uint_as_float(m[j] & 0xFFFF0000u);
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(l[j]) : "f"(lb), "f"(la));
    }
    put16(at, make_uint4(h[0], h[1], h[2], h[3]));
    put16(at + part, make_uint4(m[0], m[1], m[2], m[3]));
    put16(at + 2 * part, make_uint4(l[0], l[1], l[2], l[3]));
}

template <int KIND>
constexpr int kBlockK = KIND == kEight ? 128 : KIND == kHalf ? 64 : 32;       // values of a stage along k

// Bytes of a 16- or 8-bit operand's tile: `extent` values across, a stage's values along k.
template <bool DOWN>
__host__ __device__ constexpr uint32_t part_bytes(int extent) {
    return DOWN ? (uint32_t)((extent + 63) / 64) * 64u * kRowBytes : (uint32_t)extent * kRowBytes;
}

// Order of the tiles: bands of 8 rows of tiles, down the band first, so that the tiles in flight share operands in L2.
// In 32 bits throughout: with 64-bit quotients per stage and tile the threads that issue copies and products spent more time
// dividing than anything else.
struct Tile {
    int m, n, split, blocks;      // blocks: stages along k
    int64_t k0;
};
__device__ __forceinline__ Tile tile_of(const GemmArgs& g, uint32_t item) {
    Tile t{(int)item, 0, 0, 0, 0};
    if (g.splits > 1) {
        t.split = (int)(item / g.tiles);
        item -= (uint32_t)t.split * g.tiles;
        t.m = (int)item;
    }
    if (g.tiles_n > 1) {
        const uint32_t band = item / (8u * g.tiles_n), in = item - band * 8u * g.tiles_n;
        const uint32_t high = min(8u, g.tiles_m - band * 8u);
        t.n = (int)(in / high);
        t.m = (int)(band * 8u + in - (uint32_t)t.n * high);
    }
    t.k0 = (int64_t)t.split * g.split_blocks * g.block_k;
    t.blocks = (int)min(g.split_blocks, g.blocks_k - (uint32_t)t.split * g.split_blocks);
    return t;
}

// A place in the ring of stages, or of the tiles in tensor memory, and the parity of its next phase.
struct Turn {
    int at = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next(int size) {
        if (++at == size) {
            at = 0;
            parity ^= 1u;
        }
    }
};

// The sums of a warp's 32 x 32 block, from registers (a row a thread) through shared memory to memory (rows whole).
__device__ __forceinline__ void put_block(float* block, int lane, const float (&r)[32]) {
#pragma unroll
    for (int q = 0; q < 8; ++q)
        *reinterpret_cast<float4*>(block + lane * 32 + ((q ^ (lane & 7)) << 2)) =
                make_float4(r[4 * q], r[4 * q + 1], r[4 * q + 2], r[4 * q + 3]);
}

__device__ __forceinline__ void add_block(const float* block, int lane, float (&r)[32]) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        const float4 s = *reinterpret_cast<const float4*>(block + lane * 32 + ((q ^ (lane & 7)) << 2));
        r[4 * q] += s.x;
        r[4 * q + 1] += s.y;
        r[4 * q + 2] += s.z;
        r[4 * q + 3] += s.w;
    }
}

// What a lane of finish_wide wants besides the sums, fetched before they are waited for: its columns' bias and scales, and the
// residuals of the first four of its eight passes.
template <class T>
struct Ahead {
    using Four = typename Word<4 * sizeof(T)>::type;
    Four bias, residual[4];
    float4 scales;
    __device__ __forceinline__ void fetch(const Finish& f, int lane, int64_t row0, int64_t col0, int64_t m, int64_t n) {
        if (!f.wide) return;
        const int64_t col = col0 + 4 * (lane & 7);
        if (col >= n) return;
        if (f.bias) bias = __ldg(reinterpret_cast<const Four*>(static_cast<const T*>(f.bias) + col));
        if (f.b_scales) scales = __ldg(reinterpret_cast<const float4*>(f.b_scales + col));
        if (f.residual) {
            const int64_t row = row0 + (lane >> 3);
            const T* p = static_cast<const T*>(f.residual) + row * f.residual_stride + col;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (row + 4 * i < m) residual[i] = __ldg(reinterpret_cast<const Four*>(p + 4 * i * f.residual_stride));
        }
    }
};

// Four values a lane, four rows a pass, two passes a round.  A loop, so that its code stays where instructions are fetched
// from (in one piece of eight passes half of the cycles went by waiting for code), with the next round's sums and the round
// after that's residuals under way: what a round stores may be the same memory for all that the compiler knows, so a read
// written after it would wait for it.
template <class T, int ACT, bool SLOPE>
__device__ __forceinline__ void finish_wide(const Finish& f, const float* block, Ahead<T>& ahead, int lane, int64_t row0,
                                            int64_t col0, int64_t m, int64_t n) {
    constexpr bool kRounded = sizeof(T) == 2;
    const int q = lane & 7, sub = lane >> 3;
    const int64_t col = col0 + 4 * q;
    if (col >= n) return;
    float b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (f.bias) {
        const T* t = reinterpret_cast<const T*>(&ahead.bias);
#pragma unroll
        for (int k = 0; k < 4; ++k) b[k] = to_float(t[k]);
    }
    const int left = (int)min((int64_t)32, m - row0) - sub;      // of this lane's rows, four apart
    T* out = static_cast<T*>(f.out) + (row0 + sub) * n + col;
    using S = SlopeOf<T, ACT>;
    S* slopes = SLOPE ? static_cast<S*>(f.slope) + (row0 + sub) * n + col : nullptr;
    const T* residual = f.residual ? static_cast<const T*>(f.residual) + (row0 + sub + 16) * f.residual_stride + col : nullptr;
    const float* scale = f.b_scales ? f.a_scales + row0 + sub : nullptr;
    // rows sub and sub + 4 of every eight: two places in the block, a round 8 rows on
    const float4* at0 = reinterpret_cast<const float4*>(block + sub * 32 + ((q ^ sub) << 2));
    const float4* at1 = reinterpret_cast<const float4*>(block + (sub + 4) * 32 + ((q ^ (sub + 4)) << 2));
    float4 next[2] = {at0[0], at1[0]};
#pragma unroll 1
    for (int in = 0; in < 32; in += 8) {      // rows beyond the last are worked on and not stored
        float z[2][4] = {{next[0].x, next[0].y, next[0].z, next[0].w}, {next[1].x, next[1].y, next[1].z, next[1].w}}, d[2][4];
        if (in < 24) {
            next[0] = at0[(in + 8) * 8];
            next[1] = at1[(in + 8) * 8];
        }
        if (scale) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const float sa = in + 4 * p < left ? __ldg(scale + in + 4 * p) : 0.0f;
                z[p][0] *= sa * ahead.scales.x;
                z[p][1] *= sa * ahead.scales.y;
                z[p][2] *= sa * ahead.scales.z;
                z[p][3] *= sa * ahead.scales.w;
            }
        }
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int k = 0; k < 4; ++k) z[p][k] += b[k];
        activate<ACT, SLOPE, kRounded>(f.omega, z[0], d[0]);
        activate<ACT, SLOPE, kRounded>(f.omega, z[1], d[1]);
        if (f.residual) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const T* r = reinterpret_cast<const T*>(&ahead.residual[p]);
#pragma unroll
                for (int k = 0; k < 4; ++k) z[p][k] += to_float(r[k]);
                ahead.residual[p] = ahead.residual[p + 2];
                if (in < 16 && in + 16 + 4 * p < left)
                    ahead.residual[p + 2] = __ldg(reinterpret_cast<const typename Ahead<T>::Four*>(residual + 4 * p * f.residual_stride));
            }
            residual += 8 * f.residual_stride;
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            if (in + 4 * p < left) {
                if (SLOPE) store_n<S, 4>(slopes + 4 * p * n, d[p]);
                store_n<T, 4>(out + 4 * p * n, z[p]);
            }
        }
        out += 8 * n;
        if (SLOPE) slopes += 8 * n;
    }
}

// A value a lane, a row a pass; eight rows' values are read before any is stored.
template <class T, int ACT, bool SLOPE>
__device__ __forceinline__ void finish_narrow(const Finish& f, const float* block, int lane, int64_t row0, int64_t col0, int64_t m,
                                              int64_t n) {
    constexpr bool kRounded = sizeof(T) == 2;
    const int64_t col = col0 + lane;
    if (col >= n) return;
    const float b = f.bias ? to_float(static_cast<const T*>(f.bias)[col]) : 0.0f, sb = f.b_scales ? f.b_scales[col] : 1.0f;
    const int left = (int)min((int64_t)32, m - row0);
    T* out = static_cast<T*>(f.out) + row0 * n + col;
    using S = SlopeOf<T, ACT>;
    S* slopes = SLOPE ? static_cast<S*>(f.slope) + row0 * n + col : nullptr;
    const T* residual = f.residual ? static_cast<const T*>(f.residual) + row0 * f.residual_stride + col : nullptr;
#pragma unroll 1
    for (int first = 0; first < left; first += 8) {
        float z[8], d[8], r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int in = first + i, row = min(in, left - 1);
            z[i] = block[in * 32 + (((lane >> 2) ^ (in & 7)) << 2) + (lane & 3)];
            if (f.b_scales) z[i] *= f.a_scales[row0 + row] * sb;
            z[i] += b;
            r[i] = residual ? to_float(residual[row * f.residual_stride]) : 0.0f;
        }
        activate<ACT, SLOPE, kRounded>(f.omega, z, d);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (first + i < left) {
                if (SLOPE) *slopes = from_float<S>(d[i]);
                *out = from_float<T>(z[i] + r[i]);
            }
            out += n;
            if (SLOPE) slopes += n;
        }
    }
}

__device__ __forceinline__ void finish_partial(const Finish& f, float* partial, const float* block, int lane, int64_t row0, int64_t col0,
                                               int64_t m, int64_t n) {
    const int64_t col = col0 + lane;
    if (col >= n) return;
    partial += row0 * n + col;
    const int left = (int)min((int64_t)32, m - row0);
    const float sb = f.b_scales ? f.b_scales[col] : 1.0f;
#pragma unroll
    for (int first = 0; first < 32; first += 8) {
        float z[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int in = first + i;
            z[i] = block[in * 32 + (((lane >> 2) ^ (in & 7)) << 2) + (lane & 3)];
            if (f.b_scales) z[i] *= f.a_scales[row0 + min(in, left - 1)] * sb;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (first + i < left) partial[(first + i) * n] = z[i];
    }
}

template <class T, int ACT, bool SLOPE>
__device__ __forceinline__ void finish_as(const GemmArgs& g, const float* block, Ahead<T>& r, int lane, int64_t row0,
                                          int64_t col0) {
    if (g.f.wide) finish_wide<T, ACT, SLOPE>(g.f, block, r, lane, row0, col0, g.m, g.n);
    else finish_narrow<T, ACT, SLOPE>(g.f, block, lane, row0, col0, g.m, g.n);
}

// FORWARD: the layer's own product; the gradients' have no activation.
template <int KIND, bool FORWARD, class T>
__device__ __forceinline__ void finish_typed(const GemmArgs& g, const float* block, Ahead<T>& r, int lane,
                                             int64_t row0, int64_t col0) {
    if constexpr (!FORWARD) {
        finish_as<T, kNone, false>(g, block, r, lane, row0, col0);
    } else {
        by_activation(g.f.activation, [&](auto act) {
            constexpr int ACT = decltype(act)::value;
            if constexpr (KIND != kEight && ACT != kNone) {
                if (g.f.slope) {
                    finish_as<T, ACT, true>(g, block, r, lane, row0, col0);
                    return;
                }
            }
            finish_as<T, ACT, false>(g, block, r, lane, row0, col0);
        });
    }
}

// What is fetched ahead is in words: of 16-bit values held as bf16 whichever of the two they are.
template <int KIND>
struct AheadOf { using type = Ahead<__nv_bfloat16>; };
template <>
struct AheadOf<kSplit> { using type = Ahead<float>; };

template <class T>
__device__ __forceinline__ Ahead<T> as_type(const Ahead<__nv_bfloat16>& a) {
    Ahead<T> t;
    t.bias = a.bias;
    t.scales = a.scales;
#pragma unroll
    for (int i = 0; i < 4; ++i) t.residual[i] = a.residual[i];
    return t;
}

template <int KIND, bool FORWARD>
__device__ __forceinline__ void finish(const GemmArgs& g, const float* block, typename AheadOf<KIND>::type& r, int lane,
                                       int64_t row0, int64_t col0, int split) {
    if (g.f.partial) {
        finish_partial(g.f, g.f.partial + split * g.m * g.n, block, lane, row0, col0, g.m, g.n);
        return;
    }
    if constexpr (KIND == kSplit) {
        finish_typed<KIND, FORWARD, float>(g, block, r, lane, row0, col0);
    } else {
        if constexpr (KIND == kEight) {
            if (g.f.type == ASHB_F32) {
                Ahead<float> wide;
                wide.fetch(g.f, lane, row0, col0, g.m, g.n);
                finish_typed<KIND, FORWARD, float>(g, block, wide, lane, row0, col0);
                return;
            }
        }
        if (g.f.type == ASHB_F16) {
            Ahead<__half> h = as_type<__half>(r);
            finish_typed<KIND, FORWARD, __half>(g, block, h, lane, row0, col0);
        } else finish_typed<KIND, FORWARD, __nv_bfloat16>(g, block, r, lane, row0, col0);
    }
}

// ---- finishing by bulk copies -------------------------------------------------------------------------------------------
// Where rows of the output (and slope and residual) are multiples of 16 bytes: a lane keeps the row of the tile that tensor
// memory gives it, takes the columns' biases from shared memory, where all lanes read the same word, writes its row to a
// swizzled block there and one lane sends the block off as a tile; residuals come in the same way, into the block they leave
// from.  No addresses, no bounds and no second pass through shared memory: a third of the instructions of a block that leaves
// by stores of its own.
struct FinishMaps {
    CUtensorMap out, slope, residual;
};

template <class T>
__device__ __forceinline__ uint32_t block_word(uint32_t row, int lane, int word) {      // 16-byte word of a lane's row
    return row + (uint32_t)((word ^ (sizeof(T) == 4 ? lane & 7 : (lane >> 1) & 3)) << 4);
}
__device__ __forceinline__ uint4 get_word(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
// Eight values of a lane's row, from column 8 j.
template <class T>
__device__ __forceinline__ void put_eight(uint32_t row, int lane, int j, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        put16(block_word<T>(row, lane, 2 * j), make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])));
        put16(block_word<T>(row, lane, 2 * j + 1), make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])));
    } else {
        uint4 w;
        T* t = reinterpret_cast<T*>(&w);
#pragma unroll
        for (int k = 0; k < 8; ++k) t[k] = from_float<T>(v[k]);
        put16(block_word<T>(row, lane, j), w);
    }
}
template <class T>
__device__ __forceinline__ void add_eight(uint32_t row, int lane, int j, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const uint4 a = get_word(block_word<T>(row, lane, 2 * j)), b = get_word(block_word<T>(row, lane, 2 * j + 1));
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] += __uint_as_float(w[k]);
    } else {
        const uint4 a = get_word(block_word<T>(row, lane, j));
        const T* t = reinterpret_cast<const T*>(&a);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] += to_float(t[k]);
    }
}

// 32 columns of the warp's lanes, from tensor memory to the blocks at `out` and `slope`.  A short loop: its code stays where
// instructions are fetched from.  columns: the biases (and e4m3 scales, 128 bytes on) of the columns.
template <int KIND, class T, int ACT, bool SLOPE>
__device__ __forceinline__ void bulk_block(const GemmArgs& g, uint32_t sums, uint32_t out, uint32_t slope, uint32_t columns, float row_scale,
                                           int lane) {
    const bool has_residual = g.f.residual != nullptr, has_bias = g.f.bias != nullptr;
    using S = SlopeOf<T, ACT>;
    const uint32_t out_row = out + (uint32_t)lane * (32 * sizeof(T)), slope_row = slope + (uint32_t)lane * (32 * sizeof(S));
#pragma unroll 1
    for (int j = 0; j < 4; ++j) {
        float z[8], d[8];
        if constexpr (KIND == kSplit) {
            float small[8];
            tmem_load8_twice(sums + 8u * j, sums + (uint32_t)g.bn + 8u * j, z, small);
#pragma unroll
            for (int k = 0; k < 8; ++k) z[k] += small[k];
        } else {
            tmem_load8(sums + 8u * j, z);
        }
        if constexpr (KIND == kEight) {
            const uint4 a = get_word(columns + 128u + 32u * j), b = get_word(columns + 144u + 32u * j);
            const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int k = 0; k < 8; ++k) z[k] *= row_scale * __uint_as_float(w[k]);
        }
        if (has_bias) {
            const uint4 a = get_word(columns + 32u * j), b = get_word(columns + 16u + 32u * j);
            const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int k = 0; k < 8; ++k) z[k] += __uint_as_float(w[k]);
        }
        activate<ACT, SLOPE, sizeof(T) == 2>(g.f.omega, z, d);
        if (SLOPE) put_eight<S>(slope_row, lane, j, d);
        if (has_residual) add_eight<T>(out_row, lane, j, z);
        put_eight<T>(out_row, lane, j, z);
    }
}

template <int KIND, bool FORWARD, class T>
__device__ __forceinline__ void bulk_typed(const GemmArgs& g, uint32_t sums, uint32_t out, uint32_t slope, uint32_t columns, float row_scale,
                                           int lane) {
    if constexpr (!FORWARD) {
        bulk_block<KIND, T, kNone, false>(g, sums, out, slope, columns, row_scale, lane);
    } else {
        by_activation(g.f.activation, [&](auto act) {
            constexpr int ACT = decltype(act)::value;
            if constexpr (KIND != kEight && ACT != kNone) {
                if (g.f.slope) {
                    bulk_block<KIND, T, ACT, true>(g, sums, out, slope, columns, row_scale, lane);
                    return;
                }
            }
            bulk_block<KIND, T, ACT, false>(g, sums, out, slope, columns, row_scale, lane);
        });
    }
}

// The finishers of a kernel, by warp: `number` of 4 * groups.  scratch: this warp's blocks (g.bufs of out, then as many of
// slope) and columns; arrivals: its g.bufs barriers for residuals.  A tile's blocks of 32 columns go to the groups in turn.
template <int KIND, bool FORWARD>
__device__ __forceinline__ void finish_bulk(const GemmArgs& g, const FinishMaps& maps, int number, int lane, uint32_t tmem,
                                            uint32_t slot_columns, uint32_t sums_full, uint32_t sums_empty, uint32_t scratch,
                                            uint32_t arrivals, const Waits& waits) {
    const int quarter = threadIdx.x >> 5 & 3, n_blocks = (g.bn + 31) >> 5;
    const uint32_t block = g.f.partial || g.f.type == ASHB_F32 ? 4096u : 2048u;
    const uint32_t slopes = scratch + block * g.bufs, columns = slopes + g.slope_bytes * g.bufs;
    const bool fetches = FORWARD && g.f.residual != nullptr;
    // the next place among the groups' blocks, and how many tiles on it is
    const auto settle = [&](uint32_t& item, int& blk) {
        int tiles = 0;
        while (blk >= n_blocks) {
            blk -= n_blocks;
            item += gridDim.x;
            ++tiles;
        }
        return tiles;
    };
    const auto fetch = [&](uint32_t to, uint32_t bar, int col, int row0) {
        bar_expect(bar, block);
        tma_load_3d(to, &maps.residual, col, row0, 0, bar);
    };
    Turn slot, buf;
    uint32_t item = blockIdx.x;
    int blk = number >> 2;
    for (int n = settle(item, blk); n > 0; --n) slot.next(g.slots);
    Tile t{};
    if (item < g.items) t = tile_of(g, item);
    bool under_way = false;      // this block's residuals, fetched while the block before was worked on
    while (item < g.items) {
        const int row0 = t.m * kTileM + quarter * 32, col = t.n * g.bn + blk * 32;
        const bool inside = row0 < g.m && col < g.n;
        uint32_t next_item = item;
        int next_blk = blk + g.groups;
        const int tiles = settle(next_item, next_blk);
        Tile next = t;
        if (tiles && next_item < g.items) next = tile_of(g, next_item);
        const uint32_t out = scratch + block * buf.at, slope = slopes + g.slope_bytes * buf.at;
        const Turn here = buf;
        float row_scale = 1.0f;
        bool next_under_way = false;
        if (inside) {
            buf.next(g.bufs);
            if (lane == 0 && !under_way) {      // what left from this block has been read
                if (g.bufs == 2) tma_wait_read<1>();
                else tma_wait_read<0>();
                if (fetches) fetch(out, arrivals + 8 * here.at, col, row0);
            }
            if (fetches && g.bufs == 2 && next_item < g.items) {
                const int next_row = next.m * kTileM + quarter * 32, next_col = next.n * g.bn + next_blk * 32;
                next_under_way = next_row < g.m && next_col < g.n;
                if (next_under_way && lane == 0) {
                    tma_wait_read<0>();
                    fetch(scratch + block * buf.at, arrivals + 8 * buf.at, next_col, next_row);
                }
            }
            __syncwarp();
            if (FORWARD) {
                const int mine = col + lane;
                float b = 0.0f;
                if (g.f.bias && mine < g.n) {
                    if (g.f.type == ASHB_F32) b = __ldg(static_cast<const float*>(g.f.bias) + mine);
                    else if (g.f.type == ASHB_F16) b = to_float(static_cast<const __half*>(g.f.bias)[mine]);
                    else b = to_float(static_cast<const __nv_bfloat16*>(g.f.bias)[mine]);
                }
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(columns + 4u * lane), "f"(b) : "memory");
                if constexpr (KIND == kEight) {
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(columns + 128u + 4u * lane), "f"(mine < g.n ? __ldg(g.f.b_scales + mine) : 0.0f)
                                 : "memory");
                    row_scale = row0 + lane < g.m ? __ldg(g.f.a_scales + row0 + lane) : 0.0f;
                }
                __syncwarp();
            }
        }
        bool ok = bar_wait(sums_full + 8 * slot.at, slot.parity, waits);
        if (fetches && inside) ok = bar_wait(arrivals + 8 * here.at, here.parity, waits) && ok;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {      // the copies still under way end before the CTA does
            if (fetches && inside) bar_drain(arrivals + 8 * here.at, here.parity);
            if (next_under_way) bar_drain(arrivals + 8 * buf.at, buf.parity);
            break;
        }
        tc_fence_after();
        if (inside) {
            const uint32_t sums = tmem + (uint32_t)slot.at * slot_columns + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(blk * 32);
            if (g.f.partial) bulk_block<KIND, float, kNone, false>(g, sums, out, slope, columns, row_scale, lane);
            else if (KIND == kSplit || (KIND == kEight && g.f.type == ASHB_F32))
                bulk_typed<KIND, FORWARD, float>(g, sums, out, slope, columns, row_scale, lane);
            else if (g.f.type == ASHB_F16) bulk_typed<KIND, FORWARD, __half>(g, sums, out, slope, columns, row_scale, lane);
            else bulk_typed<KIND, FORWARD, __nv_bfloat16>(g, sums, out, slope, columns, row_scale, lane);
            tc_fence_before();
            fence_async_shared();
        }
        __syncwarp();
        if (lane == 0) {
            bar_arrive(sums_empty + 8 * slot.at);
            if (inside) {
                tma_store_3d(&maps.out, col, row0, t.split, out);
                if (FORWARD && g.f.slope) tma_store_3d(&maps.slope, col, row0, 0, slope);
                tma_commit();
            }
        }
        for (int n = tiles; n > 0; --n) slot.next(g.slots);
        item = next_item;
        blk = next_blk;
        t = next;
        under_way = next_under_way;
    }
    if (lane == 0) tma_wait_read<0>();
}

// Split products: a warp's share of a tile, the blocks `which` and `which` + 2 of 32 columns.  The two sums of a phase are added
// in registers, those of later phases to what the block holds in shared memory (`block`: 32 x 32 values, of each block where
// there are several phases).  False: a wait gave up.
template <bool FORWARD>
__device__ __forceinline__ bool finish_split(const GemmArgs& g, const Tile& t, int phase_blocks, Turn& slot, uint32_t tmem,
                                             uint32_t sums_full, uint32_t sums_empty, const Waits& waits, float* block,
                                             int quarter, int which, int lane) {
    const int n_blocks = (g.bn + 31) >> 5;
    const int64_t row0 = (int64_t)t.m * kTileM + quarter * 32, col0 = (int64_t)t.n * g.bn;
    const bool several = t.blocks > phase_blocks;
    Ahead<float> ahead;
#pragma unroll 1
    for (int b0 = 0; b0 < t.blocks; b0 += phase_blocks, slot.next(g.slots)) {
        const bool last = b0 + phase_blocks >= t.blocks;
        if (!__all_sync(0xffffffffu, bar_wait(sums_full + 8 * slot.at, slot.parity, waits))) return false;
        tc_fence_after();
        const uint32_t at = tmem + (uint32_t)(slot.at * 2 * g.bn) + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
        for (int mine = which; mine < n_blocks; mine += 2) {
            float* place = block + (several ? (mine >> 1) * 1024 : 0);
            if (FORWARD && last) ahead.fetch(g.f, lane, row0, col0 + mine * 32, g.m, g.n);
            float r[32], small[32];
            tmem_load32(at + (uint32_t)(mine * 32), r);
            tmem_load32(at + (uint32_t)(g.bn + mine * 32), small);
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] += small[j];
            if (b0 > 0) add_block(place, lane, r);
            put_block(place, lane, r);
            __syncwarp();
            if (mine + 2 >= n_blocks) {
                tc_fence_before();
                if (lane == 0) bar_arrive(sums_empty + 8 * slot.at);
            }
            if (last) {
                finish<kSplit, FORWARD>(g, place, ahead, lane, row0, col0 + mine * 32, t.split);
                __syncwarp();
            }
        }
        if (which >= n_blocks && lane == 0) bar_arrive(sums_empty + 8 * slot.at);
    }
    return true;
}

struct GemmShared {
    uint64_t full[kMaxStages], empty[kMaxStages], sums_full[kMaxSlots], sums_empty[kMaxSlots], residual[24], drained;
    uint32_t tmem;
    int gave_up;
};

// Barriers: full[s] by the copies' bytes, empty[s] by the products that read stage s, sums_full / sums_empty of the tiles in
// tensor memory.  Every role walks the same items and blocks.
template <int KIND, bool A_DOWN, bool B_DOWN>
__global__ void __launch_bounds__(kGemmThreads, 1) layer_gemm_kernel(const GemmArgs g, const __grid_constant__ CUtensorMap map_a,
                                                                     const __grid_constant__ CUtensorMap map_b,
                                                                     const __grid_constant__ FinishMaps maps) {
    extern __shared__ __align__(1024) uint8_t dynamic[];
    __shared__ GemmShared sh;
    constexpr int kBlock = kBlockK<KIND>, kStep = KIND == kEight ? 32 : 16;
    constexpr bool kForward = !A_DOWN && !B_DOWN;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_of(dynamic) + 1023u) & ~1023u;
    const uint32_t a_bytes = part_bytes<A_DOWN>(kTileM), b_bytes = part_bytes<B_DOWN>(g.bn), stage_bytes = a_bytes + b_bytes;
    float* blocks = reinterpret_cast<float*>(dynamic + (base - smem_of(dynamic)) + (size_t)stage_bytes * g.stages);
    const Waits waits{&sh.gave_up, g.polls};
    const uint32_t full = smem_of(sh.full), empty = smem_of(sh.empty);
    const uint32_t sums_full = smem_of(sh.sums_full), sums_empty = smem_of(sh.sums_empty);

    if (threadIdx.x == 0) {
        sh.gave_up = 0;
        for (int s = 0; s < g.stages; ++s) {
            bar_init(full + 8 * s, 1);
            bar_init(empty + 8 * s, 1);
        }
        for (int h = 0; h < g.slots; ++h) {
            bar_init(sums_full + 8 * h, 1);
            bar_init(sums_empty + 8 * h, 4 * ((g.bn + 31) >> 5));
        }
        for (int i = 0; i < 24; ++i) bar_init(smem_of(sh.residual) + 8 * i, 1);
        bar_init(smem_of(&sh.drained), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(smem_of(&sh.tmem), (uint32_t)g.columns);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;

    if (warp == 0) {
        if (lane == 0) {
            Turn turn;
            int fills = 0;      // up to the number of stages
            bool ok = true;
            for (uint32_t item = blockIdx.x; item < g.items && ok; item += gridDim.x) {
                const Tile t = tile_of(g, item);
                int k = (int)t.k0;
                for (int b = 0; b < t.blocks; ++b, k += kBlock, turn.next(g.stages)) {
                    if (!(ok = bar_wait(empty + 8 * turn.at, turn.parity ^ 1u, waits))) break;
                    const bool with_b = !g.b_stays || fills < g.stages;
                    if (fills < g.stages) ++fills;
                    const uint32_t tile_a = base + (uint32_t)turn.at * stage_bytes, tile_b = tile_a + a_bytes;
                    const uint32_t bar = full + 8 * turn.at;
                    bar_expect(bar, a_bytes + (with_b ? b_bytes : 0u));
                    if constexpr (A_DOWN) {
                        for (int box = 0; box < kTileM / 64; ++box)
                            tma_load_2d(tile_a + box * 64 * kRowBytes, &map_a, t.m * kTileM + box * 64, k, bar);
                    } else {
                        tma_load_2d(tile_a, &map_a, k, t.m * kTileM, bar);
                    }
                    if (with_b) {
                        if constexpr (B_DOWN) {
                            for (int box = 0; box * 64 < g.bn; ++box)
                                tma_load_2d(tile_b + box * 64 * kRowBytes, &map_b, t.n * g.bn + box * 64, k, bar);
                        } else {
                            tma_load_2d(tile_b, &map_b, k, t.n * g.bn, bar);
                        }
                    }
                }
            }
            // The copies still under way end before the CTA does: those that it has products for have ended by then, the
            // others where a wait ran out in whatever role.
            for (; fills > 0; --fills) {
                if (turn.at == 0) turn.parity ^= 1u;
                turn.at = (turn.at == 0 ? g.stages : turn.at) - 1;
                bar_drain(full + 8 * turn.at, turn.parity);
            }
        }
    } else if (warp == 1) {
        const uint32_t mine = elected();
        Turn turn, slot;
        bool ok = true;
        for (uint32_t item = blockIdx.x; item < g.items && ok; item += gridDim.x, slot.next(g.slots)) {
            const Tile t = tile_of(g, item);
            int left = (int)min((int64_t)t.blocks * kBlock, g.k - t.k0);      // values along k
            const uint32_t sums = tmem + (uint32_t)(slot.at * g.bn);
            if (!(ok = bar_wait(sums_empty + 8 * slot.at, slot.parity ^ 1u, waits))) break;
            tc_fence_after();
            bool add = false;
            for (int b = 0; b < t.blocks; ++b, left -= kBlock, turn.next(g.stages)) {
                if (!(ok = bar_wait(full + 8 * turn.at, turn.parity, waits))) break;
                tc_fence_after();
                const int steps = (min(kBlock, left) + kStep - 1) / kStep;
                const uint32_t tile_a = base + (uint32_t)turn.at * stage_bytes;
                // a step along k: 32 bytes along rows, 16 rows down them
                constexpr uint64_t a_step = (A_DOWN ? 16 * kRowBytes : 32) >> 4, b_step = (B_DOWN ? 16 * kRowBytes : 32) >> 4;
                uint64_t at = tile_desc(tile_a, 64 * kRowBytes), bt = tile_desc(tile_a + a_bytes, 64 * kRowBytes);
                for (int i = 0; i < steps; ++i, at += a_step, bt += b_step) {
                    product<KIND == kEight>(mine, sums, at, bt, g.desc, add);
                    add = true;
                }
                products_done(mine, empty + 8 * turn.at);
            }
            if (ok) products_done(mine, sums_full + 8 * slot.at);
        }
        // Tensor memory is not given back, nor shared memory left, under products still running: finishers that gave up have not
        // waited for them.
        products_done(mine, smem_of(&sh.drained));
        bar_drain(smem_of(&sh.drained), 0);
    } else if (warp >= kFirstFinisher && warp < kFirstFinisher + 4 * g.groups) {
        const int number = warp - kFirstFinisher;
        if (g.bulk_out) {
            finish_bulk<KIND, kForward>(g, maps, number, lane, tmem, (uint32_t)g.bn, sums_full, sums_empty,
                                        smem_of(blocks) + (uint32_t)(number * g.finish_bytes), smem_of(sh.residual) + 16 * number, waits);
        } else {
            // lanes of tensor memory that the warp may read; the blocks of 32 columns go to the groups in turn
            const int quarter = warp & 3, n_blocks = (g.bn + 31) >> 5;
            float* block = blocks + (size_t)number * 1024;
            Turn slot;
            Ahead<__nv_bfloat16> ahead;
            int blk = number >> 2;
            bool ok = true;
            for (uint32_t item = blockIdx.x; item < g.items && ok; item += gridDim.x, blk -= n_blocks, slot.next(g.slots)) {
                const Tile t = tile_of(g, item);
                const int64_t row0 = (int64_t)t.m * kTileM + quarter * 32, col0 = (int64_t)t.n * g.bn;
                for (; blk < n_blocks; blk += g.groups) {
                    if (kForward) ahead.fetch(g.f, lane, row0, col0 + blk * 32, g.m, g.n);
                    ok = __all_sync(0xffffffffu, bar_wait(sums_full + 8 * slot.at, slot.parity, waits));
                    if (!ok) break;
                    tc_fence_after();
                    float r[32];
                    tmem_load32(tmem + (uint32_t)(slot.at * g.bn) + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(blk * 32), r);
                    put_block(block, lane, r);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(sums_empty + 8 * slot.at);
                    finish<KIND, kForward>(g, block, ahead, lane, row0, col0 + blk * 32, t.split);
                    __syncwarp();
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_free(tmem, (uint32_t)g.columns);
    if (threadIdx.x == 0 && *waits.gave_up) tell_timeout(g.told);
}

// ---- split products from bulk copies ---------------------------------------------------------------------------------------
// The product kernel of float32 operands.  The copies bring values as they are into a ring
// of their own, 32 along k a stage, so that several tiles are under way without a register; six warps split them into the
// parts' tiles by a short loop.  Splitting on the way from registers instead took 40 registers for a tile under way and a loop
// so long that it and the finishers' did not fit the instruction cache together (1M rows 64 -> 64: 145 us, 123 this way).
constexpr int kSplitBlock = 32, kSplitPhase = 512 / kSplitBlock, kSplitters = 6;
constexpr int kMaxRaws = 6;

struct SplitShared {
    uint64_t raw_full[kMaxRaws], raw_empty[kMaxRaws], full[kMaxStages], empty[kMaxStages], sums_full[kMaxSlots],
            sums_empty[kMaxSlots], residual[24], drained;
    uint32_t tmem;
    int gave_up;
};

// Bytes of one part of a tile of `extent` values across and 32 along k.
template <bool DOWN>
__host__ __device__ constexpr uint32_t split_bytes(int extent) {
    return DOWN ? (uint32_t)((extent + 63) / 64) * 4096u : (uint32_t)extent * 64u;
}

__device__ __forceinline__ float4 get16(uint32_t at) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
    return v;
}

// Eight values a step.  Along rows: the raw tile has `extent` rows of 32 values, a part as many of 64 bytes.  Down rows: boxes of
// 32 rows of 32 values, a part boxes of 32 rows of 64.  Both sides swizzled: two lanes of eight share a bank at most.
template <bool DOWN>
__device__ __forceinline__ void split_tile(uint32_t raw, uint32_t parts, int extent, int thread) {
    const uint32_t part = split_bytes<DOWN>(extent);
#pragma unroll 2
    for (int i = thread; i < extent * 4; i += kSplitters * 32) {
        const int r = i >> 2, c = i & 3;
        const uint32_t row = raw + (uint32_t)r * 128u;      // rows of boxes follow one another too
        const float4 a = get16(row + (uint32_t)(((2 * c) ^ (r & 7)) << 4)), b = get16(row + (uint32_t)(((2 * c + 1) ^ (r & 7)) << 4));
        const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        uint32_t to;
        if (DOWN) {
            const int box = r >> 5, k = r & 31, word = (box & 1) * 4 + c;
            to = parts + (uint32_t)(box >> 1) * 4096u + (uint32_t)k * 128u + (uint32_t)((word ^ (k & 7)) << 4);
        } else {
            to = parts + (uint32_t)r * 64u + (uint32_t)((c ^ ((r >> 1) & 3)) << 4);
        }
        put_parts(to, part, v);
    }
}

template <bool A_DOWN, bool B_DOWN>
__global__ void __launch_bounds__(kGemmThreads, 1) split_gemm_kernel(const GemmArgs g, const __grid_constant__ CUtensorMap map_a,
                                                                     const __grid_constant__ CUtensorMap map_b,
                                                                     const __grid_constant__ FinishMaps maps) {
    extern __shared__ __align__(1024) uint8_t dynamic[];
    __shared__ SplitShared sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_of(dynamic) + 1023u) & ~1023u;
    const uint32_t a_part = split_bytes<A_DOWN>(kTileM), b_part = split_bytes<B_DOWN>(g.bn);
    const uint32_t raw_a = kTileM * 128u, raw_b = (uint32_t)g.bn * 128u;
    // raw stages, parts' stages, all of B's parts where it stays, the finishers' blocks
    const uint32_t raw_bytes = raw_a + (g.b_stays ? 0u : raw_b), stage_bytes = 3 * (a_part + (g.b_stays ? 0u : b_part));
    const uint32_t raws = base, stages = raws + raw_bytes * g.raws, all_b = stages + stage_bytes * g.stages;
    float* blocks = reinterpret_cast<float*>(dynamic + (all_b - smem_of(dynamic)) + (g.b_stays ? (size_t)3 * b_part * g.blocks_k : 0));
    const Waits waits{&sh.gave_up, g.polls};
    const uint32_t raw_full = smem_of(sh.raw_full), raw_empty = smem_of(sh.raw_empty), full = smem_of(sh.full),
                   empty = smem_of(sh.empty), sums_full = smem_of(sh.sums_full), sums_empty = smem_of(sh.sums_empty);

    if (threadIdx.x == 0) {
        sh.gave_up = 0;
        for (int s = 0; s < g.raws; ++s) {
            bar_init(raw_full + 8 * s, 1);
            bar_init(raw_empty + 8 * s, kSplitters);
        }
        for (int s = 0; s < g.stages; ++s) {
            bar_init(full + 8 * s, kSplitters);
            bar_init(empty + 8 * s, 1);
        }
        for (int h = 0; h < g.slots; ++h) {
            bar_init(sums_full + 8 * h, 1);
            bar_init(sums_empty + 8 * h, g.bulk_out ? 4 * ((g.bn + 31) >> 5) : 8);
        }
        for (int i = 0; i < 24; ++i) bar_init(smem_of(sh.residual) + 8 * i, 1);
        bar_init(smem_of(&sh.drained), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(smem_of(&sh.tmem), (uint32_t)g.columns);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;

    if (warp == 0) {
        if (lane == 0) {
            Turn raw;
            int fills = 0;      // up to the ring's size
            bool ok = true;
            const auto room = [&](uint32_t bytes) {
                if (!(ok = bar_wait(raw_empty + 8 * raw.at, raw.parity ^ 1u, waits))) return false;
                bar_expect(raw_full + 8 * raw.at, bytes);
                fills = min(fills + 1, g.raws);
                return true;
            };
            const auto load = [&](auto down, const CUtensorMap* map, uint32_t to, int across, int extent, int k) {
                if constexpr (decltype(down)::value) {
                    for (int box = 0; box * 32 < extent; ++box)
                        tma_load_2d(to + box * 4096, map, across + box * 32, k, raw_full + 8 * raw.at);
                } else {
                    tma_load_2d(to, map, k, across, raw_full + 8 * raw.at);
                }
            };
            if (g.b_stays)
                for (int b = 0; b < (int)g.blocks_k && ok; ++b) {
                    if (!room(raw_b)) break;
                    load(std::integral_constant<bool, B_DOWN>{}, &map_b, raws + raw.at * raw_bytes, 0, g.bn, b * kSplitBlock);
                    raw.next(g.raws);
                }
            for (uint32_t item = blockIdx.x; item < g.items && ok; item += gridDim.x) {
                const Tile t = tile_of(g, item);
                int k = (int)t.k0;
                for (int b = 0; b < t.blocks; ++b, k += kSplitBlock) {
                    if (!room(raw_bytes)) break;
                    const uint32_t to = raws + raw.at * raw_bytes;
                    load(std::integral_constant<bool, A_DOWN>{}, &map_a, to, t.m * kTileM, kTileM, k);
                    if (!g.b_stays) load(std::integral_constant<bool, B_DOWN>{}, &map_b, to + raw_a, t.n * g.bn, g.bn, k);
                    raw.next(g.raws);
                }
            }
            for (; fills > 0; --fills) {      // the copies still under way end before the CTA does
                if (raw.at == 0) raw.parity ^= 1u;
                raw.at = (raw.at == 0 ? g.raws : raw.at) - 1;
                bar_drain(raw_full + 8 * raw.at, raw.parity);
            }
        }
    } else if (warp == 1) {
        {
            const uint32_t mine = elected();
            Turn turn, slot;
            bool ok = true;
            // a step along k: 32 bytes along rows, 16 rows of 128 bytes down them
            constexpr uint64_t a_step = (A_DOWN ? 2048 : 32) >> 4, b_step = (B_DOWN ? 2048 : 32) >> 4;
            const uint64_t ap = a_part >> 4, bp = b_part >> 4;
            for (uint32_t item = blockIdx.x; item < g.items && ok; item += gridDim.x) {
                const Tile t = tile_of(g, item);
                int left = (int)min((int64_t)t.blocks * kSplitBlock, g.k - t.k0);
                for (int b0 = 0; b0 < t.blocks && ok; slot.next(g.slots)) {
                    const int b1 = min(t.blocks, b0 + kSplitPhase);
                    const uint32_t sums = tmem + (uint32_t)(slot.at * 2 * g.bn), small = sums + (uint32_t)g.bn;
                    if (!(ok = bar_wait(sums_empty + 8 * slot.at, slot.parity ^ 1u, waits))) break;
                    bool add = false;
                    for (; b0 < b1; ++b0, left -= kSplitBlock, turn.next(g.stages)) {
                        if (!(ok = bar_wait(full + 8 * turn.at, turn.parity, waits))) break;
                        tc_fence_after();
                        const uint32_t at = stages + (uint32_t)turn.at * stage_bytes;
                        const uint32_t at_b = g.b_stays ? all_b + (uint32_t)b0 * 3u * b_part : at + 3 * a_part;
                        uint64_t a = tile_desc<A_DOWN ? 128 : 64>(at, 4096), b = tile_desc<B_DOWN ? 128 : 64>(at_b, 4096);
                        const int steps = left > 16 ? 2 : 1;
                        for (int i = 0; i < steps; ++i, a += a_step, b += b_step) {
                            product<false>(mine, sums, a, b, g.desc, add);
                            product<false>(mine, small, a + 2 * ap, b, g.desc, add);
                            product<false>(mine, small, a, b + 2 * bp, g.desc, true);
                            product<false>(mine, small, a + ap, b + bp, g.desc, true);
                            product<false>(mine, small, a + ap, b, g.desc, true);
                            product<false>(mine, small, a, b + bp, g.desc, true);
                            add = true;
                        }
                        products_done(mine, empty + 8 * turn.at);
                    }
                    if (ok) products_done(mine, sums_full + 8 * slot.at);
                }
            }
            products_done(mine, smem_of(&sh.drained));      // as in layer_gemm_kernel
            bar_drain(smem_of(&sh.drained), 0);
        }
    } else if (warp < 2 + kSplitters) {
        const int thread = threadIdx.x - 64;
        Turn raw, turn;
        bool ok = true;
        // a warp is done with a raw stage, or has its share of a stage of parts in place
        const auto tell = [&](uint32_t bar) {
            __syncwarp();
            if (lane == 0) bar_arrive(bar);
        };
        if (g.b_stays)
            for (int b = 0; b < (int)g.blocks_k && ok; ++b) {
                ok = __all_sync(0xffffffffu, bar_wait(raw_full + 8 * raw.at, raw.parity, waits));
                if (!ok) break;
                split_tile<B_DOWN>(raws + raw.at * raw_bytes, all_b + (uint32_t)b * 3u * b_part, g.bn, thread);
                tell(raw_empty + 8 * raw.at);
                raw.next(g.raws);
            }
        for (uint32_t item = blockIdx.x; item < g.items && ok; item += gridDim.x) {
            const Tile t = tile_of(g, item);
            for (int b = 0; b < t.blocks && ok; ++b) {
                ok = __all_sync(0xffffffffu, bar_wait(empty + 8 * turn.at, turn.parity ^ 1u, waits) &&
                                                     bar_wait(raw_full + 8 * raw.at, raw.parity, waits));
                if (!ok) break;
                const uint32_t from = raws + raw.at * raw_bytes, to = stages + (uint32_t)turn.at * stage_bytes;
                split_tile<A_DOWN>(from, to, kTileM, thread);
                if (!g.b_stays) split_tile<B_DOWN>(from + raw_a, to + 3 * a_part, g.bn, thread);
                fence_async_shared();
                tell(raw_empty + 8 * raw.at);
                if (lane == 0) bar_arrive(full + 8 * turn.at);
                raw.next(g.raws);
                turn.next(g.stages);
            }
        }
    } else {
        const int quarter = warp & 3, which = (warp - kFirstSplitFinisher) >> 2;
        if (g.bulk_out)
            finish_bulk<kSplit, !A_DOWN && !B_DOWN>(g, maps, warp - 8, lane, tmem, 2u * g.bn, sums_full, sums_empty,
                                                    smem_of(blocks) + (uint32_t)((warp - 8) * g.finish_bytes),
                                                    smem_of(sh.residual) + 16 * (warp - 8), waits);
        float* block = blocks + (size_t)(warp - 8) * 1024 * g.places;
        Turn slot;
        for (uint32_t item = blockIdx.x; item < g.items && !g.bulk_out; item += gridDim.x) {
            const Tile t = tile_of(g, item);
            if (!finish_split<!A_DOWN && !B_DOWN>(g, t, kSplitPhase, slot, tmem, sums_full, sums_empty, waits, block, quarter, which,
                                                  lane))
                break;
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_free(tmem, (uint32_t)g.columns);
    if (threadIdx.x == 0 && *waits.gave_up) tell_timeout(g.told);
}

// ---- rows of whole words ------------------------------------------------------------------------------------------------
// Operands whose rows do not begin at multiples of 16 bytes are copied to where they do: bulk copies take no others.  Two
// operands a launch; a lane gathers a word of each of four rows.  Reading such rows by loads of the product kernels' own, as
// they once did, waits for memory at every stage along k: 500 rows 4001 -> 301 of bfloat16 134 us against 27, 67k rows 47 -> 375
// 156 against 120.  A million rows of 63 values gain nothing by the copy: bfloat16 63 -> 63 162 us both ways, float32 63 -> 64
// 121 us then and 181 now.
struct Padding {
    const void* from;
    void* to;
    int64_t rows, cols, stride, words;      // words: of a row where it goes
    int lanes;                              // of a row: the power of two that covers its words, 32 at most
    uint32_t units;                         // of work of a CTA: `lanes` words of as many rows as it has lanes for, four times
    unsigned blocks;
};
constexpr int kPadRows = 4;      // of a thread under way
template <class V>
__global__ void __launch_bounds__(256) pad_kernel(const Padding first, const Padding second) {
    constexpr int kValues = 16 / sizeof(V);
    const bool is_first = blockIdx.x < first.blocks;
    const Padding& p = is_first ? first : second;
    const int lanes = p.lanes, sub = threadIdx.x & (lanes - 1), groups = 256 / lanes;
    // in turn: the next `lanes` words of the same rows, then the next rows
    const uint32_t pieces = (uint32_t)((p.words + lanes - 1) / lanes);
    for (uint32_t unit = is_first ? blockIdx.x : blockIdx.x - first.blocks; unit < p.units; unit += p.blocks) {
        const uint32_t rows = unit / pieces;
        const int64_t row0 = (int64_t)rows * groups * kPadRows + threadIdx.x / lanes;
        const int64_t word = (int64_t)(unit - rows * pieces) * lanes + sub, col = word * kValues;
        const int left = (int)max(min(p.cols - col, (int64_t)kValues), (int64_t)0);
        uint4 w[kPadRows];
#pragma unroll
        for (int i = 0; i < kPadRows; ++i) {
            const int64_t row = row0 + i * groups;
            const V* from = static_cast<const V*>(p.from) + row * p.stride + col;
            V v[kValues];
#pragma unroll
            for (int k = 0; k < kValues; ++k) v[k] = row < p.rows && k < left ? __ldg(from + k) : (V)0;
            uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < kValues; ++k) u[k * (int)sizeof(V) / 4] |= (uint32_t)v[k] << (8 * (k * (int)sizeof(V) % 4));
            w[i] = make_uint4(u[0], u[1], u[2], u[3]);
        }
#pragma unroll
        for (int i = 0; i < kPadRows; ++i)
            if (row0 + i * groups < p.rows && word < p.words) static_cast<uint4*>(p.to)[(row0 + i * groups) * p.words + word] = w[i];
    }
}

// ---- products of few tiles -------------------------------------------------------------------------------------------------
// Where a layer has fewer tiles than the GPU has SMs its sums along k are split over several of them; the parts are added
// here, in their order, and become the layer's results (500 rows 4001 -> 301 of bfloat16
// 27 us without splits, 17 with them; of float32 104 and 32).
template <class T>
__global__ void __launch_bounds__(256) join_layer_kernel(const Finish f, const float* __restrict__ partial, int splits, int64_t m, int64_t n) {
    constexpr bool kRounded = sizeof(T) == 2;
    const int64_t total = m * n;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / n, col = i - row * n;
        float z[1] = {0.0f}, d[1];
#pragma unroll 8
        for (int s = 0; s < splits; ++s) z[0] += partial[s * total + i];
        if (f.bias) z[0] += to_float(static_cast<const T*>(f.bias)[col]);
        const float r = f.residual ? to_float(static_cast<const T*>(f.residual)[row * f.residual_stride + col]) : 0.0f;
        by_activation(f.activation, [&](auto act) {
            constexpr int ACT = decltype(act)::value;
            if (f.slope) {
                activate<ACT, true, kRounded>(f.omega, z, d);
                static_cast<SlopeOf<T, ACT>*>(f.slope)[i] = from_float<SlopeOf<T, ACT>>(d[0]);
            } else activate<ACT, false, kRounded>(f.omega, z, d);
        });
        static_cast<T*>(f.out)[i] = from_float<T>(z[0] + r);
    }
}

// ---- few rows ------------------------------------------------------------------------------------------------------
// Up to kFewRows rows: the weights are all there is to read, so a warp takes one output at a time, 16 bytes a lane and
// load, and keeps a float32 sum per row of x.  A 128-row tile would load as much and pad the rest; from five rows on the
// arithmetic of this form costs more than that.
constexpr int kFewRows = 4;

template <class T>
__device__ __forceinline__ void words_to_floats(uint4 w, float (&v)[16 / sizeof(T)]) {
    const T* t = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int j = 0; j < (int)(16 / sizeof(T)); ++j) v[j] = to_float(t[j]);
}
struct E4M3 { uint8_t code; };
__device__ __forceinline__ float to_float(E4M3 c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(c.code, __NV_E4M3))); }

template <class T, class OUT, bool ROUNDED>
__global__ void __launch_bounds__(256) few_rows_kernel(const GemmArgs g, bool wide) {
    constexpr int kVec = 16 / sizeof(T);
    const int lane = threadIdx.x & 31;
    const T* x = static_cast<const T*>(g.a.at);
    const int rows = (int)g.m;
    for (int64_t n = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); n < g.n; n += (int64_t)gridDim.x * 8) {
        const T* w = static_cast<const T*>(g.b.at) + n * g.b.stride;
        float sum[kFewRows] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (wide) {
#pragma unroll 4
            for (int64_t k = lane * kVec; k < g.k; k += 32 * kVec) {
                float wv[kVec];
                words_to_floats<T>(__ldcs(reinterpret_cast<const uint4*>(w + k)), wv);
#pragma unroll
                for (int r = 0; r < kFewRows; ++r) {
                    if (r >= rows) break;
                    float xv[kVec];
                    words_to_floats<T>(__ldg(reinterpret_cast<const uint4*>(x + r * g.a.stride + k)), xv);
#pragma unroll
                    for (int j = 0; j < kVec; ++j) sum[r] = fmaf(wv[j], xv[j], sum[r]);
                }
            }
        } else {
#pragma unroll 4
            for (int64_t k = lane; k < g.k; k += 32) {
                const float wv = to_float(w[k]);
#pragma unroll
                for (int r = 0; r < kFewRows; ++r)
                    if (r < rows) sum[r] = fmaf(wv, to_float(x[r * g.a.stride + k]), sum[r]);
            }
        }
        float mine = 0.0f;
#pragma unroll
        for (int r = 0; r < kFewRows; ++r) {
            float v = sum[r];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            if (lane == r) mine = v;
        }
        if (lane < rows) {
            const Finish& f = g.f;
            float z[1] = {mine}, d[1] = {1.0f};
            if (f.b_scales) z[0] *= f.a_scales[lane] * f.b_scales[n];
            if (f.bias) z[0] += to_float(static_cast<const OUT*>(f.bias)[n]);
            const float r = f.residual ? to_float(static_cast<const OUT*>(f.residual)[lane * f.residual_stride + n]) : 0.0f;
            const int64_t at = lane * g.n + n;
            by_activation(f.activation, [&](auto act) {
                constexpr int ACT = decltype(act)::value;
                if (f.slope) {
                    activate<ACT, true, ROUNDED>(f.omega, z, d);
                    static_cast<SlopeOf<OUT, ACT>*>(f.slope)[at] = from_float<SlopeOf<OUT, ACT>>(d[0]);
                } else activate<ACT, false, ROUNDED>(f.omega, z, d);
            });
            static_cast<OUT*>(f.out)[at] = from_float<OUT>(z[0] + r);
        }
    }
}

// ---- few outputs ---------------------------------------------------------------------------------------------------
// Heads of one to three outputs (a distance, a colour) on narrow rows, and of four in float32 or where rows are no whole 16-byte
// words: their tiles are nearly empty, and but for four leave value by value.  Four lanes have a row, and two rows at a time,
// which share the weights that they fetch from L1; with more lanes a row's shuffles and its way out cost more than its products.  The four sums of a row are
// joined by halves: lanes give two away and keep two, then one, and end with an output each.
// A million rows of 64 into one output: float32 64 us (tiles 156), bf16 43 (87); into four float32 68 (100);
// 16 into three 36 (140) and 39 (85); 100k rows of 63 into three 23 (38, a copy to whole rows included) and 19 (28).  Bf16 rows of 64 into four gain nothing (59 against 52), nor do
// wider rows, where four lanes are too few and more do too much beside (162 into four 182 against 152).
constexpr int kFewOutputs = 4, kNarrowRow = 64, kRowLanes = 4;

template <class T, bool ROUNDED>
__global__ void __launch_bounds__(256) few_outputs_kernel(const GemmArgs g, bool wide) {
    constexpr int kVec = 16 / sizeof(T), kRows = 2, lanes = kRowLanes;
    const int sub = threadIdx.x & (lanes - 1), outputs = (int)g.n;
    const int64_t groups = (int64_t)gridDim.x * (256 / lanes), me = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
    const int64_t rounds = (g.m + groups * kRows - 1) / (groups * kRows);      // of all lanes alike, for the shuffles
    const T* weights = static_cast<const T*>(g.b.at);
    const bool upper = sub & 2, second = sub & 1;
    const int n = sub;                                                         // this lane's output
    for (int64_t round = 0; round < rounds; ++round) {
        const int64_t row0 = (round * groups + me) * kRows;
        const T* x[kRows];
        float sum[kRows][kFewOutputs];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            x[i] = static_cast<const T*>(g.a.at) + min(row0 + i, g.m - 1) * g.a.stride;
#pragma unroll
            for (int r = 0; r < kFewOutputs; ++r) sum[i][r] = 0.0f;
        }
        if (wide) {
#pragma unroll 2
            for (int64_t k = sub * kVec; k < g.k; k += lanes * kVec) {
                float xv[kRows][kVec];
#pragma unroll
                for (int i = 0; i < kRows; ++i) words_to_floats<T>(__ldg(reinterpret_cast<const uint4*>(x[i] + k)), xv[i]);
#pragma unroll
                for (int r = 0; r < kFewOutputs; ++r) {
                    if (r >= outputs) break;
                    float wv[kVec];
                    words_to_floats<T>(__ldg(reinterpret_cast<const uint4*>(weights + r * g.b.stride + k)), wv);
#pragma unroll
                    for (int i = 0; i < kRows; ++i)
#pragma unroll
                        for (int j = 0; j < kVec; ++j) sum[i][r] = fmaf(wv[j], xv[i][j], sum[i][r]);
                }
            }
        } else {
#pragma unroll 4
            for (int64_t k = sub; k < g.k; k += lanes) {
                float xv[kRows];
#pragma unroll
                for (int i = 0; i < kRows; ++i) xv[i] = to_float(x[i][k]);
#pragma unroll
                for (int r = 0; r < kFewOutputs; ++r) {
                    if (r >= outputs) break;
                    const float wv = to_float(weights[r * g.b.stride + k]);
#pragma unroll
                    for (int i = 0; i < kRows; ++i) sum[i][r] = fmaf(wv, xv[i], sum[i][r]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            float (&s)[kFewOutputs] = sum[i];
            const float a = (upper ? s[2] : s[0]) + __shfl_xor_sync(0xffffffffu, upper ? s[0] : s[2], 2);
            const float b = (upper ? s[3] : s[1]) + __shfl_xor_sync(0xffffffffu, upper ? s[1] : s[3], 2);
            const float v = (second ? b : a) + __shfl_xor_sync(0xffffffffu, second ? a : b, 1);
            if (row0 + i >= g.m || n >= outputs) continue;
            const Finish& f = g.f;
            float z[1] = {v}, d[1] = {1.0f};
            if (f.bias) z[0] += to_float(static_cast<const T*>(f.bias)[n]);
            const float r = f.residual ? to_float(static_cast<const T*>(f.residual)[(row0 + i) * f.residual_stride + n]) : 0.0f;
            const int64_t at = (row0 + i) * outputs + n;
            by_activation(f.activation, [&](auto act) {
                constexpr int ACT = decltype(act)::value;
                if (f.slope) {
                    activate<ACT, true, ROUNDED>(f.omega, z, d);
                    static_cast<SlopeOf<T, ACT>*>(f.slope)[at] = from_float<SlopeOf<T, ACT>>(d[0]);
                } else activate<ACT, false, ROUNDED>(f.omega, z, d);
            });
            static_cast<T*>(f.out)[at] = from_float<T>(z[0] + r);
        }
    }
}

// ---- dz and its column sums -------------------------------------------------------------------------------------------
// dz = dy * slope (slope kind 1, float32) or dy where slope is positive (kind 2: relu's slope or, without a residual, its
// output); column sums of it (kind 0: of dy) over the rows of a CTA go to partial[CTA][outputs].  dz is rounded to the layer's
// type, being an operand of two products of that type: in two parts it would double them.  A row has as many lanes as it has
// accesses, 32 at most; blockIdx.x picks the columns of wider rows.
template <int N>
__device__ __forceinline__ void load_floats(const float* __restrict__ p, float (&v)[N]) {
    if constexpr (N == 8) {
        float a[4], b[4];
        load_n<float, 4>(p, a);
        load_n<float, 4>(p + 4, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = a[j];
            v[j + 4] = b[j];
        }
    } else {
        load_n<float, N>(p, v);
    }
}
template <class T, int VEC, int SLOPE_KIND>
__global__ void __launch_bounds__(256) slope_kernel(const T* __restrict__ dy, const std::conditional_t<SLOPE_KIND == 1, float, T>* __restrict__ slope,
                                                    int64_t rows, int64_t n, int lanes, T* __restrict__ dz,
                                                    int64_t dz_stride, float* __restrict__ partial) {
    __shared__ float sums[256 * VEC];
    const int sub = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes, groups = 256 / lanes;
    const int64_t col = ((int64_t)blockIdx.x * lanes + sub) * VEC;
    float total[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) total[j] = 0.0f;
    if (col < n) {
#pragma unroll 4
        for (int64_t r = (int64_t)blockIdx.y * groups + group; r < rows; r += (int64_t)gridDim.y * groups) {
            float g[VEC], s[VEC];
            load_n<T, VEC>(dy + r * n + col, g);
            if (SLOPE_KIND != 0) {
                if constexpr (SLOPE_KIND == 1) load_floats<VEC>(slope + r * n + col, s);
                else load_n<T, VEC>(slope + r * n + col, s);
#pragma unroll
                for (int j = 0; j < VEC; ++j) g[j] = SLOPE_KIND == 1 ? g[j] * s[j] : s[j] > 0.0f ? g[j] : 0.0f;
                if (dz != nullptr) store_n<T, VEC>(dz + r * dz_stride + col, g);
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) total[j] += g[j];
        }
    }
    if (partial == nullptr) return;
#pragma unroll
    for (int j = 0; j < VEC; ++j) sums[threadIdx.x * VEC + j] = total[j];
    __syncthreads();
    for (int c = threadIdx.x; c < lanes * VEC; c += 256) {
        float v = 0.0f;
        for (int i = 0; i < groups; ++i) v += sums[i * lanes * VEC + c];
        const int64_t at = (int64_t)blockIdx.x * lanes * VEC + c;
        if (at < n) partial[blockIdx.y * n + at] = v;
    }
}

// ---- gradients of a small layer ------------------------------------------------------------------------------------------
// All gradients in one launch, for layers whose backward pass is launches and little else: a CTA has a 32 x 32 tile of dx or of
// dW and walks the summed dimension 32 at a time, both operands as float32 in shared memory, dz made on the way (and not
// rounded); the tiles of dW at the first inputs sum the columns of dz too.  A call takes 15 us of the host where four or five
// launches and their maps take 30.  The GPU needs about 2.7 us for 32 of a sum: 22 us for 250 x 256 x 256 against 24 of the tensor
// cores' kernels, but 38 for sums of 500, so these are the limits.
constexpr int64_t kSmallLayer = (int64_t)1 << 24, kSmallSum = 256;

struct SmallGrads {
    const void *dy, *slope, *x, *weight;
    void *dx, *dw, *db;
    int64_t x_stride, weight_stride;
    int rows, inputs, outputs, kind;
    int dx_tiles;      // the first blocks', then dW's
};

template <class T>
__global__ void __launch_bounds__(256) small_grads_kernel(const SmallGrads s) {
    // left by the summed index, so that a thread's four values are one read that all lanes share
    __shared__ __align__(16) float left[32][36];
    __shared__ float right[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const bool is_dx = (int)blockIdx.x < s.dx_tiles;
    const int tile = is_dx ? blockIdx.x : blockIdx.x - s.dx_tiles, across = (s.inputs + 31) / 32;
    const int first = tile / across * 32, k0 = tile % across * 32;      // rows of x, or outputs; inputs
    const int length = is_dx ? s.outputs : s.rows;
    const T* dy = static_cast<const T*>(s.dy);
    const T* other = static_cast<const T*>(is_dx ? s.weight : s.dw ? s.x : nullptr);
    const int64_t stride = is_dx ? s.weight_stride : s.x_stride;
    const bool sums = !is_dx && k0 == 0 && s.db != nullptr;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, total = 0.0f, a[4], b[4];
    // dz of a row and output, and the other operand: rows of 32, the next ones fetched while these are multiplied
    const auto fetch = [&](int at) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = ty + 8 * i;
            const int row = is_dx ? first + r : at + r, out = is_dx ? at + tx : first + tx;
            a[i] = b[i] = 0.0f;
            if (row < s.rows && out < s.outputs) {
                const int64_t e = (int64_t)row * s.outputs + out;
                a[i] = to_float(dy[e]);
                if (s.kind == 1) a[i] *= static_cast<const float*>(s.slope)[e];
                else if (s.kind == 2) a[i] = to_float(static_cast<const T*>(s.slope)[e]) > 0.0f ? a[i] : 0.0f;
            }
            if (other != nullptr && at + r < length && k0 + tx < s.inputs) b[i] = to_float(other[(at + r) * stride + k0 + tx]);
        }
    };
    fetch(0);
    for (int at = 0; at < length; at += 32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (is_dx) left[tx][ty + 8 * i] = a[i];
            else left[ty + 8 * i][tx] = a[i];
            right[ty + 8 * i][tx] = b[i];
        }
        __syncthreads();
        if (at + 32 < length) fetch(at + 32);
#pragma unroll 8
        for (int j = 0; j < 32; ++j) {
            const float r = right[j][tx];
            const float4 l = *reinterpret_cast<const float4*>(&left[j][4 * ty]);
            acc[0] = fmaf(l.x, r, acc[0]);
            acc[1] = fmaf(l.y, r, acc[1]);
            acc[2] = fmaf(l.z, r, acc[2]);
            acc[3] = fmaf(l.w, r, acc[3]);
        }
        if (sums && ty == 0) {
#pragma unroll 8
            for (int j = 0; j < 32; ++j) total += left[j][tx];
        }
        __syncthreads();
    }
    T* out = static_cast<T*>(is_dx ? s.dx : s.dw);
    const int most = is_dx ? s.rows : s.outputs;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (out != nullptr && first + 4 * ty + i < most && k0 + tx < s.inputs)
            out[(int64_t)(first + 4 * ty + i) * s.inputs + k0 + tx] = from_float<T>(acc[i]);
    if (sums && ty == 0 && first + tx < s.outputs) static_cast<T*>(s.db)[first + tx] = from_float<T>(total);
}

static bool is_small_layer(int64_t rows, int64_t inputs, int64_t outputs) {
    return rows <= kSmallSum && outputs <= kSmallSum && inputs <= kSmallLayer && rows * outputs * inputs <= kSmallLayer;
}
static void launch_small_grads(int type, SmallGrads s, cudaStream_t st) {
    const int across = (s.inputs + 31) / 32;
    s.dx_tiles = s.dx ? (s.rows + 31) / 32 * across : 0;
    // dW's tiles; where only the columns' sums are wanted too, of which those at the first inputs do the work
    const int dw_tiles = s.dw || s.db ? (s.outputs + 31) / 32 * across : 0;
    const unsigned blocks = (unsigned)(s.dx_tiles + dw_tiles);
    if (blocks == 0) return;
    if (type == ASHB_F32) small_grads_kernel<float><<<blocks, 256, 0, st>>>(s);
    else if (type == ASHB_F16) small_grads_kernel<__half><<<blocks, 256, 0, st>>>(s);
    else small_grads_kernel<__nv_bfloat16><<<blocks, 256, 0, st>>>(s);
}

// ---- plans --------------------------------------------------------------------------------------------------------------
static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Plan {
    int bn, stages, raws, slots, groups, places, bulk_out, bufs, b_stays, columns;
    int64_t finish_bytes;
    size_t stage;
    int64_t tiles_m, tiles_n, splits, split_blocks;
    size_t shared;
};

// Cycles of a launch, to choose between tile widths and splits: a stage costs what its copies take at about 50 bytes a
// cycle and SM or what its products take, whichever is more, a tile's end about 12 cycles a column; both overlap but
// for the first and the last tile.
static double cycles(int kind, int bn, int64_t blocks, int64_t items, int sms) {
    const double copies = (128.0 + bn) * (kind == kSplit ? 256 : 128) / 50.0, products = bn * (kind == kSplit ? 12.0 : 2.0);
    const double body = (double)blocks * std::max(copies, products) + 600.0, end = 12.0 * bn + 400.0;
    const double waves = (double)ceil_div(items, sms);
    return waves * std::max(body, end) + std::min(body, end);
}

static Plan plan_product(int kind, bool a_down, bool b_down, int64_t m, int64_t n, int64_t k, bool may_split) {
    const int block = kind == kEight ? 128 : 64, sms = sm_count();
    const int widest = kind == kSplit ? 128 : 256;
    Plan best{};
    double least = 0.0;
    for (int bn = 32; bn <= widest; bn += 32) {
        if (bn > 32 && bn - 32 >= n) break;                    // no wider than the columns there are
        if (bn > 128 && bn != 256 && bn < n) continue;          // between, only what covers all columns
        if (bn < 128 && bn != 32 && bn != 64 && bn < n) continue;
        Plan p{};
        p.bn = bn;
        p.tiles_m = ceil_div(m, kTileM);
        p.tiles_n = ceil_div(n, bn);
        const int64_t tiles = p.tiles_m * p.tiles_n, blocks = ceil_div(k, block);
        const int64_t most = may_split ? std::max<int64_t>(1, blocks / 4) : 1;
        // no splits, or as many as make one or two rounds of the SMs
        const int64_t tries[3] = {1, std::min(most, sms / tiles), std::min(most, 2 * sms / tiles)};
        for (int i = 0; i < 3; ++i) {
            if (tries[i] < 1 || (i > 0 && tries[i] <= tries[i - 1])) continue;
            const int64_t per = ceil_div(blocks, tries[i]), splits = ceil_div(blocks, per);
            // a split writes and reads its sums once more: 8 bytes a value at about 3000 bytes a cycle of the whole GPU
            const double join = splits > 1 ? 8.0 * splits * m * n / 3000.0 + 3000.0 : 0.0;
            const double c = cycles(kind, bn, per, tiles * splits, sms) + join;
            if (least == 0.0 || c < least) {
                least = c;
                p.splits = splits;
                p.split_blocks = per;
                best = p;
            }
        }
    }
    best.stage = (a_down ? part_bytes<true>(kTileM) : part_bytes<false>(kTileM)) +
                 (b_down ? part_bytes<true>(best.bn) : part_bytes<false>(best.bn));
    best.b_stays = !a_down && best.tiles_n == 1 && best.splits == 1;      // if the stages hold all of it
    return best;
}

// As many tiles' sums as tensor memory holds: with two, a narrow tile waits for the round trip of one through the products, a
// barrier, the way out and a barrier back (1.5k cycles).
static void plan_slots(Plan* p, int columns) {
    p->slots = std::min(kMaxSlots, 512 / columns);
    p->columns = 32;
    while (p->columns < columns * p->slots) p->columns <<= 1;
}

// A finisher's shared memory: blocks that leave by bulk copies, and their columns' biases and scales, or a block (two, where
// sums of several phases wait in them) whose values are stored.
static size_t finisher_bytes(const Plan& p, int block, int slope) {
    return p.bulk_out ? (size_t)((block + slope) * p.bufs + 1024) : (size_t)4096 * p.places;
}

// Stages and finishers once it is known how results are stored.  block, slope: bytes of one that leaves by bulk copies.
static void plan_shared(Plan* p, int64_t blocks, int block, int slope) {
    const size_t room = kSharedLimit - 2048;
    plan_slots(p, p->bn);
    p->places = 1;
    // twelve finishers and two blocks each where that leaves four stages, or three where a tile has no more than two
    const size_t stages = (p->split_blocks <= 2 ? 3 : 4) * p->stage;
    p->groups = 3;
    p->bufs = 2;
    const auto finish = [&] { return 4 * p->groups * finisher_bytes(*p, block, slope); };
    if (stages + finish() > room) p->groups = 2;
    if (stages + finish() > room) p->bufs = 1;
    p->finish_bytes = (int64_t)finisher_bytes(*p, block, slope);
    p->stages = (int)std::min<size_t>(kMaxStages, (room - finish()) / p->stage);
    p->b_stays = p->b_stays && blocks <= p->stages;
    if (p->b_stays) p->stages = (int)(p->stages / blocks * blocks);
    // more than half of the SM's shared memory: a second CTA would wait for tensor memory
    p->shared = std::max<size_t>((size_t)p->stages * p->stage + finish() + 1024, 120 * 1024);
}

// The same of split_gemm_kernel.  Blocks are half as long as the plan counts them.
static void plan_split(Plan* p, bool a_down, bool b_down, int64_t k, int slope) {
    const int64_t blocks = ceil_div(k, kSplitBlock);
    plan_slots(p, 2 * p->bn);
    p->split_blocks *= 2;
    const bool phases = p->split_blocks > kSplitPhase;
    p->bulk_out = p->bulk_out && !phases;
    p->places = phases && p->bn > 64 ? 2 : 1;
    p->groups = 2;
    const size_t a = 3 * (a_down ? split_bytes<true>(kTileM) : split_bytes<false>(kTileM));
    const size_t b = 3 * (b_down ? split_bytes<true>(p->bn) : split_bytes<false>(p->bn));
    const size_t raw_a = kTileM * 128, raw_b = (size_t)p->bn * 128, all = kSharedLimit - 2048;
    // B stays where two stages of A's parts and three of its values fit beside it and the smallest finishers
    const size_t least = 8 * (size_t)(p->bulk_out ? 4096 + slope + 1024 : 4096 * p->places);
    p->b_stays = p->b_stays && b * blocks + 2 * a + 3 * raw_a + least <= all;
    const size_t operands = p->b_stays ? b * blocks + 2 * a + 3 * raw_a : 2 * (a + b + raw_a + raw_b);
    // two blocks of a finisher, else one, else blocks that are stored value by value
    p->bufs = 2;
    if (8 * finisher_bytes(*p, 4096, slope) + operands > all) p->bufs = 1;
    if (8 * finisher_bytes(*p, 4096, slope) + operands > all) p->bulk_out = 0;
    p->finish_bytes = (int64_t)finisher_bytes(*p, 4096, slope);
    const size_t finish = 8 * (size_t)p->finish_bytes, room = all - finish;
    const size_t stay = p->b_stays ? b * blocks : 0, stage = a + (p->b_stays ? 0 : b), raw = raw_a + (p->b_stays ? 0 : raw_b);
    // stages of parts, then of values, in turn while they fit
    p->stages = 2;
    p->raws = 2;
    size_t used = stay + 2 * stage + 2 * raw;
    for (bool more = true; more;) {
        more = false;
        if (p->raws < kMaxRaws && p->raws <= p->stages + 1 && used + raw <= room) { ++p->raws; used += raw; more = true; }
        if (p->stages < 4 && used + stage <= room) { ++p->stages; used += stage; more = true; }
    }
    p->shared = std::max<size_t>(used + finish + 1024, 120 * 1024);
}

// ---- launches -----------------------------------------------------------------------------------------------------------
static PFN_cuTensorMapEncodeTiled_v12000 encode_tiled() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}

// Map of an operand for copies of `box_rows` rows of 128 bytes.
static bool operand_map(CUtensorMap* map, int kind, int type, const Operand& o, int64_t rows, int64_t cols, int box_rows) {
    const int bytes = kind == kEight ? 1 : kind == kSplit ? 4 : 2;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(o.stride * bytes)};
    const cuuint32_t box[2] = {(cuuint32_t)(kRowBytes / bytes), (cuuint32_t)box_rows}, steps[2] = {1, 1};
    const CUtensorMapDataType t = kind == kEight ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                  : kind == kSplit ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                  : type == ASHB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const auto encode = encode_tiled();
    return encode != nullptr &&
           encode(map, t, 2, const_cast<void*>(o.at), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Map of what leaves (or of residuals): blocks of 32 x 32, `splits` times m rows of n values.
static bool block_map(CUtensorMap* map, const void* at, int type, int64_t stride, int64_t m, int64_t n, int64_t splits) {
    const int bytes = value_bytes(type);
    if (((uintptr_t)at & 15) != 0 || stride * bytes % 16 != 0) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)n, (cuuint64_t)m, (cuuint64_t)splits};
    const cuuint64_t strides[2] = {(cuuint64_t)(stride * bytes), (cuuint64_t)(stride * m * bytes)};
    const cuuint32_t box[3] = {32, 32, 1}, steps[3] = {1, 1, 1};
    const CUtensorMapDataType t = type == ASHB_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                  : type == ASHB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const auto encode = encode_tiled();
    return encode != nullptr &&
           encode(map, t, 3, const_cast<void*>(at), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  bytes == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static bool finish_maps(FinishMaps* maps, const GemmArgs& g, int64_t splits) {
    const Finish& f = g.f;
    const int type = f.partial ? ASHB_F32 : f.type;
    return block_map(&maps->out, f.partial ? (const void*)f.partial : f.out, type, g.n, g.m, g.n, splits) &&
           (!f.slope || block_map(&maps->slope, f.slope, f.activation == kRelu ? type : ASHB_F32, g.n, g.m, g.n, 1)) &&
           (!f.residual || block_map(&maps->residual, f.residual, type, f.residual_stride, g.m, g.n, 1));
}

static std::atomic<int> g_wait_polls{kWaitPolls};
constexpr int kToldDevices = 64;
static std::atomic<unsigned int*> g_told{nullptr};

// The host's words for waits that ran out, one a device, which kernels reach too; null where there is no such memory.
static unsigned int* told_words() {
    static unsigned int* words = [] {
        void* p = nullptr;
        // a first call may be one that is captured, where allocations are refused unless the thread says it knows
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (cudaHostAlloc(&p, kToldDevices * sizeof(unsigned int), cudaHostAllocPortable | cudaHostAllocMapped) != cudaSuccess) {
            (void)cudaGetLastError();
            p = nullptr;
        }
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (p) std::memset(p, 0, kToldDevices * sizeof(unsigned int));
        return static_cast<unsigned int*>(p);
    }();
    g_told.store(words, std::memory_order_release);
    return words;
}
// Whether a wait has run out in an earlier launch on the current device, as far as is known without waiting: told once.
static int check_told() {
    unsigned int* words = g_told.load(std::memory_order_acquire);
    int device = 0;
    if (words == nullptr || cudaGetDevice(&device) != cudaSuccess || device >= kToldDevices) return ASHB_OK;
    volatile unsigned int* word = words + device;
    if (*word == 0) return ASHB_OK;
    *word = 0;
    set_error("a wait inside a kernel of an earlier dense layer ran out: what it returned is incomplete");
    return ASHB_ERR_TIMEOUT;
}

template <auto kernel>
static cudaError_t launch_kernel(GemmArgs g, const Plan& p, const CUtensorMap& ma, const CUtensorMap& mb,
                                 const FinishMaps& maps, cudaStream_t st) {
    // once a kernel and device: a call of the runtime less on every launch
    static std::atomic<uint64_t> told{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if (!(told.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kSharedLimit - 1024));
        if (e != cudaSuccess) return e;
        told.fetch_or(bit, std::memory_order_release);
    }
    unsigned int* words = told_words();
    g.told = words && device < kToldDevices ? words + device : nullptr;
    g.polls = g_wait_polls.load(std::memory_order_relaxed);
    kernel<<<(unsigned)std::min<int64_t>(g.items, sm_count()), kGemmThreads, p.shared, st>>>(g, ma, mb, maps);
    return cudaGetLastError();
}

// ---- operands ----------------------------------------------------------------------------------------------------------
static size_t padded(size_t bytes) { return (bytes + 255) / 256 * 256; }

static int operand_bytes(int type) { return type == ASHB_E4M3_ROWS ? 1 : value_bytes(type); }

// Values between rows that begin at multiples of 16 bytes.
static int64_t whole_stride(int type, int64_t cols) {
    const int64_t values = 16 / operand_bytes(type);
    return ceil_div(cols, values) * values;
}
static bool is_whole(int type, const void* at, int64_t stride) {
    return ((uintptr_t)at & 15) == 0 && stride * operand_bytes(type) % 16 == 0;
}

static bool takes_few_outputs(int type, const void* x, int64_t x_stride, int64_t inputs, int64_t outputs) {
    return type != ASHB_E4M3_ROWS && outputs <= kFewOutputs && inputs <= kNarrowRow &&
           (outputs < kFewOutputs || type == ASHB_F32 || !is_whole(type, x, x_stride));
}

template <class T>
static void launch_few_outputs(const GemmArgs& g, bool wide, cudaStream_t st) {
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(g.m, 2 * (256 / kRowLanes)), (int64_t)sm_count() * 8);
    few_outputs_kernel<T, sizeof(T) == 2><<<grid, 256, 0, st>>>(g, wide);
}
// Bytes of the copy that an operand needs, 0 if it is taken as it is.
static size_t copy_bytes(int type, const void* at, int64_t stride, int64_t rows, int64_t cols) {
    return is_whole(type, at, stride) ? 0 : padded((size_t)(rows * whole_stride(type, cols)) * operand_bytes(type));
}
// The operand where `to` has its copy if it needs one; the copy itself is left in *p for launch_padding.
static Operand placed(int type, const void* at, int64_t stride, int64_t rows, int64_t cols, char* to, Padding* p) {
    if (is_whole(type, at, stride)) return Operand{at, stride};
    const int64_t whole = whole_stride(type, cols);
    *p = Padding{at, to, rows, cols, stride, whole * operand_bytes(type) / 16, 1, 0, 0};
    while (p->lanes < 32 && p->lanes < p->words) p->lanes <<= 1;
    p->units = (uint32_t)(ceil_div(rows, 256 / p->lanes * kPadRows) * ceil_div(p->words, p->lanes));
    p->blocks = (unsigned)std::min<int64_t>(p->units, (int64_t)sm_count() * 16);
    return Operand{to, whole};
}
static void launch_padding(int type, const Padding& first, const Padding& second, cudaStream_t st) {
    const unsigned blocks = first.blocks + second.blocks;
    if (blocks == 0) return;
    switch (operand_bytes(type)) {
        case 1: pad_kernel<uint8_t><<<blocks, 256, 0, st>>>(first, second); break;
        case 2: pad_kernel<uint16_t><<<blocks, 256, 0, st>>>(first, second); break;
        default: pad_kernel<uint32_t><<<blocks, 256, 0, st>>>(first, second);
    }
}

// Operands' rows begin at multiples of 16 bytes.
template <int KIND, bool A_DOWN, bool B_DOWN>
static int run_product(GemmArgs g, int type, Plan p, cudaStream_t st) {
    CUtensorMap ma{}, mb{};
    const int down = KIND == kSplit ? kSplitBlock : 64;      // rows of a box that k runs down
    if (!operand_map(&ma, KIND, type, g.a, A_DOWN ? g.k : g.m, A_DOWN ? g.m : g.k, A_DOWN ? down : kTileM) ||
        !operand_map(&mb, KIND, type, g.b, B_DOWN ? g.k : g.n, B_DOWN ? g.n : g.k, B_DOWN ? down : p.bn)) {
        set_error("no tensor map of a product's operands");
        return ASHB_ERR_CUDA;
    }
    FinishMaps maps{};
    p.bulk_out = finish_maps(&maps, g, p.splits);
    constexpr int64_t kBlock = kBlockK<KIND>;
    const int block = g.f.partial || g.f.type == ASHB_F32 ? 4096 : 2048, slope = !g.f.slope ? 0 : g.f.activation == kRelu ? block : 4096;
    if (KIND == kSplit) plan_split(&p, A_DOWN, B_DOWN, g.k, slope);
    else plan_shared(&p, ceil_div(g.k, kBlock), block, slope);
    g.slope_bytes = (uint32_t)slope;
    g.bulk_out = p.bulk_out;
    g.bufs = p.bufs;
    g.finish_bytes = p.finish_bytes;
    g.bn = p.bn;
    g.stages = p.stages;
    g.slots = p.slots;
    g.groups = p.groups;
    g.places = p.places;
    g.raws = p.raws;
    g.b_stays = p.b_stays;
    g.columns = p.columns;
    ASHB_REQUIRE(p.tiles_m * p.tiles_n * p.splits < (int64_t)1 << 31, "a product of %lld x %lld values", (long long)g.m, (long long)g.n);
    g.tiles_m = (uint32_t)p.tiles_m;
    g.tiles_n = (uint32_t)p.tiles_n;
    g.tiles = g.tiles_m * g.tiles_n;
    g.splits = (uint32_t)p.splits;
    g.items = g.tiles * g.splits;
    g.blocks_k = (uint32_t)ceil_div(g.k, kBlock);
    g.split_blocks = (uint32_t)p.split_blocks;
    g.block_k = (uint32_t)kBlock;
    g.desc = product_desc(kTileM, p.bn, KIND == kEight ? 0 : KIND == kSplit || type == ASHB_BF16 ? 1 : 0, A_DOWN, B_DOWN);
    if constexpr (KIND == kSplit) ASHB_CUDA_TRY((launch_kernel<split_gemm_kernel<A_DOWN, B_DOWN>>(g, p, ma, mb, maps, st)));
    else ASHB_CUDA_TRY((launch_kernel<layer_gemm_kernel<KIND, A_DOWN, B_DOWN>>(g, p, ma, mb, maps, st)));
    return ASHB_OK;
}

template <bool A_DOWN, bool B_DOWN>
static int run_typed(const GemmArgs& g, int type, const Plan& p, cudaStream_t st) {
    return type == ASHB_F32 ? run_product<kSplit, A_DOWN, B_DOWN>(g, type, p, st)
                            : run_product<kHalf, A_DOWN, B_DOWN>(g, type, p, st);
}

template <class T, class OUT>
static void launch_few(const GemmArgs& g, bool wide, cudaStream_t st) {
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(g.n, 8), (int64_t)sm_count() * 8);
    few_rows_kernel<T, OUT, sizeof(OUT) == 2><<<grid, 256, 0, st>>>(g, wide);
}

static int kind_of(int type) { return type == ASHB_F32 ? kSplit : type == ASHB_E4M3_ROWS ? kEight : kHalf; }

struct SlopePlan {
    int vec, lanes;
    unsigned across, down;
};
static SlopePlan plan_slope(int type, int64_t rows, int64_t n, bool wide) {
    SlopePlan p{};
    p.vec = wide ? 16 / value_bytes(type) : 1;
    p.lanes = 1;
    while (p.lanes < 32 && (int64_t)p.lanes * p.vec < n) p.lanes <<= 1;
    p.across = (unsigned)ceil_div(n, (int64_t)p.lanes * p.vec);
    const int64_t groups = 256 / p.lanes;
    p.down = (unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(rows, groups * 4), ceil_div((int64_t)sm_count() * 4, p.across)));
    return p;
}
// the largest `down` of both forms, for the workspace
static int64_t slope_rows(int type, int64_t rows, int64_t n) {
    return std::max(plan_slope(type, rows, n, true).down, plan_slope(type, rows, n, false).down);
}

template <class T, int SLOPE_KIND>
static void launch_slope_kind(const SlopePlan& p, const void* dy, const void* slope, int64_t rows, int64_t n, void* dz, int64_t dz_stride,
                              float* partial, cudaStream_t st) {
    const dim3 grid(p.across, p.down);
    const T* g = static_cast<const T*>(dy);
    const auto* s = static_cast<const std::conditional_t<SLOPE_KIND == 1, float, T>*>(slope);
    if (p.vec > 1) slope_kernel<T, 16 / sizeof(T), SLOPE_KIND><<<grid, 256, 0, st>>>(g, s, rows, n, p.lanes, static_cast<T*>(dz), dz_stride, partial);
    else slope_kernel<T, 1, SLOPE_KIND><<<grid, 256, 0, st>>>(g, s, rows, n, p.lanes, static_cast<T*>(dz), dz_stride, partial);
}
template <class T>
static void launch_slope(const SlopePlan& p, const void* dy, const void* slope, int kind, int64_t rows, int64_t n, void* dz,
                         int64_t dz_stride, float* partial, cudaStream_t st) {
    if (kind == 0) launch_slope_kind<T, 0>(p, dy, nullptr, rows, n, dz, dz_stride, partial, st);
    else if (kind == 1) launch_slope_kind<T, 1>(p, dy, slope, rows, n, dz, dz_stride, partial, st);
    else launch_slope_kind<T, 2>(p, dy, slope, rows, n, dz, dz_stride, partial, st);
}

// What a layer's own product needs: copies of operands whose rows are no whole words, and the parts of split sums.
struct ForwardPlan {
    size_t weight, partial, total;      // offsets into the workspace; x's copy is first
    Plan p;
};
static ForwardPlan plan_forward(int type, const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, int64_t rows,
                                int64_t inputs, int64_t outputs) {
    ForwardPlan f{};
    f.weight = copy_bytes(type, x, x_stride, rows, inputs);
    f.partial = f.weight + copy_bytes(type, weight, weight_stride, outputs, inputs);
    f.p = plan_product(kind_of(type), false, false, rows, outputs, inputs, true);
    f.total = f.partial + (f.p.splits > 1 ? padded((size_t)(f.p.splits * rows * outputs) * sizeof(float)) : 0);
    return f;
}

// What the backward pass needs: dz where it differs from dy or dy's rows are no whole words, copies of x and the weights that
// are none, partial sums of the gradients.
struct BackwardPlan {
    size_t dz, x, weight, sums_b, sums_w, sums_x, total;      // offsets into the workspace
    bool makes_dz;
    int64_t dz_stride;
    Plan pw, px;
};
static BackwardPlan plan_backward(int type, const void* dy, const void* x, int64_t x_stride, const void* weight, int64_t weight_stride,
                                  int64_t rows, int64_t inputs, int64_t outputs, int kind, bool want_x, bool want_w, bool want_b) {
    BackwardPlan b{};
    size_t at = 0;
    const bool products = want_x || want_w;
    b.makes_dz = products && (kind != 0 || !is_whole(type, dy, outputs));
    b.dz_stride = b.makes_dz ? whole_stride(type, outputs) : outputs;
    b.dz = at;
    if (b.makes_dz) at += padded((size_t)(rows * b.dz_stride) * value_bytes(type));
    b.x = at;
    if (want_w) at += copy_bytes(type, x, x_stride, rows, inputs);
    b.weight = at;
    if (want_x) at += copy_bytes(type, weight, weight_stride, outputs, inputs);
    b.sums_b = at;
    if (want_b) at += padded((size_t)(slope_rows(type, rows, outputs) * outputs) * sizeof(float));
    b.sums_w = at;
    if (want_w) {
        b.pw = plan_product(kind_of(type), true, true, outputs, inputs, rows, true);
        if (b.pw.splits > 1) at += padded((size_t)(b.pw.splits * outputs * inputs) * sizeof(float));
    }
    b.sums_x = at;
    if (want_x) {
        b.px = plan_product(kind_of(type), false, true, rows, inputs, outputs, true);
        if (b.px.splits > 1) at += padded((size_t)(b.px.splits * rows * inputs) * sizeof(float));
    }
    b.total = at;
    return b;
}

static int check_sizes(int64_t rows, int64_t inputs, int64_t outputs) {
    const int64_t most = (int64_t)1 << 30;
    ASHB_REQUIRE(rows >= 0 && rows <= most && inputs >= 1 && inputs <= most && outputs >= 1 && outputs <= most,
                 "a layer of %lld rows, %lld inputs and %lld outputs", (long long)rows, (long long)inputs, (long long)outputs);
    return ASHB_OK;
}

}  // namespace ashb

using namespace ashb;

extern "C" {

int ashb_linear_forward(int type, const void* x, int64_t x_stride, const float* x_scales, const void* weight,
                        int64_t weight_stride, const float* weight_scales, const void* bias, const void* residual,
                        int64_t residual_stride, int64_t rows, int64_t inputs, int64_t outputs, int activation, float omega,
                        int out_type, void* y, void* slope, void* workspace, int64_t workspace_bytes, void* stream) {
    const bool eight = type == ASHB_E4M3_ROWS;
    ASHB_REQUIRE(is_value_type(type) || eight, "operand type %d", type);
    ASHB_REQUIRE(is_value_type(out_type) && (eight || out_type == type), "output type %d", out_type);
    ASHB_REQUIRE(activation >= kNone && activation <= kSin, "activation %d", activation);
    if (int rc = check_sizes(rows, inputs, outputs)) return rc;
    if (rows == 0) return ASHB_OK;
    ASHB_REQUIRE(x && weight && y && (!eight || (x_scales && weight_scales)), "null buffer");
    ASHB_REQUIRE((x_stride >= inputs || rows == 1) && weight_stride >= inputs, "rows overlap");
    if (int rc = check_told()) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    GemmArgs g{};
    g.a = Operand{x, x_stride};
    g.b = Operand{weight, weight_stride};
    g.m = rows;
    g.n = outputs;
    g.k = inputs;
    Finish& f = g.f;
    f.a_scales = eight ? x_scales : nullptr;
    f.b_scales = eight ? weight_scales : nullptr;
    f.bias = bias;
    f.residual = residual;
    f.residual_stride = residual_stride;
    f.out = y;
    f.slope = slope;
    f.type = out_type;
    f.activation = activation;
    f.omega = omega;
    const uintptr_t four = (uintptr_t)(4 * value_bytes(out_type));
    f.wide = outputs % 4 == 0 && (!residual || residual_stride % 4 == 0) &&
             (((uintptr_t)y | (uintptr_t)bias | (uintptr_t)residual) & (four - 1)) == 0 &&
             (((uintptr_t)f.b_scales | (uintptr_t)slope) & 15) == 0;
    if (rows <= kFewRows) {
        const bool wide = is_whole(type, x, rows == 1 ? 0 : x_stride) && is_whole(type, weight, weight_stride) &&
                          inputs * operand_bytes(type) % 16 == 0;
        if (type == ASHB_F32) launch_few<float, float>(g, wide, st);
        else if (type == ASHB_F16) launch_few<__half, __half>(g, wide, st);
        else if (type == ASHB_BF16) launch_few<__nv_bfloat16, __nv_bfloat16>(g, wide, st);
        else if (out_type == ASHB_F32) launch_few<E4M3, float>(g, wide, st);
        else if (out_type == ASHB_F16) launch_few<E4M3, __half>(g, wide, st);
        else launch_few<E4M3, __nv_bfloat16>(g, wide, st);
        ASHB_LAUNCH_CHECK();
        return ASHB_OK;
    }
    if (takes_few_outputs(type, x, x_stride, inputs, outputs)) {
        const bool wide = is_whole(type, x, x_stride) && is_whole(type, weight, outputs == 1 ? 0 : weight_stride) &&
                          inputs * operand_bytes(type) % 16 == 0;
        if (type == ASHB_F32) launch_few_outputs<float>(g, wide, st);
        else if (type == ASHB_F16) launch_few_outputs<__half>(g, wide, st);
        else launch_few_outputs<__nv_bfloat16>(g, wide, st);
        ASHB_LAUNCH_CHECK();
        return ASHB_OK;
    }
    const ForwardPlan fp = plan_forward(type, x, x_stride, weight, weight_stride, rows, inputs, outputs);
    ASHB_REQUIRE(fp.total == 0 || (workspace && ((uintptr_t)workspace & 255) == 0 && workspace_bytes >= (int64_t)fp.total),
                 "null, unaligned or small workspace");
    ASHB_REQUIRE(!slope || (!eight && activation != kNone), "a slope is of an activation, of operands that are not quantised");
    Padding px{}, pw{};
    char* ws = static_cast<char*>(workspace);
    g.a = placed(type, x, x_stride, rows, inputs, ws, &px);
    g.b = placed(type, weight, weight_stride, outputs, inputs, ws + fp.weight, &pw);
    launch_padding(type, px, pw, st);
    const Finish whole = f;
    if (fp.p.splits > 1) {      // scales belong to the parts, all else to their sums
        f = Finish{};
        f.a_scales = whole.a_scales;
        f.b_scales = whole.b_scales;
        f.partial = reinterpret_cast<float*>(ws + fp.partial);
    }
    if (int rc = eight ? run_product<kEight, false, false>(g, type, fp.p, st) : run_typed<false, false>(g, type, fp.p, st)) return rc;
    if (fp.p.splits > 1) {
        const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(rows * outputs, 256), (int64_t)sm_count() * 8);
        const int splits = (int)fp.p.splits;
        if (out_type == ASHB_F32) join_layer_kernel<float><<<blocks, 256, 0, st>>>(whole, f.partial, splits, rows, outputs);
        else if (out_type == ASHB_F16) join_layer_kernel<__half><<<blocks, 256, 0, st>>>(whole, f.partial, splits, rows, outputs);
        else join_layer_kernel<__nv_bfloat16><<<blocks, 256, 0, st>>>(whole, f.partial, splits, rows, outputs);
    }
    ASHB_LAUNCH_CHECK();
    return ASHB_OK;
}

int64_t ashb_linear_forward_workspace(int type, const void* x, int64_t x_stride, const void* weight, int64_t weight_stride,
                                      int64_t rows, int64_t inputs, int64_t outputs) {
    if ((!is_value_type(type) && type != ASHB_E4M3_ROWS) || check_sizes(rows, inputs, outputs) != ASHB_OK || rows <= kFewRows ||
        takes_few_outputs(type, x, x_stride, inputs, outputs))
        return 0;
    return (int64_t)plan_forward(type, x, x_stride, weight, weight_stride, rows, inputs, outputs).total;
}

int64_t ashb_linear_backward_workspace(int type, const void* dy, const void* x, int64_t x_stride, const void* weight,
                                       int64_t weight_stride, int64_t rows, int64_t inputs, int64_t outputs, int slope_kind,
                                       int want_dx, int want_dweight, int want_dbias) {
    if (!is_value_type(type) || check_sizes(rows, inputs, outputs) != ASHB_OK || rows == 0 || is_small_layer(rows, inputs, outputs))
        return 0;
    return (int64_t)plan_backward(type, dy, x, x_stride, weight, weight_stride, rows, inputs, outputs, slope_kind, want_dx != 0,
                                  want_dweight != 0, want_dbias != 0)
            .total;
}

int ashb_linear_backward(int type, const void* dy, const void* slope, int slope_kind, const void* x, int64_t x_stride,
                         const void* weight, int64_t weight_stride, int64_t rows, int64_t inputs, int64_t outputs, void* dx,
                         void* dweight, void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
    ASHB_REQUIRE(is_value_type(type), "value type %d", type);
    ASHB_REQUIRE(slope_kind >= 0 && slope_kind <= 2, "slope kind %d", slope_kind);
    if (int rc = check_sizes(rows, inputs, outputs)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const size_t e = (size_t)value_bytes(type);
    if (rows == 0) {
        if (dweight) ASHB_CUDA_TRY(cudaMemsetAsync(dweight, 0, (size_t)(outputs * inputs) * e, st));
        if (dbias) ASHB_CUDA_TRY(cudaMemsetAsync(dbias, 0, (size_t)outputs * e, st));
        return ASHB_OK;
    }
    ASHB_REQUIRE(dy && (!dx || weight) && (!dweight || x) && (slope_kind == 0) == (slope == nullptr),
                 "null buffer, or a slope that the slope kind has no use for");
    ASHB_REQUIRE(!dx || weight_stride >= inputs, "rows overlap");
    ASHB_REQUIRE(!dweight || x_stride >= inputs || rows == 1, "rows overlap");
    if (int rc = check_told()) return rc;
    if (is_small_layer(rows, inputs, outputs)) {
        launch_small_grads(type, SmallGrads{dy, slope, x, weight, dx, dweight, dbias, x_stride, weight_stride, (int)rows, (int)inputs,
                                            (int)outputs, slope_kind, 0}, st);
        ASHB_LAUNCH_CHECK();
        return ASHB_OK;
    }
    const BackwardPlan bp = plan_backward(type, dy, x, x_stride, weight, weight_stride, rows, inputs, outputs, slope_kind,
                                          dx != nullptr, dweight != nullptr, dbias != nullptr);
    ASHB_REQUIRE(bp.total == 0 || (workspace && ((uintptr_t)workspace & 255) == 0 && workspace_bytes >= (int64_t)bp.total),
                 "null, unaligned or small workspace");
    char* ws = static_cast<char*>(workspace);
    float* pb = dbias ? reinterpret_cast<float*>(ws + bp.sums_b) : nullptr;
    void* made = bp.makes_dz ? ws + bp.dz : nullptr;
    const Operand dz{made ? made : dy, bp.dz_stride};
    Padding px{}, pweight{}, pdy{};
    const Operand ox = dweight ? placed(type, x, x_stride, rows, inputs, ws + bp.x, &px) : Operand{};
    const Operand ow = dx ? placed(type, weight, weight_stride, outputs, inputs, ws + bp.weight, &pweight) : Operand{};
    launch_padding(type, px, pweight, st);
    if (made && slope_kind == 0) {
        placed(type, dy, outputs, rows, outputs, ws + bp.dz, &pdy);
        launch_padding(type, pdy, Padding{}, st);
    }
    ASHB_LAUNCH_CHECK();
    int64_t count_b = 0;
    if ((made && slope_kind != 0) || dbias) {
        const bool wide = outputs * (int64_t)e % 16 == 0 && (((uintptr_t)dy | (uintptr_t)slope) & 15) == 0;
        const SlopePlan sp = plan_slope(type, rows, outputs, wide);
        count_b = sp.down;
        if (type == ASHB_F32) launch_slope<float>(sp, dy, slope, slope_kind, rows, outputs, made, bp.dz_stride, pb, st);
        else if (type == ASHB_F16) launch_slope<__half>(sp, dy, slope, slope_kind, rows, outputs, made, bp.dz_stride, pb, st);
        else launch_slope<__nv_bfloat16>(sp, dy, slope, slope_kind, rows, outputs, made, bp.dz_stride, pb, st);
        ASHB_LAUNCH_CHECK();
    }
    const auto finish_to = [&](void* out, int64_t n) {
        Finish f{};
        f.out = out;
        f.type = type;
        f.activation = kNone;
        f.wide = n % 4 == 0 && ((uintptr_t)out & (4 * e - 1)) == 0;
        return f;
    };
    const float* px_sums = nullptr;
    if (dx) {
        GemmArgs g{};
        g.a = dz;
        g.b = ow;
        g.f = finish_to(dx, inputs);
        g.m = rows;
        g.n = inputs;
        g.k = outputs;
        if (bp.px.splits > 1) {
            g.f.partial = reinterpret_cast<float*>(ws + bp.sums_x);
            px_sums = g.f.partial;
        }
        if (int rc = run_typed<false, true>(g, type, bp.px, st)) return rc;
    }
    const float* pw = nullptr;
    if (dweight) {
        GemmArgs g{};
        g.a = dz;
        g.b = ox;
        g.f = finish_to(dweight, inputs);
        g.m = outputs;
        g.n = inputs;
        g.k = rows;
        if (bp.pw.splits > 1) {
            g.f.partial = reinterpret_cast<float*>(ws + bp.sums_w);
            pw = g.f.partial;
        }
        if (int rc = run_typed<true, true>(g, type, bp.pw, st)) return rc;
    }
    const Sums sw{pw, bp.pw.splits, outputs * inputs, dweight}, sb{pb, count_b, outputs, dbias};
    const Sums sx{px_sums, bp.px.splits, rows * inputs, dx};
    const auto sums = [&](auto value) {
        launch_sums<decltype(value)>(sw, sb, st);
        launch_sums<decltype(value)>(sx, Sums{}, st);
    };
    if (type == ASHB_F32) sums(0.0f);
    else if (type == ASHB_F16) sums(__half{});
    else sums(__nv_bfloat16{});
    ASHB_LAUNCH_CHECK();
    return ASHB_OK;
}

int ashb_layer_timeouts(unsigned int* out) {
    ASHB_REQUIRE(out != nullptr, "null output");
    // of every stream: a copy on the default one does not wait for those that do not wait for it
    ASHB_CUDA_TRY(cudaDeviceSynchronize());
    ASHB_CUDA_TRY(cudaMemcpyFromSymbol(out, g_layer_timeouts, sizeof(unsigned int)));
    if (*out != 0) {
        const unsigned int none = 0;
        ASHB_CUDA_TRY(cudaMemcpyToSymbol(g_layer_timeouts, &none, sizeof(none)));
        (void)check_told();
    }
    return ASHB_OK;
}

int ashb_set_layer_wait_limit(int polls) {
    g_wait_polls.store(polls < 0 ? kWaitPolls : polls, std::memory_order_relaxed);
    return ASHB_OK;
}

}  // extern "C"
