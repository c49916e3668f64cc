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
// what is left out is below 2^-23 of a term.  Their sums are kept apart, hi hi in one accumulator and the five small
// ones in another, and both are added to float32 registers, rounded to nearest, every 512 values: the tensor cores
// truncate as they accumulate, which over thousands of steps would be seen in 32 bits.  (An infinity in float32 operands
// becomes NaN: its mid part is infinity less infinity.)
//
// Shape of a CTA, one per SM and looping over tiles of 128 x bn: loaders fill a ring of shared-memory stages, one thread
// issues the products, and eight warps finish the tile before in the other half of tensor memory.  Loaders are one thread
// with tiled bulk copies where types are 8 or 16 bits and rows are multiples of 16 bytes, else seven warps with loads of
// their own, which take any size and alignment and split float32 on the way.
// A layer's rows are long and few values wide as often as not: then the kernel is bound by memory, and a weight tile that
// serves every tile of a CTA is loaded once (`b_stays`).
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstring>

#include "rowformat.cuh"
#include "tensorcore.cuh"

namespace ashb {

constexpr int kRowBytes = 128;            // of a tile row: 64 values of 16 bits, 128 of 8
constexpr int kTileM = 128;
constexpr int kLoaders = 7, kFinishers = 8;             // warps; the one between them issues the products: 16 in all, 128 registers
constexpr int kGemmThreads = (kLoaders + kFinishers + 1) * 32;
constexpr int kPhaseBlocks = 8;           // blocks of 64 between the float32 sums of split products
constexpr int kMaxStages = 8;
constexpr size_t kSharedLimit = 232448;
constexpr size_t kFinishBytes = kFinishers * 32 * 32 * sizeof(float);

enum Activation { kNone = ASHB_ACT_NONE, kRelu = ASHB_ACT_RELU, kSilu = ASHB_ACT_SILU, kGelu = ASHB_ACT_GELU, kSin = ASHB_ACT_SIN };

__device__ unsigned int g_layer_timeouts = 0;

// ---- activations -----------------------------------------------------------------------------------------------------
// act(z) and, where SLOPE, act'(z).  ROUNDED: the results are rounded to 16 bits, for which the hardware's exponential
// (2^-21 of the value) is exact enough; float32 results take the library's.
template <int ACT, bool SLOPE, bool ROUNDED>
__device__ __forceinline__ float activate(float omega, float z, float& slope) {
    if constexpr (ACT == kRelu) {
        if (SLOPE) slope = z > 0.0f ? 1.0f : 0.0f;
        return z < 0.0f ? 0.0f : z;      // a NaN stays
    } else if constexpr (ACT == kSilu) {
        const float e = ROUNDED ? __expf(-z) : expf(-z);
        const float p = ROUNDED ? __fdividef(1.0f, 1.0f + e) : 1.0f / (1.0f + e);
        if (SLOPE) slope = p * fmaf(z, 1.0f - p, 1.0f);
        return z * p;
    } else if constexpr (ACT == kGelu) {
        const float c = 0.5f * (1.0f + erff(z * 0.70710678f));
        if (SLOPE) slope = fmaf(z * 0.39894228f, ROUNDED ? __expf(-0.5f * z * z) : expf(-0.5f * z * z), c);
        return z * c;
    } else if constexpr (ACT == kSin) {
        if (SLOPE) {
            float s, co;
            sincosf(omega * z, &s, &co);
            slope = omega * co;
            return s;
        }
        return sinf(omega * z);
    } else {
        if (SLOPE) slope = 1.0f;
        return z;
    }
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
    int wide;            // rows start at multiples of 16 bytes
};

struct Finish {          // what becomes of the sums
    const float *a_scales, *b_scales;      // e4m3: of the rows of A and B
    const void *bias, *residual;           // of out's type
    void *out, *slope;
    float* partial;                        // float32 sums instead of out: [splits][m][n]
    int64_t residual_stride;
    int type, activation, wide;            // of out; quadruples are aligned everywhere
    float omega;
};

struct GemmArgs {
    Operand a, b;
    Finish f;
    int64_t m, n, k, k_split;              // k_split: of a split, a multiple of a stage's
    int64_t tiles_m, tiles_n, items;
    uint32_t desc;
    int bn, stages, b_stays, columns;      // columns: tensor memory to allocate
};

// Eight consecutive values of an operand as one 16-byte word per part.
struct Eight32 { float v[8]; };
struct Eight16 { uint4 w; };

template <bool WIDE>
__device__ __forceinline__ void fetch8(Eight32& e, const Operand& o, int64_t row, int64_t col, int64_t rows, int64_t cols) {
    const float* p = static_cast<const float*>(o.at) + row * o.stride + col;
    if (WIDE && row < rows && col + 8 <= cols) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
        e.v[0] = a.x; e.v[1] = a.y; e.v[2] = a.z; e.v[3] = a.w;
        e.v[4] = b.x; e.v[5] = b.y; e.v[6] = b.z; e.v[7] = b.w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) e.v[j] = row < rows && col + j < cols ? __ldg(p + j) : 0.0f;
    }
}
template <bool WIDE>
__device__ __forceinline__ void fetch8(Eight16& e, const Operand& o, int64_t row, int64_t col, int64_t rows, int64_t cols) {
    const uint16_t* p = static_cast<const uint16_t*>(o.at) + row * o.stride + col;
    if (WIDE && row < rows && col + 8 <= cols) {
        e.w = __ldg(reinterpret_cast<const uint4*>(p));
    } else {
        uint32_t h[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = row < rows && col + j < cols ? (uint32_t)__ldg(p + j) : 0u;
        e.w = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    }
}
// e4m3: sixteen values.
struct Sixteen8 { uint4 w; };
template <bool WIDE>
__device__ __forceinline__ void fetch8(Sixteen8& e, const Operand& o, int64_t row, int64_t col, int64_t rows, int64_t cols) {
    const uint8_t* p = static_cast<const uint8_t*>(o.at) + row * o.stride + col;
    if (WIDE && row < rows && col + 16 <= cols) {
        e.w = __ldg(reinterpret_cast<const uint4*>(p));
    } else {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (row < rows && col + j < cols) w[j / 4] |= (uint32_t)__ldg(p + j) << (8 * (j % 4));
        e.w = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

__device__ __forceinline__ void put16(uint32_t at, uint4 w) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
}
__device__ __forceinline__ void put8(uint32_t at, uint32_t, const Eight16& e) { put16(at, e.w); }
__device__ __forceinline__ void put8(uint32_t at, uint32_t, const Sixteen8& e) { put16(at, e.w); }
// hi is truncated, so that the largest finite value stays finite; what follows is exact, v = hi + mid + lo.
__device__ __forceinline__ void put8(uint32_t at, uint32_t part, const Eight32& e) {
    uint32_t h[4], m[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t a = __float_as_uint(e.v[2 * j]), b = __float_as_uint(e.v[2 * j + 1]);
        h[j] = __byte_perm(a, b, 0x7632);
        const float ra = e.v[2 * j] - __uint_as_float(a & 0xFFFF0000u), rb = e.v[2 * j + 1] - __uint_as_float(b & 0xFFFF0000u);
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(m[j]) : "f"(rb), "f"(ra));
        const float la = ra - __uint_as_float(m[j] << 16), lb = rb - __uint_as_float(m[j] & 0xFFFF0000u);
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(l[j]) : "f"(lb), "f"(la));
    }
    put16(at, make_uint4(h[0], h[1], h[2], h[3]));
    put16(at + part, make_uint4(m[0], m[1], m[2], m[3]));
    put16(at + 2 * part, make_uint4(l[0], l[1], l[2], l[3]));
}

template <int KIND>
struct KindOf { using Chunk = Eight16; };
template <>
struct KindOf<kSplit> { using Chunk = Eight32; };
template <>
struct KindOf<kEight> { using Chunk = Sixteen8; };

template <int KIND>
constexpr int kBlockK = KIND == kEight ? 128 : 64;       // values of a stage along k
template <int KIND>
constexpr int kParts = KIND == kSplit ? 3 : 1;

// Bytes of one part of an operand's tile: `extent` values across, a stage's values along k.
template <bool DOWN>
__host__ __device__ constexpr uint32_t part_bytes(int extent) {
    return DOWN ? (uint32_t)((extent + 63) / 64) * 64u * kRowBytes : (uint32_t)extent * kRowBytes;
}

// A stage's tile of an operand by loads of the loader warps' own: CHUNKS chunks a thread.
// Chunk `i` of a tile: along rows, row i / 8 and word i % 8; down rows, word i % 8 of row (i / 8) % 64 of box i / 512.
template <int KIND, bool DOWN, int CHUNKS>
struct TileFetch {
    using Chunk = typename KindOf<KIND>::Chunk;
    static constexpr int kValues = KIND == kEight ? 16 : 8;
    Chunk c[CHUNKS];

    // across0, k0: first value across and along k; words: 16-byte words along k that the products will read (of 8).
    __device__ __forceinline__ void fetch(const Operand& o, int thread, int total, int64_t across0, int64_t across, int64_t k0,
                                          int64_t k, int words) {
        if (o.wide) fetch_as<true>(o, thread, total, across0, across, k0, k, words);
        else fetch_as<false>(o, thread, total, across0, across, k0, k, words);
    }
    template <bool WIDE>
    __device__ __forceinline__ void fetch_as(const Operand& o, int thread, int total, int64_t across0, int64_t across,
                                             int64_t k0, int64_t k, int words) {
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) {
            const int i = thread + j * kLoaders * 32;
            if (i >= total) break;
            if (DOWN) {
                const int r = (i >> 3) & 63;
                if (r < words * 8) fetch8<WIDE>(c[j], o, k0 + r, across0 + (int64_t)(i >> 9) * 64 + (i & 7) * 8, k, across);
            } else if ((i & 7) < words) {
                fetch8<WIDE>(c[j], o, across0 + (i >> 3), k0 + (int64_t)(i & 7) * kValues, across, k);
            }
        }
    }
    __device__ __forceinline__ void put(uint32_t tile, uint32_t part, int thread, int total, int words) {
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) {
            const int i = thread + j * kLoaders * 32;
            if (i >= total) break;
            const int r = i >> 3;             // tile rows of a box follow one another: 64 of 128 bytes
            const int w = (i & 7) ^ (r & 7);
            if (DOWN ? (r & 63) < words * 8 : (i & 7) < words) put8(tile + (uint32_t)r * kRowBytes + (uint32_t)w * 16, part, c[j]);
        }
    }
};

// Order of the tiles: bands of 8 rows of tiles, down the band first, so that the tiles in flight share operands in L2.
__device__ __forceinline__ void tile_of(const GemmArgs& g, int64_t item, int64_t& tm, int64_t& tn, int64_t& split) {
    const int64_t tiles = g.tiles_m * g.tiles_n;
    split = item / tiles;
    const int64_t t = item - split * tiles;
    const int64_t band = t / (8 * g.tiles_n), in = t - band * 8 * g.tiles_n;
    const int64_t high = min((int64_t)8, g.tiles_m - band * 8);
    tn = in / high;
    tm = band * 8 + in - tn * high;
}

// The sums of a warp's 32 x 32 block, from registers (a row a thread) through shared memory to memory (rows whole).
__device__ __forceinline__ void put_block(float* block, int lane, const float (&r)[32]) {
#pragma unroll
    for (int q = 0; q < 8; ++q)
        *reinterpret_cast<float4*>(block + lane * 32 + ((q ^ (lane & 7)) << 2)) =
                make_float4(r[4 * q], r[4 * q + 1], r[4 * q + 2], r[4 * q + 3]);
}

// Four values a lane, four rows a pass.  The residuals of four passes are fetched together.
template <class T, int ACT, bool SLOPE>
__device__ __forceinline__ void finish_wide(const Finish& f, const float* block, int lane, int64_t row0, int64_t col0, int64_t m,
                                            int64_t n) {
    constexpr bool kRounded = sizeof(T) == 2;
    const int q = lane & 7, sub = lane >> 3;
    const int64_t col = col0 + 4 * q;
    if (col >= n) return;
    float b[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sb[4] = {1.0f, 1.0f, 1.0f, 1.0f};
    if (f.bias) load_n<T, 4>(static_cast<const T*>(f.bias) + col, b);
    if (f.b_scales) load_n<float, 4>(f.b_scales + col, sb);
    const int64_t row = row0 + sub;
    const int left = (int)min((int64_t)32, m - row0);
    T* out = static_cast<T*>(f.out) + row * n + col;
    T* slopes = SLOPE ? static_cast<T*>(f.slope) + row * n + col : nullptr;
    const T* residual = f.residual ? static_cast<const T*>(f.residual) + row * f.residual_stride + col : nullptr;
#pragma unroll 1
    for (int first = sub; first < left; first += 16) {
        float r[4][4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
#pragma unroll
            for (int k = 0; k < 4; ++k) r[p][k] = 0.0f;
            if (residual && first + 4 * p < left) load_n<T, 4>(residual + 4 * p * f.residual_stride, r[p]);
        }
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const int in = first + 4 * p;
            if (in >= left) break;
            const float4 z4 = *reinterpret_cast<const float4*>(block + in * 32 + ((q ^ (in & 7)) << 2));
            float z[4] = {z4.x, z4.y, z4.z, z4.w}, d[4];
            if (f.b_scales) {
                const float sa = __ldg(f.a_scales + row0 + in);
#pragma unroll
                for (int k = 0; k < 4; ++k) z[k] *= sa * sb[k];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) z[k] = activate<ACT, SLOPE, kRounded>(f.omega, z[k] + b[k], d[k]) + r[p][k];
            if (SLOPE) store_n<T, 4>(slopes + 4 * p * n, d);
            store_n<T, 4>(out + 4 * p * n, z);
        }
        out += 16 * n;
        if (SLOPE) slopes += 16 * n;
        if (residual) residual += 16 * f.residual_stride;
    }
}

// A value a lane, a row a pass.
template <class T, int ACT, bool SLOPE>
__device__ __forceinline__ void finish_narrow(const Finish& f, const float* block, int lane, int64_t row0, int64_t col0, int64_t m,
                                              int64_t n) {
    constexpr bool kRounded = sizeof(T) == 2;
    const int64_t col = col0 + lane;
    if (col >= n) return;
    const float b = f.bias ? to_float(static_cast<const T*>(f.bias)[col]) : 0.0f, sb = f.b_scales ? f.b_scales[col] : 1.0f;
    const int left = (int)min((int64_t)32, m - row0);
    T* out = static_cast<T*>(f.out) + row0 * n + col;
    T* slopes = SLOPE ? static_cast<T*>(f.slope) + row0 * n + col : nullptr;
    const T* residual = f.residual ? static_cast<const T*>(f.residual) + row0 * f.residual_stride + col : nullptr;
#pragma unroll 4
    for (int in = 0; in < left; ++in) {
        const float r = residual ? to_float(residual[in * f.residual_stride]) : 0.0f;
        float z = block[in * 32 + (((lane >> 2) ^ (in & 7)) << 2) + (lane & 3)], d;
        if (f.b_scales) z *= f.a_scales[row0 + in] * sb;
        z = activate<ACT, SLOPE, kRounded>(f.omega, z + b, d) + r;
        if (SLOPE) slopes[in * n] = from_float<T>(d);
        out[in * n] = from_float<T>(z);
    }
}

__device__ __forceinline__ void finish_partial(float* partial, const float* block, int lane, int64_t row0, int64_t col0, int64_t m,
                                               int64_t n) {
    const int64_t col = col0 + lane;
    if (col >= n) return;
#pragma unroll 8
    for (int in = 0; in < 32; ++in)
        if (row0 + in < m) partial[(row0 + in) * n + col] = block[in * 32 + (((lane >> 2) ^ (in & 7)) << 2) + (lane & 3)];
}

template <class T, int ACT, bool SLOPE>
__device__ __forceinline__ void finish_as(const GemmArgs& g, const float* block, int lane, int64_t row0, int64_t col0) {
    if (g.f.wide) finish_wide<T, ACT, SLOPE>(g.f, block, lane, row0, col0, g.m, g.n);
    else finish_narrow<T, ACT, SLOPE>(g.f, block, lane, row0, col0, g.m, g.n);
}

// FORWARD: the layer's own product; the gradients' have no activation.
template <int KIND, bool FORWARD, class T>
__device__ __forceinline__ void finish_typed(const GemmArgs& g, const float* block, int lane, int64_t row0, int64_t col0) {
    if constexpr (!FORWARD) {
        finish_as<T, kNone, false>(g, block, lane, row0, col0);
    } else {
        by_activation(g.f.activation, [&](auto act) {
            constexpr int ACT = decltype(act)::value;
            if constexpr (KIND != kEight && ACT != kNone) {
                if (g.f.slope) {
                    finish_as<T, ACT, true>(g, block, lane, row0, col0);
                    return;
                }
            }
            finish_as<T, ACT, false>(g, block, lane, row0, col0);
        });
    }
}

template <int KIND, bool FORWARD>
__device__ __forceinline__ void finish(const GemmArgs& g, const float* block, int lane, int64_t row0, int64_t col0, int64_t split) {
    if (!FORWARD && g.f.partial) {
        finish_partial(g.f.partial + split * g.m * g.n, block, lane, row0, col0, g.m, g.n);
        return;
    }
    if constexpr (KIND != kHalf) {
        if (KIND == kSplit || g.f.type == ASHB_F32) {
            finish_typed<KIND, FORWARD, float>(g, block, lane, row0, col0);
            return;
        }
    }
    if constexpr (KIND != kSplit) {
        if (g.f.type == ASHB_F16) finish_typed<KIND, FORWARD, __half>(g, block, lane, row0, col0);
        else finish_typed<KIND, FORWARD, __nv_bfloat16>(g, block, lane, row0, col0);
    }
}

struct GemmShared {
    uint64_t full[kMaxStages], empty[kMaxStages], sums_full[2], sums_empty[2], drained;
    uint32_t tmem;
    int gave_up;
};

// Barriers: full[s] by the loaders (the copies' bytes, or a count of their threads), empty[s] by the products that read
// stage s, sums_full / sums_empty of the two halves of tensor memory.  Every role walks the same items, blocks and phases.
template <int KIND, bool BULK, bool A_DOWN, bool B_DOWN>
__global__ void __launch_bounds__(kGemmThreads, 1) layer_gemm_kernel(const GemmArgs g, const __grid_constant__ CUtensorMap map_a,
                                                                     const __grid_constant__ CUtensorMap map_b) {
    extern __shared__ __align__(1024) uint8_t dynamic[];
    __shared__ GemmShared sh;
    constexpr int kBlock = kBlockK<KIND>, kPartsOf = kParts<KIND>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_of(dynamic) + 1023u) & ~1023u;
    const uint32_t a_part = part_bytes<A_DOWN>(kTileM), b_part = part_bytes<B_DOWN>(g.bn);
    const uint32_t a_bytes = a_part * kPartsOf, stage_bytes = a_bytes + b_part * kPartsOf;
    float* blocks = reinterpret_cast<float*>(dynamic + (base - smem_of(dynamic)) + (size_t)stage_bytes * g.stages);
    volatile int* gave_up = &sh.gave_up;

    if (threadIdx.x == 0) {
        sh.gave_up = 0;
        for (int s = 0; s < g.stages; ++s) {
            bar_init(smem_of(&sh.full[s]), BULK ? 1 : kLoaders * 32);
            bar_init(smem_of(&sh.empty[s]), 1);
        }
        for (int h = 0; h < 2; ++h) {
            bar_init(smem_of(&sh.sums_full[h]), 1);
            bar_init(smem_of(&sh.sums_empty[h]), kFinishers);
        }
        bar_init(smem_of(&sh.drained), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kLoaders) tmem_alloc(smem_of(&sh.tmem), (uint32_t)g.columns);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const uint32_t half_columns = (uint32_t)g.bn * (KIND == kSplit ? 2u : 1u);

    if (warp < kLoaders) {
        if (!BULK || threadIdx.x == 0) {
            int64_t fill = 0;      // stages filled so far
            bool ok = true;
            for (int64_t item = blockIdx.x; item < g.items && ok; item += gridDim.x) {
                int64_t tm, tn, split;
                tile_of(g, item, tm, tn, split);
                const int64_t k0 = split * g.k_split, k1 = min(g.k, k0 + g.k_split);
                for (int64_t k = k0; k < k1 && ok; k += kBlock, ++fill) {
                    const int s = (int)(fill % g.stages);
                    const uint32_t parity = (uint32_t)(fill / g.stages) & 1u;
                    const bool with_b = !g.b_stays || fill < g.stages;
                    const uint32_t tile_a = base + (uint32_t)s * stage_bytes, tile_b = tile_a + a_bytes;
                    const uint32_t full = smem_of(&sh.full[s]), empty = smem_of(&sh.empty[s]);
                    if constexpr (BULK) {
                        if (!(ok = bar_wait(empty, parity ^ 1u, gave_up))) break;
                        bar_expect(full, a_part + (with_b ? b_part : 0u));
                        if constexpr (A_DOWN) {
                            for (int box = 0; box < kTileM / 64; ++box)
                                tma_load_2d(tile_a + box * 64 * kRowBytes, &map_a, (int)(tm * kTileM + box * 64), (int)k, full);
                        } else {
                            tma_load_2d(tile_a, &map_a, (int)k, (int)(tm * kTileM), full);
                        }
                        if (with_b) {
                            if constexpr (B_DOWN) {
                                for (int box = 0; box * 64 < g.bn; ++box)
                                    tma_load_2d(tile_b + box * 64 * kRowBytes, &map_b, (int)(tn * g.bn + box * 64), (int)k, full);
                            } else {
                                tma_load_2d(tile_b, &map_b, (int)k, (int)(tn * g.bn), full);
                            }
                        }
                    } else {
                        constexpr int kValues = KIND == kEight ? 16 : 8, kStep = KIND == kEight ? 32 : 16;
                        const int left = (int)min((int64_t)kBlock, k1 - k);
                        const int words = (left + kStep - 1) / kStep * (kStep / kValues);
                        // 224 threads, 1024 words of A and as many of B (twice as many of 16 and 8 bits)
                        constexpr int kB = KIND == kSplit ? 5 : 10;
                        TileFetch<KIND, A_DOWN, 5> fa;
                        TileFetch<KIND, B_DOWN, kB> fb;
                        const int b_chunks = (int)(b_part / 16);
                        fa.fetch(g.a, threadIdx.x, 1024, tm * kTileM, g.m, k, k1, words);
                        if (with_b) fb.fetch(g.b, threadIdx.x, b_chunks, tn * g.bn, g.n, k, k1, words);
                        if (!(ok = bar_wait(empty, parity ^ 1u, gave_up))) break;
                        fa.put(tile_a, a_part, threadIdx.x, 1024, words);
                        if (with_b) fb.put(tile_b, b_part, threadIdx.x, b_chunks, words);
                        fence_async_shared();
                        bar_arrive(full);
                    }
                }
            }
            if (BULK && !ok)      // the copies still under way end before the CTA does
                for (int64_t f = max((int64_t)0, fill - g.stages); f < fill; ++f)
                    bar_drain(smem_of(&sh.full[f % g.stages]), (uint32_t)(f / g.stages) & 1u);
        }
    } else if (warp == kLoaders) {
        if (lane == 0) {
            int64_t fill = 0, phase = 0;
            bool ok = true;
            for (int64_t item = blockIdx.x; item < g.items && ok; item += gridDim.x) {
                int64_t tm, tn, split;
                tile_of(g, item, tm, tn, split);
                const int64_t k0 = split * g.k_split, k1 = min(g.k, k0 + g.k_split);
                const int64_t phase_k = KIND == kSplit ? (int64_t)kPhaseBlocks * kBlock : g.k_split;
                for (int64_t p0 = k0; p0 < k1 && ok; p0 += phase_k, ++phase) {
                    const int h = (int)(phase & 1);
                    const uint32_t sums = tmem + (uint32_t)h * half_columns;
                    if (!(ok = bar_wait(smem_of(&sh.sums_empty[h]), ((uint32_t)(phase >> 1) & 1u) ^ 1u, gave_up))) break;
                    tc_fence_after();
                    const int64_t p1 = min(k1, p0 + phase_k);
                    bool add = false;
                    for (int64_t k = p0; k < p1; k += kBlock, ++fill) {
                        const int s = (int)(fill % g.stages);
                        if (!(ok = bar_wait(smem_of(&sh.full[s]), (uint32_t)(fill / g.stages) & 1u, gave_up))) break;
                        tc_fence_after();
                        constexpr int kStep = KIND == kEight ? 32 : 16;
                        const int steps = (int)((min((int64_t)kBlock, k1 - k) + kStep - 1) / kStep);
                        const uint32_t tile_a = base + (uint32_t)s * stage_bytes, tile_b = tile_a + a_bytes;
                        // a step along k: 32 bytes along rows, 16 rows down them
                        constexpr uint64_t a_step = (A_DOWN ? 16 * kRowBytes : 32) >> 4, b_step = (B_DOWN ? 16 * kRowBytes : 32) >> 4;
                        const uint64_t a = tile_desc(tile_a, 64 * kRowBytes), b = tile_desc(tile_b, 64 * kRowBytes);
                        if constexpr (KIND == kSplit) {
                            const uint64_t ap = a_part >> 4, bp = b_part >> 4;
                            for (int i = 0; i < steps; ++i) {
                                const uint64_t ai = a + i * a_step, bi = b + i * b_step;
                                product<false>(sums, ai, bi, g.desc, add);
                                const uint32_t small = sums + (uint32_t)g.bn;
                                product<false>(small, ai + 2 * ap, bi, g.desc, add);
                                product<false>(small, ai, bi + 2 * bp, g.desc, true);
                                product<false>(small, ai + ap, bi + bp, g.desc, true);
                                product<false>(small, ai + ap, bi, g.desc, true);
                                product<false>(small, ai, bi + bp, g.desc, true);
                                add = true;
                            }
                        } else {
                            for (int i = 0; i < steps; ++i) {
                                product<KIND == kEight>(sums, a + i * a_step, b + i * b_step, g.desc, add);
                                add = true;
                            }
                        }
                        products_done(smem_of(&sh.empty[s]));
                    }
                    if (ok) products_done(smem_of(&sh.sums_full[h]));
                }
            }
            if (!ok) {      // tensor memory is not given back under products still running
                products_done(smem_of(&sh.drained));
                bar_drain(smem_of(&sh.drained), 0);
                atomicAdd(&g_layer_timeouts, 1u);
            }
        }
    } else {
        const int quarter = warp & 3, which = (warp - kLoaders - 1) >> 2;      // lanes of tensor memory; which of the blocks of 32 columns
        float* block = blocks + (size_t)(warp - kLoaders - 1) * 32 * 32;
        const int n_blocks = (g.bn + 31) >> 5;
        int64_t phase = 0;
        bool ok = true;
        for (int64_t item = blockIdx.x; item < g.items && ok; item += gridDim.x) {
            int64_t tm, tn, split;
            tile_of(g, item, tm, tn, split);
            const int64_t row0 = tm * kTileM + quarter * 32, col0 = tn * g.bn;
            if constexpr (KIND == kSplit) {
                float sums[2][32];
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int j = 0; j < 32; ++j) sums[c][j] = 0.0f;
                const int64_t k0 = split * g.k_split, k1 = min(g.k, k0 + g.k_split);
                for (int64_t p0 = k0; p0 < k1 && ok; p0 += (int64_t)kPhaseBlocks * kBlock, ++phase) {
                    const int h = (int)(phase & 1);
                    ok = __all_sync(0xffffffffu, bar_wait(smem_of(&sh.sums_full[h]), (uint32_t)(phase >> 1) & 1u, gave_up));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t at = tmem + (uint32_t)h * half_columns + ((uint32_t)(quarter * 32) << 16);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int blk = which + 2 * c;
                        if (blk >= n_blocks) continue;
                        float r[32];
                        tmem_load32(at + (uint32_t)(g.bn + blk * 32), r);
#pragma unroll
                        for (int j = 0; j < 32; ++j) sums[c][j] += r[j];
                        tmem_load32(at + (uint32_t)(blk * 32), r);
#pragma unroll
                        for (int j = 0; j < 32; ++j) sums[c][j] += r[j];
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(smem_of(&sh.sums_empty[h]));
                }
                if (!ok) break;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int blk = which + 2 * c;
                    if (blk >= n_blocks) continue;
                    put_block(block, lane, sums[c]);
                    __syncwarp();
                    finish<KIND, !A_DOWN && !B_DOWN>(g, block, lane, row0, col0 + blk * 32, split);
                    __syncwarp();
                }
            } else {
                const int h = (int)(phase & 1);
                ok = __all_sync(0xffffffffu, bar_wait(smem_of(&sh.sums_full[h]), (uint32_t)(phase >> 1) & 1u, gave_up));
                if (!ok) break;
                ++phase;
                tc_fence_after();
                const uint32_t at = tmem + (uint32_t)h * half_columns + ((uint32_t)(quarter * 32) << 16);
                for (int blk = which; blk < n_blocks; blk += 2) {
                    float r[32];
                    tmem_load32(at + (uint32_t)(blk * 32), r);
                    put_block(block, lane, r);
                    if (blk + 2 >= n_blocks) {      // the sums are out: the next tile but one may have their place
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) bar_arrive(smem_of(&sh.sums_empty[h]));
                    }
                    __syncwarp();
                    finish<KIND, !A_DOWN && !B_DOWN>(g, block, lane, row0, col0 + blk * 32, split);
                    __syncwarp();
                }
                if (which >= n_blocks && lane == 0) bar_arrive(smem_of(&sh.sums_empty[h]));   // had none of them
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kLoaders) tmem_free(tmem, (uint32_t)g.columns);
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
__global__ void __launch_bounds__(256) few_rows_kernel(const GemmArgs g) {
    constexpr int kVec = 16 / sizeof(T);
    const int lane = threadIdx.x & 31;
    const T* x = static_cast<const T*>(g.a.at);
    const int rows = (int)g.m;
    for (int64_t n = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); n < g.n; n += (int64_t)gridDim.x * 8) {
        const T* w = static_cast<const T*>(g.b.at) + n * g.b.stride;
        float sum[kFewRows] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (g.a.wide && g.b.wide) {
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
            float z = mine, d = 1.0f;
            if (f.b_scales) z *= f.a_scales[lane] * f.b_scales[n];
            if (f.bias) z += to_float(static_cast<const OUT*>(f.bias)[n]);
            const float r = f.residual ? to_float(static_cast<const OUT*>(f.residual)[lane * f.residual_stride + n]) : 0.0f;
            const int64_t at = lane * g.n + n;
            by_activation(f.activation, [&](auto act) {
                constexpr int ACT = decltype(act)::value;
                z = f.slope ? activate<ACT, true, ROUNDED>(f.omega, z, d) : activate<ACT, false, ROUNDED>(f.omega, z, d);
            });
            if (f.slope) static_cast<OUT*>(f.slope)[at] = from_float<OUT>(d);
            static_cast<OUT*>(f.out)[at] = from_float<OUT>(z + r);
        }
    }
}

// ---- dz and its column sums -------------------------------------------------------------------------------------------
// dz = dy * slope (slope kind 1) or dy where the output is positive (kind 2: relu without a residual); column sums of it
// (kind 0: of dy) over the rows of a CTA go to partial[CTA][outputs].  A row has as many lanes as it has accesses, 32 at
// most; blockIdx.x picks the columns of wider rows.
template <class T, int VEC>
__global__ void __launch_bounds__(256) slope_kernel(const T* __restrict__ dy, const T* __restrict__ slope, int kind,
                                                    int64_t rows, int64_t n, int lanes, T* __restrict__ dz,
                                                    float* __restrict__ partial) {
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
            if (kind != 0) {
                load_n<T, VEC>(slope + r * n + col, s);
#pragma unroll
                for (int j = 0; j < VEC; ++j) g[j] = kind == 1 ? g[j] * s[j] : s[j] > 0.0f ? g[j] : 0.0f;
                store_n<T, VEC>(dz + r * n + col, g);
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

// Sums over the first dimension of `partial` [count][n] in a fixed order: the weight's gradient from the splits and the
// bias's from the CTAs above, one launch.  MANY: eight warps share the terms of 32 columns; else a thread sums a column.
template <class T>
struct Join {
    const float* partial;
    int64_t count, n;
    T* out;
    unsigned blocks;
};
template <class T>
__global__ void __launch_bounds__(256) join_kernel(const Join<T> first, const Join<T> second) {
    __shared__ float mine[8][32];
    const bool is_first = blockIdx.x < first.blocks;
    const Join<T>& j = is_first ? first : second;
    const int64_t block = is_first ? blockIdx.x : blockIdx.x - first.blocks;
    if (j.count <= 8) {
        const int64_t col = block * 256 + threadIdx.x;
        if (col >= j.n) return;
        float v = 0.0f;
        for (int64_t i = 0; i < j.count; ++i) v += j.partial[i * j.n + col];
        j.out[col] = from_float<T>(v);
        return;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t col = block * 32 + lane;
    float v = 0.0f;
    if (col < j.n) {
#pragma unroll 8
        for (int64_t i = warp; i < j.count; i += 8) v += j.partial[i * j.n + col];
    }
    mine[warp][lane] = v;
    __syncthreads();
    if (warp != 0 || col >= j.n) return;
    float t = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) t += mine[w][lane];
    j.out[col] = from_float<T>(t);
}

// ---- plans --------------------------------------------------------------------------------------------------------------
static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Plan {
    int bn, stages, b_stays, columns;
    int64_t tiles_m, tiles_n, splits, k_split;
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
    const int block = kind == kEight ? 128 : 64, parts = kind == kSplit ? 3 : 1, sms = sm_count();
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
        const int64_t most = may_split ? std::min<int64_t>(std::max<int64_t>(1, blocks / 4), ceil_div(2 * sms, tiles)) : 1;
        for (int64_t s = 1; s <= most; ++s) {
            const int64_t per = ceil_div(blocks, s), splits = ceil_div(blocks, per);
            // a split writes and reads its sums once more: 8 bytes a value at about 3000 bytes a cycle of the whole GPU
            const double join = splits > 1 ? 8.0 * splits * m * n / 3000.0 + 3000.0 : 0.0;
            const double c = cycles(kind, bn, per, tiles * splits, sms) + join;
            if (least == 0.0 || c < least) {
                least = c;
                p.splits = splits;
                p.k_split = per * block;
                best = p;
            }
        }
    }
    const size_t stage = (size_t)parts * ((a_down ? part_bytes<true>(kTileM) : part_bytes<false>(kTileM)) +
                                          (b_down ? part_bytes<true>(best.bn) : part_bytes<false>(best.bn)));
    const size_t room = kSharedLimit - 2048 - kFinishBytes;
    best.stages = (int)std::min<size_t>(kMaxStages, room / stage);
    const int64_t blocks = ceil_div(k, block);
    if (best.tiles_n == 1 && best.splits == 1 && blocks <= best.stages) {
        best.b_stays = 1;
        best.stages = (int)(best.stages / blocks * blocks);
    }
    // more than half of the SM's shared memory: a second CTA would wait for tensor memory
    best.shared = std::max<size_t>((size_t)best.stages * stage + kFinishBytes + 1024, 120 * 1024);
    const int columns = 2 * best.bn * (kind == kSplit ? 2 : 1);
    best.columns = 32;
    while (best.columns < columns) best.columns <<= 1;
    return best;
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
    const int bytes = kind == kEight ? 1 : 2;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(o.stride * bytes)};
    const cuuint32_t box[2] = {(cuuint32_t)(kRowBytes / bytes), (cuuint32_t)box_rows}, steps[2] = {1, 1};
    const CUtensorMapDataType t = kind == kEight ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                  : type == ASHB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const auto encode = encode_tiled();
    return encode != nullptr &&
           encode(map, t, 2, const_cast<void*>(o.at), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int KIND, bool BULK, bool A_DOWN, bool B_DOWN>
static cudaError_t launch_product(const GemmArgs& g, const Plan& p, const CUtensorMap& ma, const CUtensorMap& mb, cudaStream_t st) {
    const auto kernel = layer_gemm_kernel<KIND, BULK, A_DOWN, B_DOWN>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kSharedLimit - 1024));
    if (e != cudaSuccess) return e;
    kernel<<<(unsigned)std::min<int64_t>(g.items, sm_count()), kGemmThreads, p.shared, st>>>(g, ma, mb);
    return cudaGetLastError();
}

template <int KIND, bool A_DOWN, bool B_DOWN>
static int run_product(GemmArgs g, int type, const Plan& p, cudaStream_t st) {
    constexpr int kBytes = KIND == kEight ? 1 : KIND == kSplit ? 4 : 2;
    const auto wide = [&](const Operand& o) { return ((uintptr_t)o.at & 15) == 0 && o.stride * kBytes % 16 == 0; };
    g.a.wide = wide(g.a);
    g.b.wide = wide(g.b);
    g.bn = p.bn;
    g.stages = p.stages;
    g.b_stays = p.b_stays;
    g.columns = p.columns;
    g.tiles_m = p.tiles_m;
    g.tiles_n = p.tiles_n;
    g.k_split = p.k_split;
    g.items = p.tiles_m * p.tiles_n * p.splits;
    g.desc = product_desc(kTileM, p.bn, KIND == kEight ? 0 : KIND == kSplit || type == ASHB_BF16 ? 1 : 0, A_DOWN, B_DOWN);
    CUtensorMap ma{}, mb{};
    cudaError_t e;
    const bool bulk = KIND != kSplit && g.a.wide && g.b.wide &&
                      operand_map(&ma, KIND, type, g.a, A_DOWN ? g.k : g.m, A_DOWN ? g.m : g.k, A_DOWN ? 64 : kTileM) &&
                      operand_map(&mb, KIND, type, g.b, B_DOWN ? g.k : g.n, B_DOWN ? g.n : g.k, B_DOWN ? 64 : p.bn);
    if constexpr (KIND != kSplit) {
        e = bulk ? launch_product<KIND, true, A_DOWN, B_DOWN>(g, p, ma, mb, st)
                 : launch_product<KIND, false, A_DOWN, B_DOWN>(g, p, ma, mb, st);
    } else {
        e = launch_product<KIND, false, A_DOWN, B_DOWN>(g, p, ma, mb, st);
    }
    ASHB_CUDA_TRY(e);
    return ASHB_OK;
}

template <bool A_DOWN, bool B_DOWN>
static int run_typed(const GemmArgs& g, int type, const Plan& p, cudaStream_t st) {
    return type == ASHB_F32 ? run_product<kSplit, A_DOWN, B_DOWN>(g, type, p, st)
                            : run_product<kHalf, A_DOWN, B_DOWN>(g, type, p, st);
}

static int kind_of(int type) { return type == ASHB_F32 ? kSplit : type == ASHB_E4M3_ROWS ? kEight : kHalf; }

template <class T, class OUT>
static void launch_few(const GemmArgs& g, cudaStream_t st) {
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(g.n, 8), (int64_t)sm_count() * 8);
    few_rows_kernel<T, OUT, sizeof(OUT) == 2><<<grid, 256, 0, st>>>(g);
}

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
    p.down = (unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(rows, groups * 4), ceil_div((int64_t)sm_count() * 8, p.across)));
    return p;
}
// the largest `down` of both forms, for the workspace
static int64_t slope_rows(int type, int64_t rows, int64_t n) {
    return std::max(plan_slope(type, rows, n, true).down, plan_slope(type, rows, n, false).down);
}

template <class T>
static void launch_slope(const SlopePlan& p, const void* dy, const void* slope, int kind, int64_t rows, int64_t n, void* dz,
                         float* partial, cudaStream_t st) {
    const dim3 grid(p.across, p.down);
    const T *g = static_cast<const T*>(dy), *s = static_cast<const T*>(slope);
    if (p.vec > 1) slope_kernel<T, 16 / sizeof(T)><<<grid, 256, 0, st>>>(g, s, kind, rows, n, p.lanes, static_cast<T*>(dz), partial);
    else slope_kernel<T, 1><<<grid, 256, 0, st>>>(g, s, kind, rows, n, p.lanes, static_cast<T*>(dz), partial);
}

template <class T>
static void launch_join(const float* pw, int64_t count_w, int64_t n_w, void* dw, const float* pb, int64_t count_b, int64_t n_b,
                        void* db, cudaStream_t st) {
    const auto make = [](const float* p, int64_t count, int64_t n, void* out) {
        return Join<T>{p, count, n, static_cast<T*>(out), p ? (unsigned)ceil_div(n, count <= 8 ? 256 : 32) : 0u};
    };
    const Join<T> w = make(pw, count_w, n_w, dw), b = make(pb, count_b, n_b, db);
    if (w.blocks + b.blocks) join_kernel<T><<<w.blocks + b.blocks, 256, 0, st>>>(w, b);
}

static size_t padded(size_t bytes) { return (bytes + 255) / 256 * 256; }

struct BackwardPlan {
    size_t dz, bias, weight, total;      // offsets into the workspace
    Plan pw;
};
static BackwardPlan plan_backward(int type, int64_t rows, int64_t inputs, int64_t outputs, int kind, bool want_w, bool want_b) {
    BackwardPlan b{};
    size_t at = 0;
    b.dz = at;
    if (kind != 0) at += padded((size_t)(rows * outputs) * value_bytes(type));
    b.bias = at;
    if (want_b) at += padded((size_t)(slope_rows(type, rows, outputs) * outputs) * sizeof(float));
    b.weight = at;
    if (want_w) {
        b.pw = plan_product(kind_of(type), true, true, outputs, inputs, rows, true);
        if (b.pw.splits > 1) at += padded((size_t)(b.pw.splits * outputs * inputs) * sizeof(float));
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
                        int out_type, void* y, void* slope, void* stream) {
    const bool eight = type == ASHB_E4M3_ROWS;
    ASHB_REQUIRE(is_value_type(type) || eight, "operand type %d", type);
    ASHB_REQUIRE(is_value_type(out_type) && (eight || out_type == type), "output type %d", out_type);
    ASHB_REQUIRE(activation >= kNone && activation <= kSin, "activation %d", activation);
    if (int rc = check_sizes(rows, inputs, outputs)) return rc;
    if (rows == 0) return ASHB_OK;
    ASHB_REQUIRE(x && weight && y && (!eight || (x_scales && weight_scales)), "null buffer");
    ASHB_REQUIRE((x_stride >= inputs || rows == 1) && weight_stride >= inputs, "rows overlap");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    GemmArgs g{};
    g.a = Operand{x, x_stride, 0};
    g.b = Operand{weight, weight_stride, 0};
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
             (((uintptr_t)y | (uintptr_t)slope | (uintptr_t)bias | (uintptr_t)residual) & (four - 1)) == 0 &&
             ((uintptr_t)f.b_scales & 15) == 0;
    if (rows <= kFewRows) {
        const int bytes = eight ? 1 : value_bytes(type);
        const auto wide = [&](const Operand& o) {
            return ((uintptr_t)o.at & 15) == 0 && o.stride * bytes % 16 == 0 && inputs * bytes % 16 == 0;
        };
        g.a.wide = wide(g.a);
        g.b.wide = wide(g.b);
        if (type == ASHB_F32) launch_few<float, float>(g, st);
        else if (type == ASHB_F16) launch_few<__half, __half>(g, st);
        else if (type == ASHB_BF16) launch_few<__nv_bfloat16, __nv_bfloat16>(g, st);
        else if (out_type == ASHB_F32) launch_few<E4M3, float>(g, st);
        else if (out_type == ASHB_F16) launch_few<E4M3, __half>(g, st);
        else launch_few<E4M3, __nv_bfloat16>(g, st);
        ASHB_LAUNCH_CHECK();
        return ASHB_OK;
    }
    const Plan p = plan_product(kind_of(type), false, false, rows, outputs, inputs, false);
    ASHB_REQUIRE(!slope || (!eight && activation != kNone), "a slope is of an activation, of operands that are not quantised");
    if (eight) return run_product<kEight, false, false>(g, type, p, st);
    return run_typed<false, false>(g, type, p, st);
}

int64_t ashb_linear_workspace(int type, int64_t rows, int64_t inputs, int64_t outputs, int slope_kind, int want_dweight,
                              int want_dbias) {
    if (!is_value_type(type) || check_sizes(rows, inputs, outputs) != ASHB_OK || rows == 0) return 0;
    return (int64_t)plan_backward(type, rows, inputs, outputs, slope_kind, want_dweight != 0, want_dbias != 0).total;
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
    const BackwardPlan bp = plan_backward(type, rows, inputs, outputs, slope_kind, dweight != nullptr, dbias != nullptr);
    ASHB_REQUIRE(bp.total == 0 || (workspace && ((uintptr_t)workspace & 255) == 0 && workspace_bytes >= (int64_t)bp.total),
                 "null, unaligned or small workspace");
    char* ws = static_cast<char*>(workspace);
    const void* dz = slope_kind != 0 ? ws + bp.dz : dy;
    float* pb = dbias ? reinterpret_cast<float*>(ws + bp.bias) : nullptr;
    int64_t count_b = 0;
    if (slope_kind != 0 || dbias) {
        const bool wide = outputs * (int64_t)e % 16 == 0 && (((uintptr_t)dy | (uintptr_t)slope) & 15) == 0;
        const SlopePlan sp = plan_slope(type, rows, outputs, wide);
        count_b = sp.down;
        if (type == ASHB_F32) launch_slope<float>(sp, dy, slope, slope_kind, rows, outputs, ws + bp.dz, pb, st);
        else if (type == ASHB_F16) launch_slope<__half>(sp, dy, slope, slope_kind, rows, outputs, ws + bp.dz, pb, st);
        else launch_slope<__nv_bfloat16>(sp, dy, slope, slope_kind, rows, outputs, ws + bp.dz, pb, st);
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
    if (dx) {
        GemmArgs g{};
        g.a = Operand{dz, outputs, 0};
        g.b = Operand{weight, weight_stride, 0};
        g.f = finish_to(dx, inputs);
        g.m = rows;
        g.n = inputs;
        g.k = outputs;
        const Plan p = plan_product(kind_of(type), false, true, rows, inputs, outputs, false);
        if (int rc = run_typed<false, true>(g, type, p, st)) return rc;
    }
    const float* pw = nullptr;
    if (dweight) {
        GemmArgs g{};
        g.a = Operand{dz, outputs, 0};
        g.b = Operand{x, x_stride, 0};
        g.f = finish_to(dweight, inputs);
        g.m = outputs;
        g.n = inputs;
        g.k = rows;
        if (bp.pw.splits > 1) {
            g.f.partial = reinterpret_cast<float*>(ws + bp.weight);
            pw = g.f.partial;
        }
        if (int rc = run_typed<true, true>(g, type, bp.pw, st)) return rc;
    }
    if (type == ASHB_F32) launch_join<float>(pw, bp.pw.splits, outputs * inputs, dweight, pb, count_b, outputs, dbias, st);
    else if (type == ASHB_F16) launch_join<__half>(pw, bp.pw.splits, outputs * inputs, dweight, pb, count_b, outputs, dbias, st);
    else launch_join<__nv_bfloat16>(pw, bp.pw.splits, outputs * inputs, dweight, pb, count_b, outputs, dbias, st);
    ASHB_LAUNCH_CHECK();
    return ASHB_OK;
}

int ashb_layer_timeouts(unsigned int* out) {
    ASHB_REQUIRE(out != nullptr, "null output");
    ASHB_CUDA_TRY(cudaMemcpyFromSymbol(out, g_layer_timeouts, sizeof(unsigned int)));
    return ASHB_OK;
}

}  // extern "C"
