// The sm_100a tensor-core instructions that the dense-layer kernels use: mbarriers with bounded waits, tiled bulk copies,
// tensor memory, and tcgen05 products of shared-memory tiles in the 128-byte swizzle.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace ashb {

__device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// ---- mbarriers ---------------------------------------------------------------------------------------------------
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// The thread may sleep for up to a microsecond inside: polling without it takes issue slots from the warps that work.
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t"
            "}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
    return ok != 0;
}

// Polls of a barrier before a wait gives up: between a tenth of a second and four seconds, where the longest wait of a healthy
// launch, for the products of one tile, is milliseconds.
constexpr int kWaitPolls = 1 << 22;

// A CTA's waits: how many polls each may take, and whether one has run out.
struct Waits {
    volatile int* gave_up;
    int polls;
};

// Waits for phase `parity`.  False once the limit has run out here (`gave_up` is set) or anywhere else in the CTA.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, const Waits& waits) {
    if (bar_try(bar, parity)) return true;
    for (int i = 0; i < waits.polls; ++i) {
        if (bar_try(bar, parity)) return true;
        if (*waits.gave_up) return false;
    }
    *waits.gave_up = 1;
    return false;
}
// The same for what must end before the CTA does, whatever has failed in it: only the full limit ends it.
__device__ __forceinline__ void bar_drain(uint32_t bar, uint32_t parity) {
    for (int i = 0; i < kWaitPolls && !bar_try(bar, parity); ++i) {
    }
}

// ---- bulk copies ---------------------------------------------------------------------------------------------------
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, int x, int y, int z, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x), "r"(y), "r"(z),
                 "r"(src)
                 : "memory");
}
__device__ __forceinline__ void tma_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// Until all but the last PENDING groups of this thread's stores have read their shared memory.
template <int PENDING>
__device__ __forceinline__ void tma_wait_read() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(PENDING) : "memory");
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- tensor memory -------------------------------------------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t where, uint32_t columns) {   // one warp; columns: a power of two, 32..512
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t columns) {       // the same warp
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of the warp's 32 lanes: r[c] is column c of this thread's lane.
__device__ __forceinline__ void tmem_load32(uint32_t at, float (&r)[32]) {
    uint32_t u[32];
    asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
            "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
            "tcgen05.wait::ld.sync.aligned;"
            : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
              "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]),
              "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]),
              "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
            : "r"(at)
            : "memory");
#pragma unroll
    for (int c = 0; c < 32; ++c) r[c] = __uint_as_float(u[c]);
}

// Eight columns.
__device__ __forceinline__ void tmem_load8(uint32_t at, float (&r)[8]) {
    uint32_t u[8];
    asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
            "tcgen05.wait::ld.sync.aligned;"
            : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7])
            : "r"(at)
            : "memory");
#pragma unroll
    for (int c = 0; c < 8; ++c) r[c] = __uint_as_float(u[c]);
}
// Eight columns of each of two sums.
__device__ __forceinline__ void tmem_load8_twice(uint32_t at, uint32_t at2, float (&r)[8], float (&s)[8]) {
    uint32_t u[8], v[8];
    asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%16];\n\t"
            "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%17];\n\t"
            "tcgen05.wait::ld.sync.aligned;"
            : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(v[0]), "=r"(v[1]),
              "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
            : "r"(at), "r"(at2)
            : "memory");
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        r[c] = __uint_as_float(u[c]);
        s[c] = __uint_as_float(v[c]);
    }
}

// ---- products --------------------------------------------------------------------------------------------------------
// A shared-memory tile in a swizzle of rows of ROW_BYTES: groups of 8 rows follow one another, the 16-byte word w of row r at
// word w ^ (r & 7) of rows of 128 bytes, at w ^ (r / 2 & 3) of rows of 64.  Rows are the tile's rows where the summed
// dimension runs along them; where the other dimension does (64 values in 128 bytes), `box` is the distance between blocks of
// 64 of them.  The tile starts at a multiple of 1024 bytes (512 for rows of 64).
template <int ROW_BYTES = 128>
__device__ __forceinline__ uint64_t tile_desc(uint32_t at, uint32_t box) {
    static_assert(ROW_BYTES == 128 || ROW_BYTES == 64, "");
    return (uint64_t)((at >> 4) & 0x3FFFu) | (uint64_t)((box >> 4) & 0x3FFFu) << 16 | (uint64_t)((8u * ROW_BYTES) >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)(ROW_BYTES == 128 ? 2 : 4) << 61;
}

// Instruction word: float32 sums of an M x N tile.  `format` of both operands: f16 0, bf16 1 (kind::f16); e4m3 0
// (kind::f8f6f4).  a_rows / b_rows: the summed dimension runs down the rows of the tile instead of along them.
constexpr uint32_t product_desc(int m, int n, int format, bool a_rows, bool b_rows) {
    return 1u << 4 | (uint32_t)format << 7 | (uint32_t)format << 10 | (uint32_t)a_rows << 15 | (uint32_t)b_rows << 16 |
           (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}

// The warp that issues products runs as a whole and one lane of it issues: what the instructions take then stays in registers
// that the warp shares, where a branch for one lane has every operand moved there first (a product of 64 columns took 85
// cycles to issue, and 32 to run).
__device__ __forceinline__ uint32_t elected() {
    uint32_t mine;
    asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "elect.sync _|p, 0xffffffff;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t"
            "}"
            : "=r"(mine));
    return mine;
}

template <bool EIGHT_BITS>
__device__ __forceinline__ void product(uint32_t mine, uint32_t to, uint64_t a, uint64_t b, uint32_t desc, bool add) {
    if constexpr (EIGHT_BITS)
        asm volatile(
                "{\n\t"
                ".reg .pred p, q;\n\t"
                "setp.ne.b32 p, %4, 0;\n\t"
                "setp.ne.b32 q, %5, 0;\n\t"
                "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
                "}" ::"r"(to), "l"(a), "l"(b), "r"(desc), "r"((uint32_t)add), "r"(mine)
                : "memory");
    else
        asm volatile(
                "{\n\t"
                ".reg .pred p, q;\n\t"
                "setp.ne.b32 p, %4, 0;\n\t"
                "setp.ne.b32 q, %5, 0;\n\t"
                "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
                "}" ::"r"(to), "l"(a), "l"(b), "r"(desc), "r"((uint32_t)add), "r"(mine)
                : "memory");
}
// Arrives on `bar` once the products issued before are done.
__device__ __forceinline__ void products_done(uint32_t mine, uint32_t bar) {
    asm volatile(
            "{\n\t"
            ".reg .pred q;\n\t"
            "setp.ne.b32 q, %1, 0;\n\t"
            "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t"
            "}" ::"r"(bar), "r"(mine)
            : "memory");
}

}  // namespace ashb
