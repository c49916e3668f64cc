// Feature rows in 8 bits: the value tables of a hash map quantised as keys are inserted and read back as keys are
// looked up, and the same for rows that lie in order or are named by their numbers.
//
// Both directions are bound by memory: a key moves its 12 bytes, a 16-byte slot of the table at a random place, and
// its row.
// Writing takes two launches: the keys are placed, their rows' numbers noted, then rows are quantised by as many lanes as
// they have quadruples of values (32 at most), four rows of a group under way.  In one launch the registers of the
// second part leave an SM one CTA for the first, whose chains of dependent accesses want many (1M keys with 32 values:
// 331 us against 47 and 48).
// Reading takes one: a CTA looks 128 keys up and notes their rows and scales in shared memory, then its threads walk the
// 128 rows of output as one run of quadruples, four of a thread under way, so that stores are contiguous whatever the width.
// Sixteen CTAs an SM read 4M keys' rows of 64 int8 values, half of them misses, in 291 us (4.4 TB/s); eight of 256 keys, 297 us;
// six with eight quadruples under way, 303 us; lanes of a group per row, 336 us.
#include <algorithm>
#include <cstring>

#include "hashmap.cuh"
#include "rowformat.cuh"

namespace ashb {

constexpr int kMaxRowTables = 16;

struct RowTable {
    const void* src;     // insertion: the batch's values; reading: the codes
    void* dst;           // insertion: the codes (or the rows themselves where format is 0); reading: the values
    float* scales;
    int64_t width;       // values a row (format 0: bytes a row)
    int format;          // 0: copied as bytes
    int dtype;           // of the values
    int wide;            // quadruples are aligned on both sides
    int long_rows;       // reading: a CTA's run has too many places for 32 bits
    uint32_t reciprocal; // reading: of a row's steps, for a place's row in a run (0: one step a row)
};
struct RowTables {
    int n;
    RowTable t[kMaxRowTables];
};

template <class T>
__device__ __forceinline__ void load4(const T* __restrict__ row, int64_t col, int64_t width, bool wide, float (&v)[4]) {
    if (wide) {
        load_n<T, 4>(row + col, v);
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = col + k < width ? to_float(row[col + k]) : 0.0f;
}

__device__ __forceinline__ void store_codes(uint8_t* __restrict__ row, int64_t col, int64_t width, bool wide, uint32_t w) {
    if (wide) {
        *reinterpret_cast<uint32_t*>(row + col) = w;
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (col + k < width) row[col + k] = (uint8_t)(w >> (8 * k));
}

// ---- writing rows ------------------------------------------------------------------------------------------------------
// Row r of the values, r < n, to row row_of[r] of the table (negative: left out; null: to row r).  A row has `lanes` lanes,
// the power of two that covers its quadruples, 32 at most.  QUADS quadruples a lane and ROWS rows stay in registers; a
// longer row is read a second time, from L1.
template <class T, int QUADS, int ROWS>
__global__ void __launch_bounds__(256, 5) quantize_rows_kernel(int64_t n, const int32_t* __restrict__ row_of, int lanes,
                                                            const __grid_constant__ RowTable t) {
    const int sub = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes, groups = 256 / lanes;
    const T* src = static_cast<const T*>(t.src);
    uint8_t* codes = static_cast<uint8_t*>(t.dst);
    const int64_t first = (int64_t)blockIdx.x * groups * ROWS + group;
    float v[ROWS][QUADS][4];
    int to[ROWS];
    uint32_t amax[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int64_t r = first + i * groups;
        to[i] = r < n ? (row_of ? row_of[r] : (int)r) : -1;
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const T* row = src + (first + i * groups) * t.width;
        amax[i] = 0;
#pragma unroll
        for (int q = 0; q < QUADS; ++q) {
            const int64_t col = ((int64_t)q * lanes + sub) * 4;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[i][q][k] = 0.0f;
            if (to[i] >= 0 && col < t.width) load4(row, col, t.width, t.wide, v[i][q]);
        }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
#pragma unroll
        for (int q = 0; q < QUADS; ++q)
#pragma unroll
            for (int k = 0; k < 4; ++k) amax[i] = max(amax[i], magnitude_bits(v[i][q][k]));
        if (to[i] >= 0) {
            const T* row = src + (first + i * groups) * t.width;
            for (int64_t col = ((int64_t)QUADS * lanes + sub) * 4; col < t.width; col += lanes * 4) {
                float u[4];
                load4(row, col, t.width, t.wide, u);
#pragma unroll
                for (int k = 0; k < 4; ++k) amax[i] = max(amax[i], magnitude_bits(u[k]));
            }
        }
        for (int o = lanes >> 1; o > 0; o >>= 1) amax[i] = max(amax[i], __shfl_xor_sync(0xffffffffu, amax[i], o));
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        if (to[i] < 0) continue;
        const RowScale s(amax[i], t.format);
        uint8_t* out = codes + to[i] * t.width;
#pragma unroll
        for (int q = 0; q < QUADS; ++q) {
            const int64_t col = ((int64_t)q * lanes + sub) * 4;
            if (col < t.width) store_codes(out, col, t.width, t.wide, encode4(v[i][q], s.inverse, t.format));
        }
        const T* row = src + (first + i * groups) * t.width;
        for (int64_t col = ((int64_t)QUADS * lanes + sub) * 4; col < t.width; col += lanes * 4) {
            float u[4];
            load4(row, col, t.width, t.wide, u);
            store_codes(out, col, t.width, t.wide, encode4(u, s.inverse, t.format));
        }
        if (sub == 0) t.scales[to[i]] = s.scale;
    }
}

// ---- reading rows ------------------------------------------------------------------------------------------------------
// The rows of kReaders keys or numbers: rows[i] of the codes (negative: zeros) to row first + i of the values, i < have.
// UNIT values a step of a thread: four, or one where rows are not multiples of four or not aligned.
constexpr int kReadsAhead = 4, kReaders = 128;
template <class T, int UNIT>
__device__ __forceinline__ void read_run(const RowTable& t, int64_t first, int have, const int* rows, const float* scales) {
    const uint8_t* codes = static_cast<const uint8_t*>(t.src);
    T* out = static_cast<T*>(t.dst) + first * t.width;
    const uint32_t per_row = (uint32_t)t.width / UNIT, total = per_row * (uint32_t)have;
    for (uint32_t e0 = threadIdx.x; e0 < total; e0 += kReaders * kReadsAhead) {
        uint32_t w[kReadsAhead];
        float scale[kReadsAhead];
#pragma unroll
        for (int i = 0; i < kReadsAhead; ++i) {
            const uint32_t e = e0 + kReaders * i;
            w[i] = 0;
            scale[i] = 0.0f;
            if (e >= total) continue;
            const uint32_t r = t.reciprocal ? __umulhi(e, t.reciprocal) : e;
            const int row = rows[r];
            if (row < 0) continue;
            const uint8_t* p = codes + row * t.width + (e - r * per_row) * UNIT;
            w[i] = UNIT == 4 ? __ldg(reinterpret_cast<const uint32_t*>(p)) : (uint32_t)__ldg(p);
            scale[i] = scales[r];
        }
#pragma unroll
        for (int i = 0; i < kReadsAhead; ++i) {
            const uint32_t e = e0 + kReaders * i;
            if (e >= total) continue;
            float v[4];
            decode4(w[i], scale[i], t.format, v);
            if constexpr (UNIT == 4) store_n_passing<T, 4>(out + (size_t)e * 4, v);
            else out[e] = from_float<T>(v[0]);
        }
    }
}

// Rows too wide for 32-bit positions in a CTA's run: a row at a time.
template <class T>
__device__ __noinline__ void read_long(const RowTable& t, int64_t first, int have, const int* rows, const float* scales) {
    const uint8_t* codes = static_cast<const uint8_t*>(t.src);
    T* out = static_cast<T*>(t.dst);
    for (int r = 0; r < have; ++r)
        for (int64_t c = threadIdx.x; c < t.width; c += kReaders) {
            float v[4];
            decode4(rows[r] >= 0 ? (uint32_t)codes[rows[r] * t.width + c] : 0u, scales[r], t.format, v);
            out[(first + r) * t.width + c] = from_float<T>(v[0]);
        }
}

template <class T>
__device__ __forceinline__ void read_typed(const RowTable& t, int64_t first, int have, const int* rows, const float* scales) {
    if (t.long_rows) read_long<T>(t, first, have, rows, scales);
    else if (t.wide) read_run<T, 4>(t, first, have, rows, scales);
    else read_run<T, 1>(t, first, have, rows, scales);
}

// All of the CTA: the row of this thread's key is `mine` (negative: none).
__device__ __forceinline__ void read_rows_of(const RowTables& tables, int64_t first, int64_t n, int mine) {
    __shared__ int rows[kReaders];
    __shared__ float scales[kReaders];
    const int have = (int)min((int64_t)kReaders, n - first);
    rows[threadIdx.x] = mine;
    for (int j = 0; j < tables.n; ++j) {
        const RowTable& t = tables.t[j];
        scales[threadIdx.x] = mine >= 0 ? __ldg(t.scales + mine) : 0.0f;
        __syncthreads();
        if (t.dtype == ASHB_F32) read_typed<float>(t, first, have, rows, scales);
        else if (t.dtype == ASHB_F16) read_typed<__half>(t, first, have, rows, scales);
        else read_typed<__nv_bfloat16>(t, first, have, rows, scales);
        __syncthreads();
    }
}

// ---- the hash map's tables -------------------------------------------------------------------------------------
// The keys of insertion: row_of[i] becomes the row of key i if it is new, -1 if not.  Tables of format 0 are copied here, a row
// a thread.  A new key's index is published before its row is written: within a launch nobody reads rows, and the next
// launches of the stream see both.
template <class Table, int DIM>
__global__ void __launch_bounds__(256) insert_rows_kernel(Table t, const int32_t* __restrict__ keys, int64_t n,
                                                          int32_t* __restrict__ heap, int32_t* counter, int32_t capacity,
                                                          int32_t* __restrict__ row_of, const __grid_constant__ RowTables tables) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    int64_t slot = -1;
    if (i < n) {
        int k0, k1, k2, k3;
        load_key<DIM>(keys, i, k0, k1, k2, k3);
        bool present = false;
        slot = emplace(t, k0, k1, k2, k3, kPending, &present);
    }
    const int idx = pop_index_for_slot_cta(t, slot, heap, counter, capacity);
    if (idx >= 0) publish_index(t, slot, idx);
    if (i >= n) return;
    row_of[i] = idx;
    if (idx < 0) return;
    for (int j = 0; j < tables.n; ++j) {
        const RowTable& v = tables.t[j];
        if (v.format != 0) continue;
        const char* src = static_cast<const char*>(v.src) + i * v.width;
        char* dst = static_cast<char*>(v.dst) + idx * v.width;
        if (v.wide)
            for (int64_t b = 0; b < v.width; b += 4) *reinterpret_cast<int*>(dst + b) = *reinterpret_cast<const int*>(src + b);
        else
            for (int64_t b = 0; b < v.width; ++b) dst[b] = src[b];
    }
}

template <class Table, int DIM, bool FILTER>
__global__ void __launch_bounds__(kReaders, 2048 / kReaders) find_rows_kernel(Table t, const int32_t* __restrict__ keys, int64_t n,
                                                        int64_t* __restrict__ indices, uint8_t* __restrict__ masks,
                                                        const __grid_constant__ RowTables tables) {
    const int64_t first = (int64_t)blockIdx.x * kReaders, i = first + threadIdx.x;
    int found = -1;
    if (i < n) {
        int k0, k1, k2, k3;
        load_key<DIM>(keys, i, k0, k1, k2, k3);
        uint32_t s = hash_key(k0, k1, k2, k3) & t.mask;
        bool absent = false;
        if constexpr (FILTER) absent = t.never_used(s);
        for (uint32_t probe = 0; !absent && probe <= t.mask; ++probe) {
            Entry e;
            if constexpr (FILTER) e = t.read_const_passing(s);
            else e = t.read_const(s);
            if (e.val == kEmpty) break;
            if (e.val >= 0 && key_match(e, k0, k1, k2, k3)) {
                found = e.val;
                break;
            }
            s = (s + 1) & t.mask;
        }
        if (indices) __stcs(indices + i, found >= 0 ? (int64_t)found : 0);
        __stcs(masks + i, (uint8_t)(found >= 0));
    }
    read_rows_of(tables, first, n, found);
}

// ---- rows in order, or by number -------------------------------------------------------------------------------
// A number outside 0 .. n_rows - 1 reads zeros.
__global__ void __launch_bounds__(kReaders, 2048 / kReaders) read_rows_kernel(int64_t n, const int64_t* __restrict__ numbers, int64_t n_rows,
                                                        const __grid_constant__ RowTables tables) {
    const int64_t first = (int64_t)blockIdx.x * kReaders, i = first + threadIdx.x;
    const int64_t row = i < n ? (numbers ? numbers[i] : i) : -1;
    read_rows_of(tables, first, n, row >= 0 && row < n_rows ? (int)row : -1);
}

template <class T>
static void launch_quantize(int64_t n, const int32_t* row_of, const RowTable& t, cudaStream_t st) {
    int lanes = 1;
    while (lanes < 32 && (int64_t)lanes * 4 < t.width) lanes <<= 1;
    const int groups = 256 / lanes;
    // rows of up to 128 values: one quadruple a lane, four rows under way; else four quadruples of one row
    if (t.width <= 128) quantize_rows_kernel<T, 1, 4><<<(unsigned)((n + 4 * groups - 1) / (4 * groups)), 256, 0, st>>>(n, row_of, lanes, t);
    else quantize_rows_kernel<T, 4, 1><<<(unsigned)((n + groups - 1) / groups), 256, 0, st>>>(n, row_of, lanes, t);
}

static void quantize_table(int64_t n, const int32_t* row_of, const RowTable& t, cudaStream_t st) {
    if (t.dtype == ASHB_F32) launch_quantize<float>(n, row_of, t, st);
    else if (t.dtype == ASHB_F16) launch_quantize<__half>(n, row_of, t, st);
    else launch_quantize<__nv_bfloat16>(n, row_of, t, st);
}

}  // namespace ashb

using namespace ashb;

static int check_table(const ashb_row_table* in, bool reading, bool may_copy, RowTable* out) {
    std::memset(out, 0, sizeof(*out));
    ASHB_REQUIRE(in->src && in->dst && in->width > 0, "row table: null pointer or empty row");
    ASHB_REQUIRE(in->format == ASHB_E4M3 || in->format == ASHB_INT8 || (may_copy && in->format == 0),
                 "row table: format %d", in->format);
    out->src = in->src;
    out->dst = in->dst;
    out->scales = in->scales;
    out->width = in->width;
    out->format = in->format;
    out->dtype = in->dtype;
    if (in->format == 0) {
        out->wide = (((uintptr_t)in->src | (uintptr_t)in->dst | (uintptr_t)in->width) & 3) == 0;
        return ASHB_OK;
    }
    ASHB_REQUIRE(in->scales != nullptr, "row table: null scales");
    ASHB_REQUIRE(is_value_type(in->dtype), "row table: value type %d", in->dtype);
    const uintptr_t values = (uintptr_t)(reading ? in->dst : in->src), codes = (uintptr_t)(reading ? in->src : in->dst);
    ASHB_REQUIRE((values & (value_bytes(in->dtype) - 1)) == 0, "row table: values not aligned to their type");
    out->wide = in->width % 4 == 0 && (values & (4 * value_bytes(in->dtype) - 1)) == 0 && (codes & 3) == 0;
    // e * ceil(2^32 / steps) >> 32 is e / steps while e * steps < 2^32, e being below 256 * steps (kReaders is no more)
    const int64_t steps = out->wide ? in->width / 4 : in->width;
    out->long_rows = steps >= 4096;
    out->reciprocal = steps == 1 || out->long_rows ? 0u : (uint32_t)(((1ull << 32) + (uint64_t)steps - 1) / (uint64_t)steps);
    return ASHB_OK;
}

static int check_tables(int n, const ashb_row_table* in, bool reading, bool may_copy, RowTables* out) {
    std::memset(out, 0, sizeof(*out));
    ASHB_REQUIRE(n >= 0 && n <= kMaxRowTables, "%d row tables, at most %d", n, kMaxRowTables);
    ASHB_REQUIRE(n == 0 || in != nullptr, "null row tables");
    out->n = n;
    for (int j = 0; j < n; ++j)
        if (int rc = check_table(in + j, reading, may_copy, &out->t[j])) return rc;
    return ASHB_OK;
}

static int tile_count(int64_t n, unsigned* grid) {
    ASHB_REQUIRE(n >= 0 && n / kReaders < 0x7FFFFFFF, "%lld rows", (long long)n);
    *grid = (unsigned)((n + 255) / 256);
    return ASHB_OK;
}

extern "C" {

int ashb_map_insert_rows(ashb_map* m, const int32_t* keys, int64_t n, int n_tables, const ashb_row_table* tables, int32_t* row_of,
                         void* stream) {
    ASHB_REQUIRE(m != nullptr && m->slots != nullptr, "null or destroyed map");
    unsigned grid;
    if (int rc = tile_count(n, &grid)) return rc;
    if (n == 0) return ASHB_OK;
    ASHB_REQUIRE(keys && row_of, "null buffer");
    RowTables v;
    if (int rc = check_tables(n_tables, tables, false, true, &v)) return rc;
    DeviceGuard guard(m->device);
    ASHB_REQUIRE(guard.ok, "cannot select device %d", m->device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int32_t cap = (int32_t)m->capacity;
    const Table16 t = table16_of(m);
    switch (m->key_dim) {
        case 1: insert_rows_kernel<Table16, 1><<<grid, 256, 0, st>>>(t, keys, n, m->heap, m->counter, cap, row_of, v); break;
        case 2: insert_rows_kernel<Table16, 2><<<grid, 256, 0, st>>>(t, keys, n, m->heap, m->counter, cap, row_of, v); break;
        case 3: insert_rows_kernel<Table16, 3><<<grid, 256, 0, st>>>(t, keys, n, m->heap, m->counter, cap, row_of, v); break;
        default: {
            const Table32 t4{static_cast<Slot32*>(m->slots), (uint32_t)(m->n_slots - 1), m->status};
            insert_rows_kernel<Table32, 4><<<grid, 256, 0, st>>>(t4, keys, n, m->heap, m->counter, cap, row_of, v);
        }
    }
    for (int j = 0; j < v.n; ++j)
        if (v.t[j].format != 0) quantize_table(n, row_of, v.t[j], st);
    ASHB_LAUNCH_CHECK();
    return ASHB_OK;
}

int ashb_map_find_rows(ashb_map* m, const int32_t* keys, int64_t n, int64_t* indices, uint8_t* masks, int n_tables,
                       const ashb_row_table* tables, void* stream) {
    ASHB_REQUIRE(m != nullptr && m->slots != nullptr, "null or destroyed map");
    unsigned grid;
    if (int rc = tile_count(n, &grid)) return rc;
    if (n == 0) return ASHB_OK;
    ASHB_REQUIRE(keys && masks, "null buffer");
    RowTables v;
    if (int rc = check_tables(n_tables, tables, true, false, &v)) return rc;
    DeviceGuard guard(m->device);
    ASHB_REQUIRE(guard.ok, "cannot select device %d", m->device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const Table16 t = table16_of(m);
    // as find: tables beyond L2 ask the occupancy bits first
    const bool filter = m->occupied != nullptr && m->n_slots * m->slot_bytes >= (size_t)64 << 20;
    const unsigned readers = (unsigned)((n + kReaders - 1) / kReaders);
#define ASHB_FIND_ROWS(DIM)                                                                                              \
    if (filter) find_rows_kernel<Table16, DIM, true><<<readers, kReaders, 0, st>>>(t, keys, n, indices, masks, v);                \
    else find_rows_kernel<Table16, DIM, false><<<readers, kReaders, 0, st>>>(t, keys, n, indices, masks, v)
    switch (m->key_dim) {
        case 1: ASHB_FIND_ROWS(1); break;
        case 2: ASHB_FIND_ROWS(2); break;
        case 3: ASHB_FIND_ROWS(3); break;
        default: {
            const Table32 t4{static_cast<Slot32*>(m->slots), (uint32_t)(m->n_slots - 1), m->status};
            find_rows_kernel<Table32, 4, false><<<readers, kReaders, 0, st>>>(t4, keys, n, indices, masks, v);
        }
    }
#undef ASHB_FIND_ROWS
    ASHB_LAUNCH_CHECK();
    return ASHB_OK;
}

int ashb_quantize_rows(int64_t n, const ashb_row_table* table, void* stream) {
    if (n == 0) return ASHB_OK;
    ASHB_REQUIRE(n > 0 && table != nullptr, "null row table");
    ASHB_REQUIRE(n <= 0x7FFFFFFF, "%lld rows", (long long)n);
    RowTable t;
    if (int rc = check_table(table, false, false, &t)) return rc;
    quantize_table(n, nullptr, t, static_cast<cudaStream_t>(stream));
    ASHB_LAUNCH_CHECK();
    return ASHB_OK;
}

int ashb_read_rows(int64_t n, const int64_t* numbers, int64_t n_rows, const ashb_row_table* table, void* stream) {
    unsigned grid;
    if (int rc = tile_count(n, &grid)) return rc;
    if (n == 0) return ASHB_OK;
    ASHB_REQUIRE(table != nullptr && n_rows >= 0 && n_rows <= 0x7FFFFFFF, "bad row table");
    ASHB_REQUIRE(numbers != nullptr || n <= n_rows, "more rows than the table has");
    RowTables t;
    if (int rc = check_tables(1, table, true, false, &t)) return rc;
    read_rows_kernel<<<(unsigned)((n + kReaders - 1) / kReaders), kReaders, 0, static_cast<cudaStream_t>(stream)>>>(n, numbers, n_rows, t);
    ASHB_LAUNCH_CHECK();
    return ASHB_OK;
}

}  // extern "C"
