// Feature rows in 8 bits: the value tables of a hash map quantised as keys are inserted and read back as keys are
// looked up, and the same for rows that lie in order or are named by their numbers.
//
// Both directions are bound by memory: a key moves its 12 bytes, a 16-byte slot of the table at a random place, and
// its row.  One launch does all of it.  The 256 threads of a CTA first place or look up a key each, then take the 256
// rows together: a row is served by as many lanes as it has quadruples of values (32 at most), so that codes and
// values move in whole sectors whatever the width, and a group of lanes has four rows in flight.  A thread copying its
// own row instead, as rows of 64 bytes are copied elsewhere, touches a sector per lane and instruction.
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
};
struct RowTables {
    int n;
    RowTable t[kMaxRowTables];
};

// Lanes that share a row: the power of two that covers its quadruples, 32 at most.
__device__ __forceinline__ int lanes_of(int64_t width) {
    int lanes = 1;
    while (lanes < 32 && (int64_t)lanes * 4 < width) lanes <<= 1;
    return lanes;
}

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

// Rows `first .. first + 255` of a batch of n, row r of them to row index_of(r) of the table (negative: left out).
// QUADS quadruples a lane and ROWS rows stay in registers; a longer row is read a second time, from L1.
template <class T, int QUADS, int ROWS, class IndexOf>
__device__ __forceinline__ void quantize_tile(const RowTable& t, int64_t first, int lanes, IndexOf index_of) {
    const int sub = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes, groups = 256 / lanes;
    const T* src = static_cast<const T*>(t.src);
    uint8_t* codes = static_cast<uint8_t*>(t.dst);
    for (int r0 = 0; r0 < lanes; r0 += ROWS) {      // 256 rows over `groups` groups: `lanes` rows each
        float v[ROWS][QUADS][4];
        int64_t to[ROWS];
        uint32_t amax[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int r = (r0 + i) * groups + group;
            to[i] = r0 + i < lanes ? index_of(r) : -1;
            amax[i] = 0;
            if (to[i] < 0) continue;
            const T* row = src + (first + r) * t.width;
#pragma unroll
            for (int q = 0; q < QUADS; ++q) {
                const int64_t col = ((int64_t)q * lanes + sub) * 4;
                if (col < t.width) {
                    load4(row, col, t.width, t.wide, v[i][q]);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[i][q][k] = 0.0f;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            if (to[i] >= 0) {
#pragma unroll
                for (int q = 0; q < QUADS; ++q)
#pragma unroll
                    for (int k = 0; k < 4; ++k) amax[i] = max(amax[i], magnitude_bits(v[i][q][k]));
                const T* row = src + (first + (r0 + i) * groups + group) * t.width;
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
            const T* row = src + (first + (r0 + i) * groups + group) * t.width;
            for (int64_t col = ((int64_t)QUADS * lanes + sub) * 4; col < t.width; col += lanes * 4) {
                float u[4];
                load4(row, col, t.width, t.wide, u);
                store_codes(out, col, t.width, t.wide, encode4(u, s.inverse, t.format));
            }
            if (sub == 0) t.scales[to[i]] = s.scale;
        }
    }
}

template <class T, class IndexOf>
__device__ __forceinline__ void quantize_typed(const RowTable& t, int64_t first, IndexOf index_of) {
    const int lanes = lanes_of(t.width);
    if (t.width <= 128) quantize_tile<T, 1, 4>(t, first, lanes, index_of);
    else quantize_tile<T, 4, 1>(t, first, lanes, index_of);
}

template <class IndexOf>
__device__ __forceinline__ void quantize_rows_of(const RowTable& t, int64_t first, IndexOf index_of) {
    if (t.dtype == ASHB_F32) quantize_typed<float>(t, first, index_of);
    else if (t.dtype == ASHB_F16) quantize_typed<__half>(t, first, index_of);
    else quantize_typed<__nv_bfloat16>(t, first, index_of);
}

// Row index_of(r) of the codes to row first + r of the values, r < have; zeros where it is negative.
template <class T, class IndexOf>
__device__ __forceinline__ void read_typed(const RowTable& t, int64_t first, int have, IndexOf index_of) {
    constexpr int ROWS = 4;
    const int lanes = lanes_of(t.width);
    const int sub = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes, groups = 256 / lanes;
    const uint8_t* codes = static_cast<const uint8_t*>(t.src);
    T* out = static_cast<T*>(t.dst);
    for (int r0 = 0; r0 < lanes; r0 += ROWS) {
        int64_t from[ROWS];
        float scale[ROWS];
        bool live[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int r = (r0 + i) * groups + group;
            live[i] = r0 + i < lanes && r < have;
            from[i] = live[i] ? index_of(r) : -1;
            scale[i] = from[i] >= 0 ? __ldg(t.scales + from[i]) : 0.0f;
        }
        for (int64_t col = (int64_t)sub * 4; col < t.width; col += lanes * 4) {
            uint32_t w[ROWS];
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                w[i] = 0;
                if (from[i] < 0) continue;
                const uint8_t* row = codes + from[i] * t.width + col;
                if (t.wide) {
                    w[i] = __ldg(reinterpret_cast<const uint32_t*>(row));
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (col + k < t.width) w[i] |= (uint32_t)__ldg(row + k) << (8 * k);
                }
            }
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                if (!live[i]) continue;
                float v[4];
                decode4(w[i], scale[i], t.format, v);
                T* row = out + (first + (r0 + i) * groups + group) * t.width + col;
                if (t.wide) {
                    store_n<T, 4>(row, v);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (col + k < t.width) row[k] = from_float<T>(v[k]);
                }
            }
        }
    }
}

template <class IndexOf>
__device__ __forceinline__ void read_rows_of(const RowTable& t, int64_t first, int have, IndexOf index_of) {
    if (t.dtype == ASHB_F32) read_typed<float>(t, first, have, index_of);
    else if (t.dtype == ASHB_F16) read_typed<__half>(t, first, have, index_of);
    else read_typed<__nv_bfloat16>(t, first, have, index_of);
}

// ---- the hash map's tables -------------------------------------------------------------------------------------
// A new key's index is published before its row is written: within a launch nobody reads rows, and the next launch
// of the stream sees both.
template <class Table, int DIM>
__global__ void __launch_bounds__(256) insert_rows_kernel(Table t, const int32_t* __restrict__ keys, int64_t n,
                                                          int32_t* __restrict__ heap, int32_t* counter, int32_t capacity,
                                                          const __grid_constant__ RowTables tables) {
    __shared__ int row_of[256];
    const int64_t first = (int64_t)blockIdx.x * 256, i = first + threadIdx.x;
    int64_t slot = -1;
    if (i < n) {
        int k0, k1, k2, k3;
        load_key<DIM>(keys, i, k0, k1, k2, k3);
        bool present = false;
        slot = emplace(t, k0, k1, k2, k3, kPending, &present);
    }
    const int idx = pop_index_for_slot_cta(t, slot, heap, counter, capacity);
    if (idx >= 0) publish_index(t, slot, idx);
    row_of[threadIdx.x] = idx;
    __syncthreads();
    for (int j = 0; j < tables.n; ++j) {
        const RowTable& v = tables.t[j];
        if (v.format != 0) {
            quantize_rows_of(v, first, [&](int r) { return (int64_t)row_of[r]; });
        } else if (idx >= 0) {
            const char* src = static_cast<const char*>(v.src) + i * v.width;
            char* dst = static_cast<char*>(v.dst) + idx * v.width;
            if (v.wide)
                for (int64_t b = 0; b < v.width; b += 4) *reinterpret_cast<int*>(dst + b) = *reinterpret_cast<const int*>(src + b);
            else
                for (int64_t b = 0; b < v.width; ++b) dst[b] = src[b];
        }
    }
}

template <class Table, int DIM, bool FILTER>
__global__ void __launch_bounds__(256) find_rows_kernel(Table t, const int32_t* __restrict__ keys, int64_t n,
                                                        int64_t* __restrict__ indices, uint8_t* __restrict__ masks,
                                                        const __grid_constant__ RowTables tables) {
    __shared__ int row_of[256];
    const int64_t first = (int64_t)blockIdx.x * 256, i = first + threadIdx.x;
    int found = -1;
    if (i < n) {
        int k0, k1, k2, k3;
        load_key<DIM>(keys, i, k0, k1, k2, k3);
        uint32_t s = hash_key(k0, k1, k2, k3) & t.mask;
        bool absent = false;
        if constexpr (FILTER) absent = t.never_used(s);
        for (uint32_t probe = 0; !absent && probe <= t.mask; ++probe) {
            const Entry e = t.read_const(s);
            if (e.val == kEmpty) break;
            if (e.val >= 0 && key_match(e, k0, k1, k2, k3)) {
                found = e.val;
                break;
            }
            s = (s + 1) & t.mask;
        }
        if (indices) indices[i] = found >= 0 ? (int64_t)found : 0;
        masks[i] = (uint8_t)(found >= 0);
    }
    row_of[threadIdx.x] = found;
    __syncthreads();
    const int have = (int)min((int64_t)256, n - first);
    for (int j = 0; j < tables.n; ++j) read_rows_of(tables.t[j], first, have, [&](int r) { return (int64_t)row_of[r]; });
}

// ---- rows in order, or by number -------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) quantize_rows_kernel(int64_t n, const __grid_constant__ RowTable t) {
    const int64_t first = (int64_t)blockIdx.x * 256;
    quantize_rows_of(t, first, [&](int r) { return first + r < n ? first + r : (int64_t)-1; });
}

// A number outside 0 .. n_rows - 1 reads zeros.
__global__ void __launch_bounds__(256) read_rows_kernel(int64_t n, const int64_t* __restrict__ numbers, int64_t n_rows,
                                                        const __grid_constant__ RowTable t) {
    const int64_t first = (int64_t)blockIdx.x * 256;
    const int have = (int)min((int64_t)256, n - first);
    read_rows_of(t, first, have, [&](int r) {
        const int64_t i = numbers ? numbers[first + r] : first + r;
        return i < n_rows ? i : (int64_t)-1;
    });
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
    ASHB_REQUIRE(n >= 0 && (n + 255) / 256 <= 0x7FFFFFFF, "%lld rows", (long long)n);
    *grid = (unsigned)((n + 255) / 256);
    return ASHB_OK;
}

extern "C" {

int ashb_map_insert_rows(ashb_map* m, const int32_t* keys, int64_t n, int n_tables, const ashb_row_table* tables, void* stream) {
    ASHB_REQUIRE(m != nullptr && m->slots != nullptr, "null or destroyed map");
    unsigned grid;
    if (int rc = tile_count(n, &grid)) return rc;
    if (n == 0) return ASHB_OK;
    ASHB_REQUIRE(keys != nullptr, "null keys");
    RowTables v;
    if (int rc = check_tables(n_tables, tables, false, true, &v)) return rc;
    DeviceGuard guard(m->device);
    ASHB_REQUIRE(guard.ok, "cannot select device %d", m->device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int32_t cap = (int32_t)m->capacity;
    const Table16 t = table16_of(m);
    switch (m->key_dim) {
        case 1: insert_rows_kernel<Table16, 1><<<grid, 256, 0, st>>>(t, keys, n, m->heap, m->counter, cap, v); break;
        case 2: insert_rows_kernel<Table16, 2><<<grid, 256, 0, st>>>(t, keys, n, m->heap, m->counter, cap, v); break;
        case 3: insert_rows_kernel<Table16, 3><<<grid, 256, 0, st>>>(t, keys, n, m->heap, m->counter, cap, v); break;
        default: {
            const Table32 t4{static_cast<Slot32*>(m->slots), (uint32_t)(m->n_slots - 1), m->status};
            insert_rows_kernel<Table32, 4><<<grid, 256, 0, st>>>(t4, keys, n, m->heap, m->counter, cap, v);
        }
    }
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
#define ASHB_FIND_ROWS(DIM)                                                                                              \
    if (filter) find_rows_kernel<Table16, DIM, true><<<grid, 256, 0, st>>>(t, keys, n, indices, masks, v);                \
    else find_rows_kernel<Table16, DIM, false><<<grid, 256, 0, st>>>(t, keys, n, indices, masks, v)
    switch (m->key_dim) {
        case 1: ASHB_FIND_ROWS(1); break;
        case 2: ASHB_FIND_ROWS(2); break;
        case 3: ASHB_FIND_ROWS(3); break;
        default: {
            const Table32 t4{static_cast<Slot32*>(m->slots), (uint32_t)(m->n_slots - 1), m->status};
            find_rows_kernel<Table32, 4, false><<<grid, 256, 0, st>>>(t4, keys, n, indices, masks, v);
        }
    }
#undef ASHB_FIND_ROWS
    ASHB_LAUNCH_CHECK();
    return ASHB_OK;
}

int ashb_quantize_rows(int64_t n, const ashb_row_table* table, void* stream) {
    unsigned grid;
    if (int rc = tile_count(n, &grid)) return rc;
    if (n == 0) return ASHB_OK;
    ASHB_REQUIRE(table != nullptr, "null row table");
    RowTable t;
    if (int rc = check_table(table, false, false, &t)) return rc;
    quantize_rows_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(n, t);
    ASHB_LAUNCH_CHECK();
    return ASHB_OK;
}

int ashb_read_rows(int64_t n, const int64_t* numbers, int64_t n_rows, const ashb_row_table* table, void* stream) {
    unsigned grid;
    if (int rc = tile_count(n, &grid)) return rc;
    if (n == 0) return ASHB_OK;
    ASHB_REQUIRE(table != nullptr && n_rows >= 0, "bad row table");
    ASHB_REQUIRE(numbers != nullptr || n <= n_rows, "more rows than the table has");
    RowTable t;
    if (int rc = check_table(table, true, false, &t)) return rc;
    read_rows_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(n, numbers, n_rows, t);
    ASHB_LAUNCH_CHECK();
    return ASHB_OK;
}

}  // extern "C"
