// What the attention kernels share: element types, matrix fragments, the staging of a tile of rows through LDS,
// and the work items that faith_attention_plan lays down on the host.
//
// Every product here has the query rows (forward, gradient of the queries) or the keys (gradients of keys and
// values) along the 32 columns of v_mfma_f32_32x32x{16,2}: lane l holds column l % 32, and of a result's 32 rows
// those with ((row >> 2) & 1) == l / 32, row = (r & 3) + 8 (r >> 2) + 4 (l / 32) for its register r = 0 ... 15.
// A result is thereby the second operand of the next product as it stands: the reduction over rows may run in any
// order as long as the first operand is read in the same one, so probabilities never pass through LDS.
#pragma once
#include "common.h"

#include <type_traits>

namespace faith {
namespace attn {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx4 __attribute__((ext_vector_type(4)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef short shortx8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) shortx4 lds_shortx4;

template <class T> struct Vec;
template <> struct Vec<__bf16> { typedef bf16x8 x8; typedef bf16x4 x4; };
template <> struct Vec<_Float16> { typedef halfx8 x8; typedef halfx4 x4; };

__device__ __forceinline__ floatx16 mfma(bf16x8 a, bf16x8 b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ floatx16 mfma(halfx8 a, halfx8 b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ floatx16 mfma(float a, float b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }

// the row that register r of a lane in half `half` of the wavefront holds of a 32 x 32 result
__device__ __forceinline__ constexpr int row_of(int r, int half) { return (r & 3) + 8 * (r >> 2) + 4 * half; }

// How a workgroup's wavefronts share its work: each has 32 rows of its own, or all have the same 32 and take turns at the tiles
// of the rest (KEYS; ONCE where none has a second turn: one stage, half the LDS, twice the workgroups on a compute unit)
constexpr int KIND_ROWS = 0, KIND_KEYS = 1, KIND_ONCE = 2;

// One unit of work of one key head; eight ints, read as one scalar load.
struct Item {
    int q_start, q_len;          // the sequence's queries: first packed token and how many
    int k_start, k_len;          // its keys
    int row0;                    // first row (token * group + head of the group) or first key of the tile
    int begin, end;              // keys (or tokens) that the tile goes over; end <= begin: none
    int slot;                    // where its partial result goes; -1: it is the whole result
};
static_assert(sizeof(Item) == 32, "the host writes eight ints");

// Workgroup -> (key head, item).  Workgroups are dealt to the eight XCDs round robin; a key head's items all run on one
// XCD (or, with fewer than eight key heads, on 8 / gcd of them), whose L2 then holds that head's keys and values.
struct Deal {
    int heads_apart, stripes, items_per_stripe, n_items;
};
inline Deal deal(int n_items, int kv_heads, unsigned *grid) {
    int e = 1;
    while (e < 8 && kv_heads % (2 * e) == 0) e *= 2;
    Deal d;
    d.heads_apart = e;
    d.stripes = 8 / e;
    d.items_per_stripe = (n_items + d.stripes - 1) / d.stripes;
    d.n_items = n_items;
    *grid = 8u * (unsigned)(kv_heads / e) * (unsigned)d.items_per_stripe;
    return d;
}
__device__ __forceinline__ bool dealt(const Deal &d, int *head, int *item) {
    const int x = (int)(blockIdx.x & 7), l = (int)(blockIdx.x >> 3);
    *head = x % d.heads_apart + d.heads_apart * (l / d.items_per_stripe);
    *item = x / d.heads_apart + d.stripes * (l % d.items_per_stripe);
    return *item < d.n_items;
}

// ------------------------------------------------------------------------------------------ a tile of rows in LDS
// ROWS x DP elements, rows of RB bytes in chunks of 16 bytes; chunk c of row r stands at chunk c ^ swizzle(r).  Two reads
// have to be free of bank conflicts (64 banks of 4 bytes): the same chunk of 16 consecutive rows (ROWS: 16 bytes a lane, 16
// lanes a clock), and 64 bytes of each of four (COLUMNS: the transposing read, 8 bytes a lane, 32 lanes a clock).  A tile that is
// read by columns only has the simpler swizzle, which repeats sooner: fewer addresses to hold.
enum Reads { COLUMNS, ROWS_TOO };
template <class T, int DP, Reads READS = ROWS_TOO> struct Tile {
    static constexpr int RB = DP * (int)sizeof(T), CHUNKS = RB / 16, PER = 16 / (int)sizeof(T);
    // rows until the swizzle repeats; rows of 12 chunks start at another quarter of the banks each by themselves
    static constexpr int PERIOD = READS == ROWS_TOO ? 16 : sizeof(T) == 4 || CHUNKS == 4 || CHUNKS == 12 ? 1 : 4;
    __device__ static __forceinline__ int swizzle(int r) {
        if constexpr (READS == COLUMNS) {
            if constexpr (PERIOD == 1) return 0;
            else if constexpr (CHUNKS == 8) return ((r >> 1) & 1) << 2;
            else return (r & 3) << 2;
        }
        else if constexpr (CHUNKS == 4 || CHUNKS == 12) return (r >> 2) & 3;
        else if constexpr (CHUNKS == 24) return (r >> 1) & 7;
        else if constexpr (CHUNKS == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
        else return ((r & 3) << 2) | ((r >> 2) & 3);
    }
    // element offset of chunk c of row r
    __device__ static __forceinline__ int at(int r, int c) { return r * DP + (c ^ swizzle(r)) * PER; }
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t window(const void *base, unsigned bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, (int)bytes, 0x00020000);
}

// 16 bytes a lane into LDS: lane i's land at dst + 16 i
__device__ __forceinline__ void groups_to_lds(__amdgpu_buffer_rsrc_t w, char *dst, unsigned lane_off, unsigned uniform_off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(w, (lds_void *)dst, 16, lane_off, uniform_off, 0, 0);
}

// The loads of one tile of ROWS rows by WAVES wavefronts: 1 KB an instruction, straight into LDS (lane i's 16 bytes land at
// 16 i), so the swizzle is applied to the address that a lane reads.  Rows behind the sequence's last and chunks behind the
// head's size lie outside the window and arrive as zeros.
template <class T, int DP, int ROWS, int WAVES, Reads READS = ROWS_TOO> struct Stager {
    typedef Tile<T, DP, READS> Tl;
    static constexpr int TOTAL = ROWS * Tl::RB / 1024, LOADS = (TOTAL + WAVES - 1) / WAVES;
    // Where whole rows make up a load and the swizzle has repeated, a later load's offsets are an earlier one's further on.
    static constexpr int ROWS_PER = 1024 / Tl::RB, PERIOD = ROWS_PER < Tl::PERIOD ? Tl::PERIOD / ROWS_PER : 1;
    static constexpr int PATTERNS = 1024 % Tl::RB == 0 && PERIOD < LOADS ? PERIOD : LOADS;
    static_assert(TOTAL * 1024 == ROWS * Tl::RB && LOADS % PATTERNS == 0, "whole loads");
    unsigned off[PATTERNS];
    unsigned stride;             // bytes from one row to the next

    __device__ __forceinline__ void init(int lane, int wave, int size, long long row_stride) {
        stride = (unsigned)(row_stride * (long long)sizeof(T));
#pragma unroll
        for (int i = 0; i < PATTERNS; ++i) {
            const int x = (wave * LOADS + i) * 64 + lane, r = x / Tl::CHUNKS, c = (x % Tl::CHUNKS) ^ Tl::swizzle(r);
            off[i] = c * Tl::PER < size ? (unsigned)r * stride + (unsigned)c * 16u : 0x7ffffff0u;
        }
    }
    // base: the tile's first row; rows_left: rows from there to the sequence's end (may be <= 0)
    __device__ __forceinline__ void load(T *lds, const T *base, int rows_left, int size, int wave) const {
        // a window up to the last element of the last row; never so long that the offsets outside could fall into it
        const long long n = rows_left > 0 ? (long long)((rows_left < ROWS ? rows_left : ROWS) - 1) * stride + (long long)size * (int)sizeof(T) : 0;
        const __amdgpu_buffer_rsrc_t w = window(base, (unsigned)n);
        char *dst = reinterpret_cast<char *>(lds) + wave * LOADS * 1024;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            if (TOTAL % WAVES && wave * LOADS + i >= TOTAL) break;
            groups_to_lds(w, dst + i * 1024, off[i % PATTERNS], (unsigned)((i / PATTERNS) * PATTERNS * ROWS_PER) * stride);
        }
    }
};

// n <= 64 floats into LDS, one a lane; zeros behind them
__device__ __forceinline__ void words_to_lds(float *lds, const float *src, int n, int lane) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(window(src, (unsigned)n * 4u), (lds_void *)lds, 4, (unsigned)lane * 4u, 0, 0, 0);
}

// Addresses.  Where a row's bytes are a power of two, the place of a row's chunk is that of its first one with the chunk's number
// exclusive-ored in: one instruction from one register, however many chunks, blocks and tiles are read (their starts are
// constants of the instructions).  row0: a multiple of 32.

// first operand, rows row0 ... row0 + 31 of a tile (this lane: row0 + col), 16 bytes of the reduction at its chunk 2 u + half
template <class T, int DP> __device__ __forceinline__ const char *row_chunk(const T *tile, int row0, int col, int u, int half) {
    typedef Tile<T, DP> Tl;
    const int first = (half ^ Tl::swizzle(col)) * 16;
    int off;
    if constexpr ((Tl::RB & (Tl::RB - 1)) == 0) off = (col * Tl::RB + first) ^ (32 * u);
    else off = col * Tl::RB + (first ^ (32 * u));
    return reinterpret_cast<const char *>(tile) + row0 * Tl::RB + off;
}
template <class T, int DP> __device__ __forceinline__ typename Vec<T>::x8 row_fragment(const T *tile, int row0, int col, int u, int half) {
    return *reinterpret_cast<const typename Vec<T>::x8 *>(row_chunk<T, DP>(tile, row0, col, u, half));
}
template <int DP> __device__ __forceinline__ floatx4 row_fragment4(const float *tile, int row0, int col, int u, int half) {
    return *reinterpret_cast<const floatx4 *>(row_chunk<float, DP>(tile, row0, col, u, half));
}
// first operand transposed: columns 32 m ... 32 m + 31 of the tile against the 16 rows row0 + 16 u + {0 ... 15} in the order in
// which registers 0 ... 7 hold them: lane half h has rows 4h ... 4h + 3, then 8 + 4h ... 8 + 4h + 3
template <class T, int DP, Reads READS> __device__ __forceinline__ typename Vec<T>::x8 column_fragment(const T *tile, int row0, int u, int m, int lane) {
    typedef Tile<T, DP, READS> Tl;
    const int i = lane & 15, r = 4 * (lane >> 5) + (i >> 2), c = 16 * ((lane >> 4) & 1) + 4 * (i & 3);       // within the block
    shortx4 part[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int first = ((c >> 3) ^ Tl::swizzle(r)) * 16 + (c & 7) * 2, flip = (64 * m) ^ ((Tl::swizzle(8) ^ Tl::swizzle(0)) * 16 * h);
        int off;
        if constexpr ((Tl::RB & (Tl::RB - 1)) == 0) off = (r * Tl::RB + first) ^ flip;
        else off = r * Tl::RB + (READS == COLUMNS ? first + flip : (first ^ ((Tl::swizzle(8) ^ Tl::swizzle(0)) * 16 * h)) + 64 * m);
        part[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4 *)(reinterpret_cast<const char *>(tile) + (row0 + 16 * u + 8 * h) * Tl::RB + off));
    }
    const shortx8 v = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(typename Vec<T>::x8, v);
}
// one element, fp32: column 32 m + col of row row0 + row_of(r, half)
template <int DP, Reads READS> __device__ __forceinline__ float column_element(const float *tile, int row0, int r, int half, int m, int col) {
    typedef Tile<float, DP, READS> Tl;
    if constexpr ((Tl::RB & (Tl::RB - 1)) == 0) {
        // row_of(r, half) = row_of(r, 0) + 4 half, and the swizzles of the two parts have no bit in common
        const int first = ((col >> 2) ^ Tl::swizzle(4 * half)) * 16 + (col & 3) * 4;
        const int off = (half * 4 * Tl::RB + first) ^ (128 * m ^ Tl::swizzle(row_of(r, 0)) * 16);
        return *reinterpret_cast<const float *>(reinterpret_cast<const char *>(tile) + (row0 + row_of(r, 0)) * Tl::RB + off);
    } else {
        const int row = row_of(r, half), c = 32 * m + col;
        return tile[row0 * DP + Tl::at(row, c >> 2) + (c & 3)];
    }
}

// acc[r] + sum_d tile[row_of(r)][d] * b[d]: the 32 rows from row0 on against this lane's column, whose values are in `b`
template <class T, int DP> struct ColumnRegs { typename Vec<T>::x8 v[DP / 16]; };
template <int DP> struct ColumnRegs<float, DP> { floatx4 v[DP / 8]; };

template <class T, int DP> __device__ __forceinline__ floatx16 rows_by_column(const T *tile, int row0, int col, int half, const ColumnRegs<T, DP> &b, floatx16 acc) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int u = 0; u < DP / 8; ++u) {
            const floatx4 a = row_fragment4<DP>(tile, row0, col, u, half);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc = mfma(a[e], b.v[u][e], acc);
        }
    } else {
#pragma unroll
        for (int u = 0; u < DP / 16; ++u) acc = mfma(row_fragment<T, DP>(tile, row0, col, u, half), b.v[u], acc);
    }
    return acc;
}

template <class T, int DP> __device__ __forceinline__ floatx16 rows_by_column(const T *tile, int row0, int col, int half, const ColumnRegs<T, DP> &b) {
    floatx16 none;
#pragma unroll
    for (int r = 0; r < 16; ++r) none[r] = 0.f;
    return rows_by_column<T, DP>(tile, row0, col, half, b, none);
}

// the values of one row (DP of them, zero behind `size`) in the order in which rows_by_column takes them; all loads first, with
// no branch between them
template <class T, int DP> __device__ __forceinline__ ColumnRegs<T, DP> column_regs(const T *row, int half, int size) {
    ColumnRegs<T, DP> b;
    constexpr int PER = 16 / (int)sizeof(T), N = DP / (2 * PER);
    uintx4 z[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int d = (2 * u + half) * PER;
        z[u] = *reinterpret_cast<const uintx4 *>(row + (d < size ? d : 0));
    }
    if (size < DP) {
#pragma unroll
        for (int u = 0; u < N; ++u)
            if ((2 * u + half) * PER >= size) z[u] = uintx4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
        if constexpr (sizeof(T) == 4) b.v[u] = __builtin_bit_cast(floatx4, z[u]);
        else b.v[u] = __builtin_bit_cast(typename Vec<T>::x8, z[u]);
    }
    return b;
}

// this lane's column of a result, `factor` times, to a row of T
template <class T, int DP> __device__ __forceinline__ void store_column(T *dst, const floatx16 (&o)[DP / 32], float factor, int half, int size) {
    auto all = [&](auto checked) {
#pragma unroll
        for (int m = 0; m < DP / 32; ++m)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int d = 32 * m + row_of(r, half);
                if (decltype(checked)::value && d >= size) continue;
                if constexpr (sizeof(T) == 4) {
                    const floatx4 x = {o[m][r] * factor, o[m][r + 1] * factor, o[m][r + 2] * factor, o[m][r + 3] * factor};
                    *reinterpret_cast<floatx4 *>(dst + d) = x;
                } else {
                    const typename Vec<T>::x4 x = {(T)(o[m][r] * factor), (T)(o[m][r + 1] * factor), (T)(o[m][r + 2] * factor), (T)(o[m][r + 3] * factor)};
                    *reinterpret_cast<typename Vec<T>::x4 *>(dst + d) = x;
                }
            }
    };
    if (size == DP) all(std::false_type{});
    else all(std::true_type{});
}

// acc[m][r] += sum over the tile's 32 rows from row0 on of tile[row][32 m + row_of(r)] * p[row]: p is a result register set of
// this lane's column.  Products of 2-byte elements round p to that type (half a step of it, against sums in 32 bits).
template <class T, int DP, Reads READS = ROWS_TOO> __device__ __forceinline__ void columns_by_result(floatx16 (&acc)[DP / 32], const T *tile, int row0, int lane, const floatx16 &p) {
    if constexpr (sizeof(T) == 4) {
        const int half = lane >> 5, col = lane & 31;
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int m = 0; m < DP / 32; ++m) acc[m] = mfma(column_element<DP, READS>(tile, row0, r, half, m, col), p[r], acc[m]);
    } else {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            typename Vec<T>::x8 b;
#pragma unroll
            for (int e = 0; e < 8; ++e) b[e] = (T)p[8 * u + e];
#pragma unroll
            for (int m = 0; m < DP / 32; ++m) acc[m] = mfma(column_fragment<T, DP, READS>(tile, row0, u, m, lane), b, acc[m]);
        }
    }
}

// Operands in fp16.  Its five exponent bits end at 2^-14 (2^-24 with ever fewer bits) and 65504, and a probability among
// thousands of keys, or a small gradient times one, lies below.  So what is rounded to fp16 is first multiplied by a power of two, which
// the 32-bit sums it goes into are divided by at the end: both are exact.  bf16 has the exponents of 32 bits and needs none.
// Probabilities, at most 1: a constant.
template <class T> constexpr int probability_up() { return std::is_same<T, _Float16>::value ? 14 : 0; }

// over the two lanes that share a column
__device__ __forceinline__ float max_halves(float v) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const unsigned a = s[0], b = s[1];
    return __builtin_fmaxf(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ float sum_halves(float v) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const unsigned a = s[0], b = s[1];
    return __uint_as_float(a) + __uint_as_float(b);
}

// Other values (fp16): a power of two for each column, 2^up, with which s comes here, and under which the largest of the column so far
// lies at most at 2^15.  It starts higher than any value asks for (ds is at most 2^40: products of two fp16 values over 128 places) and
// only falls, to where that value lies in [2^7, 2^8); the sums follow it.  13 sequences of 37 ... 1021, 12 heads of 80, forward and
// gradients: 185 us with it, 183 without; 2048 keys and gradients of 2^-13: dq off by 0.38 %, all of it its own rounding, instead of 2.2.
constexpr int UP_MOST = 80;
template <int DP, int N> __device__ __forceinline__ void follow(floatx16 (&s)[N], floatx16 (&acc)[DP / 32], int &up) {
    float top = 0.f;
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = __builtin_fmaxf(top, __builtin_fabsf(s[b][r]));
    if (__any(top > 32768.f)) {
        top = max_halves(top);
        const int down = top > 32768.f ? 8 - __builtin_amdgcn_frexp_expf(top) : 0;
        const float f = __builtin_ldexpf(1.f, down);
        up += down;
#pragma unroll
        for (int b = 0; b < N; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[b][r] *= f;
#pragma unroll
        for (int m = 0; m < DP / 32; ++m)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[m][r] *= f;
    }
}
// acc times 2^-up
template <int DP> __device__ __forceinline__ void lower(floatx16 (&acc)[DP / 32], int up) {
#pragma unroll
    for (int m = 0; m < DP / 32; ++m)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[m][r] = __builtin_ldexpf(acc[m][r], -up);
}

// ------------------------------------------------------------------------------------------ what a mask hides
// A mask may hide anything, and the products above multiply what it hides by zero, which NaN and infinity survive.  A wavefront whose
// causal result is not finite therefore looks at what was hidden from its rows, the ends of one or two tiles, and only if that holds
// what is no number, does its rows again: every lane its own row over what the row sees, in 32 bits and on the vector units.  A NaN that is seen
// is in the first result, and costs nothing beyond the look; so does an input that is NaN throughout, whose rows know it from their sums.
// The slow way is some 140 times the first pass: 4096 causal tokens, 32 / 8 heads of 128, bf16, every value NaN and no key: 22 ms instead of 0.16.
template <class T> __device__ __forceinline__ bool rows_not_finite(const T *base, long long stride, int from, int to, int size, int lane) {
    bool bad = false;
    for (int i = from; i < to; ++i)
        for (int d = lane; d < size; d += 64) bad |= !(__builtin_fabsf((float)base[i * stride + d]) < __builtin_inff());
    return __any(bad);
}
// rows start on 16 bytes and are whole groups of them
template <class T> __device__ __forceinline__ float dot_rows(const T *a, const T *b, int size) {
    constexpr int PER = 16 / (int)sizeof(T);
    typedef T group __attribute__((ext_vector_type(PER)));
    float s = 0.f;
#pragma unroll 2
    for (int d = 0; d < size; d += PER) {
        const group x = *reinterpret_cast<const group *>(a + d), y = *reinterpret_cast<const group *>(b + d);
#pragma unroll
        for (int e = 0; e < PER; ++e) s = fmaf((float)x[e], (float)y[e], s);
    }
    return s;
}
// o += f * row, for this lane's registers (those behind the head's size are not stored)
template <class T, int DP> __device__ __forceinline__ void add_row(floatx16 (&o)[DP / 32], const T *row, float f, int half, int size) {
    typedef T four __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int m = 0; m < DP / 32; ++m) {
        __builtin_amdgcn_sched_barrier(0);           // a block's loads at a time: no registers for speed here
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int d = 32 * m + row_of(r, half);
            const four v = *reinterpret_cast<const four *>(row + (d < size ? d : 0));
#pragma unroll
            for (int i = 0; i < 4; ++i) o[m][r + i] = fmaf(f, (float)v[i], o[m][r + i]);
        }
    }
}

// Wavefronts on a SIMD that a kernel is compiled for: as many as LDS and the registers of its tiles' loop allow.  (Left to itself the compiler takes
// more registers for what comes behind the loop.)
enum Pass { FORWARD, GRAD_QUERIES, GRAD_KEYS };
constexpr int resident(Pass pass, int kind, int element_size, int padded) {
    constexpr int N[3][2][4][3] = {        // pass; elements of 2, 4 bytes; heads of 32, 64, 96, 128; ROWS, KEYS, ONCE
        {{{4, 4, 4}, {3, 2, 4}, {2, 1, 3}, {2, 1, 2}}, {{4, 2, 4}, {4, 1, 2}, {3, 1, 2}, {2, 1, 1}}},
        {{{4, 3, 5}, {4, 2, 5}, {3, 1, 3}, {2, 1, 2}}, {{4, 2, 4}, {3, 1, 2}, {1, 1, 2}, {1, 1, 1}}},
        {{{2, 3, 5}, {2, 2, 4}, {2, 1, 3}, {2, 1, 2}}, {{3, 2, 4}, {2, 1, 2}, {1, 1, 2}, {1, 1, 1}}}};
    return N[pass][element_size / 4][padded / 32 - 1][kind];
}

// Wavefronts of a workgroup that share their columns and divide the reduction, each with tiles of its own: four, unless their
// four pairs of stages would not fit LDS (fp32, heads of more than 64).
constexpr int split_waves(int element_size, int padded) { return 32 * padded * element_size * 16 <= 128 * 1024 ? 4 : 2; }
template <class T, int DP> constexpr int split_waves() { return split_waves((int)sizeof(T), DP); }

// The reduction of such a wavefront: its tiles first, first + step, ... < end, no barrier; `stage(n, i)` issues LOADS loads for
// tile i into stage n (the caller has done so for the first), `use(n, i)` works on it while the younger stage's loads stay in
// flight.
template <int LOADS, bool ONCE, class Stage, class Use> __device__ __forceinline__ void alone(int first, int step, int end, Stage stage, Use use) {
    if constexpr (ONCE) {
        if (first >= end) return;
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        use(0, first);
        return;
    }
    for (int i = first; i < end; i += 2 * step) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (i + step < end) {
            stage(1, i + step);
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        }
        use(0, i);
        if (i + step >= end) break;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (i + 2 * step < end) {
            stage(0, i + 2 * step);
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        }
        use(1, i + step);
    }
}

// Adds the wavefronts' results up in the first one, in order; lo and hi: room for them (HALF floats each).
template <int WAVES, int DP, int HALF> __device__ __forceinline__ void add_waves(floatx16 (&o)[DP / 32], float *lo, float *hi, int wave, int lane) {
    constexpr int WIDTH = DP / 32 * 16;
    static_assert((WAVES - 1) * 64 * WIDTH <= 2 * HALF, "the results fit");
    __syncthreads();
    if (wave > 0)
#pragma unroll
        for (int e = 0; e < WIDTH; ++e) {
            const int x = ((wave - 1) * WIDTH + e) * 64 + lane;
            (x < HALF ? lo[x] : hi[x - HALF]) = o[e / 16][e % 16];
        }
    __syncthreads();
    if (wave == 0)
#pragma unroll
        for (int w = 0; w < WAVES - 1; ++w)
#pragma unroll
            for (int e = 0; e < WIDTH; ++e) {
                const int x = (w * WIDTH + e) * 64 + lane;
                o[e / 16][e % 16] += x < HALF ? lo[x] : hi[x - HALF];
            }
}

// This wavefront's loads into LDS have landed and its reads are done; then the barrier.  (The compiler does not see
// other wavefronts' loads.)
__device__ __forceinline__ void landed_and_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Host checks that the three entry points share.
inline int attention_shapes(const char *fn, int heads, int kv_heads, int size, int dtype, float scale) {
    FAITH_REQUIRE(kv_heads > 0 && heads > 0 && heads % kv_heads == 0, FAITH_ERR_SHAPE, "%s: %d heads do not share %d key heads evenly", fn, heads, kv_heads);
    FAITH_REQUIRE(dtype == FAITH_F32 || dtype == FAITH_BF16 || dtype == FAITH_F16, FAITH_ERR_UNSUPPORTED, "%s: element type %d", fn, dtype);
    FAITH_REQUIRE(size > 0 && size <= 128 && size % (dtype == FAITH_F32 ? 4 : 8) == 0, FAITH_ERR_UNSUPPORTED,
                  "%s: heads of %d elements (up to 128, whole groups of 16 bytes)", fn, size);
    FAITH_REQUIRE(scale > 0.f && scale < 1e30f, FAITH_ERR_UNSUPPORTED, "%s: the scale must be positive and finite", fn);
    return FAITH_OK;
}
// a launch holds fewer than 2^32 threads
inline bool attention_grid(const char *fn, int n_items, int kv_heads) {
    unsigned grid;
    const Deal d = deal(n_items, kv_heads, &grid);
    if (8LL * (kv_heads / d.heads_apart) * d.items_per_stripe < (1LL << 24)) return true;
    set_error("%s: %d items of %d key heads are more than one launch holds", fn, n_items, kv_heads);
    return false;
}
// rows in whole 16-byte groups that neither overlap nor lie further apart than a 32-bit offset reaches over one tile
inline bool attention_rows(const char *fn, const char *name, const void *p, long long token_stride, long long head_stride, int size, int es) {
    const int per = 16 / es;
    if (p && aligned(p, 16) && token_stride % per == 0 && head_stride % per == 0 && token_stride >= size && head_stride >= 0 &&
        token_stride * es < (1LL << 24))
        return true;
    if (!p) set_error("%s: argument '%s' is NULL", fn, name);
    else set_error("%s: %s must start on 16 bytes and have strides of whole 16-byte groups, the tokens' at least %d and under 2^24 bytes", fn, name, size);
    return false;
}
// Rows and heads that are read may lie on each other; written, they would race.  Token by token, or head by head: how many tokens, and with
// that how far apart heads have to be, the items say on the device; two at least are taken for granted.
inline bool attention_heads_apart(const char *fn, const char *name, long long token_stride, long long head_stride, int heads, int size) {
    if (heads == 1 || (head_stride >= size && (token_stride >= (heads - 1) * head_stride + size || head_stride >= token_stride + size))) return true;
    set_error("%s: the rows and heads of %s, which is written, must not overlap", fn, name);
    return false;
}

}  // namespace attn
}  // namespace faith
