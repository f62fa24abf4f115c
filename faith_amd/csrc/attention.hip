// Attention of a network's concrete pass: out = softmax(scale q k^T) v over packed sequences of different lengths, with
// groups of query heads that share a key head, causal or not; one query against a long cache is the same call.
//
// One pass over the keys with the running maximum and sum of the softmax.  A row is one (token, head of the group) pair,
// row = token * group + head: all rows of a tile share the keys and values that it stages, so a group reads them once.
// Two shapes of workgroup, four wavefronts each (keys: two in fp32 with heads of more than 64), 32 rows to a wavefront:
//   rows    128 rows; every wavefront goes over every key tile (64 keys, 32 in fp32), staged once for the four
//   keys    at most 32 rows (a single token's group, a short sentence); the wavefronts take turns at the key tiles of 32
//           keys, each staged by its wavefront alone with no barrier, and join their results through LDS at the end
// Few rows against many keys leave most of the device idle: the keys are then cut into several items, whose partial
// results (maximum, sum, unnormalised output, all in fp32) a second small launch joins in a fixed order.
// Measured, 32 / 8 heads of 128 in bf16: 16384 causal tokens 1.94 ms, 1132 TFLOP/s, bound by power (1.47 ms at an earlier step with
// zeros for data, 2.07 without); one query each against 64 caches of 100 to 8192, 1.08 GB, 192 us, 5.6 TB/s, bound by HBM.
#include "attention.h"

#include <algorithm>
#include <vector>

namespace {

using namespace faith;
using namespace faith::attn;

constexpr int MFMA = 0x8, VALU = 0x2, DS_READ = 0x100;      // classes of __builtin_amdgcn_sched_group_barrier
constexpr float LOWEST = -3.402823466e38f;   // the least finite number stands for "no key yet": differences stay numbers
constexpr float LAZY = 8.f;                  // powers of two by which a row's largest score may pass its reference

struct FwdArgs {
    const void *q, *k, *v;
    void *out;
    float *lse, *part;
    const Item *items;
    Deal deal;
    long long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs, lse_hs;       // strides in elements
    int group, kv_heads, size, causal;
    float c;                                 // scale * log2(e)
};

// The output of one row over the keys that it sees, by this lane alone (see "what a mask hides" in attention.h); its reference stands, for
// a score that is hidden is replaced, not multiplied.
template <class T, int DP>
__device__ void one_row(const FwdArgs &g, const Item &it, int hk, const T *qrow, int last, int half, float ref, floatx16 (&o)[DP / 32]) {
    const T *k = reinterpret_cast<const T *>(g.k) + (long long)hk * g.k_hs, *v = reinterpret_cast<const T *>(g.v) + (long long)hk * g.v_hs;
    const int end = it.end < last + 1 ? it.end : last + 1;
#pragma unroll
    for (int m = 0; m < DP / 32; ++m)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[m][r] = 0.f;
    for (int j = it.begin; j < end; ++j) {
        const float p = __builtin_amdgcn_exp2f(fmaf(dot_rows(qrow, k + (long long)(it.k_start + j) * g.k_ts, g.size), g.c, -ref));
        add_row<T, DP>(o, v + (long long)(it.k_start + j) * g.v_ts, p, half, g.size);
    }
}

template <class T, int DP, int BN, int KIND, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, resident(FORWARD, KIND, sizeof(T), DP)) attention_forward(const FwdArgs g) {
    constexpr bool KEYS = KIND != KIND_ROWS, ONCE = KIND == KIND_ONCE;
    constexpr int TILE = BN * DP, ALL = TILE * (KEYS ? WAVES : 1);
    typedef Stager<T, DP, BN, KEYS ? 1 : 4> St;                     // keys: read by rows
    typedef Stager<T, DP, BN, KEYS ? 1 : 4, COLUMNS> Sv;            // values: by columns only
    // two stages in arrays of their own, so that the compiler sees that loads into one do not touch the other
    __shared__ __align__(16) T k0[ALL], v0[ALL], k1[ONCE ? 1 : ALL], v1[ONCE ? 1 : ALL];

    int hk, n;
    if (!dealt(g.deal, &hk, &n)) return;
    const Item it = g.items[n];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int half = lane >> 5, col = lane & 31;

    // this lane's row
    const int row = it.row0 + (KEYS ? 0 : wave * 32) + col, rows = it.q_len * g.group;
    const int at = row < rows ? row : rows - 1;                    // a row behind the last repeats it and is not stored
    const int token = at / g.group, head = hk * g.group + (at - token * g.group);
    const T *qrow = reinterpret_cast<const T *>(g.q) + (long long)(it.q_start + token) * g.q_ts + (long long)head * g.q_hs;
    const ColumnRegs<T, DP> q = column_regs<T, DP>(qrow, half, g.size);
    // the last key that it may look at (the last query stands at the last key)
    int last = it.k_len - 1;
    if (g.causal) last = last < token + it.k_len - it.q_len ? last : token + it.k_len - it.q_len;
    // first and last of the wavefront's rows: tiles that some row sees in part, tiles that no row sees
    const int row_lo = it.row0 + (KEYS ? 0 : wave * 32), row_hi = row_lo + 31 < rows ? row_lo + 31 : rows - 1;
    int all_see = it.k_len - 1, any_sees = it.k_len - 1;
    if (g.causal) {
        const int shift = it.k_len - it.q_len, a = row_lo / g.group + shift, b = row_hi / g.group + shift;
        all_see = all_see < a ? all_see : a;
        any_sees = any_sees < b ? any_sees : b;
    }
    if (row_lo >= rows) any_sees = -1;

    floatx16 o[DP / 32];
#pragma unroll
    for (int m = 0; m < DP / 32; ++m)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[m][r] = 0.f;
    float ref = LOWEST, sum = 0.f;           // the row's reference (powers of two) and this lane's part of its sum
    // fp16: the reference lies that much under the row's maximum, so that smaller probabilities keep their bits as operands; the
    // largest are then 2^(UP + LAZY) = 2^15
    constexpr float UP = probability_up<T>() ? 7.f : 0.f;

    St ks;
    Sv vs;
    ks.init(lane, KEYS ? 0 : wave, g.size, g.k_ts);
    vs.init(lane, KEYS ? 0 : wave, g.size, g.v_ts);
    const T *kb = reinterpret_cast<const T *>(g.k) + (long long)it.k_start * g.k_ts + (long long)hk * g.k_hs;
    const T *vb = reinterpret_cast<const T *>(g.v) + (long long)it.k_start * g.v_ts + (long long)hk * g.v_hs;
    const int own = KEYS ? wave * TILE : 0;

    auto stage = [&](T *kt, T *vt, int key0) {
        ks.load(kt + own, kb + (long long)key0 * g.k_ts, it.k_len - key0, g.size, KEYS ? 0 : wave);
        vs.load(vt + own, vb + (long long)key0 * g.v_ts, it.k_len - key0, g.size, KEYS ? 0 : wave);
    };
    typedef floatx16 Scores[BN / 32];
    auto scores = [&](const T *kt, Scores &s) {
#pragma unroll
        for (int b = 0; b < BN / 32; ++b) s[b] = rows_by_column<T, DP>(kt + own, 32 * b, col, half, q);
    };
    // what the mask hides of the tile, and the row's reference
    auto masked = [&](Scores &s, int key0) {
        if (key0 + BN - 1 > all_see) {
#pragma unroll
            for (int b = 0; b < BN / 32; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (key0 + 32 * b + row_of(r, half) > last) s[b][r] = -__builtin_inff();
        }
        float top = s[0][0];
#pragma unroll
        for (int b = 0; b < BN / 32; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = __builtin_fmaxf(top, s[b][r]);
        // The reference follows the maximum only when it has fallen LAZY powers of two behind: sums and outputs are then at
        // most 2^LAZY times what they would be, which costs no precision, and most tiles rescale nothing.
        if (__any(top * g.c > ref + (UP + LAZY))) {
            const float now = __builtin_fmaxf(ref, max_halves(top) * g.c - UP), f = __builtin_amdgcn_exp2f(ref - now);
            ref = now;
            sum *= f;
#pragma unroll
            for (int m = 0; m < DP / 32; ++m)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[m][r] *= f;
        }
    };
    auto values = [&](Scores &s, const T *vt) {
#pragma unroll
        for (int b = 0; b < BN / 32; ++b) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[b][r] = __builtin_amdgcn_exp2f(fmaf(s[b][r], g.c, -ref));
                sum += s[b][r];
            }
            columns_by_result<T, DP, COLUMNS>(o, vt + own, 32 * b, lane, s[b]);
        }
    };
    auto tile = [&](const T *kt, const T *vt, int key0) {
        if (key0 > any_sees) return;
        Scores s;
        scores(kt, s);
        masked(s, key0);
        values(s, vt);
    };

    if constexpr (!KEYS && sizeof(T) == 2) {
        // The scores of a tile are computed one tile ahead, beside the exponentials of the tile before: a product leaves room
        // for four vector instructions.  16384 causal tokens, 32 / 8 heads of 128: 2059 -> 2034 us; the rest is power (with
        // zeros for data, where the same instructions draw less, the same call takes 1466 us).
        auto stage_k = [&](T *kt, int key0) { ks.load(kt, kb + (long long)key0 * g.k_ts, it.k_len - key0, g.size, wave); };
        auto stage_v = [&](T *vt, int key0) { vs.load(vt, vb + (long long)key0 * g.v_ts, it.k_len - key0, g.size, wave); };
        auto step = [&](const T *k_next, const T *vt, Scores &s, Scores &next, int key0) {
            if (key0 > any_sees) return;
            masked(s, key0);
            scores(k_next, next);            // behind the last tile: of what the stage held before, and not used
            values(s, vt);
            // the order of issue: reads four products ahead, the vector instructions spread between the products
            constexpr int SCORES = BN / 32 * (DP / 16), VALUES = BN / 32 * 2 * (DP / 32);
            __builtin_amdgcn_sched_group_barrier(DS_READ, 4, 0);
#pragma unroll
            for (int i = 0; i < SCORES; ++i) {
                __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
                __builtin_amdgcn_sched_group_barrier(VALU, 4, 0);
                __builtin_amdgcn_sched_group_barrier(DS_READ, 1, 0);
            }
#pragma unroll
            for (int i = 0; i < VALUES; ++i) {
                __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
                __builtin_amdgcn_sched_group_barrier(VALU, 4, 0);
                __builtin_amdgcn_sched_group_barrier(DS_READ, 2, 0);
            }
        };
        if (it.begin < it.end) {
            Scores s0, s1;
            stage_k(k0, it.begin);
            landed_and_barrier();
            if (it.begin + BN < it.end) stage_k(k1, it.begin + BN);
            stage_v(v0, it.begin);
            scores(k0, s0);
            for (int key0 = it.begin; key0 < it.end; key0 += 2 * BN) {
                landed_and_barrier();
                if (key0 + 2 * BN < it.end) stage_k(k0, key0 + 2 * BN);
                if (key0 + BN < it.end) stage_v(v1, key0 + BN);
                step(k1, v0, s0, s1, key0);
                if (key0 + BN >= it.end) break;
                landed_and_barrier();
                if (key0 + 3 * BN < it.end) stage_k(k1, key0 + 3 * BN);
                if (key0 + 2 * BN < it.end) stage_v(v0, key0 + 2 * BN);
                step(k0, v1, s1, s0, key0 + BN);
            }
        }
    } else if constexpr (!KEYS) {
        if (it.begin < it.end) {
            stage(k0, v0, it.begin);
            for (int key0 = it.begin; key0 < it.end; key0 += 2 * BN) {
                landed_and_barrier();
                if (key0 + BN < it.end) stage(k1, v1, key0 + BN);
                tile(k0, v0, key0);
                if (key0 + BN >= it.end) break;
                landed_and_barrier();
                if (key0 + 2 * BN < it.end) stage(k0, v0, key0 + 2 * BN);
                tile(k1, v1, key0 + BN);
            }
        }
    } else {
        if (it.begin + wave * BN < it.end) stage(k0, v0, it.begin + wave * BN);
        alone<2 * St::LOADS, ONCE>(it.begin + wave * BN, WAVES * BN, it.end,
                             [&](int n, int key0) { n ? stage(k1, v1, key0) : stage(k0, v0, key0); },
                             [&](int n, int key0) { n ? tile(k1, v1, key0) : tile(k0, v0, key0); });
        // the wavefronts' results meet in LDS: each leaves (reference, sum) and its output, the first joins them
        __syncthreads();
        constexpr int WIDTH = DP / 32 * 16, HALF = ALL * (int)sizeof(T) / 4;
        static_assert((WAVES - 1) * 64 * WIDTH <= 2 * HALF, "the results fit a stage");
        __shared__ __align__(16) float ml[(WAVES - 1) * 128];
        float *lo = reinterpret_cast<float *>(k0), *hi = reinterpret_cast<float *>(v0);
        auto cell = [&](int w, int e) -> float & {                 // result w, register e of this lane
            const int x = (w * WIDTH + e) * 64 + lane;
            return x < HALF ? lo[x] : hi[x - HALF];
        };
        if (wave > 0) {
            ml[(wave - 1) * 128 + lane] = ref;
            ml[(wave - 1) * 128 + 64 + lane] = sum;
#pragma unroll
            for (int m = 0; m < DP / 32; ++m)
#pragma unroll
                for (int r = 0; r < 16; ++r) cell(wave - 1, 16 * m + r) = o[m][r];
        }
        __syncthreads();
        if (wave > 0) return;
        float now = ref;
#pragma unroll
        for (int w = 0; w < WAVES - 1; ++w) now = __builtin_fmaxf(now, ml[w * 128 + lane]);
        const float f0 = __builtin_amdgcn_exp2f(ref - now);
        sum *= f0;
#pragma unroll
        for (int m = 0; m < DP / 32; ++m)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[m][r] *= f0;
#pragma unroll
        for (int w = 0; w < WAVES - 1; ++w) {
            const float f = __builtin_amdgcn_exp2f(ml[w * 128 + lane] - now);
            sum = fmaf(ml[w * 128 + 64 + lane], f, sum);
#pragma unroll
            for (int m = 0; m < DP / 32; ++m)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[m][r] = fmaf(cell(w, 16 * m + r), f, o[m][r]);
        }
        ref = now;
    }

    sum = sum_halves(sum);
    if (g.causal) {
        float bad = sum;
#pragma unroll
        for (int m = 0; m < DP / 32; ++m)
#pragma unroll
            for (int r = 0; r < 16; ++r) bad = fmaf(0.f, o[m][r], bad);      // finite values leave it finite
        // not where every row's own scores are NaN; nor where nothing that was hidden is to blame
        if (__any(!(__builtin_fabsf(bad) < __builtin_inff())) && __any(sum == sum) &&
            rows_not_finite(vb, g.v_ts, all_see + 1 > it.begin ? all_see + 1 : it.begin, it.k_len < any_sees + BN ? it.k_len : any_sees + BN, g.size, lane))
            one_row<T, DP>(g, it, hk, qrow, last, half, ref, o);
    }
    if (row >= rows) return;
    if (it.slot >= 0) {
        // a part: (reference, sum) and the unnormalised output, DP + 2 floats a row
        constexpr int ROWS = KEYS ? 32 : 128;
        float *p = g.part + ((long long)(it.slot * g.kv_heads + hk) * ROWS + (row - it.row0)) * (DP + 4);
        if (half == 0) { p[0] = ref; p[1] = sum; }
#pragma unroll
        for (int m = 0; m < DP / 32; ++m)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const floatx4 x = {o[m][r], o[m][r + 1], o[m][r + 2], o[m][r + 3]};
                *reinterpret_cast<floatx4 *>(p + 4 + 32 * m + row_of(r, half)) = x;
            }
        return;
    }
    const float inverse = last < 0 ? 0.f : 1.f / sum;                  // no key: zeros.  (Scores of -infinity only: 0 / 0)
    T *dst = reinterpret_cast<T *>(g.out) + (long long)(it.q_start + token) * g.o_ts + (long long)head * g.o_hs;
    store_column<T, DP>(dst, o, inverse, half, g.size);
    if (g.lse && half == 0)
        g.lse[(long long)head * g.lse_hs + it.q_start + token] = last < 0 ? -__builtin_inff() : (ref + __builtin_amdgcn_logf(sum)) * 0.69314718055994531f;
}

// Joins the parts of the rows of one item: {first token, tokens, -, keys, first row, parts, -, first slot}; W wavefronts
// to a row, taking turns at its parts, their lanes along the head: four for few rows in many parts, one for 128 rows in a few.
// The order of the sums depends on the number of parts only.
template <class T, int DP, int ROWS, int W>
__global__ void __launch_bounds__(256) attention_join(const FwdArgs g, const Item *joins) {
    constexpr int N = (DP + 63) / 64;
    __shared__ __align__(16) float ml[4][2], os[3][64 * N];
    const Item it = joins[blockIdx.x];
    const int hk = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int rows = it.q_len * g.group, parts = it.begin;
    const long long step = (long long)g.kv_heads * ROWS * (DP + 4);
    const int turn = W == 1 ? 0 : wave;
    for (int i = W == 1 ? blockIdx.z * 4 + wave : blockIdx.z; i < ROWS && it.row0 + i < rows; i += (W == 1 ? 4 : 1) * gridDim.z) {
        const float *p = g.part + ((long long)(it.slot * g.kv_heads + hk) * ROWS + i) * (DP + 4);
        float ref = LOWEST, sum = 0.f, o[N] = {};
        // this wavefront's parts, 64 at a time: turn, turn + W, ...
        for (int s0 = turn; s0 < parts; s0 += 64 * W) {
            const int mine = s0 + W * lane, n = (parts - s0 + W - 1) / W < 64 ? (parts - s0 + W - 1) / W : 64;
            const float r = mine < parts ? p[mine * step] : LOWEST, l = mine < parts ? p[mine * step + 1] : 0.f;
            float now = __builtin_fmaxf(ref, r);
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) now = __builtin_fmaxf(now, __shfl_xor(now, d));
            const float old = __builtin_amdgcn_exp2f(ref - now), f = __builtin_amdgcn_exp2f(r - now);
            float add = mine < parts ? l * f : 0.f;
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) add += __shfl_xor(add, d);
            sum = fmaf(sum, old, add);
            ref = now;
#pragma unroll
            for (int e = 0; e < N; ++e) o[e] *= old;
            for (int k = 0; k < n; ++k) {
                const float w = __shfl(f, k);
                const float *q = p + (s0 + W * k) * step + 4;
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (64 * e + lane < DP) o[e] = fmaf(q[64 * e + lane], w, o[e]);
            }
        }
        float now = ref;
        if constexpr (W > 1) {
            __syncthreads();                 // the row before has been read
            if (lane == 0) { ml[wave][0] = ref; ml[wave][1] = sum; }
            if (wave > 0)
#pragma unroll
                for (int e = 0; e < N; ++e) os[wave - 1][64 * e + lane] = o[e];
            __syncthreads();
            if (wave > 0) continue;
#pragma unroll
            for (int w = 1; w < W; ++w) now = __builtin_fmaxf(now, ml[w][0]);
            float f = __builtin_amdgcn_exp2f(ref - now);
            sum *= f;
#pragma unroll
            for (int e = 0; e < N; ++e) o[e] *= f;
#pragma unroll
            for (int w = 1; w < W; ++w) {
                f = __builtin_amdgcn_exp2f(ml[w][0] - now);
                sum = fmaf(ml[w][1], f, sum);
#pragma unroll
                for (int e = 0; e < N; ++e) o[e] = fmaf(os[w - 1][64 * e + lane], f, o[e]);
            }
        }
        const int row = it.row0 + i, token = row / g.group, head = hk * g.group + (row - token * g.group);
        const bool none = it.k_len == 0 || (g.causal && token + it.k_len < it.q_len);             // sees no key
        const float inverse = none ? 0.f : 1.f / sum;
        T *dst = reinterpret_cast<T *>(g.out) + (long long)(it.q_start + token) * g.o_ts + (long long)head * g.o_hs;
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (64 * e + lane < g.size) dst[64 * e + lane] = (T)(o[e] * inverse);
        if (g.lse && lane == 0)
            g.lse[(long long)head * g.lse_hs + it.q_start + token] = none ? -__builtin_inff() : (now + __builtin_amdgcn_logf(sum)) * 0.69314718055994531f;
    }
}

template <class T, int DP> int launch_forward(const FwdArgs &g, int kind, unsigned grid, const Item *joins, int n_joins, hipStream_t stream) {
    constexpr int BN = sizeof(T) == 4 ? 32 : 64;
    constexpr int WAVES = split_waves<T, DP>();
    if (kind == KIND_ONCE) hipLaunchKernelGGL((attention_forward<T, DP, 32, KIND_ONCE, WAVES>), dim3(grid), dim3(64 * WAVES), 0, stream, g);
    else if (kind == KIND_KEYS) hipLaunchKernelGGL((attention_forward<T, DP, 32, KIND_KEYS, WAVES>), dim3(grid), dim3(64 * WAVES), 0, stream, g);
    else hipLaunchKernelGGL((attention_forward<T, DP, BN, KIND_ROWS, 4>), dim3(grid), dim3(256), 0, stream, g);
    if (n_joins > 0) {
        if (kind != KIND_ROWS) hipLaunchKernelGGL((attention_join<T, DP, 32, 4>), dim3(n_joins, g.kv_heads, g.group < 8 ? g.group : 8), dim3(256), 0, stream, g, joins);
        else hipLaunchKernelGGL((attention_join<T, DP, 128, 1>), dim3(n_joins, g.kv_heads, 32), dim3(256), 0, stream, g, joins);
    }
    return check_launch("faith_attention");
}
template <class T> int launch_forward(const FwdArgs &g, int kind, unsigned grid, const Item *joins, int n_joins, hipStream_t stream) {
    if (g.size <= 32) return launch_forward<T, 32>(g, kind, grid, joins, n_joins, stream);
    if (g.size <= 64) return launch_forward<T, 64>(g, kind, grid, joins, n_joins, stream);
    if (g.size <= 96) return launch_forward<T, 96>(g, kind, grid, joins, n_joins, stream);
    return launch_forward<T, 128>(g, kind, grid, joins, n_joins, stream);
}

}  // namespace

// ------------------------------------------------------------------------------------------ host
namespace {

struct Plan {
    std::vector<Item> items, joins;
    int kind = KIND_ROWS, slots = 0;
};

// Items of one pass, longest first.
// Wavefronts share their rows and divide the rest (KEYS) for 32 rows or fewer, and
//   backward  where workgroups of 128 rows would leave half of the compute units without one: 1000 tokens, 4 heads of 64, bf16
//             27 us instead of 52; 2048 tokens, 8 / 2 heads of 128 152 instead of 467 (95 since the group is cut, below);
//             20 sequences of 256 with 4 heads (160 workgroups) would take 33 instead of 21
//   forward   there too, in fp32, if none has a second turn: 30 sequences of 128, 4 heads of 64 11.2 us instead of 13.4.  With
//             more keys, or 2-byte elements, 128 rows and cut keys are faster (1000 tokens as above: 14 against 28).
// The gradients of keys are cut by the heads of the group where there are fewer workgroups of 128 keys than the device holds:
// 4096 tokens, 8 heads on one key head, 198 instead of 435 us.
// The forward pass cuts an item's keys where there are fewer items than compute units: into parts of equal length, as many as
// make up that number, none under 256 keys.  More parts pay for filling and draining the stages and for the join (4 queries
// against 30000 keys each, 32 / 8 heads of 128: four times as many 161 us instead of 96), and 128 rows in two parts are slower
// than whole (10 sequences of 300, 8 heads of 128: 28 against 12 us).
Plan make_plan(const int *ql, const int *kl, int n, int group, int kv_heads, int element_size, int size, int causal, int pass) {
    Plan p;
    long long qs = 0, ks = 0;
    const int cus = compute_units();
    const int waves = split_waves(element_size, (size + 31) / 32 * 32);
    long long most = 0, tall = 0;            // rows of a sequence; workgroups of 128 rows
    int keys_most = 0;
    for (int b = 0; b < n; ++b) {
        const long long rows = pass == FAITH_ATTENTION_GRAD_KEYS ? kl[b] : (long long)ql[b] * group;
        most = std::max(most, rows);
        tall += (rows + 127) / 128 * kv_heads;
        keys_most = std::max(keys_most, kl[b]);
    }
    int by_heads = 1;                        // parts of the group
    if (pass == FAITH_ATTENTION_GRAD_KEYS && tall > 0) {
        by_heads = (int)std::max<long long>(1, std::min<long long>(group, 2LL * cus / tall));
        tall *= by_heads;
    }
    if (most <= 32 || (2 * tall <= cus && (pass != FAITH_ATTENTION_FORWARD || (element_size == 4 && keys_most <= 32 * waves)))) p.kind = KIND_KEYS;
    const int rows_per = p.kind == KIND_KEYS ? 32 : 128, bn = p.kind == KIND_KEYS || element_size == 4 ? 32 : 64;
    for (int b = 0; b < n; ++b) {
        const int shift = kl[b] - ql[b];
        if (pass == FAITH_ATTENTION_GRAD_KEYS) {
            for (int key0 = 0; key0 < kl[b]; key0 += rows_per) {
                // the first token that sees a key of the tile
                const int begin = causal ? std::min(ql[b], std::max(0, key0 - shift)) : 0;
                const Item it = {(int)qs, ql[b], (int)ks, kl[b], key0, begin / 32 * 32, ql[b], -1};
                if (by_heads == 1) { p.items.push_back(it); continue; }
                Item j = it;
                j.begin = by_heads;
                j.end = 0;
                j.slot = p.slots;
                p.joins.push_back(j);
                for (int i = 0; i < by_heads; ++i) {
                    p.items.push_back(it);
                    p.items.back().slot = p.slots++;
                }
            }
        } else {
            const long long rows = (long long)ql[b] * group;
            for (long long row0 = 0; row0 < rows; row0 += rows_per) {
                const int token = (int)((std::min(rows, row0 + rows_per) - 1) / group);
                const int end = causal ? std::max(0, std::min(kl[b], token + shift + 1)) : kl[b];
                p.items.push_back({(int)qs, ql[b], (int)ks, kl[b], (int)row0, 0, end, -1});
            }
        }
        qs += ql[b];
        ks += kl[b];
    }
    const long long blocks = (long long)p.items.size() * kv_heads;
    if (pass == FAITH_ATTENTION_FORWARD && blocks > 0 && blocks < cus) {
        long long keys = 0;
        for (const Item &it : p.items) keys += it.end;
        long long chunk = (keys * kv_heads + cus - 1) / cus;
        chunk = std::max<long long>((chunk + bn - 1) / bn * bn, 256);
        std::vector<Item> cut;
        for (const Item &it : p.items) {
            const int n_parts = (int)((it.end + chunk - 1) / chunk);
            if (n_parts <= (p.kind == KIND_ROWS ? 2 : 1)) { cut.push_back(it); continue; }
            Item j = it;
            j.begin = n_parts;
            j.end = 0;
            j.slot = p.slots;
            p.joins.push_back(j);
            const int each = (int)(((it.end + n_parts - 1) / n_parts + bn - 1) / bn * bn);
            for (int i = 0; i < n_parts; ++i) {
                Item c = it;
                c.begin = std::min(it.end, i * each);
                c.end = std::min(it.end, (i + 1) * each);
                c.slot = p.slots++;
                cut.push_back(c);
            }
        }
        p.items.swap(cut);
    }
    if (p.kind == KIND_KEYS) {
        // tiles of an item, as many of which as there are wavefronts are worked on at once
        const int times = pass == FAITH_ATTENTION_GRAD_KEYS ? (group + by_heads - 1) / by_heads : 1;
        const bool once = std::all_of(p.items.begin(), p.items.end(), [&](const Item &it) { return (long long)((it.end - it.begin + 31) / 32) * times <= waves; });
        if (once) p.kind = KIND_ONCE;
    }
    std::stable_sort(p.items.begin(), p.items.end(), [](const Item &a, const Item &b) { return a.end - a.begin > b.end - b.begin; });
    return p;
}

}  // namespace

extern "C" int faith_attention_plan(const int *query_lengths, const int *key_lengths, int sequences, int heads, int kv_heads,
                                    int element_size, int size, int causal, int pass, int *items, long long capacity, long long *counts) {
    FAITH_NOT_NULL(query_lengths);
    FAITH_NOT_NULL(key_lengths);
    FAITH_NOT_NULL(counts);
    FAITH_REQUIRE(sequences > 0, FAITH_ERR_SHAPE, "%s: %d sequences", __func__, sequences);
    FAITH_REQUIRE(kv_heads > 0 && heads > 0 && heads % kv_heads == 0, FAITH_ERR_SHAPE, "%s: %d heads do not share %d key heads evenly", __func__, heads, kv_heads);
    FAITH_REQUIRE(element_size == 2 || element_size == 4, FAITH_ERR_UNSUPPORTED, "%s: elements of %d bytes", __func__, element_size);
    FAITH_REQUIRE(size > 0 && size <= 128, FAITH_ERR_UNSUPPORTED, "%s: heads of %d elements", __func__, size);
    FAITH_REQUIRE(pass >= FAITH_ATTENTION_FORWARD && pass <= FAITH_ATTENTION_GRAD_KEYS, FAITH_ERR_UNSUPPORTED, "%s: pass %d", __func__, pass);
    long long q = 0, k = 0;
    for (int b = 0; b < sequences; ++b) {
        FAITH_REQUIRE(query_lengths[b] >= 0 && key_lengths[b] >= 0, FAITH_ERR_SHAPE, "%s: sequence %d has a negative length", __func__, b);
        q += query_lengths[b];
        k += key_lengths[b];
        FAITH_REQUIRE((long long)query_lengths[b] * (heads / kv_heads) < (1LL << 30) && key_lengths[b] < (1 << 30), FAITH_ERR_SHAPE,
                      "%s: sequence %d is too long", __func__, b);
    }
    FAITH_REQUIRE(q < (1LL << 31) && k < (1LL << 31), FAITH_ERR_SHAPE, "%s: more than 2^31 tokens", __func__);
    try {
        const Plan p = make_plan(query_lengths, key_lengths, sequences, heads / kv_heads, kv_heads, element_size, size, causal, pass);
        counts[0] = (long long)p.items.size();
        counts[1] = (long long)p.joins.size();
        counts[2] = p.slots;
        counts[3] = p.kind;
        if (items) {
            FAITH_REQUIRE(capacity >= counts[0] + counts[1], FAITH_ERR_SHAPE, "%s: room for %lld items, %lld are needed", __func__, capacity, counts[0] + counts[1]);
            std::copy(p.items.begin(), p.items.end(), reinterpret_cast<Item *>(items));
            std::copy(p.joins.begin(), p.joins.end(), reinterpret_cast<Item *>(items) + p.items.size());
        }
    } catch (const std::exception &e) {
        FAITH_REQUIRE(false, FAITH_ERR_UNSUPPORTED, "%s: %s", __func__, e.what());
    }
    return FAITH_OK;
}

extern "C" int faith_attention(const void *q, const void *k, const void *v, void *out, float *lse, float *parts, const int *items,
                               int n_items, int n_joins, int kind, long long q_token_stride, long long q_head_stride,
                               long long k_token_stride, long long k_head_stride, long long v_token_stride, long long v_head_stride,
                               long long out_token_stride, long long out_head_stride, long long lse_head_stride, int heads, int kv_heads,
                               int size, int dtype, int causal, float scale, void *stream) {
    FAITH_REQUIRE(n_items >= 0 && n_joins >= 0, FAITH_ERR_SHAPE, "%s: %d items, %d joins", __func__, n_items, n_joins);
    if (n_items == 0) return FAITH_OK;
    FAITH_NOT_NULL(q);
    FAITH_NOT_NULL(out);
    FAITH_NOT_NULL(items);
    FAITH_REQUIRE(n_joins == 0 || parts, FAITH_ERR_NULL, "%s: keys are cut into parts, and there is no room for their results", __func__);
    FAITH_REQUIRE(kind >= KIND_ROWS && kind <= KIND_ONCE, FAITH_ERR_UNSUPPORTED, "%s: kind %d", __func__, kind);
    const int rc = attention_shapes(__func__, heads, kv_heads, size, dtype, scale);
    if (rc != FAITH_OK) return rc;
    const int es = dtype == FAITH_F32 ? 4 : 2;
    if (!attention_rows(__func__, "q", q, q_token_stride, q_head_stride, size, es) || !attention_rows(__func__, "k", k, k_token_stride, k_head_stride, size, es) ||
        !attention_rows(__func__, "v", v, v_token_stride, v_head_stride, size, es) || !attention_rows(__func__, "out", out, out_token_stride, out_head_stride, size, es) ||
        !attention_heads_apart(__func__, "out", out_token_stride, out_head_stride, heads, size))
        return FAITH_ERR_ALIGN;
    if (!attention_grid(__func__, n_items, kv_heads)) return FAITH_ERR_UNSUPPORTED;
    FwdArgs g;
    unsigned grid;
    g.q = q; g.k = k; g.v = v; g.out = out; g.lse = lse; g.part = parts;
    g.items = reinterpret_cast<const Item *>(items);
    g.deal = deal(n_items, kv_heads, &grid);
    g.q_ts = q_token_stride; g.q_hs = q_head_stride; g.k_ts = k_token_stride; g.k_hs = k_head_stride;
    g.v_ts = v_token_stride; g.v_hs = v_head_stride; g.o_ts = out_token_stride; g.o_hs = out_head_stride; g.lse_hs = lse_head_stride;
    g.group = heads / kv_heads; g.kv_heads = kv_heads; g.size = size; g.causal = causal;
    g.c = scale * 1.4426950408889634f;
    const Item *joins = g.items + n_items;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == FAITH_F32) return launch_forward<float>(g, kind, grid, joins, n_joins, s);
    if (dtype == FAITH_BF16) return launch_forward<__bf16>(g, kind, grid, joins, n_joins, s);
    return launch_forward<_Float16>(g, kind, grid, joins, n_joins, s);
}
