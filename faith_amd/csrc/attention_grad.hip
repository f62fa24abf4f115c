// Gradients of the attention of a network's concrete pass (attention.hip), scores and probabilities computed again:
//     p = exp(s - lse),  dp = do . v,  ds = p (dp - delta),  delta = do . out
//     dq = scale sum_j ds k,   dk = scale sum_{i, heads of the group} ds q,   dv = sum_{i, heads of the group} p do
// p and ds are held in 32 bits and rounded once, to the elements' type, as operands of the last three products (in fp16 times a
// power of two that keeps them in its range, see follow() in attention.h); delta comes from the output as it was stored.  Against
// one rounding of each result these are two or three independent ones of the same size: 1.4 times the error of a computation in 32
// bits at a few hundred keys, up to twice at a handful.
// Two launches (a third joins parts where the plan cuts) and no atomics, so that the same call gives the same bits: one goes over
// the keys for a tile of query rows (and leaves delta and the logarithm of the row's sum, in powers of two, to the other), one over
// the queries of all heads of the group for a tile of keys.  That computes s and dp twice -- seven products where five would do -- and
// needs neither an array of sums in 32 bits that many workgroups add to nor a pass that rounds it.
// Measured, 5 causal sequences of 300 to 4096, 32 / 8 heads of 128 in bf16: queries 0.60 ms, matrix units 55 % busy; keys 1.00 ms, 41 %.
#include "attention.h"

namespace {

using namespace faith;
using namespace faith::attn;

struct GradArgs {
    const void *dout, *q, *k, *v, *out;
    const float *lse;
    void *dq, *dk, *dv;
    float *stat;                             // [2][heads][lse_hs]: lse in powers of two less probability_up(); delta (fp16: -delta)
    float *part;                             // [slots][key heads][keys of an item][2 DP]: parts of dk and dv
    const Item *items;
    Deal deal;
    long long do_ts, do_hs, q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs, dq_ts, dq_hs, dk_ts, dk_hs, dv_ts, dv_hs, lse_hs;
    int group, kv_heads, size, causal, parts;
    float c, scale;                          // scale * log2(e); scale
};

template <class T> __device__ __forceinline__ const T *at(const void *base, long long row, long long ts, int head, long long hs) {
    return reinterpret_cast<const T *>(base) + row * ts + (long long)head * hs;
}

template <int DP> __device__ __forceinline__ void clear(floatx16 (&o)[DP / 32]) {
#pragma unroll
    for (int m = 0; m < DP / 32; ++m)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[m][r] = 0.f;
}
template <int DP> __device__ __forceinline__ bool any_not_finite(const floatx16 (&o)[DP / 32]) {
    float bad = 0.f;
#pragma unroll
    for (int m = 0; m < DP / 32; ++m)
#pragma unroll
        for (int r = 0; r < 16; ++r) bad = fmaf(0.f, o[m][r], bad);
    return __any(bad != 0.f);                // 0 * NaN, 0 * infinity
}
// SPLIT: the wavefronts share 32 rows and divide the keys, as in attention.hip
template <class T, int DP, int BN, int KIND, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, resident(GRAD_QUERIES, KIND, sizeof(T), DP)) attention_grad_queries(const GradArgs g) {
    constexpr bool SPLIT = KIND != KIND_ROWS, ONCE = KIND == KIND_ONCE;
    constexpr int TILE = BN * DP, ALL = TILE * (SPLIT ? WAVES : 1);
    typedef Stager<T, DP, BN, SPLIT ? 1 : WAVES> St;
    __shared__ __align__(16) T k0[ALL], v0[ALL], k1[ONCE ? 1 : ALL], v1[ONCE ? 1 : ALL];

    int hk, n;
    if (!dealt(g.deal, &hk, &n)) return;
    const Item it = g.items[n];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int half = lane >> 5, col = lane & 31;
    const int staged = SPLIT ? 0 : wave, own = SPLIT ? wave * TILE : 0;
    const int row_lo = it.row0 + (SPLIT ? 0 : wave * 32), row = row_lo + col, rows = it.q_len * g.group;
    const int mine = row < rows ? row : rows - 1;
    const int token = mine / g.group, head = hk * g.group + (mine - token * g.group);
    const long long place = it.q_start + token;
    const T *qrow = at<T>(g.q, place, g.q_ts, head, g.q_hs), *dorow = at<T>(g.dout, place, g.do_ts, head, g.do_hs);
    const ColumnRegs<T, DP> q = column_regs<T, DP>(qrow, half, g.size), d_o = column_regs<T, DP>(dorow, half, g.size);
    const ColumnRegs<T, DP> o = column_regs<T, DP>(at<T>(g.out, place, g.o_ts, head, g.o_hs), half, g.size);
    const float l = g.lse[(long long)head * g.lse_hs + place];
    int last = it.k_len - 1, all_see = it.k_len - 1, any_sees = it.k_len - 1;
    if (g.causal) {
        const int shift = it.k_len - it.q_len, row_hi = row_lo + 31 < rows ? row_lo + 31 : rows - 1;
        const int a = row_lo / g.group + shift, b = row_hi / g.group + shift;
        last = last < token + shift ? last : token + shift;
        all_see = all_see < a ? all_see : a;
        any_sees = any_sees < b ? any_sees : b;
    }
    if (row_lo >= rows) any_sees = -1;

    floatx16 dq[DP / 32];
    clear<DP>(dq);
    St ks, vs;
    ks.init(lane, staged, g.size, g.k_ts);
    vs.init(lane, staged, g.size, g.v_ts);
    const T *kb = at<T>(g.k, it.k_start, g.k_ts, hk, g.k_hs), *vb = at<T>(g.v, it.k_start, g.v_ts, hk, g.v_hs);
    auto stage = [&](T *kt, T *vt, int key0) {
        ks.load(kt + own, kb + (long long)key0 * g.k_ts, it.k_len - key0, g.size, staged);
        vs.load(vt + own, vb + (long long)key0 * g.v_ts, it.k_len - key0, g.size, staged);
    };
    // the first tile is on its way before anything waits for this lane's row
    const int first = it.begin + (SPLIT ? wave * BN : 0);
    if (first < it.end) stage(k0, v0, first);
    float delta = 0.f;
    constexpr int PER = 16 / (int)sizeof(T);
#pragma unroll
    for (int u = 0; u < DP / (2 * PER); ++u)
#pragma unroll
        for (int e = 0; e < PER; ++e) delta = fmaf((float)o.v[u][e], (float)d_o.v[u][e], delta);
    delta = sum_halves(delta);
    const float lse = last < 0 ? 0.f : l * 1.4426950408889634f;                    // a row that sees no key: every p below is masked
    int up = probability_up<T>() ? UP_MOST : 0;      // p comes out times 2^up, and so does ds
    if (row < rows && half == 0 && (!SPLIT || wave == 0)) {
        float *s = g.stat + (long long)head * g.lse_hs + place;
        s[0] = lse - probability_up<T>();
        s[(long long)g.kv_heads * g.group * g.lse_hs] = probability_up<T>() ? -delta : delta;
    }
    auto tile = [&](const T *kt, const T *vt, int key0) {
        if (key0 > any_sees) return;
        const bool part = key0 + BN - 1 > all_see;
#pragma unroll
        for (int b = 0; b < BN / 32; ++b) {
            floatx16 one[1] = {rows_by_column<T, DP>(kt + own, 32 * b, col, half, q)}, &s = one[0];
            const floatx16 dp = rows_by_column<T, DP>(vt + own, 32 * b, col, half, d_o);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], g.c, (float)up - lse)) * (dp[r] - delta);
            if (part) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (key0 + 32 * b + row_of(r, half) > last) s[r] = 0.f;
            }
            if constexpr (probability_up<T>() > 0) follow<DP>(one, dq, up);
            columns_by_result<T, DP>(dq, kt + own, 32 * b, lane, s);
        }
    };
    if constexpr (SPLIT) {
        alone<2 * St::LOADS, ONCE>(first, WAVES * BN, it.end,
                             [&](int n, int key0) { n ? stage(k1, v1, key0) : stage(k0, v0, key0); },
                             [&](int n, int key0) { n ? tile(k1, v1, key0) : tile(k0, v0, key0); });
        if constexpr (probability_up<T>() > 0) lower<DP>(dq, up);
        add_waves<WAVES, DP, ALL * (int)sizeof(T) / 4>(dq, reinterpret_cast<float *>(k0), reinterpret_cast<float *>(v0), wave, lane);
        if (wave > 0) return;
    } else if (it.begin < it.end) {
        for (int key0 = it.begin; key0 < it.end; key0 += 2 * BN) {
            landed_and_barrier();
            if (key0 + BN < it.end) stage(k1, v1, key0 + BN);
            tile(k0, v0, key0);
            if (key0 + BN >= it.end) break;
            landed_and_barrier();
            if (key0 + 2 * BN < it.end) stage(k0, v0, key0 + 2 * BN);
            tile(k1, v1, key0 + BN);
        }
        if constexpr (probability_up<T>() > 0) lower<DP>(dq, up);
    }
    if (g.causal && any_not_finite<DP>(dq) && __any(lse == lse) &&
        rows_not_finite(kb, g.k_ts, all_see + 1 > 0 ? all_see + 1 : 0, it.k_len < any_sees + BN ? it.k_len : any_sees + BN, g.size, lane)) {
        // see "what a mask hides" in attention.h
        clear<DP>(dq);
        for (int j = 0; j <= last; ++j) {
            const T *kr = kb + (long long)j * g.k_ts;
            const float p = __builtin_amdgcn_exp2f(fmaf(dot_rows(qrow, kr, g.size), g.c, -lse));
            add_row<T, DP>(dq, kr, p * (dot_rows(dorow, vb + (long long)j * g.v_ts, g.size) - delta), half, g.size);
        }
    }
    if (last == 0) {                         // p = 1 and dp = delta, exactly; what is no number stays none
#pragma unroll
        for (int m = 0; m < DP / 32; ++m)
#pragma unroll
            for (int r = 0; r < 16; ++r) dq[m][r] = fmaf(dq[m][r], 0.f, 0.f);
    }
    if (row >= rows) return;
    store_column<T, DP>(const_cast<T *>(at<T>(g.dq, place, g.dq_ts, head, g.dq_hs)), dq, g.scale, half, g.size);
}

template <class T, int DP, int BQ, int KIND, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, resident(GRAD_KEYS, KIND, sizeof(T), DP)) attention_grad_keys(const GradArgs g) {
    constexpr bool SPLIT = KIND != KIND_ROWS, ONCE = KIND == KIND_ONCE;
    constexpr int TILE = BQ * DP, EACH = SPLIT ? WAVES : 1, ALL = TILE * EACH;
    typedef Stager<T, DP, BQ, SPLIT ? 1 : WAVES> St;
    __shared__ __align__(16) T q0[ALL], d0[ALL], q1[ONCE ? 1 : ALL], d1[ONCE ? 1 : ALL];
    __shared__ __align__(16) float l0[64 * EACH], e0[64 * EACH], l1[ONCE ? 1 : 64 * EACH], e1[ONCE ? 1 : 64 * EACH];           // lse, delta of the staged queries

    int hk, n;
    if (!dealt(g.deal, &hk, &n)) return;
    const Item it = g.items[n];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int half = lane >> 5, col = lane & 31;
    const int staged = SPLIT ? 0 : wave, own = SPLIT ? wave * TILE : 0, own64 = SPLIT ? wave * 64 : 0;
    const int key_lo = it.row0 + (SPLIT ? 0 : wave * 32), key = key_lo + col, mine = key < it.k_len ? key : it.k_len - 1;
    const T *krow = at<T>(g.k, it.k_start + mine, g.k_ts, hk, g.k_hs), *vrow = at<T>(g.v, it.k_start + mine, g.v_ts, hk, g.v_hs);
    const ColumnRegs<T, DP> k = column_regs<T, DP>(krow, half, g.size);
    // The values' rows stay in LDS where registers for them would halve the wavefronts on a SIMD
    constexpr bool V_IN_LDS = !SPLIT && sizeof(T) == 2 && DP == 128;
    __shared__ __align__(16) T v_rows[V_IN_LDS ? 128 * DP : 1];
    ColumnRegs<T, DP> v;
    if constexpr (V_IN_LDS) {
        Stager<T, DP, 128, 4> vs;
        vs.init(lane, wave, g.size, g.v_ts);
        vs.load(v_rows, at<T>(g.v, it.k_start + it.row0, g.v_ts, hk, g.v_hs), it.k_len - it.row0, g.size, wave);
    } else {
        v = column_regs<T, DP>(vrow, half, g.size);
    }
    const int shift = it.k_len - it.q_len;
    // the first token that sees this lane's key, all of the wavefront's, any of them
    const int first = g.causal ? mine - shift : -1, all_see = g.causal ? key_lo + 31 - shift : -1, any_sees = key_lo >= it.k_len ? 0x7fffffff : g.causal ? key_lo - shift : -1;

    floatx16 dk[DP / 32], dv[DP / 32];
    clear<DP>(dk);
    clear<DP>(dv);
    int up = UP_MOST - probability_up<T>();  // of ds beyond that of p, fp16
    St qs, ds;
    qs.init(lane, staged, g.size, g.q_ts);
    ds.init(lane, staged, g.size, g.do_ts);
    const int span = it.end - it.begin, tiles = (span + BQ - 1) / BQ;
    // the heads of the group that this item takes: all of them, or those of one part
    const int per_part = (g.group + g.parts - 1) / g.parts, h_first = it.slot < 0 ? 0 : it.slot % g.parts * per_part;
    const int h_count = it.slot < 0 ? g.group : g.group - h_first < per_part ? g.group - h_first : per_part, total = span > 0 ? tiles * h_count : 0;
    const long long stat_hs = (long long)g.kv_heads * g.group * g.lse_hs;

    // the queries of the item's head h from token t on
    auto stage_at = [&](T *qt, T *dt, float *lt, float *et, int h, int t) {
        const int head = hk * g.group + h_first + h, left = it.q_len - t;
        qs.load(qt + own, at<T>(g.q, it.q_start + t, g.q_ts, head, g.q_hs), left, g.size, staged);
        ds.load(dt + own, at<T>(g.dout, it.q_start + t, g.do_ts, head, g.do_hs), left, g.size, staged);
        const float *s = g.stat + (long long)head * g.lse_hs + it.q_start + t;
        if (SPLIT || wave == 0) words_to_lds(lt + own64, s, left < 64 ? left : 64, lane);
        if (SPLIT || wave == 1) words_to_lds(et + own64, s + stat_hs, left < 64 ? left : 64, lane);
    };
    auto tile_at = [&](const T *qt, const T *dt, const float *lt, const float *et, int t0) {
        qt += own, dt += own, lt += own64, et += own64;
        if (t0 + BQ - 1 < any_sees) return;
        // opaque to the compiler, which would otherwise compute the tile's addresses before the loop and spill them
        int lane = (int)threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const int half = lane >> 5, col = lane & 31;
        const bool part = t0 < all_see;
        // a query that sees one key only: p = 1 and dp = delta, exactly
        const bool alone_here = it.k_len == 1 || (g.causal && t0 <= -shift && -shift < t0 + BQ);
        // all scores of the tile first, so that the exponentials of one block of 32 queries can run beside the products of
        // another, where the tile has more than one
        floatx16 s[BQ / 32], dp[BQ / 32];
#pragma unroll
        for (int b = 0; b < BQ / 32; ++b) {
            s[b] = rows_by_column<T, DP>(qt, 32 * b, col, half, k);
            if constexpr (V_IN_LDS) {
#pragma unroll
                for (int u = 0; u < DP / 16; ++u) v.v[u] = row_fragment<T, DP>(v_rows + wave * 32 * DP, 0, col, u, half);
            }
            if constexpr (probability_up<T>() > 0) {
                floatx16 minus_delta;
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const floatx4 e = *reinterpret_cast<const floatx4 *>(et + 32 * b + row_of(r, half));
#pragma unroll
                    for (int i = 0; i < 4; ++i) minus_delta[r + i] = e[i];
                }
                dp[b] = rows_by_column<T, DP>(dt, 32 * b, col, half, v, minus_delta);
            } else {
                dp[b] = rows_by_column<T, DP>(dt, 32 * b, col, half, v);
            }
        }
#pragma unroll
        for (int b = 0; b < BQ / 32; ++b) {
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const floatx4 l = *reinterpret_cast<const floatx4 *>(lt + 32 * b + row_of(r, half));
                if constexpr (probability_up<T>() > 0) {
                    const float lift = __builtin_ldexpf(1.f, up);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        s[b][r + i] = __builtin_amdgcn_exp2f(fmaf(s[b][r + i], g.c, -l[i]));
                        dp[b][r + i] *= s[b][r + i] * lift;
                    }
                } else {
                    const floatx4 e = *reinterpret_cast<const floatx4 *>(et + 32 * b + row_of(r, half));
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        s[b][r + i] = __builtin_amdgcn_exp2f(fmaf(s[b][r + i], g.c, -l[i]));
                        dp[b][r + i] = s[b][r + i] * (dp[b][r + i] - e[i]);
                    }
                }
            }
        }
        // hidden: replaced behind the exponential, whatever the row's sum and delta are
        if (part) {
#pragma unroll
            for (int b = 0; b < BQ / 32; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (t0 + 32 * b + row_of(r, half) < first) s[b][r] = dp[b][r] = 0.f;
        }
        // Rows behind the last query are staged as zeros.  Their scores are zeros too, and do no harm, unless the key is not finite: then they
        // are NaN, the last of the tile's among them
        if (t0 + BQ > it.q_len && __builtin_expect(__any(s[BQ / 32 - 1][15] != s[BQ / 32 - 1][15]), 0)) {
#pragma unroll
            for (int b = 0; b < BQ / 32; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (t0 + 32 * b + row_of(r, half) >= it.q_len) s[b][r] = dp[b][r] = 0.f;
        }
        if (alone_here) {
#pragma unroll
            for (int b = 0; b < BQ / 32; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (it.k_len == 1 || t0 + 32 * b + row_of(r, half) == -shift) dp[b][r] = fmaf(dp[b][r], 0.f, 0.f);
        }
        if constexpr (probability_up<T>() > 0) follow<DP>(dp, dk, up);
#pragma unroll
        for (int b = 0; b < BQ / 32; ++b) {
            columns_by_result<T, DP>(dv, dt, 32 * b, lane, s[b]);
            columns_by_result<T, DP>(dk, qt, 32 * b, lane, dp[b]);
        }
    };
    // step n: head n / tiles of the group, tokens from begin + (n % tiles) * BQ on
    if constexpr (SPLIT) {
        auto token = [&](int n) { return it.begin + n % tiles * BQ; };
        if (wave < total) stage_at(q0, d0, l0, e0, wave / tiles, token(wave));
        alone<2 * St::LOADS + 2, ONCE>(wave, WAVES, total,
                                 [&](int n, int i) { n ? stage_at(q1, d1, l1, e1, i / tiles, token(i)) : stage_at(q0, d0, l0, e0, i / tiles, token(i)); },
                                 [&](int n, int i) { n ? tile_at(q1, d1, l1, e1, token(i)) : tile_at(q0, d0, l0, e0, token(i)); });
        constexpr int HALF = ALL * (int)sizeof(T) / 4;
        if constexpr (probability_up<T>() > 0) {
            lower<DP>(dk, up + probability_up<T>());
            lower<DP>(dv, probability_up<T>());
        }
        add_waves<WAVES, DP, HALF>(dk, reinterpret_cast<float *>(q0), reinterpret_cast<float *>(d0), wave, lane);
        add_waves<WAVES, DP, HALF>(dv, reinterpret_cast<float *>(q0), reinterpret_cast<float *>(d0), wave, lane);
        if (wave > 0) return;
    } else if (total > 0) {
        int next_h = 0, next_t = it.begin, tok0 = it.begin;
        auto stage = [&](T *qt, T *dt, float *lt, float *et) {
            stage_at(qt, dt, lt, et, next_h, next_t);
            next_t += BQ;
            if (next_t >= it.end) { next_t = it.begin; ++next_h; }
        };
        auto tile = [&](const T *qt, const T *dt, const float *lt, const float *et) {
            tile_at(qt, dt, lt, et, tok0);
            tok0 = tok0 + BQ >= it.end ? it.begin : tok0 + BQ;
        };
        stage(q0, d0, l0, e0);
        for (int i = 0; i < total; i += 2) {
            landed_and_barrier();
            if (i + 1 < total) stage(q1, d1, l1, e1);
            tile(q0, d0, l0, e0);
            if (i + 1 >= total) break;
            landed_and_barrier();
            if (i + 2 < total) stage(q0, d0, l0, e0);
            tile(q1, d1, l1, e1);
        }
        if constexpr (probability_up<T>() > 0) {
            lower<DP>(dk, up + probability_up<T>());
            lower<DP>(dv, probability_up<T>());
        }
    }
    // hidden from some of this wavefront's keys: the queries that see the first but not the last of them, and the tile's in front of those
    auto hidden_not_finite = [&]() {
        const int from = any_sees - BQ > it.begin ? any_sees - BQ : it.begin, to = all_see < it.q_len ? all_see : it.q_len;
        // the last query sees every key: where its sum is NaN, so are all gradients
        const float last = g.stat[(long long)(hk * g.group + h_first) * g.lse_hs + it.q_start + it.q_len - 1];
        if (last != last) return false;
        bool bad = false;
        for (int h = hk * g.group + h_first; h < hk * g.group + h_first + h_count; ++h) {
            bad = bad || rows_not_finite(at<T>(g.q, it.q_start, g.q_ts, h, g.q_hs), g.q_ts, from, to, g.size, lane) ||
                  rows_not_finite(at<T>(g.dout, it.q_start, g.do_ts, h, g.do_hs), g.do_ts, from, to, g.size, lane);
        }
        return bad;
    };
    if (g.causal && (any_not_finite<DP>(dk) || any_not_finite<DP>(dv)) && hidden_not_finite()) {
        // see "what a mask hides" in attention.h
        clear<DP>(dk);
        clear<DP>(dv);
        for (int h = hk * g.group + h_first; h < hk * g.group + h_first + h_count; ++h)
            for (int i = first > 0 ? first : 0; i < it.q_len; ++i) {
                const long long place = it.q_start + i;
                const T *qr = at<T>(g.q, place, g.q_ts, h, g.q_hs), *dr = at<T>(g.dout, place, g.do_ts, h, g.do_hs);
                const float *s = g.stat + (long long)h * g.lse_hs + place;
                const float p = __builtin_amdgcn_exp2f(fmaf(dot_rows(qr, krow, g.size), g.c, -s[0] - probability_up<T>()));
                add_row<T, DP>(dv, dr, p, half, g.size);
                float grad = p * (dot_rows(dr, vrow, g.size) + (probability_up<T>() ? s[stat_hs] : -s[stat_hs]));
                if (i == -shift || it.k_len == 1) grad = fmaf(grad, 0.f, 0.f);
                add_row<T, DP>(dk, qr, grad, half, g.size);
            }
    }
    if (key >= it.k_len) return;
    if (it.slot >= 0) {
        constexpr int ROWS = SPLIT ? 32 : 128;
        float *p = g.part + ((long long)(it.slot * g.kv_heads + hk) * ROWS + (key - it.row0)) * (2 * DP);
        store_column<float, DP>(p, dk, 1.f, half, DP);
        store_column<float, DP>(p + DP, dv, 1.f, half, DP);
        return;
    }
    store_column<T, DP>(const_cast<T *>(at<T>(g.dk, it.k_start + key, g.dk_ts, hk, g.dk_hs)), dk, g.scale, half, g.size);
    store_column<T, DP>(const_cast<T *>(at<T>(g.dv, it.k_start + key, g.dv_ts, hk, g.dv_hs)), dv, 1.f, half, g.size);
}

// Adds up the parts of an item's keys in their order; a wavefront to a key.  {-, -, first key of the sequence, its keys, first key
// of the item, parts, -, first slot}
template <class T, int DP, int ROWS>
__global__ void __launch_bounds__(256) attention_grad_join(const GradArgs g, const Item *joins) {
    const Item it = joins[blockIdx.x];
    const int hk = blockIdx.y, lane = threadIdx.x & 63, i = blockIdx.z * 4 + (threadIdx.x >> 6), key = it.row0 + i;
    if (key >= it.k_len) return;
    const long long step = (long long)g.kv_heads * ROWS * (2 * DP);
    const float *p = g.part + ((long long)(it.slot * g.kv_heads + hk) * ROWS + i) * (2 * DP);
    T *dk = const_cast<T *>(at<T>(g.dk, it.k_start + key, g.dk_ts, hk, g.dk_hs)), *dv = const_cast<T *>(at<T>(g.dv, it.k_start + key, g.dv_ts, hk, g.dv_hs));
    for (int d = lane; d < g.size; d += 64) {
        float a = 0.f, b = 0.f;
        for (int s = 0; s < it.begin; ++s) {
            a += p[s * step + d];
            b += p[s * step + DP + d];
        }
        dk[d] = (T)(a * g.scale);
        dv[d] = (T)b;
    }
}

struct Items { const Item *items; int n, kind, joins; };

template <class T, int DP> int launch_backward(GradArgs g, const Items &qi, const Items &ki, hipStream_t stream) {
    constexpr int BN = sizeof(T) == 2 ? 64 : 32, BQ = sizeof(T) == 2 && DP <= 64 ? 64 : 32, W = split_waves<T, DP>();
    unsigned grid;
    if (qi.n > 0) {
        g.items = qi.items;
        g.deal = deal(qi.n, g.kv_heads, &grid);
        if (qi.kind == KIND_ONCE) hipLaunchKernelGGL((attention_grad_queries<T, DP, 32, KIND_ONCE, W>), dim3(grid), dim3(64 * W), 0, stream, g);
        else if (qi.kind == KIND_KEYS) hipLaunchKernelGGL((attention_grad_queries<T, DP, 32, KIND_KEYS, W>), dim3(grid), dim3(64 * W), 0, stream, g);
        else hipLaunchKernelGGL((attention_grad_queries<T, DP, BN, KIND_ROWS, 4>), dim3(grid), dim3(256), 0, stream, g);
    }
    if (ki.n > 0) {
        g.items = ki.items;
        g.deal = deal(ki.n, g.kv_heads, &grid);
        if (ki.kind == KIND_ONCE) hipLaunchKernelGGL((attention_grad_keys<T, DP, 32, KIND_ONCE, W>), dim3(grid), dim3(64 * W), 0, stream, g);
        else if (ki.kind == KIND_KEYS) hipLaunchKernelGGL((attention_grad_keys<T, DP, 32, KIND_KEYS, W>), dim3(grid), dim3(64 * W), 0, stream, g);
        else hipLaunchKernelGGL((attention_grad_keys<T, DP, BQ, KIND_ROWS, 4>), dim3(grid), dim3(256), 0, stream, g);
        const Item *joins = ki.items + ki.n;
        if (ki.joins > 0 && ki.kind == KIND_ROWS) hipLaunchKernelGGL((attention_grad_join<T, DP, 128>), dim3(ki.joins, g.kv_heads, 32), dim3(256), 0, stream, g, joins);
        else if (ki.joins > 0) hipLaunchKernelGGL((attention_grad_join<T, DP, 32>), dim3(ki.joins, g.kv_heads, 8), dim3(256), 0, stream, g, joins);
    }
    return check_launch("faith_attention_backward");
}
template <class T> int launch_backward(const GradArgs &g, const Items &qi, const Items &ki, hipStream_t stream) {
    if (g.size <= 32) return launch_backward<T, 32>(g, qi, ki, stream);
    if (g.size <= 64) return launch_backward<T, 64>(g, qi, ki, stream);
    if (g.size <= 96) return launch_backward<T, 96>(g, qi, ki, stream);
    return launch_backward<T, 128>(g, qi, ki, stream);
}

}  // namespace

extern "C" int faith_attention_backward(const void *dout, const void *q, const void *k, const void *v, const void *out, const float *lse,
                                        void *dq, void *dk, void *dv, float *stat, float *parts,
                                        const int *query_items, int n_query_items, int query_kind, const int *key_items,
                                        int n_key_items, int n_key_joins, int key_parts, int key_kind, const long long *strides, long long lse_head_stride,
                                        int heads, int kv_heads, int size, int dtype, int causal, float scale, void *stream) {
    FAITH_REQUIRE(n_query_items >= 0 && n_key_items >= 0, FAITH_ERR_SHAPE, "%s: %d and %d items", __func__, n_query_items, n_key_items);
    if (n_query_items == 0 && n_key_items == 0) return FAITH_OK;
    FAITH_REQUIRE(query_kind >= KIND_ROWS && query_kind <= KIND_ONCE && key_kind >= KIND_ROWS && key_kind <= KIND_ONCE, FAITH_ERR_UNSUPPORTED,
                  "%s: kinds %d and %d", __func__, query_kind, key_kind);
    FAITH_NOT_NULL(strides);
    FAITH_REQUIRE(n_key_joins >= 0 && key_parts >= 0 && (n_key_joins == 0 || key_parts > 0), FAITH_ERR_SHAPE, "%s: %d joins of %d parts", __func__, n_key_joins, key_parts);
    FAITH_REQUIRE(n_key_joins == 0 || parts, FAITH_ERR_NULL, "%s: keys are worked on in parts, and there is no room for their results", __func__);
    const int rc = attention_shapes(__func__, heads, kv_heads, size, dtype, scale);
    if (rc != FAITH_OK) return rc;
    const int es = dtype == FAITH_F32 ? 4 : 2;
    const struct { const char *name; const void *p; bool keys; } rows[8] = {{"dout", dout, false}, {"q", q, false}, {"k", k, true}, {"v", v, true},
                                                                            {"out", out, false}, {"dq", dq, false}, {"dk", dk, true}, {"dv", dv, true}};
    // a batch without queries or without keys may come without the tensors of that side
    for (int i = 0; i < 8; ++i) {
        if ((rows[i].keys ? n_key_items : n_query_items) == 0) continue;
        if (!attention_rows(__func__, rows[i].name, rows[i].p, strides[2 * i], strides[2 * i + 1], size, es)) return rows[i].p ? FAITH_ERR_ALIGN : FAITH_ERR_NULL;
        if (i >= 5 && !attention_heads_apart(__func__, rows[i].name, strides[2 * i], strides[2 * i + 1], rows[i].keys ? kv_heads : heads, size)) return FAITH_ERR_ALIGN;
    }
    FAITH_REQUIRE(n_query_items == 0 || (lse && stat && query_items), FAITH_ERR_NULL, "%s: lse, stat or the query items are NULL", __func__);
    FAITH_REQUIRE(n_key_items == 0 || key_items, FAITH_ERR_NULL, "%s: the key items are NULL", __func__);
    if (!attention_grid(__func__, n_query_items, kv_heads) || !attention_grid(__func__, n_key_items, kv_heads)) return FAITH_ERR_UNSUPPORTED;
    GradArgs g;
    g.dout = dout; g.q = q; g.k = k; g.v = v; g.out = out; g.lse = lse; g.dq = dq; g.dk = dk; g.dv = dv; g.stat = stat; g.part = parts;
    long long *to[16] = {&g.do_ts, &g.do_hs, &g.q_ts, &g.q_hs, &g.k_ts, &g.k_hs, &g.v_ts, &g.v_hs, &g.o_ts, &g.o_hs, &g.dq_ts, &g.dq_hs, &g.dk_ts, &g.dk_hs, &g.dv_ts, &g.dv_hs};
    for (int i = 0; i < 16; ++i) *to[i] = strides[i];
    g.lse_hs = lse_head_stride;
    g.group = heads / kv_heads; g.kv_heads = kv_heads; g.size = size; g.causal = causal;
    g.c = scale * 1.4426950408889634f; g.scale = scale;
    // every item is cut into as many parts
    g.parts = n_key_joins > 0 ? key_parts / n_key_joins : 1;
    const Items qi = {reinterpret_cast<const Item *>(query_items), n_query_items, query_kind, 0};
    const Items ki = {reinterpret_cast<const Item *>(key_items), n_key_items, key_kind, n_key_joins};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == FAITH_F32) return launch_backward<float>(g, qi, ki, s);
    if (dtype == FAITH_BF16) return launch_backward<__bf16>(g, qi, ki, s);
    return launch_backward<_Float16>(g, qi, ki, s);
}
