// attention_backward.hip -- gradients of softmax attention of packed sequences with grouped heads.
//
//   p_rj = exp(s_rj - lse_r),  delta_r = <do_r, o_r>,  dp_rj = <do_r, v_j>,  ds_rj = p_rj (dp_rj - delta_r)
//   dq_r = scale sum_j ds_rj k_j,  dk_j = scale sum_r ds_rj q_r,  dv_j = sum_r p_rj do_r
// with the sums over r running over all heads of the group that read key head of j.
//
// Two kernels, each of which owns what it adds up in registers, so no result is made by atomics and none depends on
// timing: one by rows (dq, and delta on its way), one by keys (dk and dv).  Scores and dp are made twice, seven products
// in all where five would do, for which no gradient is written and read again as partial sums.
//  * by rows: 128 packed rows a workgroup, 32 a wave, q and do in registers; tiles of keys and values.
//    S^T and dP^T leave a lane with its own row's scores, so lse and delta are its own scalars.
//  * by keys: 128 keys a workgroup, 32 a wave, k and v in registers; tiles of packed rows of q and do, whose lse and
//    delta come from LDS.  S and dP leave a lane with its own key's column.
// delta comes from out, whose rounding and whose weights' rounding would go into every ds of the row: an error of 2.2e-3 of dq and
// dk in bfloat16, more than rounding ds (1.8e-3) or the results (1.7e-3). But sum_j ds_rj is 0, so what the kernel by rows finds
// for it is delta's error: it hands the exact one to the kernel by keys.  For dq it sums ds as rounded, and takes that sum
// times sum_j p_rj k_j off: an eighth product, by operands that are in registers already, after which what is
// multiplied sums to 0 again, so that neither delta's error nor what rounding adds to all keys alike is left (not in 32 bits).
//
// 1 x 32768 tokens, causal, 16 / 4 heads of 128 in bfloat16: by rows 7.2 ms (four products, 1.2 PFLOP/s), by keys 8.6 (1.02),
// bound by power as the forward pass is.  8 sequences of 512 to 8192 tokens: 0.73 and 0.84 ms, and 0.04 to add up the parts of
// dk and dv into which the longest sequences' rows are cut (without: 1.04).
//
// p and ds are rounded to the operands' type for the last products, which is half a unit of each; in float16 they are held
// in powers of two of their own (p times 2^14, ds see Units).
#include "attention.h"

namespace vh {
namespace attn {
namespace {

struct BwdArgs {
    Heads q, k, v, o, go, dq, dk, dv;
    const float *lse;
    float *delta;
    Packed rows, keys;
    Group group;
    int heads, kv_heads, dim;
    bool causal;
    float scale;
    int splits;   // parts of what is summed over, each a workgroup; more than one leave `part`, which other kernels add up
    float *part;  // [split][2][token][head][DP]: dq and sum p k, or dk and dv
    float2 *off;  // [split][token][head]: sum ds, and of ds as rounded
    uint32_t first;  // workgroup of this launch
};

constexpr int kBM = 128, kBK = 128;  // rows and keys of a workgroup
template <class T>
constexpr int kBN = sizeof(T) == 2 ? 64 : 32;  // keys of a tile

// Waves of a SIMD whose registers hold all that they own: two have 256 a lane, one has 512.
template <class T, int DP>
struct RegsFor {
    static constexpr int dq = sizeof(T) == 4 && DP > 96 ? 1 : 2;
};

// The kernel by keys: 4 waves of 32 keys each, where registers allow it twice: both halves of the waves have the same
// keys, and every second block of 32 rows. The longest workgroup, not their sum, is what few long sequences wait for.
template <class T, int DP>
struct ByKeys {
    static constexpr bool wide = sizeof(T) == 4 && DP > 64;
    static constexpr int halves = wide ? 1 : 2, waves = 4 * halves;
    static constexpr int rows = wide ? 32 : sizeof(T) == 4 ? 64 : 128;  // of a tile
};

// Power of two of p where it is an operand
template <class T>
constexpr float kShift = std::is_same<T, half_t>::value ? 14.f : 0.f;

template <class T, int KS>
__device__ __forceinline__ void load_operand(typename Frag<T>::type (&f)[KS], const char *row, int dim, int half, bool neg) {
    constexpr int VEC = 16 / (int)sizeof(T);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const auto x = load_row<VEC>((const T *)row, (2 * ks + half) * VEC, dim);
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[ks][e] = neg ? -x.v[e] : x.v[e];
    }
}

template <class T, int DP, bool DMA>
__global__ __launch_bounds__(256, (RegsFor<T, DP>::dq)) void k_attn_dq(BwdArgs a) {
    constexpr int BN = kBN<T>, NS = BN / 32, RB = DP * (int)sizeof(T), KS = RB / 32, DT = DP / 32, VEC = 16 / (int)sizeof(T);
    typedef typename Frag<T>::type frag;
    typedef Tile<T, DP, BN, 4, DMA> KV;
    __shared__ __attribute__((aligned(1024))) char lds[2][2][KV::kBytes];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;

    const uint32_t id = a.first + blockIdx.x;
    const int kh = id % a.kv_heads, split = (id / a.kv_heads) % a.splits;
    const Place at = find_tile<kBM>(a.rows, a.group.size, id / a.kv_heads / a.splits);
    const Span rows = packed_span(a.rows, at.seq);
    const int n = rows.len * a.group.size;
    if (at.tile >= (n + kBM - 1) / kBM) return;
    const bool real = at.seq >= 1 && at.seq <= a.rows.count;
    const Span keys = real ? packed_span(a.keys, at.seq) : Span{0, 0};
    const int row0 = ((n + kBM - 1) / kBM - 1 - at.tile) * kBM;

    const int r = row0 + wave * 32 + (lane & 31), rc = min(r, n - 1);
    const int token = a.group.token(rc), head = kh * a.group.size + rc - token * a.group.size;
    const int64_t row = rows.begin + token;
    const int shift = keys.len - rows.len + 1;
    const int sees = a.causal ? min(keys.len, max(0, token + shift)) : keys.len;
    const int most = a.causal ? min(keys.len, max(0, a.group.token(min(row0 + kBM, n) - 1) + shift)) : keys.len;
    const int tiles = (most + BN - 1) / BN, per = (tiles + a.splits - 1) / a.splits;
    const int t0 = split * per, t1 = min(tiles, t0 + per);
    const int w0 = row0 + wave * 32, w1 = min(w0 + 32, n) - 1;
    const int all = a.causal ? min(keys.len, max(0, a.group.token(min(w0, n - 1)) + shift)) : keys.len;
    const int any = w0 >= n ? 0 : a.causal ? min(keys.len, max(0, a.group.token(w1) + shift)) : keys.len;

    const char *kb = a.k.data + keys.begin * a.k.token + kh * a.k.head, *vb = a.v.data + keys.begin * a.v.token + kh * a.v.head;
    auto load = [&](int t, int buf) {
        load_rows<KV, BN>(kb, a.k.token, t * BN, keys.len - 1, a.dim, lds[buf][0]);
        load_rows<KV, BN>(vb, a.v.token, t * BN, keys.len - 1, a.dim, lds[buf][1]);
    };
    if (t0 < t1) load(t0, 0);
    KV::clear_past(a.dim, 4 * BN, lds[0][0]);

    const int64_t at_row = row * a.heads + head;
    frag q[KS], go[KS];
    load_operand<T>(q, a.q.data + row * (int64_t)a.q.token + (int64_t)head * a.q.head, a.dim, half, a.scale < 0.f);
    load_operand<T>(go, a.go.data + row * (int64_t)a.go.token + (int64_t)head * a.go.head, a.dim, half, false);
    float delta = 0.f;
    {
        const T *p = (const T *)(a.o.data + row * (int64_t)a.o.token + (int64_t)head * a.o.head);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const auto x = load_row<VEC>(p, (2 * ks + half) * VEC, a.dim);
#pragma unroll
            for (int e = 0; e < VEC; ++e) delta = fmaf((float)go[ks][e], (float)x.v[e], delta);
        }
        delta = half_sum(delta);
    }
    const float lse = a.lse[at_row], c = fmaxf(fabsf(a.scale) * kLog2e, 1.2e-38f);
    const float base = lse == -INFINITY ? 0.f : -lse * kLog2e;

    constexpr bool EXACT = sizeof(T) == 2;  // see above
    floatx16_t dq[DT] = {}, pk[EXACT ? DT : 1] = {};
    float off = 0.f, rounded = 0.f;  // sum ds, and as rounded, in units
    Units<T> units;
    for (int t = t0; t < t1; ++t) {
        tiles_ready();
        const int buf = (t - t0) & 1;
        if (t + 1 < t1) load(t + 1, buf ^ 1);
#pragma unroll 1
        for (int j = 0; j < NS; ++j) {
            const int key0 = t * BN + 32 * j, ln = anew(lane);
            if (key0 >= any) break;
            floatx16_t s = mma_rows<T, RB>(lds[buf][0], 32 * j, q, ln);
            floatx16_t dp = mma_rows<T, RB>(lds[buf][1], 32 * j, go, ln);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, base));
                dp[i] = s[i] * (dp[i] - delta);
            }
            if (key0 + 32 > all) {
                const int left = sees - key0 - 4 * half;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (row_of(i) >= left) s[i] = dp[i] = 0.f;
            }
            frag ds[kOps<T>], p[kOps<T>];
            if constexpr (EXACT) {
                float sum[2] = {};
#pragma unroll
                for (int i = 0; i < 16; ++i) sum[i % 2] += dp[i];
                off += sum[0] + sum[1];
                to_operand<T>(s, p);
            }
            units.to_units(dp, dq, rounded);
            to_operand<T>(dp, ds);
            if constexpr (EXACT) rounded = operand_sum(ds[1], operand_sum(ds[0], rounded));
            __builtin_amdgcn_sched_barrier(0);  // operands read ahead of these would not fit the registers
            if constexpr (EXACT)
                mma_cols2<T, RB>(lds[buf][0], 32 * j, ds, dq, p, pk, ln);
            else
                mma_cols<T, RB>(lds[buf][0], 32 * j, ds, dq, ln);
        }
    }
    if (r >= n) return;
    off = half_sum(off);
    rounded = units.back(half_sum(rounded));
    if (split == 0 && half == 0) a.delta[at_row] = a.splits > 1 ? delta : delta + off;
    if (a.splits > 1) {  // k_attn_sum_rows does the rest
        const int64_t all = a.rows.tokens * a.heads;
        if (EXACT && half == 0) a.off[split * all + at_row] = make_float2(off, rounded);
        store_cols<float, DT>(a.part + (2 * split * all + at_row) * DP, dq, DP, lane, [&](float x) { return units.back(x); });
        if constexpr (EXACT)
            store_cols<float, DT>(a.part + ((2 * split + 1) * all + at_row) * DP, pk, DP, lane, [](float x) { return x; });
        return;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            dq[d][i] = units.back(dq[d][i]);
            if constexpr (EXACT) dq[d][i] = fmaf(-rounded, pk[d][i], dq[d][i]);
        }
    store_cols<T, DT>((T *)(a.dq.data + row * (int64_t)a.dq.token + (int64_t)head * a.dq.head), dq, a.dim, lane,
                      [&](float x) { return x * a.scale; });
}

template <class T, int DP, bool DMA>
__global__ __launch_bounds__((64 * ByKeys<T, DP>::waves), (ByKeys<T, DP>::halves)) void k_attn_dkv(BwdArgs a) {
    constexpr int NW = ByKeys<T, DP>::waves, HALVES = ByKeys<T, DP>::halves, BR = ByKeys<T, DP>::rows, NS = BR / 32, RB = DP * (int)sizeof(T), KS = RB / 32, DT = DP / 32;
    typedef typename Frag<T>::type frag;
    typedef Tile<T, DP, BR, NW, DMA> QG;
    __shared__ __attribute__((aligned(1024))) char lds[2][2][QG::kBytes];
    static_assert(HALVES == 1 || 4 * QG::kBytes >= 4 * DT * 4096, "room for one half's sums");
    __shared__ __attribute__((aligned(16))) float stats[2][2][BR];  // -lse in base 2, delta
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;

    const uint32_t id = a.first + blockIdx.x;
    const int kh = id % a.kv_heads, split = (id / a.kv_heads) % a.splits;
    const Place at = find_tile<kBK>(a.keys, 1, id / a.kv_heads / a.splits);
    const Span keys = packed_span(a.keys, at.seq);
    if (at.tile >= (keys.len + kBK - 1) / kBK) return;
    const bool real = at.seq >= 1 && at.seq <= a.keys.count;
    const Span rows = real ? packed_span(a.rows, at.seq) : Span{0, 0};
    const int n = rows.len * a.group.size, g = a.group.size;
    // the first keys of a sequence are seen by the most rows
    const int key0 = at.tile * kBK, w0 = key0 + (wave & 3) * 32, row_half = wave >> 2;

    // this lane's key, and the first row that sees it: of the lane, of the wave's first and last key, of the workgroup
    const int j = w0 + (lane & 31), back = rows.len - keys.len;
    auto first_row = [&](int key) { return a.causal ? min(n, max(0, key + back) * g) : 0; };
    const int first = first_row(j), wave_first = first_row(w0), wave_last = first_row(w0 + 31);
    const int b0 = first_row(key0) / BR, blocks = (n + BR - 1) / BR - b0, per = (blocks + a.splits - 1) / a.splits;
    const int t0 = b0 + split * per, t1 = min(b0 + blocks, t0 + per);

    const char *qb = a.q.data + rows.begin * a.q.token + (int64_t)kh * g * a.q.head;
    const char *gb = a.go.data + rows.begin * a.go.token + (int64_t)kh * g * a.go.head;
    float next_lse = 0.f, next_delta = 0.f;
    auto load = [&](int t, int buf) {
        const int r0 = t * BR;
        if (threadIdx.x < BR) {
            const int r = min(r0 + (int)threadIdx.x, n - 1), token = a.group.token(r);
            const int64_t i = (rows.begin + token) * a.heads + kh * g + r - token * g;
            next_lse = a.lse[i];
            next_delta = a.delta[i];
        }
        load_packed<QG, BR>(qb, a.q, a.group, r0, n - 1, a.dim, lds[buf][0]);
        load_packed<QG, BR>(gb, a.go, a.group, r0, n - 1, a.dim, lds[buf][1]);
    };
    auto put_stats = [&](int buf) {
        if (threadIdx.x < BR) {
            stats[buf][0][threadIdx.x] = next_lse == -INFINITY ? 0.f : fmaf(-next_lse, kLog2e, kShift<T>);
            stats[buf][1][threadIdx.x] = next_delta;
        }
    };
    if (t0 < t1) {
        load(t0, 0);
        put_stats(0);
    }
    QG::clear_past(a.dim, 4 * BR, lds[0][0]);

    const int jc = min(j, keys.len - 1);
    frag k[KS], v[KS];
    load_operand<T>(k, a.k.data + (keys.begin + jc) * (int64_t)a.k.token + (int64_t)kh * a.k.head, a.dim, half, a.scale < 0.f);
    load_operand<T>(v, a.v.data + (keys.begin + jc) * (int64_t)a.v.token + (int64_t)kh * a.v.head, a.dim, half, false);
    const float c = fmaxf(fabsf(a.scale) * kLog2e, 1.2e-38f);

    floatx16_t dk[DT] = {}, dv[DT] = {};
    float none = 0.f;
    Units<T> units;
    for (int t = t0; t < t1; ++t) {
        tiles_ready();
        const int buf = (t - t0) & 1;
        if (t + 1 < t1) load(t + 1, buf ^ 1);
#pragma unroll 1
        for (int h = 0; h < NS / HALVES; ++h) {
            const int b = h * HALVES + row_half, ln = anew(lane);
            const int r0 = t * BR + 32 * b;
            if (r0 + 32 <= wave_first || r0 >= n) continue;
            floatx16_t s = mma_rows<T, RB>(lds[buf][0], 32 * b, k, ln);
            floatx16_t dp = mma_rows<T, RB>(lds[buf][1], 32 * b, v, ln);
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const Pack<float, 4> l = *(const Pack<float, 4> *)&stats[buf][0][32 * b + row_of(i) + 4 * half];
                const Pack<float, 4> d = *(const Pack<float, 4> *)&stats[buf][1][32 * b + row_of(i) + 4 * half];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[i + e] = __builtin_amdgcn_exp2f(fmaf(s[i + e], c, l.v[e]));
                    dp[i + e] = s[i + e] * (dp[i + e] - d.v[e]);
                }
            }
            if (r0 < wave_last || r0 + 32 > n) {
                const int from = first - r0 - 4 * half, to = n - r0 - 4 * half;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (row_of(i) < from || row_of(i) >= to) s[i] = dp[i] = 0.f;
            }
            frag p[kOps<T>];
            to_operand<T>(s, p);
            __builtin_amdgcn_sched_barrier(0);  // operands read ahead of these would not fit the registers
            mma_cols<T, RB>(lds[buf][1], 32 * b, p, dv, ln);
            __builtin_amdgcn_sched_barrier(0);
            units.to_units(dp, dk, none);
            frag ds[kOps<T>];
            to_operand<T>(dp, ds);
            mma_cols<T, RB>(lds[buf][0], 32 * b, ds, dk, ln);
        }
        if (t + 1 < t1) put_stats(buf ^ 1);
    }
    const float shrink = kShift<T> > 0.f ? 1.f / 16384.f : 1.f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            dk[d][i] = units.back(dk[d][i]) * (a.scale * shrink);
            dv[d][i] *= shrink;
        }
    if constexpr (HALVES == 2) {  // the second half's sums go through LDS
        float *sums = (float *)&lds[0][0][0] + (wave & 3) * DT * 1024 + lane;
        auto join = [&](floatx16_t (&x)[DT]) {
            __syncthreads();
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (row_half) sums[(d * 16 + i) * 64] = x[d][i];
            __syncthreads();
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!row_half) x[d][i] += sums[(d * 16 + i) * 64];
        };
        join(dk);
        join(dv);
    }
    if (row_half || j >= keys.len) return;
    auto same = [](float x) { return x; };
    const int64_t row = keys.begin + j;
    if (a.splits > 1) {
        const int64_t all = a.keys.tokens * a.kv_heads, i = row * a.kv_heads + kh;
        store_cols<float, DT>(a.part + ((2 * split) * all + i) * DP, dk, DP, lane, same);
        store_cols<float, DT>(a.part + ((2 * split + 1) * all + i) * DP, dv, DP, lane, same);
    } else {
        store_cols<T, DT>((T *)(a.dk.data + row * (int64_t)a.dk.token + (int64_t)kh * a.dk.head), dk, a.dim, lane, same);
        store_cols<T, DT>((T *)(a.dv.data + row * (int64_t)a.dv.token + (int64_t)kh * a.dv.head), dv, a.dim, lane, same);
    }
}

// Adds up the parts of dq, in their order, and what they found for delta.
template <class T, int DP>
__global__ __launch_bounds__(256) void k_attn_sum_rows(BwdArgs a) {
    constexpr int L = DP / 4, R = kRowsOf256<DP>;
    constexpr bool EXACT = sizeof(T) == 2;
    const int64_t all = a.rows.tokens * a.heads;
    const int64_t i = (int64_t)blockIdx.x * R + threadIdx.x / L;
    const int e = threadIdx.x % L * 4;
    if (threadIdx.x >= R * L || i >= all || e >= a.dim) return;
    float sum[4] = {}, pk[4] = {}, off = 0.f, rounded = 0.f;
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
        const Pack<float, 4> p = load_any<4>(a.part + (2 * s * all + i) * DP + e);
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] += p.v[k];
        if constexpr (EXACT) {
            const Pack<float, 4> w = load_any<4>(a.part + ((2 * s + 1) * all + i) * DP + e);
#pragma unroll
            for (int k = 0; k < 4; ++k) pk[k] += w.v[k];
            const float2 o = a.off[s * all + i];
            off += o.x;
            rounded += o.y;
        }
    }
    if (EXACT && e == 0) a.delta[i] += off;
    Pack<T, 4> v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v.v[k] = (T)(fmaf(-rounded, pk[k], sum[k]) * a.scale);
    store_row<4>((T *)(a.dq.data + i / a.heads * (int64_t)a.dq.token + i % a.heads * (int64_t)a.dq.head), e, a.dim, v);
}

// Adds up the parts of dk or dv (blockIdx.y).
template <class T, int DP>
__global__ __launch_bounds__(256) void k_attn_sum_keys(BwdArgs a) {
    constexpr int L = DP / 4, R = kRowsOf256<DP>;
    const int64_t all = a.keys.tokens * a.kv_heads;
    const int64_t i = (int64_t)blockIdx.x * R + threadIdx.x / L;
    const int e = threadIdx.x % L * 4;
    if (threadIdx.x >= R * L || i >= all || e >= a.dim) return;
    float sum[4] = {};
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
        const Pack<float, 4> p = load_any<4>(a.part + ((2 * s + blockIdx.y) * all + i) * DP + e);
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] += p.v[k];
    }
    Pack<T, 4> v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v.v[k] = (T)sum[k];
    const Heads &o = blockIdx.y ? a.dv : a.dk;
    store_row<4>((T *)(o.data + i / a.kv_heads * (int64_t)o.token + i % a.kv_heads * (int64_t)o.head), e, a.dim, v);
}

// What a call works in: delta, then the parts of dq and afterwards, in the same place, those of dk and dv.
struct Work {
    int qsplits, ksplits;
    float *delta, *part;
    float2 *off;
    size_t bytes;
};
Work work_of(int dtype, const Shape &s, void *base) {
    Work w;
    w.qsplits = key_splits(dtype, s, kBM);
    // By keys a workgroup walks all rows of a group, so the longest sequence's decide. Parts cost a pass over sums of 32 bits:
    // 2048 rows at least where it is to even workgroups out, fewer where there are too few of them.
    const int64_t wgs = slot_count(s.key_tokens, s.sequences, 1, kBK) * s.kv_heads;
    const size_t along = s.tokens * (s.heads / s.kv_heads);
    const int fill = split_count(wgs, along, s.sequences, 512, 256), even = split_count(wgs, along, s.sequences, 2048, 2048);
    w.ksplits = fill > even ? fill : even;
    const size_t dp = padded(s.dim);
    const size_t q = w.qsplits > 1 ? 2 * w.qsplits * s.tokens * s.heads * dp : 0;
    const size_t k = w.ksplits > 1 ? 2 * w.ksplits * s.key_tokens * s.kv_heads * dp : 0;
    Carver c{(char *)base};
    w.delta = c.take<float>(s.tokens * s.heads);
    w.off = c.take<float2>(w.qsplits > 1 ? w.qsplits * s.tokens * s.heads : 0);
    w.part = c.take<float>(q > k ? q : k);
    w.bytes = c.used;
    return w;
}

struct Run {
    Work w;
    bool dq, dkv, dma_kv, dma_q;
    int64_t qgrid, kgrid;
    hipStream_t s;
};

template <class T, int DP>
int launch(BwdArgs a, const Run &r) {
    if (r.qgrid) {
        a.splits = r.w.qsplits;
        each_launch(r.qgrid, 256, [&](int64_t first, uint32_t n) {
            a.first = (uint32_t)first;
            if (r.dma_kv)
                k_attn_dq<T, DP, true><<<n, 256, 0, r.s>>>(a);
            else
                k_attn_dq<T, DP, false><<<n, 256, 0, r.s>>>(a);
        });
        if (a.splits > 1) k_attn_sum_rows<T, DP><<<(uint32_t)ceil_div(a.rows.tokens * a.heads, kRowsOf256<DP>), 256, 0, r.s>>>(a);
    }
    if (r.kgrid) {
        a.splits = r.w.ksplits;
        constexpr int threads = 64 * ByKeys<T, DP>::waves;
        each_launch(r.kgrid, threads, [&](int64_t first, uint32_t n) {
            a.first = (uint32_t)first;
            if (r.dma_q)
                k_attn_dkv<T, DP, true><<<n, threads, 0, r.s>>>(a);
            else
                k_attn_dkv<T, DP, false><<<n, threads, 0, r.s>>>(a);
        });
        if (a.splits > 1)
            k_attn_sum_keys<T, DP><<<dim3((uint32_t)ceil_div(a.keys.tokens * a.kv_heads, kRowsOf256<DP>), 2), 256, 0, r.s>>>(a);
    }
    return launch_status("attention launch");
}
template <class T>
int launch(const BwdArgs &a, const Run &r) {
    switch (padded(a.dim)) {
        case 32: return launch<T, 32>(a, r);
        case 64: return launch<T, 64>(a, r);
        case 96: return launch<T, 96>(a, r);
        default: return launch<T, 128>(a, r);
    }
}

}  // namespace
}  // namespace attn
}  // namespace vh

using namespace vh;
using namespace vh::attn;

extern "C" {

size_t vhip_attention_backward_workspace(int dtype, size_t tokens, size_t key_tokens, size_t heads, size_t kv_heads, size_t dim,
                                         size_t sequences) {
    if (!kv_heads || !heads || !dtype_known(dtype)) return 0;
    return work_of(dtype, {tokens, key_tokens, heads, kv_heads, dim, sequences}, nullptr).bytes;
}

int vhip_attention_backward(int ordinal, int dtype, const vhip_heads *dout, const vhip_heads *q, const vhip_heads *k,
                            const vhip_heads *v, const vhip_heads *out, const float *lse, size_t tokens, size_t key_tokens,
                            size_t heads, size_t kv_heads, size_t dim, const int64_t *offsets, const int64_t *key_offsets,
                            size_t sequences, int causal, float scale, const vhip_heads *dq, const vhip_heads *dk,
                            const vhip_heads *dv, void *workspace, size_t workspace_bytes, void *stream) {
    clear_error();
    const Shape sh{tokens, key_tokens, heads, kv_heads, dim, sequences};
    VH_CHECK(check_shape(dtype, sh, offsets, key_offsets, scale));
    VH_CHECK(check_heads("dout", dout, dtype, tokens, heads, dim));
    VH_CHECK(check_heads("q", q, dtype, tokens, heads, dim));
    VH_CHECK(check_heads("k", k, dtype, key_tokens, kv_heads, dim));
    VH_CHECK(check_heads("v", v, dtype, key_tokens, kv_heads, dim));
    VH_CHECK(check_heads("out", out, dtype, tokens, heads, dim));
    if (tokens && !lse) return set_error(VHIP_ERR_INVALID_CONFIG, "lse is null");
    VH_CHECK(check_heads("dq", dq, dtype, tokens, heads, dim));
    VH_CHECK(check_heads("dk", dk, dtype, key_tokens, kv_heads, dim));
    VH_CHECK(check_heads("dv", dv, dtype, key_tokens, kv_heads, dim));
    Run r;
    r.w = work_of(dtype, sh, workspace);
    if (r.w.bytes && (!workspace || workspace_bytes < r.w.bytes || !aligned16(workspace)))
        return set_error(VHIP_ERR_INVALID_CONFIG, "the workspace is smaller than vhip_attention_backward_workspace() or not aligned");
    const int64_t qgrid = slot_count(tokens, sequences, heads / kv_heads, kBM) * (int64_t)kv_heads * r.w.qsplits;
    const int64_t kgrid = slot_count(key_tokens, sequences, 1, kBK) * (int64_t)kv_heads * r.w.ksplits;
    if (qgrid > 0x7fffffff || kgrid > 0x7fffffff) return set_error(VHIP_ERR_INVALID_CONFIG, "too many rows or sequences");
    CallDevice dev;
    VH_CHECK(dev.enter(ordinal));
    r.qgrid = tokens ? qgrid : 0;
    r.kgrid = key_tokens ? kgrid : 0;
    r.dma_kv = whole_chunks(k, dtype, dim) && whole_chunks(v, dtype, dim);
    r.dma_q = whole_chunks(q, dtype, dim) && whole_chunks(dout, dtype, dim);
    r.s = (hipStream_t)stream;
    const BwdArgs a{to_heads(q, dtype), to_heads(k, dtype), to_heads(v, dtype), to_heads(out, dtype), to_heads(dout, dtype),
                    to_heads(dq, dtype), to_heads(dk, dtype), to_heads(dv, dtype), lse, r.w.delta,
                    {offsets, (int64_t)tokens, (int)sequences},
                    {key_offsets ? key_offsets : offsets, (int64_t)key_tokens, (int)sequences},
                    to_group(heads, kv_heads), (int)heads, (int)kv_heads, (int)dim, causal != 0, scale, 1, r.w.part, r.w.off, 0};
    switch (dtype) {
        case VHIP_DTYPE_F32: return launch<float>(a, r);
        case VHIP_DTYPE_F16: return launch<half_t>(a, r);
        default: return launch<bf16_t>(a, r);
    }
}

}  // extern "C"
