// attention_forward.hip -- softmax attention of packed sequences with grouped heads.
//
//   s_rj = scale <q_r, k_j> over the keys j that row r sees,  lse_r = log sum_j exp s_rj,
//   o_r = sum_j exp(s_rj - lse_r) v_j;  a row that sees no key has o = 0 and lse = -inf
//
// One pass over the keys: a workgroup has 128 packed rows (attention.h) of one sequence and key head, 32 to a wave,
// and walks tiles of keys and values that come by DMA into the other of two buffers while one is multiplied. A
// row's largest score m and sum l run along, in the scores' base-2 logarithms; the output and l are only scaled anew
// once a row's m has grown by more than 2^8, so most tiles take no pass over the accumulators.  Weights are rounded to the
// values' type to be multiplied (half a unit of each); their sum takes them as they were.
//
// A causal sequence of 32768 tokens, 32 / 8 heads of 128 in bfloat16: 8.5 ms, 1.03 PFLOP/s, where the library's product of
// 8192^3 reaches 1.11 to 1.33.  What bounds it is power: the clock is at 1.83 GHz of 2.4, and inputs of zeros take 6.8 ms.  Two
// other arrangements (8 waves in turns, one half multiplying while the other weighs; scores a tile ahead, weights made
// between products) kept the matrix units busier per cycle or not, at a lower clock: 8.5 to 8.9 ms.  64 columns
// multiply half as much for the same exponentials: 8 x 4096 tokens, 16 heads, both ways: 0.69 ms, 800 TFLOP/s.
//
// Few rows (a single token of each text) take parts of the keys, a workgroup each, and a second kernel joins them: five
// texts of 67177 keys together 56 us, 4.9 TB/s, and 5 to join.
#include "attention.h"

namespace vh {
namespace attn {
namespace {

struct FwdArgs {
    Heads q, k, v, out;
    float *lse;
    Packed rows, keys;
    Group group;
    int heads, kv_heads, dim;
    bool causal;
    float scale;
    int splits;     // parts of the keys, each a workgroup; more than one leave `part`, which k_attn_join or k_attn_join_few adds up
    float *part;    // [split][token][head][DP]: outputs over their row's own m
    float2 *stats;  // [split][token][head]: m, l
    uint32_t first;  // workgroup of this launch
};

constexpr int kBM = 128;
// Parts of a row that its own few threads join, all loaded at once; more of them take a workgroup a row (18 parts of 160 rows:
// 15.7 us by a loop of the row's threads, 5 by a workgroup; 2 parts of 98304 rows: 103 by a workgroup each).
constexpr int kFew = 8;

// Keys of a tile: 64, or 32 where they have 32 bits (two buffers of K and V of 128 columns in 64 KB, two workgroups a CU).
template <class T>
constexpr int kBN = sizeof(T) == 2 ? 64 : 32;

// Added to the exponents of float16's p, so that weights of 2^-20 of the largest still have all their bits: p <= 2^8
// (see above) times this stays below 2^15.
template <class T>
constexpr float kShift = std::is_same<T, half_t>::value ? 6.f : 0.f;

// Waves of a SIMD that the loop's registers allow. Without a bound the rare second pass takes more of them: 92 -> 130 us for 256
// texts of 16 to 512 tokens in 64 columns.
template <class T, int DP>
constexpr int kWaves = sizeof(T) == 4 ? (DP <= 32 ? 5 : DP <= 64 ? 3 : 2) : DP <= 32 ? 5 : DP <= 64 ? 4 : DP <= 96 ? 3 : 2;

template <class T, int DP, bool DMA>
__global__ __launch_bounds__(256, (kWaves<T, DP>)) void k_attn_forward(FwdArgs a) {
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
    // the last tile of a sequence first: it sees the most keys
    const int row0 = ((n + kBM - 1) / kBM - 1 - at.tile) * kBM;

    // this lane's row, and how many keys it sees
    const int r = row0 + wave * 32 + (lane & 31), rc = min(r, n - 1);
    const int token = a.group.token(rc), head = kh * a.group.size + rc - token * a.group.size;
    const int64_t row = rows.begin + token;
    const int shift = keys.len - rows.len + 1;
    const int sees = a.causal ? min(keys.len, max(0, token + shift)) : keys.len;
    // how many the workgroup sees, and its part of them; what all rows of the wave see, and any of them
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

    frag q[KS];
    {
        const T *p = (const T *)(a.q.data + row * (int64_t)a.q.token + (int64_t)head * a.q.head);
        const bool neg = a.scale < 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const auto x = load_row<VEC>(p, (2 * ks + half) * VEC, a.dim);
#pragma unroll
            for (int e = 0; e < VEC; ++e) q[ks][e] = neg ? -x.v[e] : x.v[e];
        }
    }
    const float c = fmaxf(fabsf(a.scale) * kLog2e, 1.2e-38f);  // s = 0 of a zero scale, and -inf of what is not seen

    floatx16_t o[DT] = {};
    float m = -INFINITY, l = 0.f;
    auto tile = [&](int t, auto careful) {
        tiles_ready();
        const int buf = (t - t0) & 1;
        if (t + 1 < t1) load(t + 1, buf ^ 1);
        const int key0 = t * BN;
        if (key0 >= any) return;

        floatx16_t s[NS];
#pragma unroll
        for (int j = 0; j < NS; ++j) s[j] = mma_rows<T, RB>(lds[buf][0], 32 * j, q, lane);
        const bool masked = key0 + BN > all;
        if (masked) {
            const int left = sees - key0 - 4 * half;
#pragma unroll
            for (int j = 0; j < NS; ++j)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (32 * j + row_of(i) >= left) s[j][i] = -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < NS; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[j][i]);
        top = half_max(top) * c;
        const bool grown = top > m + 8.f;  // a row's own matter: others of its wave may see keys that it does not
        if (__any(grown)) {
            const float next = grown ? top : m;
            const float f = __builtin_amdgcn_exp2f(m - (next == -INFINITY ? 0.f : next));
            m = next;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= f;
        }
        const float base = kShift<T> - (m == -INFINITY ? 0.f : m);
        float sum[4] = {};
#pragma unroll
        for (int j = 0; j < NS; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[j][i] = __builtin_amdgcn_exp2f(fmaf(s[j][i], c, base));
                sum[i % 4] += s[j][i];
            }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            frag p[kOps<T>];
            to_operand<T>(s[j], p);
            if constexpr (decltype(careful)::value) {
                if (masked) {
                    const int left = sees - key0 - 4 * half;
                    mma_cols_masked<T, RB>(lds[buf][1], 32 * j, p, o, lane, [&](int i) { return 32 * j + row_of(i) < left; });
                    continue;
                }
            }
            mma_cols<T, RB>(lds[buf][1], 32 * j, p, o, lane);
        }
    };
    for (int t = t0; t < t1; ++t) tile(t, std::false_type());
    if (__syncthreads_or(not_finite(o) != 0.f)) {
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = floatx16_t{};
        m = -INFINITY;
        l = 0.f;
        if (t0 < t1) load(t0, 0);
        for (int t = t0; t < t1; ++t) tile(t, std::true_type());
    }
    if (r >= n) return;
    l = half_sum(l);
    const int64_t at_row = row * a.heads + head;
    if (a.splits > 1) {
        const int64_t i = ((int64_t)split * a.rows.tokens * a.heads) + at_row;
        if (half == 0) a.stats[i] = make_float2(m, l);
        if (l != 0.f) store_cols<float, DT>(a.part + i * DP, o, DP, lane, [](float x) { return x; });
        return;
    }
    const float f = l == 0.f ? 0.f : 1.f / l;
    if (a.lse && half == 0) a.lse[at_row] = (m - kShift<T> + __builtin_amdgcn_logf(l)) * kLn2;
    store_cols<T, DT>((T *)(a.out.data + row * (int64_t)a.out.token + (int64_t)head * a.out.head), o, a.dim, lane,
                      [&](float x) { return x * f; });
}

// A row's parts: its largest m, and their outputs and sums over it.  For few parts; DP / 4 threads a row.
template <class T, int DP>
__global__ __launch_bounds__(256) void k_attn_join_few(FwdArgs a) {
    constexpr int L = DP / 4, G = kRowsOf256<DP>;
    const int64_t all = a.rows.tokens * a.heads, i = (int64_t)blockIdx.x * G + threadIdx.x / L;
    if (threadIdx.x >= G * L || i >= all) return;
    const int e = threadIdx.x % L * 4;
    float2 st[kFew];
    Pack<float, 4> p[kFew];
    float m = -INFINITY;
#pragma unroll
    for (int s = 0; s < kFew; ++s) {
        st[s] = s < a.splits ? a.stats[s * all + i] : make_float2(-INFINITY, 0.f);
        if (s < a.splits) p[s] = load_any<4>(a.part + (s * all + i) * DP + e);  // of no meaning where the part saw no key
        m = fmaxf(m, st[s].x);
    }
    float l = 0.f, o[4] = {};
#pragma unroll
    for (int s = 0; s < kFew; ++s) {
        if (st[s].y == 0.f) continue;
        const float f = __builtin_amdgcn_exp2f(st[s].x - m);
        l = fmaf(st[s].y, f, l);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = fmaf(p[s].v[k], f, o[k]);
    }
    const int64_t token = i / a.heads, head = i % a.heads;
    const float f = l == 0.f ? 0.f : 1.f / l;
    if (a.lse && e == 0) a.lse[i] = (m - kShift<T> + __builtin_amdgcn_logf(l)) * kLn2;
    Pack<T, 4> v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v.v[k] = (T)(o[k] * f);
    if (e < a.dim) store_row<4>((T *)(a.out.data + token * (int64_t)a.out.token + head * (int64_t)a.out.head), e, a.dim, v);
}

// The same for many parts, a workgroup a row: its largest m, and the parts' outputs and sums over it.  Lanes hold the parts' weights, and
// every G-th part goes to another group of threads.
template <class T, int DP>
__global__ __launch_bounds__(256) void k_attn_join(FwdArgs a) {
    constexpr int L = DP / 4, G = kRowsOf256<DP>;
    __shared__ float weight[kMaxSplits];
    __shared__ bool seen[kMaxSplits];
    __shared__ __attribute__((aligned(16))) float sums[G][DP];
    const int64_t all = a.rows.tokens * a.heads, i = blockIdx.x;
    const int lane = threadIdx.x & 63, g = threadIdx.x / L, e = threadIdx.x % L * 4;
    const float2 st = lane < a.splits ? a.stats[lane * all + i] : make_float2(-INFINITY, 0.f);
    float m = st.x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    const float w = st.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(st.x - m);  // 0: a part that saw no key
    const float l = lane_sum<64>(st.y * w);
    if (threadIdx.x < a.splits) {
        weight[threadIdx.x] = w;
        seen[threadIdx.x] = st.y != 0.f;
    }
    __syncthreads();
    float o[4] = {};
    if (g < G) {
#pragma unroll 4
        for (int s = g; s < a.splits; s += G) {
            const float f = weight[s];
            if (!seen[s]) continue;  // nothing is written there
            const Pack<float, 4> p = load_any<4>(a.part + (s * all + i) * DP + e);
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = fmaf(p.v[k], f, o[k]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) sums[g][e + k] = o[k];
    }
    __syncthreads();
    if (g) return;
#pragma unroll
    for (int q = 1; q < G; ++q)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] += sums[q][e + k];
    const int64_t token = i / a.heads, head = i % a.heads;
    const float f = l == 0.f ? 0.f : 1.f / l;
    if (a.lse && e == 0) a.lse[i] = (m - kShift<T> + __builtin_amdgcn_logf(l)) * kLn2;
    Pack<T, 4> v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v.v[k] = (T)(o[k] * f);
    if (e < a.dim) store_row<4>((T *)(a.out.data + token * (int64_t)a.out.token + head * (int64_t)a.out.head), e, a.dim, v);
}

template <class T, int DP>
int launch(FwdArgs a, bool dma, int64_t grid, hipStream_t s) {
    each_launch(grid, 256, [&](int64_t first, uint32_t n) {
        a.first = (uint32_t)first;
        if (dma)
            k_attn_forward<T, DP, true><<<n, 256, 0, s>>>(a);
        else
            k_attn_forward<T, DP, false><<<n, 256, 0, s>>>(a);
    });
    if (a.splits > kFew)
        k_attn_join<T, DP><<<(uint32_t)(a.rows.tokens * a.heads), 256, 0, s>>>(a);
    else if (a.splits > 1)
        k_attn_join_few<T, DP><<<(uint32_t)ceil_div(a.rows.tokens * a.heads, kRowsOf256<DP>), 256, 0, s>>>(a);
    return launch_status("attention launch");
}
template <class T>
int launch(const FwdArgs &a, bool dma, int64_t grid, hipStream_t s) {
    switch (padded(a.dim)) {
        case 32: return launch<T, 32>(a, dma, grid, s);
        case 64: return launch<T, 64>(a, dma, grid, s);
        case 96: return launch<T, 96>(a, dma, grid, s);
        default: return launch<T, 128>(a, dma, grid, s);
    }
}

}  // namespace

int check_shape(int dtype, const Shape &s, const int64_t *offsets, const int64_t *key_offsets, float scale) {
    if (!dtype_known(dtype)) return set_error(VHIP_ERR_INVALID_CONFIG, "unknown element type " + std::to_string(dtype));
    if (s.dim == 0 || s.dim > 128) return set_error(VHIP_ERR_INVALID_CONFIG, "dim must be in [1, 128]");
    if (s.heads == 0 || s.kv_heads == 0 || s.heads > 65536 || s.heads % s.kv_heads)
        return set_error(VHIP_ERR_INVALID_CONFIG, "heads must be a multiple of kv_heads, in [1, 65536]");
    if (!offsets) return set_error(VHIP_ERR_INVALID_CONFIG, "offsets are null");
    if (!key_offsets && s.key_tokens != s.tokens)
        return set_error(VHIP_ERR_INVALID_CONFIG, "without key_offsets there are as many keys as queries");
    if (!(fabsf(scale) <= 1e30f)) return set_error(VHIP_ERR_INVALID_CONFIG, "scale must be finite, of 1e30 at most");
    if (s.tokens > (1u << 30) || s.key_tokens > (1u << 30) || s.sequences > (1u << 28) || s.tokens * s.heads > (1u << 30))
        return set_error(VHIP_ERR_INVALID_CONFIG, "too many rows or sequences");
    return VHIP_OK;
}

int check_heads(const char *name, const vhip_heads *a, int dtype, size_t tokens, size_t heads, size_t dim) {
    const std::string who(name);
    if (!a || (tokens && !a->data)) return set_error(VHIP_ERR_INVALID_CONFIG, who + " is null");
    if ((uintptr_t)a->data % dtype_size(dtype)) return set_error(VHIP_ERR_INVALID_CONFIG, who + " is not aligned to its type");
    if ((tokens > 1 && a->token > kMmMaxLd) || (heads > 1 && a->head > ((size_t)1 << 40)))
        return set_error(VHIP_ERR_INVALID_CONFIG, who + ": tokens are more than 2^23 elements apart, or heads 2^40");
    if ((tokens > 1 && a->token < dim) || (heads > 1 && a->head < dim) ||
        (tokens > 1 && heads > 1 && a->token < (heads - 1) * a->head + dim && a->head < (tokens - 1) * a->token + dim))
        return set_error(VHIP_ERR_INVALID_CONFIG, who + ": rows overlap");
    return VHIP_OK;
}

bool whole_chunks(const vhip_heads *a, int dtype, size_t dim) {
    const size_t s = dtype_size(dtype);
    return aligned16(a->data) && a->token * s % 16 == 0 && a->head * s % 16 == 0 && dim * s % 16 == 0;
}

Heads to_heads(const vhip_heads *a, int dtype) {
    const size_t s = dtype_size(dtype);
    return {(char *)a->data, a->token * s, a->head * s};
}

}  // namespace attn
}  // namespace vh

using namespace vh;
using namespace vh::attn;

extern "C" {

size_t vhip_attention_workspace(int dtype, size_t tokens, size_t key_tokens, size_t heads, size_t kv_heads, size_t dim,
                                size_t sequences) {
    if (!kv_heads || !heads || !dtype_known(dtype)) return 0;
    const int n = key_splits(dtype, {tokens, key_tokens, heads, kv_heads, dim, sequences}, kBM);
    return n > 1 ? n * tokens * heads * (padded(dim) * sizeof(float) + sizeof(float2)) : 0;
}

int vhip_attention(int ordinal, int dtype, const vhip_heads *q, const vhip_heads *k, const vhip_heads *v, size_t tokens,
                   size_t key_tokens, size_t heads, size_t kv_heads, size_t dim, const int64_t *offsets,
                   const int64_t *key_offsets, size_t sequences, int causal, float scale, const vhip_heads *out, float *lse,
                   void *workspace, size_t workspace_bytes, void *stream) {
    clear_error();
    const Shape sh{tokens, key_tokens, heads, kv_heads, dim, sequences};
    VH_CHECK(check_shape(dtype, sh, offsets, key_offsets, scale));
    VH_CHECK(check_heads("q", q, dtype, tokens, heads, dim));
    VH_CHECK(check_heads("k", k, dtype, key_tokens, kv_heads, dim));
    VH_CHECK(check_heads("v", v, dtype, key_tokens, kv_heads, dim));
    VH_CHECK(check_heads("out", out, dtype, tokens, heads, dim));
    const int splits = key_splits(dtype, sh, kBM);
    if (splits > 1 && (!workspace || workspace_bytes < vhip_attention_workspace(dtype, tokens, key_tokens, heads, kv_heads, dim, sequences) ||
                       !aligned16(workspace)))
        return set_error(VHIP_ERR_INVALID_CONFIG, "the workspace is smaller than vhip_attention_workspace() or not aligned");
    const int64_t grid = slot_count(tokens, sequences, heads / kv_heads, kBM) * (int64_t)kv_heads * splits;
    if (grid > 0x7fffffff) return set_error(VHIP_ERR_INVALID_CONFIG, "too many rows or sequences");
    CallDevice dev;
    VH_CHECK(dev.enter(ordinal));
    if (tokens == 0) return VHIP_OK;
    FwdArgs a{to_heads(q, dtype), to_heads(k, dtype), to_heads(v, dtype), to_heads(out, dtype), lse,
              {offsets, (int64_t)tokens, (int)sequences},
              {key_offsets ? key_offsets : offsets, (int64_t)key_tokens, (int)sequences},
              to_group(heads, kv_heads), (int)heads, (int)kv_heads, (int)dim, causal != 0, scale, splits, (float *)workspace,
              (float2 *)((float *)workspace + (size_t)splits * tokens * heads * padded(dim)), 0};
    const bool dma = whole_chunks(k, dtype, dim) && whole_chunks(v, dtype, dim);
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case VHIP_DTYPE_F32: return launch<float>(a, dma, grid, s);
        case VHIP_DTYPE_F16: return launch<half_t>(a, dma, grid, s);
        default: return launch<bf16_t>(a, dma, grid, s);
    }
}

}  // extern "C"
