// head_norm.hip -- norms of queries and keys for each head with the rotation by position, and their gradients.
//
//   r = 1 / sqrt(mean x^2 + eps),  n = x r w;  pair i of a row (a, b) turns by t_i = position frequency_i:
//   a' = a cos t - b sin t,  b' = a sin t + b cos t  (columns past the pairs stay as they are)
//   backward: dn = dy turned back,  xh = x r,  u = dn w:  dx = r (u - xh mean(u xh)),  dw = sum over rows of dn xh
//
// Both passes are bound by memory: a row is read once into the registers of a few lanes, two vectors each. A lane that turns
// pairs holds both columns of them (pairs of halves: a vector of the first half and its counterpart of the second; neighbouring
// pairs: two vectors one after the other), so nothing is exchanged but the row's sums; the columns behind the pairs have lanes of
// their own. A workgroup takes a few tokens and makes their cosines and sines once in LDS, for all heads; some of its
// waves have the queries, the others the keys, in proportion to their heads.
//
// 16384 tokens of 32 + 8 heads of 128 in bfloat16: 69 us, 4.9 TB/s.  Backward, 8191 tokens of 16 + 4 heads of 80 in float16: 28 us
// (2.8 TB/s: 80 columns fill 10 of the 16 vectors of a row's 8 lanes) and 4.5 for the sums.
//
// Angles are products in 64 bits, taken modulo a quarter turn there: at position 10^6 a 32-bit product is off by 0.03.
// What is left, at most pi / 4, goes into the Taylor polynomials of sine and cosine in 32 bits, whose remainders
// (pi / 4)^11 / 11! and (pi / 4)^12 / 12! are below half a unit of them.
//
// The weights' gradients are sums over all rows: a lane keeps its columns' sums in registers over its rows, a workgroup leaves
// those of its waves in a row of the workspace, and a second kernel adds the rows in a fixed order.
#include "train_common.h"

namespace vh {
namespace {

// Tokens of a turn, at most. Forward: 16384 tokens of 40 heads of 128 in bfloat16 take 72 us by 2, 75 by 4, 84 by 8. Backward a
// workgroup ends with a sum over its rows: 8191 tokens of 20 heads of 80 in float16 take 41 us by 2, 36 by 8.
constexpr int kTokForward = 2, kTokBackward = 8;
constexpr int kMaxDim = 256, kMaxPairs = kMaxDim / 2;  // 34 lanes of 32-bit values at most: a row is a wave's
constexpr size_t kMaxParts = 1024;  // workgroups of the backward pass: rows of partial sums

struct Side {
    const char *x, *dy;  // dy: backward
    char *out;           // y, or dx
    size_t x_token, x_head, dy_token, dy_head, out_token, out_head;  // bytes
    const void *weight;
    int heads;
};

struct HeadArgs {
    Side side[2];  // queries, keys
    const int64_t *positions;
    const float *frequencies;
    float *part;  // backward: [workgroup][2][dim]
    int64_t tokens;
    int dim, pairs, lanes_log2, at_once;  // lanes of a row; tokens of a turn
    int key_waves;                        // of 4
    bool f32_params;
    float eps;
    int64_t first;  // token of this launch, forward
};

// A lane's columns of a row, two vectors: of pairs (lanes below ceil(pairs / VEC)), or of what is not turned.
template <class T, bool NEAR>
struct Columns {
    static constexpr int VEC = 16 / (int)sizeof(T);
    typedef float Values[2][VEC];
    int c[2], end[2];
    int first_pair, count;  // of the lane's pairs
    __device__ __forceinline__ Columns(int t, int dim, int pairs) {
        const int turning = (pairs + VEC - 1) / VEC, v = t * VEC;
        if (t < turning) {
            c[0] = NEAR ? 2 * v : v;
            c[1] = NEAR ? 2 * v + VEC : pairs + v;
            end[0] = NEAR ? 2 * pairs : pairs;
            end[1] = 2 * pairs;
            first_pair = v;
            count = min(VEC, pairs - v);
        } else {
            c[0] = 2 * pairs + 2 * (t - turning) * VEC;
            c[1] = c[0] + VEC;
            end[0] = end[1] = dim;
            first_pair = count = 0;
        }
    }
    template <class U>
    __device__ __forceinline__ void load(Values &v, const U *row) const {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            Pack<U, VEC> p;
#pragma unroll
            for (int e = 0; e < VEC; ++e) p.v[e] = (U)0.f;
            if (c[s] < end[s]) p = load_row<VEC>(row, c[s], end[s]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[s][e] = (float)p.v[e];
        }
    }
    __device__ __forceinline__ void store(T *row, const Values &v) const {
#pragma unroll
        for (int s = 0; s < 2; ++s)
            if (c[s] < end[s]) {
                Pack<T, VEC> p;
#pragma unroll
                for (int e = 0; e < VEC; ++e) p.v[e] = (T)v[s][e];
                store_row<VEC>(row, c[s], end[s], p);
            }
    }
    // Turns the lane's pairs by cs (cosines and sines of the row's token), or back.
    template <bool BACK>
    __device__ __forceinline__ void turn(Values &v, const float2 *cs) const {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            if (e >= count) break;
            const float2 p = cs[first_pair + e];
            const float s = BACK ? -p.y : p.y;
            float &x = NEAR ? v[2 * e / VEC][2 * e % VEC] : v[0][e], &y = NEAR ? v[2 * e / VEC][2 * e % VEC + 1] : v[1][e];
            const float a = x, b = y;
            x = a * p.x - b * s;
            y = a * s + b * p.x;
        }
    }
};

__device__ __forceinline__ float2 cos_sin(int64_t position, float frequency) {
    const double a = (double)position * (double)frequency;
    const double k = rint(a * 0.63661977236758134308);  // quarter turns
    // past 2^52 a product has no angle left
    const float r = fabs(a) <= 4503599627370496. ? (float)fma(-k, 6.123233995736766036e-17, fma(-k, 1.57079632679489661923, a)) : NAN;
    const int q = (int)((long long)k & 3);
    const float z = r * r;
    const float s = r + r * z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880))));
    const float c = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 + z * (-1.f / 3628800)))));
    const float x = q & 1 ? s : c, y = q & 1 ? c : s;
    return make_float2(q == 1 || q == 2 ? -x : x, q >= 2 ? -y : y);
}

__device__ __forceinline__ void make_turns(const HeadArgs &a, int64_t tok0, int count, float2 (*cs)[kMaxPairs]) {
    for (int i = threadIdx.x; i < count * a.pairs; i += 256) {
        const int t = i / a.pairs, p = i - t * a.pairs;
        cs[t][p] = cos_sin(a.positions[tok0 + t], a.frequencies[p]);
    }
}

__device__ __forceinline__ float row_lanes_sum(float x, int lanes_log2) {
    for (int l = 0; l < lanes_log2; ++l) x += __shfl_xor(x, 1 << l, 64);
    return x;
}

// A row's squares fit 32 bits where their mean is far from both ends of these.  Other rows (values from about 1e18 on; below
// 3e-14 where eps is as small as their squares) are taken in units of 2^k, with which the larger of their largest value and
// sqrt(eps) is near 1: x and the row's mean are replaced by theirs in these units, and the scale that comes of it is 2^k too large.
__device__ __forceinline__ bool ordinary(float mean) { return mean > 0x1p-90f && mean < 0x1p120f; }
template <int VEC>
__device__ __forceinline__ int to_units(float (&x)[2][VEC], float &mean, const HeadArgs &a, float inv) {
    float top = 0.f, sum = 0.f;
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int e = 0; e < VEC; ++e) top = fmaxf(top, fabsf(x[v][e]));
    for (int l = 0; l < a.lanes_log2; ++l) top = fmaxf(top, __shfl_xor(top, 1 << l, 64));
    int k = top > 0.f ? __builtin_amdgcn_frexp_expf(top) : -200;
    if (a.eps > 0.f) k = max(k, __builtin_amdgcn_frexp_expf(a.eps) >> 1);
    if (ordinary(mean)) k = 0;
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            x[v][e] = ldexpf(x[v][e], -k);
            sum = fmaf(x[v][e], x[v][e], sum);
        }
    sum = row_lanes_sum(sum, a.lanes_log2);
    if (!ordinary(mean)) mean = fmaf(sum, inv, ldexpf(a.eps, -2 * k));
    return k;
}

// Which side a wave has, and its place among that side's.
struct Waves {
    int side, slot, slots, t;
    __device__ __forceinline__ explicit Waves(const HeadArgs &a) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, rows = 64 >> a.lanes_log2;
        side = wave >= 4 - a.key_waves;
        slot = (side ? wave - (4 - a.key_waves) : wave) * rows + (lane >> a.lanes_log2);
        slots = (side ? a.key_waves : 4 - a.key_waves) * rows;
        t = lane & ((1 << a.lanes_log2) - 1);
    }
};

template <class T, bool NEAR>
__device__ __forceinline__ void load_weight(typename Columns<T, NEAR>::Values &w, const Columns<T, NEAR> &cols, const HeadArgs &a,
                                            const void *weight) {
    if (!weight) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int e = 0; e < Columns<T, NEAR>::VEC; ++e) w[s][e] = 1.f;
    } else if (a.f32_params) {
        cols.load(w, (const float *)weight);
    } else {
        cols.load(w, (const T *)weight);
    }
}

template <class T, bool NEAR>
__global__ __launch_bounds__(256) void k_head_forward(HeadArgs a) {
    typedef Columns<T, NEAR> Cols;
    constexpr int VEC = Cols::VEC;
    __shared__ float2 cs[kTokForward][kMaxPairs];
    const Waves at(a);
    const Cols cols(at.t, a.dim, a.pairs);
    const Side &side = a.side[at.side];
    const int64_t tok0 = a.first + (int64_t)blockIdx.x * a.at_once;
    const int count = (int)min((int64_t)a.at_once, a.tokens - tok0);
    typename Cols::Values w;
    load_weight<T, NEAR>(w, cols, a, side.weight);
    make_turns(a, tok0, count, cs);
    __syncthreads();
    const float inv = 1.f / (float)a.dim;
    for (int i = at.slot; i < count * side.heads; i += at.slots) {
        const int k = i / side.heads, h = i - k * side.heads;
        typename Cols::Values x;
        cols.load(x, (const T *)(side.x + (tok0 + k) * side.x_token + h * side.x_head));
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum = fmaf(x[v][e], x[v][e], sum);
        float mean = fmaf(row_lanes_sum(sum, a.lanes_log2), inv, a.eps);
        if (__any(!ordinary(mean))) to_units<VEC>(x, mean, a, inv);
        const float r = 1.f / sqrtf(mean);
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[v][e] *= r * w[v][e];
        cols.template turn<false>(x, cs[k]);
        cols.store((T *)(side.out + (tok0 + k) * side.out_token + h * side.out_head), x);
    }
}

template <class T, bool NEAR>
__global__ __launch_bounds__(256) void k_head_backward(HeadArgs a) {
    typedef Columns<T, NEAR> Cols;
    constexpr int VEC = Cols::VEC;
    __shared__ float2 cs[kTokBackward][kMaxPairs];
    __shared__ float sums[4][kMaxDim];
    const Waves at(a);
    const Cols cols(at.t, a.dim, a.pairs);
    const Side &side = a.side[at.side];
    const float inv = 1.f / (float)a.dim;
    typename Cols::Values w, dw = {};
    load_weight<T, NEAR>(w, cols, a, side.weight);
    for (int64_t tok0 = (int64_t)blockIdx.x * a.at_once; tok0 < a.tokens; tok0 += (int64_t)gridDim.x * a.at_once) {
        const int count = (int)min((int64_t)a.at_once, a.tokens - tok0);
        __syncthreads();
        make_turns(a, tok0, count, cs);
        __syncthreads();
        for (int i = at.slot; i < count * side.heads; i += at.slots) {
            const int k = i / side.heads, h = i - k * side.heads;
            typename Cols::Values x, g;
            cols.load(x, (const T *)(side.x + (tok0 + k) * side.x_token + h * side.x_head));
            cols.load(g, (const T *)(side.dy + (tok0 + k) * side.dy_token + h * side.dy_head));
            cols.template turn<true>(g, cs[k]);
            float sum = 0.f, dot = 0.f;
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
                for (int e = 0; e < VEC; ++e) sum = fmaf(x[v][e], x[v][e], sum);
            float mean = fmaf(row_lanes_sum(sum, a.lanes_log2), inv, a.eps);
            int units = 0;
            if (__any(!ordinary(mean))) units = to_units<VEC>(x, mean, a, inv);
            const float r = 1.f / sqrtf(mean);
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    x[v][e] *= r;
                    dw[v][e] = fmaf(g[v][e], x[v][e], dw[v][e]);
                    g[v][e] *= w[v][e];
                    dot = fmaf(x[v][e], g[v][e], dot);  // of values near 1, so that it is as large as u
                }
            const float m = row_lanes_sum(dot, a.lanes_log2) * inv;  // mean of u xh
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
                for (int e = 0; e < VEC; ++e) x[v][e] = r * (g[v][e] - x[v][e] * m);
            if (__any(units))
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) x[v][e] = ldexpf(x[v][e], -units);
            cols.store((T *)(side.out + (tok0 + k) * side.out_token + h * side.out_head), x);
        }
    }
    if (!a.part) return;
    // the sums of the workgroup's rows: over a wave's rows by exchange, then over the waves of a side
    const int lanes = 1 << a.lanes_log2;
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            for (int o = lanes; o < 64; o <<= 1) dw[v][e] += __shfl_xor(dw[v][e], o, 64);
    if ((threadIdx.x & 63) < lanes)
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (cols.c[v] + e < cols.end[v]) sums[threadIdx.x >> 6][cols.c[v] + e] = dw[v][e];
    __syncthreads();
    float *part = a.part + (size_t)blockIdx.x * 2 * a.dim;
    for (int c = threadIdx.x; c < 2 * a.dim; c += 256) {
        const int s = c >= a.dim, col = c - s * a.dim;
        float x = 0.f;
        for (int w = s ? 4 - a.key_waves : 0; w < (s ? 4 : 4 - a.key_waves); ++w) x += sums[w][col];
        part[c] = x;
    }
}

// Adds the workgroups' rows in a fixed order: 32 of the 2 dim columns a workgroup, every 32nd row a group of threads.
template <class P>
__global__ __launch_bounds__(1024) void k_head_sums(const float *part, int parts, int dim, P *dq, P *dk) {
    __shared__ float sums[32][33];
    const int g = threadIdx.x >> 5, l = threadIdx.x & 31, c = blockIdx.x * 32 + l;
    float s = 0.f;
    if (c < 2 * dim) {
#pragma unroll 4
        for (int p = g; p < parts; p += 32) s += part[(size_t)p * 2 * dim + c];
    }
    sums[g][l] = s;
    __syncthreads();
    s = sums[l][g];  // group g adds column g's
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) s += __shfl_xor(s, o, 32);
    const int at = blockIdx.x * 32 + g;
    P *out = at < dim ? dq : dk;
    if (l == 0 && at < 2 * dim && out) out[at < dim ? at : at - dim] = (P)s;
}

// Lanes of a row: a power of two of those that its pairs and its other columns take.
inline int row_lanes_log2(size_t dim, size_t rotary, int dtype) {
    const size_t vec = 16 / dtype_size(dtype);
    const size_t lanes = (rotary / 2 + vec - 1) / vec + (dim - rotary + 2 * vec - 1) / (2 * vec);
    static_assert(kMaxDim / 8 + 2 <= 64, "a row's lanes are of one wave");
    return lanes_log2(lanes);
}
// Tokens of a turn: fewer than `most` where there are not enough for two turns on every CU.
inline int tokens_at_once(size_t tokens, int most) {
    const size_t n = tokens / 512;
    return n < 1 ? 1 : n > (size_t)most ? most : (int)n;
}
// Waves of 4 that have the keys: their share of the heads, but one at least for either side that has any.
inline int key_waves(size_t heads, size_t kv_heads) {
    if (!kv_heads || !heads) return kv_heads ? 4 : 0;
    const size_t n = (4 * kv_heads + (heads + kv_heads) / 2) / (heads + kv_heads);
    return n < 1 ? 1 : n > 3 ? 3 : (int)n;
}
inline size_t part_count(size_t tokens, int at_once) {
    const size_t n = (tokens + at_once - 1) / at_once;
    return n < kMaxParts ? n : kMaxParts;
}

int check_side(const char *name, const vhip_heads *a, int dtype, size_t tokens, size_t heads, size_t dim) {
    const std::string who(name);
    if (!a || (tokens && heads && !a->data)) return set_error(VHIP_ERR_INVALID_CONFIG, who + " is null");
    if (!tokens || !heads) return VHIP_OK;
    if ((uintptr_t)a->data % dtype_size(dtype)) return set_error(VHIP_ERR_INVALID_CONFIG, who + " is not aligned to its type");
    if (a->token > ((size_t)1 << 40) || a->head > ((size_t)1 << 40))
        return set_error(VHIP_ERR_INVALID_CONFIG, who + ": rows are more than 2^40 elements apart");
    if ((tokens > 1 && a->token < dim) || (heads > 1 && a->head < dim) ||
        (tokens > 1 && heads > 1 && a->token < (heads - 1) * a->head + dim && a->head < (tokens - 1) * a->token + dim))
        return set_error(VHIP_ERR_INVALID_CONFIG, who + ": rows overlap");
    return VHIP_OK;
}

int check_common(int dtype, int param_dtype, size_t tokens, size_t heads, size_t kv_heads, size_t dim, size_t rotary,
                 const int64_t *positions, const float *frequencies, float eps) {
    if (!dtype_known(dtype)) return set_error(VHIP_ERR_INVALID_CONFIG, "unknown element type " + std::to_string(dtype));
    if (param_dtype != dtype && param_dtype != VHIP_DTYPE_F32)
        return set_error(VHIP_ERR_INVALID_CONFIG, "parameters are of the rows' type or f32");
    if (dim == 0 || dim > kMaxDim) return set_error(VHIP_ERR_INVALID_CONFIG, "dim must be in [1, 256]");
    if (rotary > dim || rotary % 2) return set_error(VHIP_ERR_INVALID_CONFIG, "rotary must be even and at most dim");
    if (heads + kv_heads == 0 || heads > 65536 || kv_heads > 65536)
        return set_error(VHIP_ERR_INVALID_CONFIG, "heads must be in [1, 65536]");
    if (tokens > (1u << 30)) return set_error(VHIP_ERR_INVALID_CONFIG, "too many tokens");
    if (rotary && ((tokens && !positions) || !frequencies)) return set_error(VHIP_ERR_INVALID_CONFIG, "positions or frequencies are null");
    if (!(eps >= 0.f)) return set_error(VHIP_ERR_INVALID_CONFIG, "eps must be >= 0");
    return VHIP_OK;
}

Side to_side(int dtype, const vhip_heads *x, const vhip_heads *dy, const vhip_heads *out, const void *weight, size_t heads) {
    const size_t s = dtype_size(dtype);
    return {(const char *)x->data, dy ? (const char *)dy->data : nullptr, (char *)out->data,
            x->token * s, x->head * s, dy ? dy->token * s : 0, dy ? dy->head * s : 0, out->token * s, out->head * s, weight, (int)heads};
}

template <class T>
int forward(HeadArgs a, bool near, hipStream_t s) {
    each_launch((a.tokens + a.at_once - 1) / a.at_once, 256, [&](int64_t first, uint32_t n) {
        a.first = first * a.at_once;
        if (near)
            k_head_forward<T, true><<<n, 256, 0, s>>>(a);
        else
            k_head_forward<T, false><<<n, 256, 0, s>>>(a);
    });
    return launch_status("head norm launch");
}

template <class T>
int backward(const HeadArgs &a, bool near, void *dqw, void *dkw, hipStream_t s) {
    const int parts = (int)part_count(a.tokens, a.at_once);
    if (parts) {
        if (near)
            k_head_backward<T, true><<<parts, 256, 0, s>>>(a);
        else
            k_head_backward<T, false><<<parts, 256, 0, s>>>(a);
    }
    if (dqw || dkw) {
        const uint32_t grid = (uint32_t)ceil_div(2 * a.dim, 32);
        if (a.f32_params)
            k_head_sums<float><<<grid, 1024, 0, s>>>(a.part, parts, a.dim, (float *)dqw, (float *)dkw);
        else
            k_head_sums<T><<<grid, 1024, 0, s>>>(a.part, parts, a.dim, (T *)dqw, (T *)dkw);
    }
    return launch_status("head norm launch");
}

}  // namespace
}  // namespace vh

using namespace vh;

extern "C" {

int vhip_qk_norm_rotary(int ordinal, int dtype, int param_dtype, const vhip_heads *q, const vhip_heads *k, size_t tokens,
                        size_t heads, size_t kv_heads, size_t dim, const void *q_weight, const void *k_weight,
                        const int64_t *positions, const float *frequencies, size_t rotary, int interleaved, float eps,
                        const vhip_heads *q_out, const vhip_heads *k_out, void *stream) {
    clear_error();
    VH_CHECK(check_common(dtype, param_dtype, tokens, heads, kv_heads, dim, rotary, positions, frequencies, eps));
    VH_CHECK(check_side("q", q, dtype, tokens, heads, dim));
    VH_CHECK(check_side("k", k, dtype, tokens, kv_heads, dim));
    VH_CHECK(check_side("q_out", q_out, dtype, tokens, heads, dim));
    VH_CHECK(check_side("k_out", k_out, dtype, tokens, kv_heads, dim));
    CallDevice dev;
    VH_CHECK(dev.enter(ordinal));
    if (tokens == 0) return VHIP_OK;
    const int l = row_lanes_log2(dim, rotary, dtype);
    const HeadArgs a{{to_side(dtype, q, nullptr, q_out, q_weight, heads), to_side(dtype, k, nullptr, k_out, k_weight, kv_heads)},
                     positions, frequencies, nullptr, (int64_t)tokens, (int)dim, (int)rotary / 2, l,
                     tokens_at_once(tokens, kTokForward), key_waves(heads, kv_heads), param_dtype == VHIP_DTYPE_F32, eps, 0};
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case VHIP_DTYPE_F32: return forward<float>(a, interleaved, s);
        case VHIP_DTYPE_F16: return forward<half_t>(a, interleaved, s);
        default: return forward<bf16_t>(a, interleaved, s);
    }
}

size_t vhip_qk_norm_rotary_backward_workspace(size_t tokens, size_t dim) {
    return 2 * sizeof(float) * dim * part_count(tokens, 1);
}

int vhip_qk_norm_rotary_backward(int ordinal, int dtype, int param_dtype, const vhip_heads *dq, const vhip_heads *dk,
                                 const vhip_heads *q, const vhip_heads *k, size_t tokens, size_t heads, size_t kv_heads,
                                 size_t dim, const void *q_weight, const void *k_weight, const int64_t *positions,
                                 const float *frequencies, size_t rotary, int interleaved, float eps, const vhip_heads *dq_out,
                                 const vhip_heads *dk_out, void *dq_weight, void *dk_weight, void *workspace,
                                 size_t workspace_bytes, void *stream) {
    clear_error();
    VH_CHECK(check_common(dtype, param_dtype, tokens, heads, kv_heads, dim, rotary, positions, frequencies, eps));
    VH_CHECK(check_side("dq", dq, dtype, tokens, heads, dim));
    VH_CHECK(check_side("dk", dk, dtype, tokens, kv_heads, dim));
    VH_CHECK(check_side("q", q, dtype, tokens, heads, dim));
    VH_CHECK(check_side("k", k, dtype, tokens, kv_heads, dim));
    VH_CHECK(check_side("dq_out", dq_out, dtype, tokens, heads, dim));
    VH_CHECK(check_side("dk_out", dk_out, dtype, tokens, kv_heads, dim));
    if ((dq_weight || dk_weight) && tokens &&
        (!workspace || workspace_bytes < vhip_qk_norm_rotary_backward_workspace(tokens, dim) || ((uintptr_t)workspace & 3)))
        return set_error(VHIP_ERR_INVALID_CONFIG,
                         "the workspace is smaller than vhip_qk_norm_rotary_backward_workspace() or not aligned");
    CallDevice dev;
    VH_CHECK(dev.enter(ordinal));
    const int l = row_lanes_log2(dim, rotary, dtype);
    const HeadArgs a{{to_side(dtype, q, dq, dq_out, q_weight, heads), to_side(dtype, k, dk, dk_out, k_weight, kv_heads)},
                     positions, frequencies, dq_weight || dk_weight ? (float *)workspace : nullptr, (int64_t)tokens, (int)dim,
                     (int)rotary / 2, l, tokens_at_once(tokens, kTokBackward), key_waves(heads, kv_heads), param_dtype == VHIP_DTYPE_F32, eps, 0};
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case VHIP_DTYPE_F32: return backward<float>(a, interleaved, dq_weight, dk_weight, s);
        case VHIP_DTYPE_F16: return backward<half_t>(a, interleaved, dq_weight, dk_weight, s);
        default: return backward<bf16_t>(a, interleaved, dq_weight, dk_weight, s);
    }
}

}  // extern "C"
