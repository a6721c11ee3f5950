// softmax_xent.hip -- softmax cross entropy of rows against every row of a table, and its gradients.
//
//   z_tv = scale <h_t, w_v> + b_v,  lse_t = log sum_v exp z_tv,  loss_t = lse_t - z_{t, y_t}
//   G_tv = c_t scale (exp(z_tv - lse_t) - [v = y_t]),  dh = G W,  dW = G^T h      (c: weights of the rows)
//
// The logits are never kept.  A first product (mm16.h) ends each 128-entry piece of a row's logits in its
// largest value and the sum of exp about it; a small kernel joins the pieces.  For the gradients G comes about
// in one of two ways, and two more products multiply it with the table and with the rows:
//  * a second product makes the same logits again and ends in G;
//  * for wide rows (kStoreDim: a product costs more than a walk through memory) the first product also stores
//    its exps about their piece's largest logit, and a kernel turns them into G where they lie.  In bfloat16
//    they are float16 for that while (11 bits before G's 8; exp_code), which holds them down to 2^-57 of their
//    piece's largest; a tile with smaller ones that a float could hold is marked and made the first way.
// Rows are taken in pieces so that G and the rows' packed copies stay below kPieceBytes; from the second piece
// on the table's gradient is added up in 32 bits. Every sum has a fixed order: results do not depend on timing.
//
// Types. float16 and bfloat16 operands are multiplied as they are; 32-bit ones as pairs of float16 (mm16.h),
// scaled by a power of two that brings the largest finite value to [2^13, 2^14), so that what a plane cannot
// hold is 2^-39 of that value: for the logits a power for each row of h, one for the entries of the table that
// are not out, and their own for those that are far smaller than the largest (kWide; where there are such
// entries G takes their powers before it multiplies the table, k_fold_powers). G is rounded to the operands'
// type (to two planes for 32-bit operands), which is as far as the gradients that are returned are rounded too.
// In float16 (and pairs) each row of G is held times 2^14 / 2^e, where 2^e is the power of two above its largest
// value, c scale (1 - p) at the target: neither small probabilities nor rows of small weight lose their bits.
// For the table's gradient the rows of h take 2^e back, times the power of two that brings the largest of all
// 2^e h to [2^13, 2^14); what a row adds to it is held to 2^-39 of the largest such product. In any type G is
// also divided by the mantissa of c scale: with the same c in every row, as a mean has it, G at a target far
// from learned is then a power of two, where rounding c would have moved every such row's gradient by the same
// 2^-9. The products' epilogues take the factors out.
//
// A row's sum of exps leaves its target out until it is joined: 1 - p at the target, and the loss
// log(1 + sum of the others / the target's), keep their bits where p is nearly one.
//
// What does not count: a row whose target is negative has loss 0 and no part in the gradients, whatever its
// values.  An entry whose bias is -inf is out of the softmax whatever its values.  A row whose target is out, or
// that has nothing left in, has loss +inf and no part in the gradients, whatever its values.  (Where sums over rows
// are made, h is replaced by zeros in rows whose G is zeros.)  A target past the table makes its row's loss and
// gradient NaN, and so the table's gradient, which is a sum over rows.
#include "xent_small.h"

#include <cmath>
#include <cstdlib>
#include <type_traits>

namespace vh {
namespace {

constexpr size_t kPieceBytes = (size_t)4 << 30;  // of G, or of what the loss alone keeps, and of packed rows
constexpr int kGBits = 14;
// Columns from which G is made of stored exps.  A product's way costs 2 (pairs: 6) dim flops a value, the walk's 4
// (8) bytes and a few operations.  4096 rows x 65536, product / walk in us: bfloat16 dim 384 1097 / 1125, 512
// 1207 / 1203, 768 1621 / 1514, 1024 2013 / 1787; 32 bits dim 256 1988 / 1784, 512 3128 / 2660, 1024 5517 / 4460.
// float16 always takes the product: its G would be rounded twice to the 11 bits that the gradients have.
constexpr size_t kStoreDim16 = 512, kStoreDim32 = 256;
inline bool stores_exps(int dtype, size_t dim) {
    return dtype == VHIP_DTYPE_F32 ? dim >= kStoreDim32 : (dtype == VHIP_DTYPE_BF16 && dim >= kStoreDim16);
}

// State of a call on the device.
struct Scalars {
    uint32_t amax_w;  // bits of the largest finite |value| of entries that are not out
    uint32_t wide;    // whether entries have powers of their own
    int least;        // least sum of a row's power (k_ranges) and of its row_power
    float mantissa;   // of weight x scale, in [1, 2)
};

// 14 - e with 2^e > x >= 2^(e-1), so that x times two to it is in [2^13, 2^14); 0 for 0.
__device__ __forceinline__ int unit_power(uint32_t bits) {
    const int e = (int)(bits >> 23) - 126;  // x < 2^e
    if (bits == 0) return 0;
    const int k = kGBits - e;
    return k > 120 ? 120 : (k < -120 ? -120 : k);
}
__device__ __forceinline__ float unit_scale(uint32_t bits) { return ldexpf(1.f, unit_power(bits)); }

// What a row of G is multiplied with is two to this (float16 and pairs: by its value at the target, rowfac's
// second) over the mantissa.  Held so that the row's weight x scale, rowfac's first, does not leave 32 bits.
__device__ __forceinline__ int row_power(float2 fac) {
    const int k = unit_power(__builtin_bit_cast(uint32_t, fac.y) & 0x7fffffffu);
    return min(k, 86 + unit_power(__builtin_bit_cast(uint32_t, fac.x) & 0x7fffffffu));
}
template <bool RANGED>
__device__ __forceinline__ float grad_unit(float2 fac, const Scalars *s) {
    return ldexpf(1.f / s->mantissa, RANGED ? row_power(fac) : 0);
}
constexpr int kNoPower = 1 << 16;  // of a row of zeros, or one that is out
// An entry has a power of its own where its largest value is less than 2^-8 of the table's: values down to 2^-15
// of it keep the 22 bits of a pair.
constexpr int kWide = 8;
__device__ __forceinline__ bool own_power(int own, int common) { return own < kNoPower && own - common > kWide; }

// The call's scalars.  The mantissa is that of the largest weight among the first rows: one that most rows have
// where it matters, and good for any others.
struct InitArgs {
    Scalars *sc;
    const float *weight;
    int rows;
    float scale;
};
__device__ void init_scalars(const InitArgs &a) {
    __shared__ float top[4];
    float m = a.weight ? 0.f : 1.f;
    if (a.weight)
        for (int t = threadIdx.x; t < min(a.rows, 4096); t += 256) {
            const float w = fabsf(a.weight[t]);
            if (w <= 3.4e38f && w > m) m = w;
        }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x != 0) return;
    const float c = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * fabsf(a.scale);
    const uint32_t u = __builtin_bit_cast(uint32_t, c);
    // 1 where c is zero, denormal or infinite
    const bool plain = u >= 0x00800000u && u < 0x7f800000u;
    *a.sc = Scalars{0, 0, 2 * kNoPower, plain ? __builtin_bit_cast(float, (u & 0x007fffffu) | 0x3f800000u) : 1.f};
}
__global__ __launch_bounds__(256) void k_xent_init(InitArgs a) { init_scalars(a); }

__global__ __launch_bounds__(256) void k_clear(uint32_t *p, int n) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = 0;
}

// The power of two of each row of h, unit_power of its largest finite |value| (blockIdx.y 0), and that of the
// table's entries that are not out, with the largest |value| of all that a workgroup sees (1).  One workgroup also
// makes the call's scalars.  Bound by memory: 100000 x 768 floats in 72 us, 4.3 TB/s.
constexpr int kRangeGroups = 1024;
template <class T>
struct RangeArgs {
    const T *h, *table;
    size_t rows, entries, ldh, ldt;
    int *power, *entry_power;
    uint32_t *tops;     // [kRangeGroups]
    const float *bias;  // or null
    int dim, lanes;     // lanes of a row, log2, 6 at most
    InitArgs init;
};
// of a row, in each of its lanes
template <class T>
__device__ __forceinline__ uint32_t largest(const T *x, int dim, int l, int lanes) {
    uint32_t m = 0;
    for (int c = l * 4; c < dim; c += 4 << lanes) {
        const Pack<T, 4> v = load_row<4>(x, c, dim);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t u = __builtin_bit_cast(uint32_t, (float)v.v[e]) & 0x7fffffffu;
            if (u < 0x7f800000u && u > m) m = u;
        }
    }
    for (int o = 1; o < 1 << lanes; o <<= 1) {
        const uint32_t v = __shfl_xor(m, o, 64);
        m = v > m ? v : m;
    }
    return m;
}
template <class T>
__global__ __launch_bounds__(256) void k_ranges(RangeArgs<T> a) {
    const int per = 256 >> a.lanes, l = threadIdx.x & ((1 << a.lanes) - 1);
    const size_t first = (size_t)blockIdx.x * per + (threadIdx.x >> a.lanes), step = (size_t)gridDim.x * per;
    if (blockIdx.y == 0) {
        for (size_t r = first; r < a.rows; r += step) {
            const uint32_t m = largest(a.h + r * a.ldh, a.dim, l, a.lanes);
            if (l == 0) a.power[r] = m ? unit_power(m) : kNoPower;
        }
        if (blockIdx.x == kRangeGroups - 1) init_scalars(a.init);
        return;
    }
    uint32_t m = 0;
    for (size_t r = first; r < a.entries; r += step) {
        const bool out = a.bias && a.bias[r] == -INFINITY;
        const uint32_t v = out ? 0 : largest(a.table + r * a.ldt, a.dim, l, a.lanes);
        if (l == 0) a.entry_power[r] = v ? unit_power(v) : kNoPower;
        m = v > m ? v : m;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t v = __shfl_xor(m, o, 64);
        m = v > m ? v : m;
    }
    __shared__ uint32_t tops[4];
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 4; ++w) m = tops[w] > m ? tops[w] : m;
        a.tops[blockIdx.x] = m;
    }
}
// The largest of k_ranges' workgroups, in each lane of a workgroup.
__device__ __forceinline__ uint32_t largest_of(const uint32_t *tops) {
    __shared__ uint32_t waves[4];
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < kRangeGroups; k += 256) m = max(m, tops[k + threadIdx.x]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) m = max(m, __shfl_xor(m, o, 64));
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = m;
    __syncthreads();
    return max(max(waves[0], waves[1]), max(waves[2], waves[3]));
}

// An operand's 16-bit form: T itself, or pairs (mm16.h) of a float times its scale.
template <class T>
struct Planes {
    typedef T type;
    static constexpr int count = 1;
};
template <>
struct Planes<float> {
    typedef half_t type;
    static constexpr int count = 2;
};

// rows x dim -> rows of kp values (or pairs), zeros past dim and in rows whose bias is -inf.  2^lanes lanes a
// row, 8 values each at a time.  Pairs are scaled by two to their row's power; `tops` (of k_ranges): by that of the
// table's largest value, or the entry's own, of which the call's scalars are told.
template <class T>
__global__ __launch_bounds__(256) void k_pack(const T *x, size_t rows, int dim, size_t ld, typename Planes<T>::type *out,
                                              int kp, int lanes, const int *power, const uint32_t *tops, Scalars *call,
                                              const float *bias) {
    typedef typename Planes<T>::type P;
    constexpr int N = Planes<T>::count;
    const int per = 256 >> lanes, l = threadIdx.x & ((1 << lanes) - 1);
    int common = 0;
    if constexpr (N == 2)
        if (tops) {
            const uint32_t m = largest_of(tops);
            common = unit_power(m);
            if (blockIdx.x == 0 && threadIdx.x == 0) call->amax_w = m;
        }
    for (size_t r = (size_t)blockIdx.x * per + (threadIdx.x >> lanes); r < rows; r += (size_t)gridDim.x * per) {
        const bool keep = !bias || bias[r] != -INFINITY;
        float sc = 1.f;
        if constexpr (N == 2) {
            int k = min(power[r], 120);
            if (tops && !own_power(power[r], common))
                k = common;
            else if (tops && l == 0)
                call->wide = 1;
            sc = ldexpf(1.f, k);
        }
        for (int c = l * 8; c < kp; c += 8 << lanes) {
            Pack<T, 8> v{};
            if (keep) v = load_row<8>(x + r * ld, c, dim);
            Pack<P, 8> hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if constexpr (N == 2) {
                    const float f = v.v[e] * sc;
                    hi.v[e] = (half_t)f;
                    lo.v[e] = (half_t)(f - (float)hi.v[e]);
                } else {
                    hi.v[e] = v.v[e];
                }
            }
            P *o = out + r * kp * N + (N == 2 ? pair_at(c) : c);
            *reinterpret_cast<Pack<P, 8> *>(o) = hi;
            if constexpr (N == 2) *reinterpret_cast<Pack<P, 8> *>(o + 32) = lo;
        }
    }
}
template <class T>
void pack(const T *x, size_t rows, int dim, size_t ld, typename Planes<T>::type *out, int kp, const int *power, const uint32_t *tops,
          Scalars *call, const float *bias, hipStream_t s) {
    const int lanes = lanes_log2(kp / 8);
    const size_t wgs = (rows + (256 >> lanes) - 1) >> (8 - lanes);
    const uint32_t grid = (uint32_t)(wgs < 8192 ? wgs : 8192);
    k_pack<T><<<grid, 256, 0, s>>>(x, rows, dim, ld, out, kp, lanes, power, tops, call, bias);
}

// rows x dim -> dim rows of rp values (or pairs), zeros past rows and where G's row is zeros.  What G's row was
// multiplied with is taken back (see the top).
template <class T>
__global__ __launch_bounds__(256) void k_pack_t(const T *x, size_t rows, int dim, size_t ld,
                                                typename Planes<T>::type *out, size_t rp, const Scalars *sc,
                                                const float2 *rowfac) {
    constexpr bool kRanged = !std::is_same_v<T, bf16_t>;
    __shared__ T tile[64][65];
    const size_t r0 = (size_t)blockIdx.x * 64;
    const int c0 = blockIdx.y * 64, tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const size_t r = r0 + ty + 4 * i;
        const int c = c0 + tx;
        T v = (T)0.f;
        if (r < rows && c < dim) v = x[r * ld + c];
        tile[ty + 4 * i][tx] = v;
    }
    __syncthreads();
    const size_t r = r0 + tx;
    const float2 fac = r < rows ? rowfac[r] : make_float2(0.f, 0.f);
    const bool on = fac.y != 0.f;
    int power = 0;
    if constexpr (kRanged) power = sc->least - row_power(fac);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int c = c0 + ty + 4 * i;
        if (c < dim && r < rp) {
            T v = on ? tile[tx][ty + 4 * i] : (T)0.f;
            if constexpr (kRanged) v = (T)ldexpf((float)v, power);
            if constexpr (Planes<T>::count == 2) {
                const float f = v;
                const half_t h = (half_t)f;
                out[c * rp * 2 + pair_at(r)] = h;
                out[c * rp * 2 + pair_at(r) + 32] = (half_t)(f - (float)h);
            } else {
                out[c * rp + r] = v;
            }
        }
    }
}

// What turns a product's sum into a logit.  SPLIT: of pairs.
template <bool SPLIT>
struct Logits {
    const float *bias;
    const Scalars *sc;
    const int *power, *entry_power;  // of the rows, of the entries
    float scale;
    __device__ __forceinline__ float factor() const { return SPLIT ? scale / unit_scale(sc->amax_w) : scale; }
    // the factor f of row t, if that is one
    __device__ __forceinline__ float of_row(float f, int t, int rows) const {
        if constexpr (SPLIT) return ldexpf(f, t < rows ? -power[t] : 0);
        return f;
    }
    // whether to_logits makes the wave's logits
    __device__ __forceinline__ bool made(int last, int table) const { return bias || last > table; }
};
// Exps in (0, 1] as float16: times 2^15, or those below 2^-28 negative and times 2^43.
__device__ __forceinline__ half_t exp_code(float p) { return (half_t)(p * (p < 0x1p-28f ? -0x1p43f : 0x1p15f)); }
__device__ __forceinline__ float exp_decode(half_t h) { return (float)h * (h < (half_t)0.f ? -0x1p-43f : 0x1p-15f); }
// Arguments of exps that exp_code would cut short, and that are not nothing in 32 bits either.
__device__ __forceinline__ bool exp_cut(float x) { return x < -39.f && x > -104.f; }

// A wave's sums to f (of the row) times them being the logits: where there is a bias, or entries past the
// table, the logits themselves (-inf where an entry is out) and f = 1 for every row.
template <int MB, int NB, bool SPLIT>
__device__ __forceinline__ float to_logits(floatx4_t (&acc)[MB][NB], const Logits<SPLIT> &lg, int m, int n, int rows, int table) {
    const float f = lg.factor();
    const int l = threadIdx.x & 63, q = l >> 4;
    if constexpr (SPLIT) {
        if (lg.sc->wide) {
            const int common = unit_power(lg.sc->amax_w);
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int v = m + 16 * i + 4 * q + e, own = v < table ? lg.entry_power[v] : kNoPower;
                    const int k = own_power(own, common) ? common - own : 0;
#pragma unroll
                    for (int j = 0; j < NB; ++j) acc[i][j][e] = ldexpf(acc[i][j][e], k);
                }
        }
    }
    if (!lg.made(m + 16 * MB, table)) return f;
    float fs[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) fs[j] = lg.of_row(f, n + 16 * j + (l & 15), rows);
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        float b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int v = m + 16 * i + 4 * q + e;
            b[e] = v < table ? (lg.bias ? lg.bias[v] : 0.f) : -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] = b[e] == -INFINITY ? -INFINITY : fmaf(acc[i][j][e], fs[j], b[e]);
    }
    return 1.f;
}

// Epilogue of the first product (A: table, B: rows): a wave's 16 MB entries of each row end in one piece.
// E: the type that the exps are stored in, void: they are not; FINE: of 32-bit operands.
template <class E, bool FINE>
struct StatEpi {
    Logits<FINE> lg;
    float2 *part;  // [piece][rows]: largest logit, sum of exp about it without the target's
    float2 *zt;    // the target's logit less its piece's largest, and that
    const int64_t *target;
    int rows, table;
    E *exps;  // [rows][vp]
    size_t vp;
    uint32_t *marks;  // [tile of N][tile of M]: exps of rows that count and that float16 cannot hold
    int mt;
    template <int MB, int NB>
    __device__ void operator()(floatx4_t (&acc)[MB][NB], int m, int n, const MmPlace &pl, char *lds) const {
        constexpr bool kHalf = std::is_same_v<E, half_t>;
        bool cut = false;
        if (m >= table) return;
        const int l = threadIdx.x & 63, q = l >> 4;
        const bool made = lg.made(m + 16 * MB, table);
        float fw = to_logits(acc, lg, m, n, rows, table);
        if (fw < 0.f) {
            fw = -fw;
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int j = 0; j < NB; ++j) acc[i][j] = -acc[i][j];
        }
        const int piece = m / (16 * MB);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int t = n + 16 * j + (l & 15);
            const bool in = t < rows;
            const float f = made ? 1.f : lg.of_row(fw, t, rows);
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                const floatx4_t a = acc[i][j];
                top = fmaxf(fmaxf(fmaxf(top, a[0]), fmaxf(a[1], a[2])), a[3]);
            }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64)) * f;
            const float about = top == -INFINITY ? 0.f : top;
            // the target's place among this lane's values, past them where it is not here
            const int64_t y = in ? target[t] : -1;
            const int d = y >= m && y < m + 16 * MB && y < table ? (int)(y - m) - 4 * q : -1;
            float sum = 0.f;
            bool wide = false;
            auto add = [&](float &v, bool skip) {
                const float x = fmaf(v, f, -about);
                const float p = FINE ? exp_fine(x) : exp_neg(x);
                if constexpr (kHalf) wide |= exp_cut(x);
                sum += skip ? 0.f : p;
                if (skip) zt[t] = make_float2(x, about);
                return p;
            };
            if (__any(d >= 0)) {
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float v = acc[i][j][e];
                        v = add(v, d == 16 * i + e);
                        if constexpr (!std::is_void_v<E>) acc[i][j][e] = v;
                    }
            } else {
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float v = acc[i][j][e];
                        v = add(v, false);
                        if constexpr (!std::is_void_v<E>) acc[i][j][e] = v;
                    }
            }
            if constexpr (kHalf) cut |= wide && y >= 0 && !(lg.bias && y < table && lg.bias[y] == -INFINITY);
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
            if (in && q == 0) part[(size_t)piece * rows + t] = make_float2(top, sum);
        }
        if constexpr (!std::is_void_v<E>) {
            constexpr int PER = 16 / (int)sizeof(E);
            if (kHalf && __any(cut) && l == 0) marks[(size_t)pl.tn * mt + pl.tm] = 1;
            rows_through_lds<E, MB, NB>(
                lds,
                [&](int i, int j, int e) {
                    if constexpr (kHalf)
                        return exp_code(acc[i][j][e]);
                    else
                        return acc[i][j][e];
                },
                [&](int r, int c, const Pack<E, PER> &v) {
                    if (n + r < rows && (size_t)(m + c) < vp) *reinterpret_cast<Pack<E, PER> *>(exps + (size_t)(n + r) * vp + m + c) = v;
                });
        }
    }
};

// Joins the pieces: R rows a workgroup, 256 / R lanes of a row each taking every (256 / R)th piece.
template <int R>
__global__ __launch_bounds__(256) void k_xent_join(const float2 *part, int pieces, int rows, const float2 *zt,
                                                   const int64_t *target, int64_t table, const float *weight,
                                                   float scale, float *loss, float *lse, float2 *stat,
                                                   float2 *rowfac, const int *power, Scalars *sc) {
    constexpr int L0 = 256 / R;
    __shared__ float s_top[L0][R + 1], s_sum[L0][R + 1];
    const int k = threadIdx.x % R, g = threadIdx.x / R, t = blockIdx.x * R + k;
    float top = -INFINITY, sum = 0.f;
    if (t < rows) {
        for (int p = g; p < pieces; p += L0) {
            const float2 v = part[(size_t)p * rows + t];
            const float m = fmaxf(top, v.x), about = m == -INFINITY ? 0.f : m;
            sum = sum * exp_neg(top - about) + v.y * exp_neg(v.x - about);
            top = m;
        }
    }
    s_top[g][k] = top;
    s_sum[g][k] = sum;
    for (int h = L0 / 2; h > 0; h /= 2) {
        __syncthreads();
        if (g < h) {
            const float m2 = s_top[g + h][k], m = fmaxf(top, m2), about = m == -INFINITY ? 0.f : m;
            sum = sum * exp_neg(top - about) + s_sum[g + h][k] * exp_neg(m2 - about);
            top = m;
            s_top[g][k] = top;
            s_sum[g][k] = sum;
        }
    }
    if (g != 0) return;
    const float about = top == -INFINITY ? 0.f : top;
    const int64_t y = t < rows ? target[t] : -1;
    float total = sum, ls = 0.f, fac = 0.f, rest = 0.f;
    if (y >= table) {
        ls = fac = NAN;
    } else if (y >= 0) {
        const float2 z = zt[t];
        const float d = (about - z.y) - z.x;  // of the target's logit below the largest
        total += exp_fine(-d);
        if (total == 0.f || z.x == -INFINITY) {
            ls = INFINITY;
        } else {
            const float u = sum * exp_fine(d);  // the others' share in units of the target's
            ls = u < 1e30f ? log1pf(u) : d + logf(total);
            rest = u < 1e30f ? u / (1.f + u) : (u == u ? 1.f : u);
            fac = (weight ? weight[t] : 1.f) * scale;
        }
    }
    const float L = total == 0.f ? -INFINITY : about + logf(total);
    if (t < rows) {
        if (loss) loss[t] = ls;
        if (lse) lse[t] = L;
        if (rowfac) {
            stat[t] = make_float2(about, 1.f / total);
            rowfac[t] = make_float2(fac, fac * rest);
        }
    }
    if (sc) {
        const float2 f = make_float2(fac, fac * rest);
        const uint32_t u = __builtin_bit_cast(uint32_t, f.y) & 0x7fffffffu;
        int least = u && u < 0x7f800000u ? power[t] + row_power(f) : 2 * kNoPower;
#pragma unroll
        for (int o = 1; o < R; o <<= 1) least = min(least, __shfl_xor(least, o, 64));
        if (k == 0 && least < kNoPower) atomicMin(&sc->least, least);
    }
}

__global__ __launch_bounds__(256) void k_zero_rows(char *p, size_t rows, size_t row_bytes, size_t ld_bytes) {
    for (size_t r = blockIdx.x; r < rows; r += gridDim.x)
        for (size_t i = threadIdx.x; i < row_bytes; i += 256) p[r * ld_bytes + i] = 0;
}

// Epilogue of the second product: G, SPLIT: in pairs.
template <class G, bool SPLIT>
struct GradEpi {
    Logits<SPLIT> lg;
    const float2 *stat;   // the row's largest logit, 1 / sum of exp about it
    const float2 *rowfac; // weight x scale, and times 1 - p at the target
    const int64_t *target;
    G *g;  // [tp][vp] values or pairs
    size_t vp;
    int rows, tp, table;
    template <int MB, int NB>
    __device__ void operator()(floatx4_t (&acc)[MB][NB], int m, int n, const MmPlace &, char *lds) const {
        if ((size_t)m >= vp) return;
        const int l = threadIdx.x & 63, q = l >> 4;
        const bool made = lg.made(m + 16 * MB, table);
        const float fw = to_logits(acc, lg, m, n, rows, table);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int t = n + 16 * j + (l & 15);
            const bool in = t < rows;
            const float f = made ? 1.f : lg.of_row(fw, t, rows);
            const float2 st = in ? stat[t] : make_float2(0.f, 0.f);
            const float2 fac = in ? rowfac[t] : make_float2(0.f, 0.f);
            const float unit = grad_unit<!std::is_same_v<G, bf16_t>>(fac, lg.sc);
            const float c = fac.x * unit, cs = c * st.y;
            if constexpr (SPLIT) {
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = cs * exp_fine(fmaf(acc[i][j][e], f, -st.x));
            } else {
                const float f2 = f * kLog2e, a2 = st.x * kLog2e;
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = cs * __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], f2, -a2));
            }
            const int64_t y = in ? target[t] : -1;
            const int d = y >= m && y < m + 16 * MB ? (int)(y - m) - 4 * q : -1;
            if (__any(d >= 0)) {
                const float own = -fac.y * unit;
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = d == 16 * i + e ? own : acc[i][j][e];
            }
            if (__any(c == 0.f)) {  // whatever such a row's logits are
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = c == 0.f ? 0.f : acc[i][j][e];
            }
        }
        G *const to = g;  // nothing of this struct goes through memory
        const size_t ld = vp;
        const int last = tp;
        auto store = [=](int low) {
            return [=](int r, int c, const Pack<G, 8> &v) {
                if (n + r >= last || (size_t)(m + c) >= ld) return;
                G *o = SPLIT ? to + (size_t)(n + r) * ld * 2 + pair_at(m + c) + low : to + (size_t)(n + r) * ld + m + c;
                *reinterpret_cast<Pack<G, 8> *>(o) = v;
            };
        };
        rows_through_lds<G, MB, NB>(lds, [&](int i, int j, int e) { return (G)acc[i][j][e]; }, store(0));
        if constexpr (SPLIT)
            rows_through_lds<G, MB, NB>(
                lds, [&](int i, int j, int e) { return (G)(acc[i][j][e] - (float)(G)acc[i][j][e]); }, store(32));
    }
};

// Stored exps (E) into G where they lie: bfloat16 for float16, pairs for float.  A row a workgroup and
// gridDim.y parts of it; `cols` entries a piece.  Rows from `rows` on become zeros.
template <class E>
__global__ __launch_bounds__(256) void k_exps_to_grad(void *g, const float2 *part, int cols, const float2 *stat,
                                                      const float2 *rowfac, const int64_t *target, int rows, int table,
                                                      size_t vp, const Scalars *sc) {
    constexpr int N = 16 / (int)sizeof(E);  // values of a lane
    const int t = blockIdx.x;
    const bool in = t < rows;
    const float2 fac = in ? rowfac[t] : make_float2(0.f, 0.f);
    const float unit = grad_unit<std::is_same_v<E, float>>(fac, sc);
    const float c = fac.x * unit;
    const float2 st = in ? stat[t] : make_float2(0.f, 0.f);
    const int64_t y = in ? target[t] : -1;
    for (size_t v = ((size_t)blockIdx.y * 256 + threadIdx.x) * N; v < vp; v += (size_t)gridDim.y * 256 * N) {
        E *at = (E *)g + (size_t)t * vp + v;
        float x[N];
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = 0.f;
        if (c != 0.f) {
            const Pack<E, N> p = *reinterpret_cast<const Pack<E, N> *>(at);
            const float f = c * st.y * exp_fine(part[v / cols * rows + t].x - st.x);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if constexpr (std::is_same_v<E, half_t>)
                    x[e] = exp_decode(p.v[e]) * f;
                else
                    x[e] = p.v[e] * f;
            }
            if (y >= (int64_t)v && y < (int64_t)v + N && y < table) {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (y == (int64_t)v + e) x[e] = -fac.y * unit;
            }
        }
        if constexpr (std::is_same_v<E, half_t>) {
            Pack<bf16_t, N> o;
#pragma unroll
            for (int e = 0; e < N; ++e) o.v[e] = (bf16_t)x[e];
            *reinterpret_cast<Pack<bf16_t, N> *>(at) = o;
        } else {
            // 8 lanes hold a block of 32; they are of one wave, so its values are read before any is written
            Pack<half_t, N> hi, lo;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                hi.v[e] = (half_t)x[e];
                lo.v[e] = (half_t)(x[e] - (float)hi.v[e]);
            }
            half_t *o = (half_t *)g + (size_t)t * vp * 2 + pair_at(v);
            __builtin_amdgcn_wave_barrier();
            *reinterpret_cast<Pack<half_t, N> *>(o) = hi;
            *reinterpret_cast<Pack<half_t, N> *>(o + 32) = lo;
        }
    }
}

// Where entries have powers of their own: a row of G (pairs) takes them back before it multiplies the table, and
// then the power of two that brings the largest of what is left to [2^13, 2^14).  A row a workgroup, which walks it
// twice.  Without such entries an early exit is all (5 us of 2048 x 100000 x 768's 2,817).
__global__ __launch_bounds__(256) void k_fold_powers(half_t *g, size_t vp, int table, const int *entry_power, const Scalars *sc, int *boost) {
    if (!sc->wide) return;
    __shared__ uint32_t tops[4];
    half_t *row = g + (size_t)blockIdx.x * vp * 2;
    const int common = unit_power(sc->amax_w);
    // calls f(value, power to take back, hi, lo) for this lane's values
    auto walk = [&](auto &&f) {
        for (size_t v = (size_t)threadIdx.x * 8; v < vp; v += 256 * 8) {
            half_t *at = row + pair_at(v);
            Pack<half_t, 8> hi = *reinterpret_cast<Pack<half_t, 8> *>(at), lo = *reinterpret_cast<Pack<half_t, 8> *>(at + 32);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int own = (int)v + e < table ? entry_power[v + e] : kNoPower;
                f((float)hi.v[e] + (float)lo.v[e], own_power(own, common) ? common - own : 0, hi.v[e], lo.v[e]);
            }
            *reinterpret_cast<Pack<half_t, 8> *>(at) = hi;
            *reinterpret_cast<Pack<half_t, 8> *>(at + 32) = lo;
        }
    };
    uint32_t m = 0;
    walk([&](float x, int k, half_t &, half_t &) {
        const uint32_t u = __builtin_bit_cast(uint32_t, ldexpf(x, k)) & 0x7fffffffu;
        if (u < 0x7f800000u && u > m) m = u;
    });
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t v = __shfl_xor(m, o, 64);
        m = v > m ? v : m;
    }
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) m = tops[w] > m ? tops[w] : m;
    const int up = unit_power(m);
    walk([&](float x, int k, half_t &hi, half_t &lo) {
        x = ldexpf(x, k + up);
        hi = (half_t)x;
        lo = (half_t)(x - (float)hi);
    });
    if (threadIdx.x == 0) boost[blockIdx.x] = up;
}

// What a gradient's product still has to be multiplied with: factor() and two to power() of the row of the result.
template <class O>
struct OutScale {
    const Scalars *sc;     // null: nothing
    const float2 *rowfac;  // null: the table's gradient
    const int *boost;      // of k_fold_powers
    __device__ __forceinline__ float factor() const { return sc ? sc->mantissa : 1.f; }
    __device__ __forceinline__ int power(int r, int rows) const {
        if (std::is_same_v<O, bf16_t> || !sc) return 0;
        if (!rowfac) return -sc->least;
        if (r >= rows) return 0;
        int k = row_power(rowfac[r]);
        if constexpr (std::is_same_v<O, float>) k += unit_power(sc->amax_w) + (sc->wide ? boost[r] : 0);
        return -k;
    }
    static __device__ __forceinline__ float apply(float v, float f, int k) {
        if constexpr (std::is_same_v<O, bf16_t>) return v * f;
        return ldexpf(v * f, k);
    }
};

// Epilogue of the gradients' products (A: columns, B: rows of the result): out, a part of a split K loop,
// or the 32-bit sum over pieces.
template <class O>
struct OutEpi {
    OutScale<O> sc;
    O *out;
    size_t ld;
    float *part;  // [part][rows][cols4], or null
    float *sum;   // [rows][cols4], or null
    int cols, rows, cols4;
    bool first, last;
    template <int MB, int NB>
    __device__ void operator()(floatx4_t (&acc)[MB][NB], int m, int n, const MmPlace &pl, char *lds) const {
        const float f = sc.factor();
        int k[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) k[j] = sc.power(n + 16 * j + ((int)threadIdx.x & 15), rows);
        if (part || sum) {
            float *to = part ? part + (size_t)pl.part * rows * cols4 : sum;
            rows_through_lds<float, MB, NB>(
                lds, [&](int i, int j, int e) { return part ? acc[i][j][e] : sc.apply(acc[i][j][e], f, k[j]); },
                [&](int r, int c, const Pack<float, 4> &v) {
                    if (n + r >= rows || m + c >= cols) return;
                    Pack<float, 4> *s = reinterpret_cast<Pack<float, 4> *>(to + (size_t)(n + r) * cols4 + m + c);
                    if (part || (first && !last)) {
                        *s = v;
                        return;
                    }
                    Pack<float, 4> u = *s;
#pragma unroll
                    for (int e = 0; e < 4; ++e) u.v[e] += v.v[e];
                    if (!last) {
                        *s = u;
                        return;
                    }
                    Pack<O, 4> o;
#pragma unroll
                    for (int e = 0; e < 4; ++e) o.v[e] = (O)u.v[e];
                    store_row<4>(out + (size_t)(n + r) * ld, m + c, cols, o);
                });
            return;
        }
        constexpr int PER = 16 / (int)sizeof(O);
        rows_through_lds<O, MB, NB>(
            lds, [&](int i, int j, int e) { return (O)sc.apply(acc[i][j][e], f, k[j]); },
            [&](int r, int c, const Pack<O, PER> &v) {
                if (n + r >= rows || m + c >= cols) return;
                store_row<PER>(out + (size_t)(n + r) * ld, m + c, cols, v);
            });
    }
};

// Adds the parts of a split K loop: 32 vectors of four values a workgroup, its 8 groups of lanes every
// eighth part.
template <class O>
__global__ __launch_bounds__(256) void k_join_parts(const float *part, int parts, int rows, int cols, int cols4,
                                                    OutScale<O> sc, O *out, size_t ld) {
    __shared__ floatx4_t sums[8][32];
    const int l = threadIdx.x & 31, g = threadIdx.x >> 5;
    const size_t at = (size_t)blockIdx.x * 32 + l, n = (size_t)rows * (cols4 / 4);
    floatx4_t v = {0.f, 0.f, 0.f, 0.f};
    if (at < n) {
#pragma unroll 4
        for (int p = g; p < parts; p += 8) v += *reinterpret_cast<const floatx4_t *>(part + (p * n + at) * 4);
    }
    sums[g][l] = v;
    __syncthreads();
    if (g != 0 || at >= n) return;
#pragma unroll
    for (int p = 1; p < 8; ++p) v += sums[p][l];
    const int r = (int)(at / (cols4 / 4)), c = (int)(at % (cols4 / 4)) * 4;
    const float f = sc.factor();
    const int power = sc.power(r, rows);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (c + e < cols) out[(size_t)r * ld + c + e] = (O)sc.apply(v[e], f, power);
}
template <class O>
void join_parts(const float *part, int parts, int rows, int cols, int cols4, OutScale<O> sc, O *out, size_t ld, hipStream_t s) {
    const size_t n = (size_t)rows * (cols4 / 4);
    k_join_parts<O><<<(uint32_t)((n + 31) / 32), 256, 0, s>>>(part, parts, rows, cols, cols4, sc, out, ld);
}

struct Sizes {
    int dtype;
    size_t rows, table, dim;
    bool grad;
    size_t kp, vp, piece_rows, tp, cols4;
    bool small;       // few rows: xent_small.h
    bool stat_big;
    int pieces;       // of a row's logits
    MmShape dh_tile, dw_tile;
    int ksplit;
};

inline size_t piece_bytes() {
    const char *e = std::getenv("VHIP_XENT_PIECE_BYTES");
    const unsigned long long v = e ? std::strtoull(e, nullptr, 10) : 0;
    return v ? (size_t)v : kPieceBytes;
}

inline Sizes sizes_of(int dtype, size_t rows, size_t table, size_t dim, bool grad) {
    Sizes z{};
    rows = rows ? rows : 1;  // an empty call gets the smallest workspace
    table = table ? table : 1;
    dim = dim ? dim : 1;
    z.dtype = dtype;
    z.rows = rows;
    z.table = table;
    z.dim = dim;
    z.grad = grad;
    z.kp = round_up(dim, kMmK);
    z.vp = round_up(table, kMmK);
    z.cols4 = round_up(dim, 4);
    z.small = few_rows(dtype, rows, table, dim);
    if (z.small) {
        z.piece_rows = rows;
        const size_t groups = ceil_div(table, small_turn(rows, table)), tiles = (table + kSmallEntries - 1) / kSmallEntries, ny = ceil_div(dim, kSmallCols);
        z.pieces = (int)(groups < 2048 ? groups : 2048);
        size_t gx = 1024 / ny;
        if (gx < 64) gx = 64;
        z.ksplit = (int)(tiles < gx ? tiles : gx);
        return z;
    }
    // what a row needs: G, or the pieces of its logits, and its packed copies
    const size_t operand = dtype == VHIP_DTYPE_F32 ? 4 : 2;
    const size_t per = (grad ? (z.vp + dim) * operand : (table + 63) / 64 * sizeof(float2)) + z.kp * operand;
    size_t fit = piece_bytes() / per / 256 * 256;
    // the rows are K of the table's gradient, which a product reads as rows of kMmMaxLd at most
    const size_t longest = kMmMaxLd / (dtype == VHIP_DTYPE_F32 ? 2 : 1);
    if (grad && fit > longest) fit = longest;
    if (fit < 256) fit = 256;
    z.piece_rows = rows <= fit ? rows : fit;
    z.tp = round_up(z.piece_rows, kMmK);
    z.stat_big = mm_big_tiles(table, z.piece_rows, 1);
    z.pieces = ceil_div(table, z.stat_big ? 128 : 64);
    const bool large = dim > 128 && z.piece_rows > 128;
    z.dh_tile = !large ? k128x128 : mm_narrow(dim) ? k192x256 : k256x256;
    const size_t tiles = (size_t)ceil_div(dim, z.dh_tile == k192x256 ? 192 : large ? 256 : 128) * ceil_div(z.piece_rows, large ? 256 : 128);
    const size_t want = large ? 256 : 512, ks = z.vp / kMmK;  // at least 8 stages a part
    size_t k = want / tiles;
    if (k > ks / 8) k = ks / 8;
    z.ksplit = (int)(k < 1 ? 1 : k);
    z.dw_tile = mm_shape(dim, table, 1);
    return z;
}

// Tiles of the logits.
inline size_t mark_count(const Sizes &z) {
    const size_t b = z.stat_big ? 256 : 128;
    return ((z.table + b - 1) / b) * ((z.piece_rows + b - 1) / b);
}

struct Parts {
    Scalars *sc;
    float2 *part;
    float2 *stat, *zt, *rowfac;
    float *split, *sum;
    float *z;  // few rows: the logits
    uint32_t *marks;
    int *power, *entry_power;  // of the rows of h, of the table's (k_ranges)
    int *boost;
    uint32_t *tops;
    void *hp, *wp, *ht, *g;
};

inline Parts carve(Carver &c, const Sizes &z) {
    const size_t planes = z.dtype == VHIP_DTYPE_F32 ? 2 : 1;
    Parts p{};
    p.sc = c.take<Scalars>(1);
    p.part = c.take<float2>((size_t)z.pieces * z.piece_rows);
    p.zt = c.take<float2>(z.piece_rows);
    if (z.small) {
        if (z.grad) {
            p.stat = c.take<float2>(z.rows);
            p.rowfac = c.take<float2>(z.rows);
            p.z = c.take<float>(z.rows * z.vp);
            p.split = c.take<float>((size_t)z.ksplit * z.rows * z.cols4);
        }
        return p;
    }
    if (planes == 2 || (z.grad && z.dtype == VHIP_DTYPE_F16)) p.power = c.take<int>(z.rows);
    if (planes == 2) {
        p.entry_power = c.take<int>(z.table);
        p.tops = c.take<uint32_t>(kRangeGroups);
    }
    p.hp = c.take<uint16_t>(planes * z.piece_rows * z.kp);
    p.wp = c.take<uint16_t>(planes * z.table * z.kp);
    if (z.grad) {
        if (planes == 2) p.boost = c.take<int>(z.tp);
        p.stat = c.take<float2>(z.piece_rows);
        p.rowfac = c.take<float2>(z.piece_rows);
        p.ht = c.take<uint16_t>(planes * z.dim * z.tp);
        p.g = c.take<uint16_t>(planes * z.tp * z.vp);
        p.marks = c.take<uint32_t>(mark_count(z));
        if (z.ksplit > 1) p.split = c.take<float>((size_t)z.ksplit * z.piece_rows * z.cols4);
        if (z.piece_rows < z.rows) p.sum = c.take<float>(z.table * z.cols4);
    }
    return p;
}

struct Call {
    const void *h, *table, *bias;
    size_t ldh, ldt;
    float scale;
    const int64_t *target;
    const float *row_weight;
    float *loss, *lse;
    void *dh, *dtable;
    size_t lddh, lddt;
};

// The pieces' join: as many rows a workgroup as still fill the chip.
inline void join_pieces(const Parts &p, const Sizes &z, size_t rows, const int64_t *target, const float *weight, float scale,
                        float *loss, float *lse, const int *power, hipStream_t s) {
    Scalars *sc = z.grad && !z.small && z.dtype != VHIP_DTYPE_BF16 ? p.sc : nullptr;
#define JOIN(R)                                                                                                       \
    k_xent_join<R><<<(uint32_t)ceil_div(rows, R), 256, 0, s>>>(p.part, z.pieces, (int)rows, p.zt, target, (int64_t)z.table, \
                                                               weight, scale, loss, lse, p.stat, p.rowfac, power, sc)
    if (rows <= 512)
        JOIN(1);
    else if (rows <= 8192)
        JOIN(4);
    else
        JOIN(16);
#undef JOIN
}

template <class T>
int xent_small(const Call &c, const Sizes &z, const Parts &p, hipStream_t s) {
    const int dim = (int)z.dim, table = (int)z.table, rows = (int)z.rows;
    small_stat<T>(SmallStat{c.h, c.table, (const float *)c.bias, c.target, p.part, p.zt, p.z, c.ldh, c.ldt, z.vp, rows, table, dim, c.scale},
                  (uint32_t)z.pieces, s);
    join_pieces(p, z, z.rows, c.target, c.row_weight, c.scale, c.loss, c.lse, nullptr, s);
    if (z.grad) {
        small_grad<T>(SmallGrad{c.h, c.table, (const float *)c.bias, p.z, p.stat, p.rowfac, c.target, c.dtable, c.dh ? p.split : nullptr,
                                c.ldh, c.ldt, c.lddt, z.vp, rows, table, dim, (int)z.cols4},
                      (uint32_t)z.ksplit, s);
        if (c.dh) join_parts<T>(p.split, z.ksplit, rows, dim, (int)z.cols4, OutScale<T>{}, (T *)c.dh, c.lddh, s);
    }
    return launch_status("softmax launch");
}

// Whether rows can be multiplied where they lie.
template <class T>
bool direct(const void *p, size_t ld, size_t dim) {
    return Planes<T>::count == 1 && dim % kMmK == 0 && ld % 8 == 0 && aligned16(p) && ld <= kMmMaxLd;
}

template <class T>
int xent(const Call &c, const Sizes &z, const Parts &p, hipStream_t s) {
    typedef typename Planes<T>::type P;
    constexpr bool kSplit = Planes<T>::count == 2;
    constexpr MmMode kMode = kSplit ? kPairs : kPlain;
    const int dim = (int)z.dim, table = (int)z.table;
    const T *h = (const T *)c.h, *w = (const T *)c.table;

    const InitArgs init{p.sc, c.row_weight, (int)z.rows, c.scale};
    if (p.power) {
        const int lanes = lanes_log2((z.dim + 3) / 4);
        const RangeArgs<T> m{h, w, z.rows, z.table, c.ldh, c.ldt, p.power, p.entry_power, p.tops, (const float *)c.bias, dim,
                             lanes < 6 ? lanes : 6, init};
        k_ranges<T><<<dim3(kRangeGroups, kSplit ? 2 : 1), 256, 0, s>>>(m);
    } else if (z.grad) {
        k_xent_init<<<1, 256, 0, s>>>(init);
    }
    const P *wp = (const P *)c.table;
    size_t ldw = c.ldt;
    if (!direct<T>(c.table, c.ldt, z.dim) || (z.grad && c.bias)) {
        pack<T>(w, z.table, dim, c.ldt, (P *)p.wp, (int)z.kp, p.entry_power, p.tops, p.sc, (const float *)c.bias, s);
        wp = (const P *)p.wp;
        ldw = z.kp * Planes<T>::count;
    }

    for (size_t r0 = 0; r0 < z.rows; r0 += z.piece_rows) {
        const size_t rows = z.rows - r0 < z.piece_rows ? z.rows - r0 : z.piece_rows;
        const T *hr = h + r0 * c.ldh;
        const int64_t *target = c.target + r0;
        const int *power = p.power ? p.power + r0 : nullptr;
        const P *hp = (const P *)(const void *)hr;
        size_t ldh = c.ldh;
        if (!direct<T>(hr, c.ldh, z.dim)) {
            pack<T>(hr, rows, dim, c.ldh, (P *)p.hp, (int)z.kp, power, nullptr, nullptr, nullptr, s);
            hp = (const P *)p.hp;
            ldh = z.kp * Planes<T>::count;
        }
        MmArgs g{};
        g.a = wp;
        g.b = hp;
        g.lda = ldw;
        g.ldb = ldh;
        g.M = table;
        g.N = (int)rows;
        g.K = (int)z.kp;
        g.alo = g.blo = true;
        g.ksplit = g.batch = 1;
        const Logits<kSplit> lg{(const float *)c.bias, p.sc, power, p.entry_power, c.scale};
        typedef std::conditional_t<kSplit, float, half_t> E;
        const bool store = z.grad && stores_exps(z.dtype, z.dim);
        if (store) {
            const StatEpi<E, kSplit> se{lg, p.part, p.zt, target, (int)rows, table, (E *)p.g, z.vp, p.marks, ceil_div(table, z.stat_big ? 256 : 128)};
            if (!kSplit) k_clear<<<(uint32_t)ceil_div(mark_count(z), 256), 256, 0, s>>>(p.marks, (int)mark_count(z));
            VH_CHECK((mm_launch<P, kMode, false, false>)(g, z.stat_big, se, s));
        } else {
            const StatEpi<void, kSplit> se{lg, p.part, p.zt, target, (int)rows, table, nullptr, 0, nullptr, 0};
            VH_CHECK((mm_launch<P, kMode, false, false>)(g, z.stat_big, se, s));
        }
        join_pieces(p, z, rows, target, c.row_weight ? c.row_weight + r0 : nullptr, c.scale, c.loss ? c.loss + r0 : nullptr,
                    c.lse ? c.lse + r0 : nullptr, power, s);
        VH_CHECK(launch_status("softmax launch"));
        if (!z.grad) continue;
        const size_t tp = round_up(rows, kMmK);
        if (store) {
            const size_t parts = (z.vp * sizeof(E) / 16 + 1023) / 1024;  // four turns of a workgroup each
            k_exps_to_grad<E><<<dim3((uint32_t)tp, (uint32_t)(parts < 64 ? parts : 64)), 256, 0, s>>>(
                p.g, p.part, z.stat_big ? 128 : 64, p.stat, p.rowfac, target, (int)rows, table, z.vp, p.sc);
        }
        if (!store || !kSplit) {
            GradEpi<P, kSplit> ge{};
            ge.lg = lg;
            ge.stat = p.stat;
            ge.rowfac = p.rowfac;
            ge.target = target;
            ge.g = (P *)p.g;
            ge.vp = z.vp;
            ge.rows = (int)rows;
            ge.tp = (int)tp;
            ge.table = table;
            MmArgs gg = g;
            gg.only = store ? p.marks : nullptr;
            VH_CHECK((mm_launch<P, kMode, false, false>)(gg, z.stat_big, ge, s));
        }
        const P *gg = (const P *)p.g;
        if (c.dtable) {
            // K the rows: those past the last are zeros in both operands, those that do not count in the first
            k_pack_t<T><<<dim3((uint32_t)(tp / 64), (uint32_t)ceil_div(dim, 64)), 256, 0, s>>>(
                hr, rows, dim, c.ldh, (P *)p.ht, tp, p.sc, p.rowfac);
            MmArgs d{};
            d.a = p.ht;
            d.b = gg;
            d.lda = tp * Planes<T>::count;
            d.ldb = z.vp * Planes<T>::count;
            d.M = dim;
            d.N = table;
            d.K = (int)tp;
            d.alo = d.blo = true;
            d.ksplit = d.batch = 1;
            const bool many = z.piece_rows < z.rows;
            OutEpi<T> oe{OutScale<T>{p.sc, nullptr, nullptr}, (T *)c.dtable, c.lddt, nullptr, many ? p.sum : nullptr, dim, table,
                         (int)z.cols4, r0 == 0, r0 + rows >= z.rows};
            VH_CHECK((mm_launch<P, kMode, false, true>)(d, z.dw_tile, oe, s));
        }
        if (c.dh) {
            if constexpr (kSplit) k_fold_powers<<<(uint32_t)rows, 256, 0, s>>>((half_t *)p.g, z.vp, table, p.entry_power, p.sc, p.boost);
            // columns of the table, K its rows: G's columns past the table are zeros
            MmArgs d = g;
            d.b = gg;
            d.ldb = z.vp * Planes<T>::count;
            d.M = dim;
            d.N = (int)rows;
            d.K = table;
            d.ksplit = z.ksplit;
            const OutScale<T> os{p.sc, p.rowfac, p.boost};
            T *out = (T *)c.dh + r0 * c.lddh;
            OutEpi<T> oe{os, out, c.lddh, z.ksplit > 1 ? p.split : nullptr, nullptr, dim, (int)rows, (int)z.cols4,
                         true, true};
            VH_CHECK((mm_launch<P, kMode, true, false>)(d, z.dh_tile, oe, s));
            if (z.ksplit > 1)
                join_parts<T>(p.split, z.ksplit, (int)rows, dim, (int)z.cols4, os, out, c.lddh, s);
        }
        VH_CHECK(launch_status("gradient launch"));
    }
    return VHIP_OK;
}

int check_call(int dtype, const Call &c, size_t rows, size_t table, size_t dim, bool grad) {
    if (!dtype_known(dtype)) return set_error(VHIP_ERR_INVALID_CONFIG, "unknown element type " + std::to_string(dtype));
    if (dim == 0 || dim > 65536) return set_error(VHIP_ERR_INVALID_CONFIG, "dim must be in [1, 65536]");
    if (table == 0 || table > kMmMaxLd / 2 - kMmK) return set_error(VHIP_ERR_INVALID_CONFIG, "the table must have 1 to 2^22 - 64 rows");
    if (rows > 0x3fffffff) return set_error(VHIP_ERR_INVALID_CONFIG, "too many rows");
    if ((rows && (!c.h || !c.target)) || !c.table) return set_error(VHIP_ERR_INVALID_CONFIG, "an input is null");
    if (c.ldh < dim || c.ldt < dim || (c.dh && c.lddh < dim) || (c.dtable && c.lddt < dim))
        return set_error(VHIP_ERR_INVALID_CONFIG, "rows are closer than dim");
    if (!std::isfinite(c.scale)) return set_error(VHIP_ERR_INVALID_CONFIG, "scale must be finite");
    if (grad && !c.dh && !c.dtable) return set_error(VHIP_ERR_INVALID_CONFIG, "no gradient is asked for");
    return VHIP_OK;
}

int run(int ordinal, int dtype, const Call &c, size_t rows, size_t table, size_t dim, bool grad, void *ws, size_t ws_bytes,
        void *stream) {
    clear_error();
    VH_CHECK(check_call(dtype, c, rows, table, dim, grad));
    const Sizes z = sizes_of(dtype, rows, table, dim, grad);
    Carver cv{(char *)ws, 0};
    const Parts p = carve(cv, z);
    if (!ws || !aligned16(ws) || ws_bytes < cv.used)
        return set_error(VHIP_ERR_INVALID_CONFIG, "the workspace is smaller than vhip_softmax_xent_workspace() (" +
                                                      std::to_string(cv.used) + " bytes) or not aligned to 16 bytes");
    CallDevice dev;
    VH_CHECK(dev.enter(ordinal));
    hipStream_t s = (hipStream_t)stream;
    if (rows == 0) {
        if (!grad || !c.dtable) return VHIP_OK;
        const size_t es = dtype_size(dtype);
        k_zero_rows<<<(uint32_t)(table < 4096 ? table : 4096), 256, 0, s>>>((char *)c.dtable, table, dim * es, c.lddt * es);
        return launch_status("gradient launch");
    }
    if (z.small) {
        switch (dtype) {
            case VHIP_DTYPE_F32: return xent_small<float>(c, z, p, s);
            case VHIP_DTYPE_F16: return xent_small<half_t>(c, z, p, s);
            default: return xent_small<bf16_t>(c, z, p, s);
        }
    }
    switch (dtype) {
        case VHIP_DTYPE_F32: return xent<float>(c, z, p, s);
        case VHIP_DTYPE_F16: return xent<half_t>(c, z, p, s);
        default: return xent<bf16_t>(c, z, p, s);
    }
}

}  // namespace
}  // namespace vh

using namespace vh;

extern "C" {

size_t vhip_softmax_xent_workspace(int dtype, size_t rows, size_t table_rows, size_t dim, int gradients) {
    Carver cv;
    carve(cv, sizes_of(dtype, rows, table_rows, dim, gradients != 0));
    return cv.used;
}

int vhip_softmax_xent(int ordinal, int dtype, const void *h, size_t rows, size_t ldh, const void *table, size_t table_rows,
                      size_t ldt, size_t dim, const int64_t *target, const float *bias, float scale, float *loss,
                      float *lse, void *workspace, size_t workspace_bytes, void *stream) {
    Call c{};
    c.h = h;
    c.table = table;
    c.bias = bias;
    c.ldh = ldh;
    c.ldt = ldt;
    c.scale = scale;
    c.target = target;
    c.loss = loss;
    c.lse = lse;
    return run(ordinal, dtype, c, rows, table_rows, dim, false, workspace, workspace_bytes, stream);
}

int vhip_softmax_xent_grad(int ordinal, int dtype, const void *h, size_t rows, size_t ldh, const void *table,
                           size_t table_rows, size_t ldt, size_t dim, const int64_t *target, const float *bias,
                           const float *row_weight, float scale, float *loss, float *lse, void *dh, size_t lddh,
                           void *dtable, size_t lddt, void *workspace, size_t workspace_bytes, void *stream) {
    Call c{};
    c.h = h;
    c.table = table;
    c.bias = bias;
    c.ldh = ldh;
    c.ldt = ldt;
    c.scale = scale;
    c.target = target;
    c.row_weight = row_weight;
    c.loss = loss;
    c.lse = lse;
    c.dh = dh;
    c.dtable = dtable;
    c.lddh = lddh;
    c.lddt = lddt;
    return run(ordinal, dtype, c, rows, table_rows, dim, true, workspace, workspace_bytes, stream);
}

}  // extern "C"
