// newton_schulz.hip -- orthogonalises update matrices by Newton-Schulz products.
//
//   X = M / (|M|_F + eps)  (of M^T where M has more rows than columns),  then `steps` times
//   A = X X^T,  B = a I + b A + c A A,  X <- B X
//
// which drives the singular values towards one while the singular vectors stay.  A direction whose singular
// value is small grows by `a` a step, and what rounding puts into it grows as much, so X, A and B are held
// in pairs of float16 (22 bits, mm16.h) and multiplied as three products with 32-bit sums, at a third of the
// 16-bit matrix rate (300 x 768, five steps: off by 1.3e-6 of the result, plain 32-bit products by 1.9e-6).  X is held times 2^10 and A and B times 2^8, or by smaller
// powers of two where the coefficients let them leave float16's range (ns_scales).
// The first X is the matrix times the power of two that brings |M|_F to [2^12, 2^13); what is left of the
// norm goes into the first step's epilogues, so 16-bit matrices are exact in the high halves and their
// first products have no low ones to multiply.  Where the result is rounded to bfloat16 (2^-9), the last
// step's B X multiplies high halves alone: no later step amplifies its 2^-12.  (Its A and A A do not: B is a
// difference of terms several times its size.)
// X's halves reach down to 2^-34: a matrix whose norm is below 2^-34 of eps comes out as zero.
//
// A and A A are symmetric: only tiles on and above the diagonal are computed, and stored twice.  a X is part
// of B's diagonal.
#include "mm16.h"

#include <cmath>
#include <type_traits>

namespace vh {
namespace {

constexpr float kXScale = 1024.f;  // of the first X
constexpr int kNormParts = 64;

__device__ __forceinline__ void split(float x, half_t &hi, half_t &lo) {
    hi = (half_t)x;
    lo = (half_t)(x - (float)hi);
}

// Partial sums of squares, in 64 bits: values of any magnitude neither overflow nor vanish.  2^lanes lanes a
// row, 16 bytes each at a time.
template <class T>
__global__ __launch_bounds__(256) void k_ns_norm(const T *in, int rows, int cols, size_t ld, size_t stride, int lanes, double *part) {
    constexpr int V = 16 / (int)sizeof(T);
    __shared__ double lds[4];
    const T *p = in + blockIdx.y * stride;
    const int per = 256 >> lanes, l = threadIdx.x & ((1 << lanes) - 1);
    double s = 0.0;
    for (int r = blockIdx.x * per + (threadIdx.x >> lanes); r < rows; r += kNormParts * per) {
        for (int c = l * V; c < cols; c += V << lanes) {
            const Pack<T, V> v = load_row<V>(p + (size_t)r * ld, c, cols);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const double x = (double)(float)v.v[e];
                s += x * x;
            }
        }
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.y * kNormParts + blockIdx.x] = lds[0] + lds[1] + lds[2] + lds[3];
}

// A stack of matrices in pairs (mm16.h).
struct Pairs {
    half_t *p;
    size_t cols;        // values of a row, a multiple of 64
    size_t ld, stride;  // halves
};

// The matrix times a power of two as x [m][np], zeros past n; BOTH: and its transpose xt [n][mp].
// gain: what is left to multiply for M / (|M| + eps) times kXScale.
template <class T, bool BOTH>
__global__ __launch_bounds__(256) void k_ns_start(const T *in, int rows, int cols, size_t ld, size_t stride, bool tall,
                                                  const double *part, float eps, Pairs x, Pairs xt, float *gain) {
    __shared__ float tile[64][65];
    __shared__ float s_inv;
    const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64, tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    const T *p = in + blockIdx.z * stride;
    float v[16];  // on their way while the norm is added up
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int r = r0 + ty + 4 * i, c = c0 + tx;
        v[i] = r < rows && c < cols ? (float)p[(size_t)r * ld + c] : 0.f;
    }
    if (threadIdx.x < 64) {
        double s = part[blockIdx.z * kNormParts + threadIdx.x];
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
        if (threadIdx.x == 0) {
            const double norm = sqrt(s);
            int e = 0;
            (void)frexp(norm, &e);  // norm < 2^e
            const double up = norm > 0.0 && norm <= 1e300 ? ldexp(1.0, 13 - e) : 1.0;
            // a power of two that a float holds: what is past its range goes into the gain as well
            s_inv = (float)fmin(fmax(up, 0x1p-126), 0x1p126);
            // zeros over a small eps are zeros, though the gain's square may leave 32 bits
            const double left = norm == 0.0 && eps > 0.f ? 0.0 : (double)kXScale / ((norm + (double)eps) * (double)s_inv);
            if (blockIdx.x == 0 && blockIdx.y == 0) gain[blockIdx.z] = (float)left;
        }
    }
    __syncthreads();
    const float inv = s_inv;
#pragma unroll
    for (int i = 0; i < 16; ++i) tile[tall ? tx : ty + 4 * i][tall ? ty + 4 * i : tx] = v[i] * inv;
    __syncthreads();
    const int m0 = tall ? c0 : r0, n0 = tall ? r0 : c0, m = tall ? cols : rows, n = tall ? rows : cols;
    half_t *o = x.p + blockIdx.z * x.stride;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int r = m0 + ty + 4 * i, c = n0 + tx;
        if (r < m && (size_t)c < x.cols) {
            half_t hi, lo;
            split(tile[ty + 4 * i][tx], hi, lo);
            o[(size_t)r * x.ld + pair_at(c)] = hi;
            o[(size_t)r * x.ld + pair_at(c) + 32] = lo;
        }
    }
    if constexpr (BOTH) {
        o = xt.p + blockIdx.z * xt.stride;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int r = n0 + ty + 4 * i, c = m0 + tx;
            if (r < n && (size_t)c < xt.cols) {
                half_t hi, lo;
                split(tile[tx][ty + 4 * i], hi, lo);
                o[(size_t)r * xt.ld + pair_at(c)] = hi;
                o[(size_t)r * xt.ld + pair_at(c) + 32] = lo;
            }
        }
    }
}

// A wave's blocks as pairs of rows [r0, rows) and columns from c0 on.
template <int MB, int NB>
__device__ __forceinline__ void store_pairs(const floatx4_t (&acc)[MB][NB], char *lds, half_t *p, const Pairs &to, int r0, int rows, int c0) {
    auto store = [=](int low) {
        return [=](int r, int c, const Pack<half_t, 8> &v) {
            if (r0 + r < rows && (size_t)(c0 + c) < to.cols)
                *reinterpret_cast<Pack<half_t, 8> *>(p + (size_t)(r0 + r) * to.ld + pair_at(c0 + c) + low) = v;
        };
    };
    rows_through_lds<half_t, MB, NB>(lds, [&](int i, int j, int e) { return (half_t)acc[i][j][e]; }, store(0));
    rows_through_lds<half_t, MB, NB>(
        lds, [&](int i, int j, int e) { return (half_t)(acc[i][j][e] - (float)(half_t)acc[i][j][e]); }, store(32));
}

// Epilogue of the symmetric products: out = alpha acc + beta add + diag I, stored at both places.
struct SymEpi {
    Pairs out, add;   // add.p null: none
    const float *gain;  // null: 1
    float alpha, beta, diag;
    int m;
    template <int MB, int NB>
    __device__ void operator()(floatx4_t (&acc)[MB][NB], int mw, int nw, const MmPlace &pl, char *lds) const {
        const int l = threadIdx.x & 63, q = l >> 4;
        half_t *o = out.p + pl.batch * out.stride;
        const half_t *ad = add.p ? add.p + pl.batch * add.stride : nullptr;
        const bool mirror = pl.tm != pl.tn;
        const float al = gain ? gain[pl.batch] * gain[pl.batch] * alpha : alpha;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int c = nw + 16 * j + (l & 15);
            int rq = mw + 4 * q;
            if constexpr (MB * NB > 16) asm volatile("" : "+v"(rq));  // see rows_through_lds
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                const int r = rq + 16 * i;
                floatx4_t v = acc[i][j] * al;
                if (ad && c < m && (size_t)r < add.cols) {
                    const Pack<half_t, 4> h = *reinterpret_cast<const Pack<half_t, 4> *>(ad + (size_t)c * add.ld + pair_at(r));
                    const Pack<half_t, 4> w = *reinterpret_cast<const Pack<half_t, 4> *>(ad + (size_t)c * add.ld + pair_at(r) + 32);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = fmaf(beta, (float)h.v[e] + (float)w.v[e], v[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = v[e] + (r + e == c ? diag : 0.f);
                    if (r + e >= m || c >= m) x = 0.f;
                    acc[i][j][e] = x;
                    if (mirror && r + e < m && (size_t)c < out.cols) {
                        half_t hi, lo;
                        split(x, hi, lo);
                        o[(size_t)(r + e) * out.ld + pair_at(c)] = hi;
                        o[(size_t)(r + e) * out.ld + pair_at(c) + 32] = lo;
                    }
                }
            }
        }
        store_pairs(acc, lds, o, out, nw, m, mw);
    }
};

// Epilogue of B X: the next X (A operand X across, B operand B), or the result in the order that the A
// operand's rows have (B where the matrix is tall).
template <class T>
struct StepEpi {
    Pairs x;
    const float *gain;  // null: 1
    float alpha;
    int cols, rows;  // of what is stored
    T *out;          // null: not the last step
    size_t ldo, so;
    template <int MB, int NB>
    __device__ void operator()(floatx4_t (&acc)[MB][NB], int mw, int nw, const MmPlace &pl, char *lds) const {
        const float al = gain ? gain[pl.batch] * alpha : alpha;
        if (!out) {
            const int l = threadIdx.x & 63, q = l >> 4;
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int j = 0; j < NB; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = mw + 16 * i + 4 * q + e < cols ? acc[i][j][e] * al : 0.f;
            store_pairs(acc, lds, x.p + pl.batch * x.stride, x, nw, rows, mw);
            return;
        }
        constexpr int PER = 16 / (int)sizeof(T);
        T *o = out + pl.batch * so;
        rows_through_lds<T, MB, NB>(
            lds, [&](int i, int j, int e) { return (T)(acc[i][j][e] * al); },
            [&](int r, int c, const Pack<T, PER> &v) {
                if (nw + r >= rows || mw + c >= cols) return;
                store_row<PER>(o + (size_t)(nw + r) * ldo, mw + c, cols, v);
            });
    }
};

// ---- small matrices ------------------------------------------------------------------------------
// With few tiles a product is bound by how long one workgroup takes for its K loop.  Here a workgroup of
// 8 waves computes a tile of 64 x 64, or of 32 x 32 where there are few, each wave all of it over every eighth
// 32 of K, from operands that it loads straight into registers (K contiguous in both: X is kept in both
// orders); the waves' sums meet in LDS.
struct SmallArgs {
    Pairs a, b;  // tile rows m of a, n of b
    int M, N, K;
    bool alo, blo;  // whether their low halves count
    bool upper;
    // out[n][m..] = alpha acc + beta add[n][m..] + diag I
    Pairs out, add, out_t;  // out_t: and the transpose; add.p, out_t.p null: none
    const float *gain;
    int gains;      // powers of the gain in alpha
    float alpha, beta, diag;
    void *result;   // in T instead of out
    size_t ldr, sr;
    bool result_t;  // result[m][n]
};

template <class T, int TB>  // blocks of 16 along a tile's side
__global__ __launch_bounds__(512) void k_ns_small(SmallArgs g) {
    typedef MmVec<half_t>::v8 v8;
    constexpr int SIDE = 16 * TB, V = SIDE * SIDE / 512;  // values of a lane in the end
    __shared__ __align__(16) float s_part[8][SIDE][SIDE + 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, q = lane >> 4;
    int tm = blockIdx.x, tn = blockIdx.y;
    if (g.upper) {
        tn = 0;
        while ((tn + 1) * (tn + 2) / 2 <= (int)blockIdx.x) ++tn;
        tm = blockIdx.x - tn * (tn + 1) / 2;
    }
    const int m0 = tm * SIDE, n0 = tn * SIDE;
    const half_t *pa = g.a.p + blockIdx.z * g.a.stride + q * 8, *pb = g.b.p + blockIdx.z * g.b.stride + q * 8;
    size_t ra[TB], rb[TB];
#pragma unroll
    for (int i = 0; i < TB; ++i) {
        ra[i] = (size_t)min(m0 + 16 * i + i16, g.M - 1) * g.a.ld;
        rb[i] = (size_t)min(n0 + 16 * i + i16, g.N - 1) * g.b.ld;
    }
    floatx4_t acc[TB][TB];
#pragma unroll
    for (int i = 0; i < TB; ++i)
#pragma unroll
        for (int j = 0; j < TB; ++j) acc[i][j] = floatx4_t{0.f, 0.f, 0.f, 0.f};
    const int steps = (g.K + 31) / 32;  // rows are zero from K to the next multiple of 64
#pragma unroll (TB == 4 ? 2 : 4)
    for (int s = wave; s < steps; s += 8) {
        v8 ah[TB], al[TB], bh[TB], bl[TB];
#pragma unroll
        for (int i = 0; i < TB; ++i) {
            ah[i] = *reinterpret_cast<const v8 *>(pa + ra[i] + s * 64);
            bh[i] = *reinterpret_cast<const v8 *>(pb + rb[i] + s * 64);
            if (g.alo) al[i] = *reinterpret_cast<const v8 *>(pa + ra[i] + s * 64 + 32);
            if (g.blo) bl[i] = *reinterpret_cast<const v8 *>(pb + rb[i] + s * 64 + 32);
        }
#pragma unroll
        for (int i = 0; i < TB; ++i)
#pragma unroll
            for (int j = 0; j < TB; ++j) {
                acc[i][j] = MmVec<half_t>::mfma(ah[i], bh[j], acc[i][j]);
                if (g.blo) acc[i][j] = MmVec<half_t>::mfma(ah[i], bl[j], acc[i][j]);
                if (g.alo) acc[i][j] = MmVec<half_t>::mfma(al[i], bh[j], acc[i][j]);
            }
    }
#pragma unroll
    for (int i = 0; i < TB; ++i)
#pragma unroll
        for (int j = 0; j < TB; ++j) *reinterpret_cast<floatx4_t *>(&s_part[wave][16 * j + i16][16 * i + 4 * q]) = acc[i][j];
    __syncthreads();
    // V values of m of one n a lane
    const int ln = threadIdx.x / (SIDE / V), lm = threadIdx.x % (SIDE / V) * V, n = n0 + ln, m = m0 + lm;
    float v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) x += s_part[w][ln][lm + e];
        v[e] = x;
    }
    float alpha = g.alpha;
    for (int k = 0; k < g.gains; ++k) alpha *= g.gain[blockIdx.z];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] *= alpha;
    if (g.result) {
        T *o = (T *)g.result + blockIdx.z * g.sr;
        if (n < g.N)
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (m + e < g.M) o[g.result_t ? (size_t)(m + e) * g.ldr + n : (size_t)n * g.ldr + m + e] = (T)v[e];
        return;
    }
    if (g.add.p && n < g.N && m < g.M) {
        const half_t *ad = g.add.p + blockIdx.z * g.add.stride + (size_t)n * g.add.ld + pair_at(m);
        const Pack<half_t, V> h = *reinterpret_cast<const Pack<half_t, V> *>(ad), l = *reinterpret_cast<const Pack<half_t, V> *>(ad + 32);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = fmaf(g.beta, (float)h.v[e] + (float)l.v[e], v[e]);
    }
    Pack<half_t, V> hi, lo;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        if (m + e == n) v[e] += g.diag;
        split(n < g.N && m + e < g.M ? v[e] : 0.f, hi.v[e], lo.v[e]);
    }
    if (n < g.N && (size_t)m < g.out.cols) {
        half_t *o = g.out.p + blockIdx.z * g.out.stride + (size_t)n * g.out.ld + pair_at(m);
        *reinterpret_cast<Pack<half_t, V> *>(o) = hi;
        *reinterpret_cast<Pack<half_t, V> *>(o + 32) = lo;
    }
    // the other order: X^T, or the mirror image of a symmetric product's tile
    const Pairs &t = g.upper ? g.out : g.out_t;
    if ((g.upper && tm != tn) || (!g.upper && t.p)) {
        half_t *o = t.p + blockIdx.z * t.stride;
        if ((size_t)n < t.cols)
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (m + e < g.M) {
                    o[(size_t)(m + e) * t.ld + pair_at(n)] = hi.v[e];
                    o[(size_t)(m + e) * t.ld + pair_at(n) + 32] = lo.v[e];
                }
    }
}

template <class T>
void ns_small_product(const SmallArgs &g, size_t count, hipStream_t s) {
    // tiles reach to the next multiple of 64, where rows of pairs end: what is past M and N is stored as zeros
    auto grid = [&](int side) {
        const uint32_t tm = ceil_div(round_up(g.M, kMmK), side), tn = ceil_div(round_up(g.N, kMmK), side);
        return g.upper ? dim3(tm * (tm + 1) / 2, 1, (uint32_t)count) : dim3(tm, tn, (uint32_t)count);
    };
    const dim3 few = grid(32);
    if ((size_t)few.x * few.y * few.z <= 512)
        k_ns_small<T, 2><<<few, 512, 0, s>>>(g);
    else
        k_ns_small<T, 4><<<grid(64), 512, 0, s>>>(g);
}

// Where the 64 x 64 tiles of all matrices are at most one round of workgroups.  Tiles of mm16.h / this way in us,
// 32 bits: 1 x 300 x 768 (60 tiles) 154 / 126, 1 x 1024 x 1024 (256) 369 / 328, 4 x 512 x 512 (256) 238 / 228,
// 2 x 768 x 768 (288) 305 / 352, 8 x 256 x 1024 (512) 223 / 256.
inline bool ns_small(size_t count, size_t m, size_t n) {
    const size_t tm = (m + 63) / 64, tn = (n + 63) / 64;
    return count * tm * tn <= 256;
}

// What X, A and B of a step are held times.
struct NsScale {
    double x, a, b;
};
constexpr int kMaxSteps = 100;
// The scales of `steps` steps and of the X after them.  The singular values of X start at 1 at most, and a step takes
// s to |a s + b s^3 + c s^5|: the largest of that over [0, s] bounds the next ones, and the values of each matrix
// are at most its norm.  False where they may pass 2^30.
inline bool ns_scales(double a, double b, double c, int steps, NsScale *out) {
    auto held = [](double bound, double usual) {
        while (usual * bound > 0x1p15) usual /= 2;
        return usual;
    };
    // largest |p0 + p1 u + p2 u^2| over [0, top], times sqrt(u) where ROOT
    auto largest = [&](double top, bool root) {
        auto at = [&](double u) { return std::fabs(a + b * u + c * u * u) * (root ? std::sqrt(u) : 1.0); };
        double m = std::fmax(at(0.0), at(top));
        auto see = [&](double u) {
            if (u > 0.0 && u < top) m = std::fmax(m, at(u));
        };
        // where the derivative is zero: q0 + q1 u + q2 u^2
        const double q0 = root ? a : b, q1 = root ? 3 * b : 2 * c, q2 = root ? 5 * c : 0.0;
        if (q2 != 0.0) {
            const double d = q1 * q1 - 4 * q0 * q2;
            if (d >= 0.0) {
                // the root of larger size without cancellation, the other by the product of both
                const double big = -0.5 * (q1 + std::copysign(std::sqrt(d), q1));
                see(big / q2);
                if (big != 0.0) see(q0 / big);
            }
        } else if (q1 != 0.0) {
            see(-q0 / q1);
        }
        return m;
    };
    double s = 1.0;
    for (int i = 0; i <= steps; ++i) {
        const double bound = largest(s * s, false);
        if (!(s <= 0x1p30 && (i == steps || bound <= 0x1p30))) return false;
        out[i] = {held(s, kXScale), held(s * s, 256.0), held(bound, 256.0)};
        s = largest(s * s, true);
    }
    return true;
}

struct NsParts {
    double *norm;
    float *gain;
    Pairs x[2], xt[2], a, b;  // xt for small matrices alone
};

inline Pairs pairs(Carver &c, size_t count, size_t rows, size_t cols) {
    Pairs p{};
    p.cols = cols;
    p.ld = 2 * cols;
    p.stride = rows * p.ld;
    p.p = c.take<half_t>(count * p.stride);
    return p;
}

inline NsParts carve(Carver &c, size_t count, size_t m, size_t n) {
    NsParts p{};
    const size_t mp = round_up(m, kMmK), np = round_up(n, kMmK);
    p.norm = c.take<double>(count * kNormParts);
    p.gain = c.take<float>(count);
    for (Pairs &x : p.x) x = pairs(c, count, m, np);
    if (ns_small(count, m, n))
        for (Pairs &x : p.xt) x = pairs(c, count, n, mp);
    p.a = pairs(c, count, m, mp);
    p.b = pairs(c, count, m, mp);
    return p;
}

// C of stacks a and b; alo, blo: whether their low halves count.
template <bool TA, bool TB, class Epi>
int multiply(const Pairs &a, int M, const Pairs &b, int N, int K, bool alo, bool blo, size_t count, bool upper, const Epi &epi,
             hipStream_t s) {
    MmArgs g{};
    g.a = a.p;
    g.b = b.p;
    g.lda = a.ld;
    g.ldb = b.ld;
    g.sa = a.stride;
    g.sb = b.stride;
    g.M = M;
    g.N = N;
    g.K = K;
    g.alo = alo;
    g.blo = blo;
    g.ksplit = 1;
    g.batch = (int)count;
    g.upper = upper;
    // 256 x 256 tiles read and store with the whole CU idle; a K loop of 64 stages makes up for it (one
    // matrix of 4096 x 4096: 3.52 ms, 3.73 with 128 x 128; of K = 1024, eight matrices of 4096 x 1024 take
    // 1.81 ms either way, 32 of 1024 x 1024 2.72 and 2.48, and eight of 1500 x 1500 2.33 and 2.03).
    const bool big = K >= 2048 && mm_big_tiles(M, N, count, upper);
    return alo || blo ? mm_launch<half_t, kPairs, TA, TB>(g, big, epi, s) : mm_launch<half_t, kHigh, TA, TB>(g, big, epi, s);
}

struct NsCall {
    const void *in;
    size_t count, rows, cols, ldi, si;
    int steps;
    float a, b, c, eps;
    const NsScale *scale;
    void *out;
    size_t ldo, so;
};

template <class T>
int newton_schulz(const NsCall &k, const NsParts &p, hipStream_t s) {
    const bool tall = k.rows > k.cols, small = p.xt[0].p != nullptr;
    const int m = (int)(tall ? k.cols : k.rows), n = (int)(tall ? k.rows : k.cols);
    const uint32_t count = (uint32_t)k.count;
    // symmetric products of few tiles: a workgroup a 32 or 64 tile, its waves sharing K (1 x 1024 x 4096: 691 us
    // with 36 workgroups of 128 x 128 each, 513 so; at 78 tiles the two are even)
    const size_t side = (size_t)ceil_div(m, 128);
    const bool few = small || k.count * side * (side + 1) / 2 <= 48;
    const T *in = (const T *)k.in;
    k_ns_norm<T><<<dim3(kNormParts, count), 256, 0, s>>>(in, (int)k.rows, (int)k.cols, k.ldi, k.si, lanes_log2((k.cols * sizeof(T) + 15) / 16), p.norm);
    const dim3 tiles((uint32_t)ceil_div(k.rows, 64), (uint32_t)ceil_div(k.cols, 64), count);
    if (small)
        k_ns_start<T, true><<<tiles, 256, 0, s>>>(in, (int)k.rows, (int)k.cols, k.ldi, k.si, tall, p.norm, k.eps, p.x[0], p.xt[0], p.gain);
    else
        k_ns_start<T, false><<<tiles, 256, 0, s>>>(in, (int)k.rows, (int)k.cols, k.ldi, k.si, tall, p.norm, k.eps, p.x[0], p.x[0], p.gain);
    VH_CHECK(launch_status("orthogonalize launch"));
    for (int i = 0; i < k.steps; ++i) {
        const bool first = i == 0, last = i + 1 == k.steps;
        const float *gain = first ? p.gain : nullptr;
        // which low halves count: X's are empty at first where the matrix has 16 bits
        const bool low = !(last && !first && std::is_same_v<T, bf16_t>);  // in B X
        const bool xlow = !(first && sizeof(T) == 2);
        const Pairs &x = p.x[i & 1], &xn = p.x[(i & 1) ^ 1], &xt = p.xt[i & 1], &xtn = p.xt[(i & 1) ^ 1];
        SmallArgs ga{}, gb{};
        ga.gain = p.gain;
        ga.a = ga.b = x;
        ga.M = ga.N = m;
        ga.K = n;
        ga.alo = ga.blo = xlow;
        ga.upper = true;
        ga.out = p.a;
        const NsScale &sc = k.scale[i];
        ga.alpha = (float)(sc.a / (sc.x * sc.x));
        ga.gains = first ? 2 : 0;
        gb = ga;
        gb.a = gb.b = gb.add = p.a;
        gb.K = m;
        gb.alo = gb.blo = true;
        gb.out = p.b;
        gb.alpha = (float)(k.c * sc.b / (sc.a * sc.a));
        gb.beta = (float)(k.b * sc.b / sc.a);
        gb.diag = (float)(k.a * sc.b);
        const float alpha = (float)((last ? 1.0 : k.scale[i + 1].x) / (sc.b * sc.x));  // of B X
        gb.gains = 0;
        if (few) {
            ns_small_product<T>(ga, k.count, s);
            ns_small_product<T>(gb, k.count, s);
            VH_CHECK(launch_status("orthogonalize launch"));
        } else {
            SymEpi ea{p.a, Pairs{}, gain, ga.alpha, 0.f, 0.f, m};
            VH_CHECK((multiply<false, false>)(x, m, x, m, n, xlow, xlow, k.count, true, ea, s));
            SymEpi eb{p.b, p.a, nullptr, gb.alpha, gb.beta, gb.diag, m};
            VH_CHECK((multiply<false, false>)(p.a, m, p.a, m, m, true, true, k.count, true, eb, s));
        }
        if (small) {
            SmallArgs h{};
            h.gain = p.gain;
            h.a = xt;
            h.b = p.b;
            h.M = n;
            h.N = h.K = m;
            h.alo = low && xlow;
            h.blo = low;
            h.out = xn;
            h.out_t = xtn;
            h.alpha = alpha;
            h.gains = first ? 1 : 0;
            if (last) {
                h.result = k.out;
                h.ldr = k.ldo;
                h.sr = k.so;
                h.result_t = tall;
            }
            ns_small_product<T>(h, k.count, s);
            VH_CHECK(launch_status("orthogonalize launch"));
            continue;
        }
        StepEpi<T> es{xn, gain, alpha, n, m, nullptr, 0, 0};
        if (last) {
            es.out = (T *)k.out;
            es.ldo = k.ldo;
            es.so = k.so;
        }
        if (last && tall) {
            es.cols = m;
            es.rows = n;
            VH_CHECK((multiply<false, true>)(p.b, m, x, n, m, low, low && xlow, k.count, false, es, s));
        } else {
            VH_CHECK((multiply<true, false>)(x, n, p.b, m, m, low && xlow, low, k.count, false, es, s));
        }
    }
    return VHIP_OK;
}

}  // namespace
}  // namespace vh

using namespace vh;

extern "C" {

size_t vhip_orthogonalize_workspace(size_t count, size_t rows, size_t cols) {
    Carver c;
    carve(c, count, rows < cols ? rows : cols, rows < cols ? cols : rows);
    return c.used;
}

int vhip_orthogonalize(int ordinal, int dtype, const void *in, size_t count, size_t rows, size_t cols, size_t ld_in,
                       size_t stride_in, int steps, float a, float b, float c, float eps, void *out, size_t ld_out,
                       size_t stride_out, void *workspace, size_t workspace_bytes, void *stream) {
    clear_error();
    if (!dtype_known(dtype)) return set_error(VHIP_ERR_INVALID_CONFIG, "unknown element type " + std::to_string(dtype));
    if (rows > 65536 || cols > 65536 || count > 65535)
        return set_error(VHIP_ERR_INVALID_CONFIG, "at most 65535 matrices of 65536 rows and columns");
    if (steps < 1 || steps > kMaxSteps) return set_error(VHIP_ERR_INVALID_CONFIG, "steps must be in [1, 100]");
    if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return set_error(VHIP_ERR_INVALID_CONFIG, "coefficients must be finite");
    NsScale scale[kMaxSteps + 1];
    if (!ns_scales(a, b, c, steps, scale))
        return set_error(VHIP_ERR_INVALID_CONFIG, "the coefficients let singular values grow past 2^30");
    if (!(eps >= 0.f)) return set_error(VHIP_ERR_INVALID_CONFIG, "eps must be >= 0");
    const bool empty = count == 0 || rows == 0 || cols == 0;
    if (!empty) {
        if (!in || !out) return set_error(VHIP_ERR_INVALID_CONFIG, "a matrix is null");
        if (ld_in < cols || ld_out < cols) return set_error(VHIP_ERR_INVALID_CONFIG, "rows are closer than cols");
        if (count > 1 && (stride_in < (rows - 1) * ld_in + cols || stride_out < (rows - 1) * ld_out + cols))
            return set_error(VHIP_ERR_INVALID_CONFIG, "matrices overlap");
    }
    const size_t m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
    Carver cv{(char *)workspace, 0};
    const NsParts p = carve(cv, count, m, n);
    if (!empty && (!workspace || !aligned16(workspace) || workspace_bytes < cv.used))
        return set_error(VHIP_ERR_INVALID_CONFIG, "the workspace is smaller than vhip_orthogonalize_workspace() (" +
                                                      std::to_string(cv.used) + " bytes) or not aligned to 16 bytes");
    CallDevice dev;
    VH_CHECK(dev.enter(ordinal));
    if (empty) return VHIP_OK;
    const NsCall k{in, count, rows, cols, ld_in, stride_in, steps, a, b, c, eps, scale, out, ld_out, stride_out};
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case VHIP_DTYPE_F32: return newton_schulz<float>(k, p, s);
        case VHIP_DTYPE_F16: return newton_schulz<half_t>(k, p, s);
        default: return newton_schulz<bf16_t>(k, p, s);
    }
}

}  // extern "C"
