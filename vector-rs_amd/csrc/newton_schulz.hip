// newton_schulz.hip -- orthogonalises update matrices by Newton-Schulz products.
//
//   X = M / (|M|_F + eps)  (of M^T where M has more rows than columns),  then `steps` times
//   A = X X^T,  B = a I + b A + c A A,  X <- B X
//
// which drives the singular values towards one while the singular vectors stay.  A direction whose singular
// value is small grows by `a` a step, and what rounding puts into it grows as much, so X, A and B are held
// as two float16 planes each (22 bits, mm16.h) and multiplied as three products with 32-bit sums: as exact as
// 32-bit products, at a third of the 16-bit matrix rate.  X is held times 2^10 and A and B times 2^8: the
// singular values stay below 2 for any useful coefficients, so neither leaves float16's range.
//
// A and A A are symmetric: only tiles on and above the diagonal are computed, and stored twice.  a X is part
// of B's diagonal.
#include "mm16.h"

#include <cmath>

namespace vh {
namespace {

constexpr float kXScale = 1024.f, kAScale = 256.f;
constexpr int kNormParts = 64;

__device__ __forceinline__ void split(float x, half_t &hi, half_t &lo) {
    hi = (half_t)x;
    lo = (half_t)(x - (float)hi);
}

// Partial sums of squares, in 64 bits: values of any magnitude neither overflow nor vanish.
template <class T>
__global__ __launch_bounds__(256) void k_ns_norm(const T *in, size_t rows, size_t cols, size_t ld, size_t stride,
                                                 double *part) {
    __shared__ double lds[4];
    const T *p = in + blockIdx.y * stride;
    double s = 0.0;
    const size_t n = rows * cols;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)kNormParts * 256) {
        const double v = (double)(float)p[i / cols * ld + i % cols];
        s += v * v;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.y * kNormParts + blockIdx.x] = lds[0] + lds[1] + lds[2] + lds[3];
}

struct Planes2 {
    half_t *p;
    size_t plane;  // from the high to the low plane
    size_t ld, stride;
};

// The scaled matrix x [m][np], zeros past n.
template <class T>
__global__ __launch_bounds__(256) void k_ns_start(const T *in, int rows, int cols, size_t ld, size_t stride, bool tall,
                                                  const double *part, float eps, Planes2 x) {
    __shared__ float tile[64][65];
    __shared__ float s_inv;
    if (threadIdx.x < 64) {
        double s = part[blockIdx.z * kNormParts + threadIdx.x];
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
        if (threadIdx.x == 0) s_inv = (float)((double)kXScale / (sqrt(s) + (double)eps));
    }
    __syncthreads();
    const float inv = s_inv;
    const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64, tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    const T *p = in + blockIdx.z * stride;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int r = r0 + ty + 4 * i, c = c0 + tx;
        const float v = r < rows && c < cols ? (float)p[(size_t)r * ld + c] * inv : 0.f;
        tile[tall ? tx : ty + 4 * i][tall ? ty + 4 * i : tx] = v;
    }
    __syncthreads();
    const int m0 = tall ? c0 : r0, n0 = tall ? r0 : c0, m = tall ? cols : rows;
    half_t *o = x.p + blockIdx.z * x.stride;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int r = m0 + ty + 4 * i, c = n0 + tx;
        if (r < m && (size_t)c < x.ld) {
            half_t hi, lo;
            split(tile[ty + 4 * i][tx], hi, lo);
            o[(size_t)r * x.ld + c] = hi;
            o[x.plane + (size_t)r * x.ld + c] = lo;
        }
    }
}

// A wave's blocks as both planes of rows [r0, rows) and columns [c0, ld).
template <int MB, int NB>
__device__ __forceinline__ void store_planes(const floatx4_t (&acc)[MB][NB], char *lds, half_t *p, size_t plane, size_t ld,
                                             int r0, int rows, int c0) {
    auto store = [=](half_t *to) {
        return [=](int r, int c, const Pack<half_t, 8> &v) {
            if (r0 + r < rows && (size_t)(c0 + c) < ld) *reinterpret_cast<Pack<half_t, 8> *>(to + (size_t)(r0 + r) * ld + c0 + c) = v;
        };
    };
    rows_through_lds<half_t, MB, NB>(lds, [&](int i, int j, int e) { return (half_t)acc[i][j][e]; }, store(p));
    rows_through_lds<half_t, MB, NB>(
        lds, [&](int i, int j, int e) { return (half_t)(acc[i][j][e] - (float)(half_t)acc[i][j][e]); }, store(p + plane));
}

// Epilogue of the symmetric products: out = alpha acc + beta add + diag I, stored at both places.
struct SymEpi {
    Planes2 out, add;  // add.p null: none
    float alpha, beta, diag;
    int m;
    template <int MB, int NB>
    __device__ void operator()(floatx4_t (&acc)[MB][NB], int mw, int nw, const MmPlace &pl, char *lds) const {
        const int l = threadIdx.x & 63, q = l >> 4;
        half_t *o = out.p + pl.batch * out.stride;
        const half_t *ad = add.p ? add.p + pl.batch * add.stride : nullptr;
        const bool mirror = pl.tm != pl.tn;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int c = nw + 16 * j + (l & 15);
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                const int r = mw + 16 * i + 4 * q;
                floatx4_t v = acc[i][j] * alpha;
                if (ad && c < m && (size_t)r < add.ld) {
                    const Pack<half_t, 4> h = *reinterpret_cast<const Pack<half_t, 4> *>(ad + (size_t)c * add.ld + r);
                    const Pack<half_t, 4> w = *reinterpret_cast<const Pack<half_t, 4> *>(ad + add.plane + (size_t)c * add.ld + r);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = fmaf(beta, (float)h.v[e] + (float)w.v[e], v[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = v[e] + (r + e == c ? diag : 0.f);
                    if (r + e >= m || c >= m) x = 0.f;
                    acc[i][j][e] = x;
                    if (mirror && r + e < m && (size_t)c < out.ld) {
                        half_t hi, lo;
                        split(x, hi, lo);
                        o[(size_t)(r + e) * out.ld + c] = hi;
                        o[out.plane + (size_t)(r + e) * out.ld + c] = lo;
                    }
                }
            }
        }
        store_planes(acc, lds, o, out.plane, out.ld, nw, m, mw);
    }
};

// Epilogue of B X: the next X (A operand X across, B operand B), or the result in the order that the A
// operand's rows have (B where the matrix is tall).
template <class T>
struct StepEpi {
    Planes2 x;
    float alpha;
    int cols, rows;  // of what is stored
    T *out;          // null: not the last step
    size_t ldo, so;
    bool vec;
    template <int MB, int NB>
    __device__ void operator()(floatx4_t (&acc)[MB][NB], int mw, int nw, const MmPlace &pl, char *lds) const {
        if (!out) {
            const int l = threadIdx.x & 63, q = l >> 4;
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int j = 0; j < NB; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = mw + 16 * i + 4 * q + e < cols ? acc[i][j][e] * alpha : 0.f;
            store_planes(acc, lds, x.p + pl.batch * x.stride, x.plane, x.ld, nw, rows, mw);
            return;
        }
        constexpr int PER = 16 / (int)sizeof(T);
        T *o = out + pl.batch * so;
        rows_through_lds<T, MB, NB>(
            lds, [&](int i, int j, int e) { return (T)(acc[i][j][e] * alpha); },
            [&](int r, int c, const Pack<T, PER> &v) {
                if (nw + r >= rows || mw + c >= cols) return;
                T *p = o + (size_t)(nw + r) * ldo + mw + c;
                if (vec && mw + c + PER <= cols) {
                    *reinterpret_cast<Pack<T, PER> *>(p) = v;
                } else {
#pragma unroll
                    for (int e = 0; e < PER; ++e)
                        if (mw + c + e < cols) p[e] = v.v[e];
                }
            });
    }
};

struct NsParts {
    double *norm;
    Planes2 x[2], a, b;
};

inline Planes2 planes(Carver &c, size_t count, size_t rows, size_t ld) {
    Planes2 p{};
    p.ld = ld;
    p.stride = rows * ld;
    p.plane = count * rows * ld;
    p.p = c.take<half_t>(2 * p.plane);
    return p;
}

inline NsParts carve(Carver &c, size_t count, size_t m, size_t n) {
    NsParts p{};
    const size_t mp = round_up(m, kMmK), np = round_up(n, kMmK);
    p.norm = c.take<double>(count * kNormParts);
    p.x[0] = planes(c, count, m, np);
    p.x[1] = planes(c, count, m, np);
    p.a = planes(c, count, m, mp);
    p.b = planes(c, count, m, mp);
    return p;
}

inline void operand(const Planes2 &p, const void *(&pl)[2], size_t &ld, size_t &stride) {
    pl[0] = p.p;
    pl[1] = p.p + p.plane;
    ld = p.ld;
    stride = p.stride;
}

// K rows of an operand across, or 0 where K is contiguous.
template <bool TA, bool TB, class Epi>
int multiply(const Planes2 &a, int M, const Planes2 &b, int N, int K, size_t count, bool upper, const Epi &epi, hipStream_t s) {
    MmArgs g{};
    operand(a, g.a, g.lda, g.sa);
    operand(b, g.b, g.ldb, g.sb);
    g.M = M;
    g.N = N;
    g.ktiles = ceil_div(K, kMmK);
    g.ka = g.kb = K;
    g.nseg = 3;
    g.ksplit = 1;
    g.batch = (int)count;
    g.upper = upper;
    return mm_launch<half_t, TA, TB>(g, mm_big_tiles(M, N, count, upper), epi, s);
}

struct NsCall {
    const void *in;
    size_t count, rows, cols, ldi, si;
    int steps;
    float a, b, c, eps;
    void *out;
    size_t ldo, so;
};

template <class T>
int newton_schulz(const NsCall &k, const NsParts &p, hipStream_t s) {
    const bool tall = k.rows > k.cols;
    const int m = (int)(tall ? k.cols : k.rows), n = (int)(tall ? k.rows : k.cols);
    const T *in = (const T *)k.in;
    k_ns_norm<T><<<dim3(kNormParts, (uint32_t)k.count), 256, 0, s>>>(in, k.rows, k.cols, k.ldi, k.si, p.norm);
    k_ns_start<T><<<dim3((uint32_t)ceil_div(k.rows, 64), (uint32_t)ceil_div(k.cols, 64), (uint32_t)k.count), 256, 0, s>>>(
        in, (int)k.rows, (int)k.cols, k.ldi, k.si, tall, p.norm, k.eps, p.x[0]);
    VH_CHECK(launch_status("orthogonalize launch"));
    for (int i = 0; i < k.steps; ++i) {
        const Planes2 &from = p.x[i & 1], &to = p.x[(i & 1) ^ 1];
        SymEpi ea{p.a, Planes2{}, kAScale / (kXScale * kXScale), 0.f, 0.f, m};
        VH_CHECK((multiply<false, false>)(from, m, from, m, n, k.count, true, ea, s));
        SymEpi eb{p.b, p.a, k.c / kAScale, k.b, k.a * kAScale, m};
        VH_CHECK((multiply<false, false>)(p.a, m, p.a, m, m, k.count, true, eb, s));
        StepEpi<T> es{to, 1.f / kAScale, n, m, nullptr, 0, 0, false};
        if (i + 1 < k.steps) {
            VH_CHECK((multiply<true, false>)(from, n, p.b, m, m, k.count, false, es, s));
            continue;
        }
        es.alpha /= kXScale;
        es.out = (T *)k.out;
        es.ldo = k.ldo;
        es.so = k.so;
        es.vec = k.ldo % (16 / sizeof(T)) == 0 && (k.count == 1 || k.so % (16 / sizeof(T)) == 0) && aligned16(k.out);
        if (tall) {
            es.cols = m;
            es.rows = n;
            VH_CHECK((multiply<false, true>)(p.b, m, from, n, m, k.count, false, es, s));
        } else {
            VH_CHECK((multiply<true, false>)(from, n, p.b, m, m, k.count, false, es, s));
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
    if (steps < 1 || steps > 100) return set_error(VHIP_ERR_INVALID_CONFIG, "steps must be in [1, 100]");
    if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return set_error(VHIP_ERR_INVALID_CONFIG, "coefficients must be finite");
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
    const NsCall k{in, count, rows, cols, ld_in, stride_in, steps, a, b, c, eps, out, ld_out, stride_out};
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case VHIP_DTYPE_F32: return newton_schulz<float>(k, p, s);
        case VHIP_DTYPE_F16: return newton_schulz<half_t>(k, p, s);
        default: return newton_schulz<bf16_t>(k, p, s);
    }
}

}  // extern "C"
