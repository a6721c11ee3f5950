// layer_norm.hip -- layer norm's forward and backward pass.
//
//   forward   mu = sum x / D,  v = sum (x - mu)^2 / D,  r = 1 / sqrt(v + eps),  y = (x - mu) r g + b
//   backward  xh = (x - mu) r,  a = dy g:  dx = r (a - mean(a) - xh mean(a xh)),
//             dg = sum over rows of dy xh,  db = sum over rows of dy
//
// Both passes are bound by memory. A row is held in the registers of the lanes that own it, so x (and dy) are
// read once: the variance is the mean of squares about the mean, not a difference of two sums, at no further
// read. The mean is rounded (values near 10^4: by 10^-3, a third of y where all are equal and eps is 10^-5), so
// the deviations from it are summed beside their squares, and their own mean, d, comes off: mu + d, sum (x -
// mu)^2 / D - d^2, y = (x - mu - d) r g + b (8192 x 4096 in bfloat16: 24.4 us, 23.6 without). Rows of up to 4
// vectors a lane belong to one wave (no barrier, four rows a workgroup), longer ones to a workgroup of 4 or 16
// waves; rows past that are walked in three passes (2048 x 16384 floats: 96 us forward, 153 backward). All sums
// are in 32 bits.
//
// The parameters' gradients are sums over all rows: each workgroup walks every gridDim-th row and keeps its
// columns' two sums in registers, which go to a row of the workspace at its end; a second kernel adds those
// rows in a fixed order, so the result does not depend on timing.
#include "train_common.h"

namespace vh {
namespace {

// Values of a lane's vector: 16 bytes of T, at whatever alignment the rows have.  TAIL: the row ends inside one.
template <class T>
constexpr int kVec = 16 / (int)sizeof(T);

template <int N, bool TAIL, class T>
__device__ __forceinline__ void load_vec(float (&o)[N], const T *row, int c, int dim) {
    const Pack<T, N> v = TAIL ? load_row<N>(row, c, dim) : load_any<N>(row + c);
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = (float)v.v[e];
}
template <int N, bool TAIL, class T>
__device__ __forceinline__ void store_vec(T *row, int c, int dim, const float (&o)[N]) {
    Pack<T, N> v;
#pragma unroll
    for (int e = 0; e < N; ++e) v.v[e] = (T)o[e];
    if (TAIL)
        store_row<N>(row, c, dim, v);
    else
        store_any<N>(row + c, v);
}

// Sum of a value over the G lanes that hold a row: a wave by itself, or through LDS.  `slot` alternates between
// two buffers, so one barrier a sum is enough: a buffer is written again only after the barrier of the sum
// between.  row_sums: of two values, in a buffer of their own.
template <int G>
__device__ __forceinline__ float row_sum(float x, float *lds, int slot) {
    x = lane_sum<64>(x);
    if constexpr (G > 64) {
        constexpr int W = G / 64;
        float *b = lds + (slot & 1) * W;
        if ((threadIdx.x & 63) == 0) b[threadIdx.x >> 6] = x;
        __syncthreads();
        x = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) x += b[w];
    }
    return x;
}

template <int G>
__device__ __forceinline__ float2 row_sums(float x, float y, float2 *lds) {
    x = lane_sum<64>(x);
    y = lane_sum<64>(y);
    if constexpr (G > 64) {
        constexpr int W = G / 64;
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = make_float2(x, y);
        __syncthreads();
        x = y = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            x += lds[w].x;
            y += lds[w].y;
        }
    }
    return make_float2(x, y);
}

// The mean's correction d and 1 / std from the sums of deviations and of their squares.
__device__ __forceinline__ float2 row_scale(float2 s, float n, float eps) {
    const float d = s.x * n, v = fmaf(-d, d, s.y * n);
    return make_float2(d, 1.f / sqrtf((v < 0.f ? 0.f : v) + eps));  // NaN stays
}

struct FwdArgs {
    const void *x, *weight, *bias;
    void *y;
    float *mean, *rstd;
    size_t rows, ldx, ldy;
    int dim;
    float eps;
};

template <class T, class P, int G, bool TAIL, int NV>
__global__ __launch_bounds__(G > 256 ? G : 256) void k_ln_forward(FwdArgs a) {
    constexpr int B = G > 256 ? G : 256, R = B / G, VEC = kVec<T>;
    __shared__ float lds[G / 64];
    __shared__ float2 lds2[G / 64];
    const size_t row = (size_t)blockIdx.x * R + threadIdx.x / G;
    if (row >= a.rows) return;  // G lanes at once: whole waves, and G > 64 has one row a workgroup
    const int t = threadIdx.x % G;
    const T *x = (const T *)a.x + row * a.ldx;
    const P *w = (const P *)a.weight, *b = (const P *)a.bias;
    float v[NV][VEC];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * G + t) * VEC;
        if (c < a.dim) {
            load_vec<VEC, TAIL>(v[i], x, c, a.dim);
#pragma unroll
            for (int e = 0; e < VEC; ++e) s += v[i][e];
        }
    }
    const float n = 1.f / (float)a.dim;
    const float mu = row_sum<G>(s, lds, 0) * n;
    float s2 = 0.f;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * G + t) * VEC;
        if (c < a.dim) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                v[i][e] = TAIL && c + e >= a.dim ? 0.f : v[i][e] - mu;
                s += v[i][e];
                s2 = fmaf(v[i][e], v[i][e], s2);
            }
        }
    }
    const float2 sc = row_scale(row_sums<G>(s, s2, lds2), n, a.eps);
    const float d = sc.x, r = sc.y;
    T *y = (T *)a.y + row * a.ldy;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * G + t) * VEC;
        if (c < a.dim) {
            float p[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[i][e] = (v[i][e] - d) * r;
            if (w) {
                load_vec<VEC, TAIL>(p, w, c, a.dim);
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[i][e] *= p[e];
            }
            if (b) {
                load_vec<VEC, TAIL>(p, b, c, a.dim);
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[i][e] += p[e];
            }
            store_vec<VEC, TAIL>(y, c, a.dim, v[i]);
        }
    }
    if (t == 0) {
        if (a.mean) a.mean[row] = mu + d;
        if (a.rstd) a.rstd[row] = r;
    }
}

// Rows of any length, one workgroup of 1024 each: the second and third walk find the row in the L2.
template <class T, class P>
__global__ __launch_bounds__(1024) void k_ln_forward_long(FwdArgs a) {
    __shared__ float lds[16];
    __shared__ float2 lds2[16];
    const size_t row = blockIdx.x;
    const T *x = (const T *)a.x + row * a.ldx;
    const P *w = (const P *)a.weight, *b = (const P *)a.bias;
    T *y = (T *)a.y + row * a.ldy;
    const float n = 1.f / (float)a.dim;
    float s = 0.f;
    for (int c = threadIdx.x; c < a.dim; c += 1024) s += (float)x[c];
    const float mu = row_sum<1024>(s, lds, 0) * n;
    float s2 = 0.f;
    s = 0.f;
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
        const float v = (float)x[c] - mu;
        s += v;
        s2 = fmaf(v, v, s2);
    }
    const float2 sc = row_scale(row_sums<1024>(s, s2, lds2), n, a.eps);
    const float d = sc.x, r = sc.y;
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
        float v = ((float)x[c] - mu - d) * r;
        if (w) v *= (float)w[c];
        if (b) v += (float)b[c];
        y[c] = (T)v;
    }
    if (threadIdx.x == 0) {
        if (a.mean) a.mean[row] = mu + d;
        if (a.rstd) a.rstd[row] = r;
    }
}

struct BwdArgs {
    const void *dy, *x, *weight;
    const float *mean, *rstd;
    void *dx;
    float *part;  // [2][parts][dim]: dg rows, then db rows; null where neither is wanted
    size_t rows, lddy, ldx, lddx;
    int dim, parts;
};

template <class T, class P, int G, bool TAIL, int NV>
__global__ __launch_bounds__(G > 256 ? G : 256) void k_ln_backward(BwdArgs a) {
    constexpr int B = G > 256 ? G : 256, R = B / G, VEC = kVec<T>;
    __shared__ float lds[4 * (G / 64)];
    const int t = threadIdx.x % G, sub = threadIdx.x / G;
    const P *w = (const P *)a.weight;
    const float n = 1.f / (float)a.dim;
    float g[NV][VEC], dg[NV][VEC], db[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * G + t) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) g[i][e] = 1.f, dg[i][e] = 0.f, db[i][e] = 0.f;
        if (w && c < a.dim) load_vec<VEC, TAIL>(g[i], w, c, a.dim);
    }
    int turn = 0;
    for (size_t row = (size_t)blockIdx.x * R + sub; row < a.rows; row += (size_t)gridDim.x * R, ++turn) {
        const T *x = (const T *)a.x + row * a.ldx, *dy = (const T *)a.dy + row * a.lddy;
        const float mu = a.mean[row], r = a.rstd[row];
        float xv[NV][VEC], d[NV][VEC];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + t) * VEC;
            if (c < a.dim) {
                load_vec<VEC, TAIL>(xv[i], x, c, a.dim);
                load_vec<VEC, TAIL>(d[i], dy, c, a.dim);
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if ((i * G + t) * VEC < a.dim) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    xv[i][e] = (xv[i][e] - mu) * r;
                    dg[i][e] = fmaf(d[i][e], xv[i][e], dg[i][e]);
                    db[i][e] += d[i][e];
                    d[i][e] *= g[i][e];
                    s1 += d[i][e];
                    s2 = fmaf(d[i][e], xv[i][e], s2);
                }
            }
        }
        if (!a.dx) continue;
        s1 = lane_sum<64>(s1);
        s2 = lane_sum<64>(s2);
        if constexpr (G > 64) {
            constexpr int W = G / 64;
            float *b = lds + (turn & 1) * 2 * W;
            if ((threadIdx.x & 63) == 0) {
                b[threadIdx.x >> 6] = s1;
                b[W + (threadIdx.x >> 6)] = s2;
            }
            __syncthreads();
            s1 = s2 = 0.f;
#pragma unroll
            for (int k = 0; k < W; ++k) {
                s1 += b[k];
                s2 += b[W + k];
            }
        }
        s1 *= n;
        s2 *= n;
        T *dx = (T *)a.dx + row * a.lddx;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + t) * VEC;
            if (c < a.dim) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) d[i][e] = r * (d[i][e] - s1 - xv[i][e] * s2);
                store_vec<VEC, TAIL>(dx, c, a.dim, d[i]);
            }
        }
    }
    if (!a.part) return;
    if constexpr (R == 1) {
        float *pg = a.part + (size_t)blockIdx.x * a.dim, *pb = pg + (size_t)a.parts * a.dim;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + t) * VEC;
            if (c < a.dim) {
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (!TAIL || c + e < a.dim) pg[c + e] = dg[i][e], pb[c + e] = db[i][e];
            }
        }
    } else {
        // the workgroup's rows (one a wave) are added in LDS, one vector of columns after the other
        __shared__ float sums[R][2][64 * VEC];
        float *pg = a.part + (size_t)blockIdx.x * a.dim, *pb = pg + (size_t)a.parts * a.dim;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                sums[sub][0][t * VEC + e] = dg[i][e];
                sums[sub][1][t * VEC + e] = db[i][e];
            }
            __syncthreads();
            for (int k = threadIdx.x; k < 64 * VEC; k += B) {
                const int c = i * 64 * VEC + k;
                if (c < a.dim) {
                    float u = 0.f, v = 0.f;
#pragma unroll
                    for (int q = 0; q < R; ++q) {
                        u += sums[q][0][k];
                        v += sums[q][1][k];
                    }
                    pg[c] = u;
                    pb[c] = v;
                }
            }
            __syncthreads();
        }
    }
}

// dx of rows of any length.
template <class T, class P>
__global__ __launch_bounds__(1024) void k_ln_backward_long(BwdArgs a) {
    __shared__ float lds[2 * 16];
    const size_t row = blockIdx.x;
    const T *x = (const T *)a.x + row * a.ldx, *dy = (const T *)a.dy + row * a.lddy;
    const P *w = (const P *)a.weight;
    const float n = 1.f / (float)a.dim, mu = a.mean[row], r = a.rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
        const float d = (float)dy[c] * (w ? (float)w[c] : 1.f);
        s1 += d;
        s2 = fmaf(d, ((float)x[c] - mu) * r, s2);
    }
    s1 = row_sum<1024>(s1, lds, 0) * n;
    s2 = row_sum<1024>(s2, lds, 1) * n;
    T *dx = (T *)a.dx + row * a.lddx;
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
        const float d = (float)dy[c] * (w ? (float)w[c] : 1.f);
        dx[c] = (T)(r * (d - s1 - ((float)x[c] - mu) * r * s2));
    }
}

// The parameters' sums of long rows: a workgroup takes 256 columns and every gridDim.y-th row.
template <class T>
__global__ __launch_bounds__(256) void k_ln_columns(BwdArgs a) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.dim) return;
    float dg = 0.f, db = 0.f;
    for (size_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float d = (float)((const T *)a.dy)[row * a.lddy + c];
        const float xh = ((float)((const T *)a.x)[row * a.ldx + c] - a.mean[row]) * a.rstd[row];
        dg = fmaf(d, xh, dg);
        db += d;
    }
    a.part[(size_t)blockIdx.y * a.dim + c] = dg;
    a.part[((size_t)a.parts + blockIdx.y) * a.dim + c] = db;
}

// Adds the workspace's rows: 32 columns a workgroup, its 32 groups of lanes every 32nd row, four loads in
// flight (16384 x 2048: 37.7 us with 8 groups and one load).
template <class P>
__global__ __launch_bounds__(1024) void k_ln_reduce(const float *part, int parts, int dim, P *dweight, P *dbias) {
    __shared__ float sums[32][33];
    const int l = threadIdx.x & 31, c = blockIdx.x * 32 + l, g = threadIdx.x >> 5;
    P *out = blockIdx.y ? dbias : dweight;
    if (!out) return;
    const float *p = part + (size_t)blockIdx.y * parts * dim + c;
    float s = 0.f;
    if (c < dim) {
        int k = g;
        float u[4] = {0.f, 0.f, 0.f, 0.f};
        for (; k + 96 < parts; k += 128) {
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] += p[(size_t)(k + 32 * i) * dim];
        }
        for (; k < parts; k += 32) u[0] += p[(size_t)k * dim];
        s = (u[0] + u[1]) + (u[2] + u[3]);
    }
    sums[g][l] = s;
    __syncthreads();
    // group g adds column g's 32 sums
    s = sums[l][g];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) s += __shfl_xor(s, o, 32);
    if (l == 0 && blockIdx.x * 32 + g < dim) out[blockIdx.x * 32 + g] = (P)s;
}

// Workgroups of the backward pass, each with one row of partial sums: enough that every CU has eight waves
// or more in flight, few enough that the partial sums stay a small part of what is read.
constexpr size_t kParts = 512;
inline int ln_parts(size_t rows, int rows_per_wg) {
    const size_t wgs = (rows + rows_per_wg - 1) / rows_per_wg;
    return (int)(wgs < kParts ? (wgs ? wgs : 1) : kParts);
}

// The lanes and vectors that hold a row: one wave or 4 waves up to 4 vectors a lane, 16 waves up to 2 (the
// backward pass keeps five values an element, and 16 waves have 128 registers a lane); 0 where the row is
// longer.
struct Shape {
    int group, nv;
};
inline Shape ln_shape(size_t dim, int vec) {
    for (int g : {64, 256, 1024}) {
        const size_t nv = (dim + (size_t)g * vec - 1) / ((size_t)g * vec);
        if (nv <= (g == 1024 ? 2 : 4)) return {g, (int)nv};
    }
    return {0, 0};
}

#define LN_DISPATCH(KERNEL, T, P, TAIL)                                      \
    switch (sh.group * 8 + sh.nv) {                                          \
        case 64 * 8 + 1: LN_LAUNCH((KERNEL<T, P, 64, TAIL, 1>), 64); break;   \
        case 64 * 8 + 2: LN_LAUNCH((KERNEL<T, P, 64, TAIL, 2>), 64); break;   \
        case 64 * 8 + 3: LN_LAUNCH((KERNEL<T, P, 64, TAIL, 3>), 64); break;   \
        case 64 * 8 + 4: LN_LAUNCH((KERNEL<T, P, 64, TAIL, 4>), 64); break;   \
        case 256 * 8 + 1: LN_LAUNCH((KERNEL<T, P, 256, TAIL, 1>), 256); break; \
        case 256 * 8 + 2: LN_LAUNCH((KERNEL<T, P, 256, TAIL, 2>), 256); break; \
        case 256 * 8 + 3: LN_LAUNCH((KERNEL<T, P, 256, TAIL, 3>), 256); break; \
        case 256 * 8 + 4: LN_LAUNCH((KERNEL<T, P, 256, TAIL, 4>), 256); break; \
        case 1024 * 8 + 1: LN_LAUNCH((KERNEL<T, P, 1024, TAIL, 1>), 1024); break; \
        default: LN_LAUNCH((KERNEL<T, P, 1024, TAIL, 2>), 1024); break;       \
    }

template <class T, class P>
int forward(const FwdArgs &a, hipStream_t s) {
    const Shape sh = ln_shape(a.dim, kVec<T>);
    if (!sh.group) {
        if (a.rows > 0x7fffffff) return set_error(VHIP_ERR_INVALID_CONFIG, "too many rows");
        k_ln_forward_long<T, P><<<(uint32_t)a.rows, 1024, 0, s>>>(a);
        return launch_status("layer norm launch");
    }
    const int per = sh.group == 64 ? 4 : 1;
    const size_t grid = (a.rows + per - 1) / per;
    if (grid > 0x7fffffff) return set_error(VHIP_ERR_INVALID_CONFIG, "too many rows");
#define LN_LAUNCH(K, G) K<<<(uint32_t)grid, G > 256 ? G : 256, 0, s>>>(a)
    if (a.dim % kVec<T>) {
        LN_DISPATCH(k_ln_forward, T, P, true)
    } else {
        LN_DISPATCH(k_ln_forward, T, P, false)
    }
#undef LN_LAUNCH
    return launch_status("layer norm launch");
}

template <class T, class P>
int backward(BwdArgs a, P *dweight, P *dbias, float *ws, hipStream_t s) {
    const bool sums = dweight || dbias;
    const Shape sh = ln_shape(a.dim, kVec<T>);
    a.part = sums ? ws : nullptr;
    if (a.rows == 0) {
        a.parts = 0;  // the sums of no rows
    } else if (!sh.group) {
        if (a.rows > 0x7fffffff) return set_error(VHIP_ERR_INVALID_CONFIG, "too many rows");
        if (a.dx) k_ln_backward_long<T, P><<<(uint32_t)a.rows, 1024, 0, s>>>(a);
        if (sums) {
            a.parts = (int)(a.rows < 64 ? a.rows : 64);
            k_ln_columns<T><<<dim3((uint32_t)ceil_div(a.dim, 256), a.parts), 256, 0, s>>>(a);
        }
    } else {
        a.parts = ln_parts(a.rows, sh.group == 64 ? 4 : 1);
#define LN_LAUNCH(K, G) K<<<(uint32_t)a.parts, G > 256 ? G : 256, 0, s>>>(a)
        if (a.dim % kVec<T>) {
            LN_DISPATCH(k_ln_backward, T, P, true)
        } else {
            LN_DISPATCH(k_ln_backward, T, P, false)
        }
#undef LN_LAUNCH
    }
    if (sums)
        k_ln_reduce<P><<<dim3((uint32_t)ceil_div(a.dim, 32), 2), 1024, 0, s>>>(a.part, a.parts, a.dim, dweight, dbias);
    return launch_status("layer norm launch");
}

int check_types(int dtype, int param_dtype) {
    if (!dtype_known(dtype)) return set_error(VHIP_ERR_INVALID_CONFIG, "unknown element type " + std::to_string(dtype));
    if (param_dtype != dtype && param_dtype != VHIP_DTYPE_F32)
        return set_error(VHIP_ERR_INVALID_CONFIG, "parameters are of the rows' type or f32");
    return VHIP_OK;
}

int check_rows(const char *name, const void *p, size_t rows, size_t dim, size_t ld) {
    if (rows && !p) return set_error(VHIP_ERR_INVALID_CONFIG, std::string(name) + " is null");
    if (ld < dim) return set_error(VHIP_ERR_INVALID_CONFIG, std::string(name) + ": rows are closer than dim");
    return VHIP_OK;
}

}  // namespace
}  // namespace vh

using namespace vh;

extern "C" {

int vhip_layer_norm(int ordinal, int dtype, int param_dtype, const void *x, size_t rows, size_t dim, size_t ldx,
                    const void *weight, const void *bias, float eps, void *y, size_t ldy, float *mean, float *rstd,
                    void *stream) {
    clear_error();
    VH_CHECK(check_types(dtype, param_dtype));
    if (dim == 0 || dim > 0x3fffffff) return set_error(VHIP_ERR_INVALID_CONFIG, "dim must be in [1, 2^30)");
    if (!(eps >= 0.f)) return set_error(VHIP_ERR_INVALID_CONFIG, "eps must be >= 0");
    VH_CHECK(check_rows("x", x, rows, dim, ldx));
    VH_CHECK(check_rows("y", y, rows, dim, ldy));
    CallDevice dev;
    VH_CHECK(dev.enter(ordinal));
    if (rows == 0) return VHIP_OK;
    const FwdArgs a{x, weight, bias, y, mean, rstd, rows, ldx, ldy, (int)dim, eps};
    hipStream_t s = (hipStream_t)stream;
    const bool f32p = param_dtype == VHIP_DTYPE_F32;
    switch (dtype) {
        case VHIP_DTYPE_F32: return forward<float, float>(a, s);
        case VHIP_DTYPE_F16: return f32p ? forward<half_t, float>(a, s) : forward<half_t, half_t>(a, s);
        default: return f32p ? forward<bf16_t, float>(a, s) : forward<bf16_t, bf16_t>(a, s);
    }
}

size_t vhip_layer_norm_backward_workspace(size_t rows, size_t dim) {
    return 2 * sizeof(float) * dim * (rows < kParts ? rows : kParts);
}

int vhip_layer_norm_backward(int ordinal, int dtype, int param_dtype, const void *dy, size_t lddy, const void *x,
                             size_t ldx, const void *weight, const float *mean, const float *rstd, size_t rows,
                             size_t dim, void *dx, size_t lddx, void *dweight, void *dbias, void *workspace,
                             size_t workspace_bytes, void *stream) {
    clear_error();
    VH_CHECK(check_types(dtype, param_dtype));
    if (dim == 0 || dim > 0x3fffffff) return set_error(VHIP_ERR_INVALID_CONFIG, "dim must be in [1, 2^30)");
    VH_CHECK(check_rows("dy", dy, rows, dim, lddy));
    VH_CHECK(check_rows("x", x, rows, dim, ldx));
    if (dx) VH_CHECK(check_rows("dx", dx, rows, dim, lddx));
    if (rows && (!mean || !rstd)) return set_error(VHIP_ERR_INVALID_CONFIG, "mean and rstd are needed");
    if ((dweight || dbias) && rows &&
        (!workspace || workspace_bytes < vhip_layer_norm_backward_workspace(rows, dim) || ((uintptr_t)workspace & 3)))
        return set_error(VHIP_ERR_INVALID_CONFIG,
                         "the workspace is smaller than vhip_layer_norm_backward_workspace() or not aligned");
    CallDevice dev;
    VH_CHECK(dev.enter(ordinal));
    if (!dx && !dweight && !dbias) return VHIP_OK;
    const BwdArgs a{dy, x, weight, mean, rstd, dx, nullptr, rows, lddy, ldx, lddx, (int)dim, 0};
    hipStream_t s = (hipStream_t)stream;
    float *ws = (float *)workspace;
    const bool f32p = param_dtype == VHIP_DTYPE_F32;
    switch (dtype) {
        case VHIP_DTYPE_F32: return backward<float, float>(a, (float *)dweight, (float *)dbias, ws, s);
        case VHIP_DTYPE_F16:
            return f32p ? backward<half_t, float>(a, (float *)dweight, (float *)dbias, ws, s)
                        : backward<half_t, half_t>(a, (half_t *)dweight, (half_t *)dbias, ws, s);
        default:
            return f32p ? backward<bf16_t, float>(a, (float *)dweight, (float *)dbias, ws, s)
                        : backward<bf16_t, bf16_t>(a, (bf16_t *)dweight, (bf16_t *)dbias, ws, s);
    }
}

}  // extern "C"
