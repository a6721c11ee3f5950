// xent_small.h -- softmax cross entropy of few rows (included by softmax_xent.hip).
//
// With few rows the table is what costs: the products of softmax_xent.hip would run tiles that are mostly
// clamped rows, and 32-bit tables would first be turned into planes.  Here the table is read from memory
// straight into matrix operands, twice in all for the gradients:
//  * k_small_stat makes the logits, and keeps them where gradients follow (64 rows of them are less than a
//    table of 64 columns).  A workgroup takes 16 or 32 entries at a time; its four waves share the K loop, so a CU
//    has enough loads in flight for short tables too.  32-bit operands are multiplied as they are, in the
//    32-bit matrix instruction (157 TFLOP/s: above the memory's rate up to 48 rows).
//  * k_small_grad turns 32 entries' logits into G in LDS, writes these entries' rows of the table's gradient
//    and adds the rows' gradient up in registers; the workgroups' sums are joined afterwards.  G is not
//    rounded here, and 16-bit operands are widened.
#pragma once

#include "mm16.h"

namespace vh {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;
__device__ __forceinline__ float exp_neg(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
// exp to 32-bit accuracy: what x log2(e) loses in rounding is put back to first order
__device__ __forceinline__ float exp_fine(float x) {
    const float t = x * kLog2e;
    const float r = fmaf(x, kLog2e, -t) + x * 1.925963033500e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    return t > -150.f && t < 128.f ? fmaf(e, r * 0.693147182f, e) : e;
}

// Whether a call takes this way.  32-bit rows, tiles / this way in us, loss and with gradients: 16 x 10000 x 128
// 26, 72 / 15, 25; 64 x 10000 x 768 50, 101 / 27, 78; 64 x 200003 x 300 272, 536 / 119, 423; 64 x 131072 x 1024
// 475, 817 / 263, 738; 100 x 50000 x 512 90, 208 / 115, 350.  16-bit rows, whose tables the tiles read as they
// are: 16 x 10000 x 128 15, 42 / 14, 24; 32 x 10000 x 768 17, 56 / 15, 50; 64 x 10000 x 768 18, 58 / 17, 68;
// 16 x 131072 x 1024 55, 230 / 69, 286: only while launches are what counts.
constexpr size_t kSmallRows = 64, kSmallWork16 = 250'000'000;
inline bool few_rows(int dtype, size_t rows, size_t table, size_t dim) {
    return rows <= kSmallRows && (dtype == VHIP_DTYPE_F32 || rows * table * dim <= kSmallWork16);
}

// Entries of a workgroup's turn.  The rows are read from the caches again for each turn: from 17 rows on with
// more of them than of the table, so a turn takes 32 entries, where enough turns for every CU are left
// (float32, 16 / 32 entries, us: 32 x 95296 x 731 129, 97; 64 x 95296 x 768 194, 148; 32 x 40000 x 768 52, 39;
// 64 x 20000 x 256 24, 20; 17 x 10000 x 768 19, 20; bfloat16: 40 x 30000 x 200 16.0, 14.7; 17 x 200000 x 64 20.7, 19.7;
// 32 x 100000 x 64 15.8, 14.9; up to 20,000 entries both are the time of the call).
inline size_t small_turn(size_t rows, size_t table) { return rows > 16 && table >= 8192 ? 32 : 16; }

// Values of one lane in a K step of the logits.
template <class T>
struct SmallStep {
    typedef typename MmVec<T>::v8 vec;
    static constexpr int E = 8, K = 32;
    static __device__ __forceinline__ floatx4_t mfma(vec a, vec b, floatx4_t c) { return MmVec<T>::mfma(a, b, c); }
};
template <>
struct SmallStep<float> {
    typedef floatx4_t vec;
    static constexpr int E = 4, K = 16;
    static __device__ __forceinline__ floatx4_t mfma(vec a, vec b, floatx4_t c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};

// E values of a row from column c on; TAIL: zeros past dim.
template <class T, bool TAIL>
__device__ __forceinline__ typename SmallStep<T>::vec small_load(const T *row, int c, int dim) {
    constexpr int E = SmallStep<T>::E;
    return __builtin_bit_cast(typename SmallStep<T>::vec, TAIL ? load_row<E>(row, c, dim) : load_any<E>(row + c));
}

struct SmallStat {
    const void *h, *w;
    const float *bias;
    const int64_t *target;
    float2 *part, *zt;
    float *z;  // [rows][vp], null: not kept
    size_t ldh, ldw, vp;
    int rows, table, dim;
    float scale;
};

template <class T, int NB, int GB>  // blocks of 16 rows, of 16 entries of a turn
__global__ __launch_bounds__(256) void k_small_stat(SmallStat a) {
    typedef SmallStep<T> S;
    constexpr int BUFS = GB == 1 ? 2 : 1;
    __shared__ floatx4_t s_acc[BUFS][4][NB][GB][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
    const T *hr[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) hr[j] = (const T *)a.h + (size_t)min(16 * j + i, a.rows - 1) * a.ldh;
    const int steps = a.dim / S::K;  // whole ones
    // wave w ends rows 16 w .. 16 w + 15
    const int t = 16 * wave + i;
    const bool mine = wave < NB && t < a.rows;
    const int64_t y = mine ? a.target[t] : -1;
    float top = -INFINITY, sum = 0.f;
    int buf = 0;
    const int groups = (a.table + 16 * GB - 1) / (16 * GB);
    for (int g = blockIdx.x; g < groups; g += gridDim.x) {
        const T *wr[GB];
#pragma unroll
        for (int b = 0; b < GB; ++b) wr[b] = (const T *)a.w + (size_t)min(16 * (GB * g + b) + i, a.table - 1) * a.ldw;
        floatx4_t acc[NB][GB];
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int b = 0; b < GB; ++b) acc[j][b] = floatx4_t{0.f, 0.f, 0.f, 0.f};
        auto step = [&](int c, auto tail) {
            constexpr bool TAIL = decltype(tail)::value;
            typename S::vec x[GB];
#pragma unroll
            for (int b = 0; b < GB; ++b) x[b] = small_load<T, TAIL>(wr[b], c, a.dim);
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const typename S::vec y = small_load<T, TAIL>(hr[j], c, a.dim);
#pragma unroll
                for (int b = 0; b < GB; ++b) acc[j][b] = S::mfma(x[b], y, acc[j][b]);
            }
        };
#pragma unroll 4
        for (int s = wave; s < steps; s += 4) step(s * S::K + q * S::E, std::false_type());
        if (steps * S::K < a.dim && wave == (steps & 3)) step(steps * S::K + q * S::E, std::true_type());
        if (BUFS == 1) __syncthreads();  // the last turn's sums are read
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int b = 0; b < GB; ++b) s_acc[buf][wave][j][b][lane] = acc[j][b];
        __syncthreads();  // with two buffers the other one is written next: one barrier a turn is enough
        const int from = buf;
        buf = (buf + 1) % BUFS;
        if (wave >= NB) continue;
#pragma unroll
        for (int b = 0; b < GB; ++b) {
            const floatx4_t v = (s_acc[from][0][wave][b][lane] + s_acc[from][1][wave][b][lane]) +
                                (s_acc[from][2][wave][b][lane] + s_acc[from][3][wave][b][lane]);
            const int e0 = 16 * (GB * g + b) + 4 * q;
            floatx4_t z;
            float m = top;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float off = e0 + e < a.table ? (a.bias ? a.bias[e0 + e] : 0.f) : -INFINITY;
                z[e] = off == -INFINITY ? -INFINITY : fmaf(v[e], a.scale, off);
                m = fmaxf(m, z[e]);
            }
            const float about = m == -INFINITY ? 0.f : m;
            sum *= exp_neg(top - about);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += e0 + e == y ? 0.f : exp_neg(z[e] - about);
            top = m;
            if (mine) {
                if (a.z) *reinterpret_cast<floatx4_t *>(a.z + (size_t)t * a.vp + e0) = z;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e0 + e == y && e0 + e < a.table) a.zt[t] = make_float2(z[e], 0.f);
            }
        }
    }
    if (wave >= NB) return;
#pragma unroll
    for (int o = 16; o < 64; o <<= 1) {
        const float m2 = __shfl_xor(top, o, 64), s2 = __shfl_xor(sum, o, 64), m = fmaxf(top, m2);
        const float about = m == -INFINITY ? 0.f : m;
        sum = sum * exp_neg(top - about) + s2 * exp_neg(m2 - about);
        top = m;
    }
    if (mine && q == 0) a.part[(size_t)blockIdx.x * a.rows + t] = make_float2(top, sum);
}

struct SmallGrad {
    const void *h, *w;
    const float *bias, *z;
    const float2 *stat, *rowfac;
    const int64_t *target;
    void *dtable;  // null: not wanted
    float *part;   // [gridDim.x][rows][cols4], null: the rows' gradient is not wanted
    size_t ldh, ldw, ldo, vp;
    int rows, table, dim, cols4;
};

constexpr int kSmallCols = 128;    // columns of a workgroup
constexpr int kSmallEntries = 32;  // entries of a turn

// Wave w: entries 16 (w & 1) .. of a turn, columns 64 (w >> 1) .. of the workgroup's.
template <class T, int TB, bool TAIL>  // TAIL: rows end inside four columns
__global__ __launch_bounds__(256) void k_small_grad(SmallGrad a) {
    constexpr int R = 16 * TB, NV = kSmallEntries, GP = NV + 4, HP = kSmallCols + 4, NZ = R * NV / 256;
    __shared__ __align__(16) float s_g[R * GP], s_h[R * HP];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 15, q = lane >> 4;
    const int sub = 16 * (wave & 1), cw = 64 * (wave >> 1), d0 = blockIdx.y * kSmallCols;

    // four columns of a row, zeros where it does not count
    auto four = [&](float (&o)[4], const T *row, int col, bool on) {
        Pack<T, 4> p{};
        if (TAIL)
            p = load_row<4>(row, col, a.dim);
        else if (col < a.dim)
            p = load_any<4>(row + col);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = on ? (float)p.v[e] : 0.f;
    };
    // this thread's logits of a turn: rows tz + 8 k, entry vz
    const int tz = tid / NV, vz = tid % NV;
    float zr[NZ], wr[4][4];
    auto fetch = [&](int v0) {
#pragma unroll
        for (int k = 0; k < NZ; ++k) {
            const int t = tz + 256 / NV * k;
            zr[k] = t < a.rows && v0 + vz < a.table ? a.z[(size_t)t * a.vp + v0 + vz] : -INFINITY;
        }
        if (!a.part) return;
        const int col = d0 + cw + 4 * i;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int v = v0 + sub + 4 * q + k;
            const bool on = v < a.table && !(a.bias && a.bias[v] == -INFINITY);
            four(wr[k], (const T *)a.w + (size_t)(on ? v : 0) * a.ldw, col, on);
        }
    };
    fetch(blockIdx.x * NV);
    float cs[NZ], cc[NZ], cy[NZ], about[NZ];
    int yy[NZ];
#pragma unroll
    for (int k = 0; k < NZ; ++k) {
        const int t = tz + 256 / NV * k;
        const bool in = t < a.rows;
        const float2 st = in ? a.stat[t] : make_float2(0.f, 0.f);
        const int64_t y = in ? a.target[t] : -1;
        const float2 fac = in ? a.rowfac[t] : make_float2(0.f, 0.f);
        cc[k] = fac.x;
        cy[k] = fac.y;
        cs[k] = cc[k] * st.y;
        about[k] = st.x;
        yy[k] = y < a.table ? (int)y : -1;
    }
    // h of the workgroup's columns, zeros in rows that do not count: every load before the first store
    constexpr int HV = kSmallCols / 4, NH = R * HV / 256;
    float hr[NH][4];
#pragma unroll
    for (int k = 0; k < NH; ++k) {
        const int t = tid / HV + 256 / HV * k, col = d0 + tid % HV * 4;
        const int in = min(t, a.rows - 1);
        four(hr[k], (const T *)a.h + (size_t)in * a.ldh, col, t < a.rows && a.rowfac[in].y != 0.f);
    }
#pragma unroll
    for (int k = 0; k < NH; ++k)
        *reinterpret_cast<floatx4_t *>(s_h + (tid / HV + 256 / HV * k) * HP + tid % HV * 4) = floatx4_t{hr[k][0], hr[k][1], hr[k][2], hr[k][3]};
    floatx4_t dh[TB][4];
#pragma unroll
    for (int j = 0; j < TB; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) dh[j][e] = floatx4_t{0.f, 0.f, 0.f, 0.f};

    // A wave's 64 columns are four MFMA blocks: block e's row r is column 4 r + e, so that operands and
    // results are four neighbouring columns a lane.
    for (int v0 = blockIdx.x * NV; v0 < a.table; v0 += gridDim.x * NV) {
        __syncthreads();  // s_h (first turn), the last turn's s_g
#pragma unroll
        for (int k = 0; k < NZ; ++k) {
            float g = 0.f;
            if (cc[k] != 0.f) g = v0 + vz == yy[k] ? -cy[k] : cs[k] * exp_fine(zr[k] - about[k]);
            if (v0 + vz >= a.table) g = 0.f;
            s_g[(tz + 256 / NV * k) * GP + vz] = g;
        }
        __syncthreads();
        if (a.part) {
            floatx4_t g[TB];  // rows 16 j + i, entries sub + 4 q ..
#pragma unroll
            for (int j = 0; j < TB; ++j) g[j] = *reinterpret_cast<const floatx4_t *>(s_g + (16 * j + i) * GP + sub + 4 * q);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int j = 0; j < TB; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        dh[j][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(wr[k][e], g[j][k], dh[j][e], 0, 0, 0);
        }
        if (v0 + gridDim.x * NV < (size_t)a.table) fetch(v0 + gridDim.x * NV);
        if (!a.dtable || d0 + cw >= a.dim) continue;
        floatx4_t dw[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) dw[e] = floatx4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4 * TB; ++k) {
            const floatx4_t x = *reinterpret_cast<const floatx4_t *>(s_h + (4 * k + q) * HP + cw + 4 * i);
            const float g = s_g[(4 * k + q) * GP + sub + i];
#pragma unroll
            for (int e = 0; e < 4; ++e) dw[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], g, dw[e], 0, 0, 0);
        }
        const int v = v0 + sub + i;
        if (v >= a.table) continue;
        T *o = (T *)a.dtable + (size_t)v * a.ldo;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int col = d0 + cw + 16 * q + 4 * x;
            Pack<T, 4> p;
#pragma unroll
            for (int e = 0; e < 4; ++e) p.v[e] = (T)dw[e][x];
            if (TAIL)
                store_row<4>(o, col, a.dim, p);
            else if (col < a.dim)
                store_any<4>(o + col, p);
        }
    }
    if (!a.part) return;
    // the two waves of a column range, one after the other
    for (int w = 0; w < 2; ++w) {
        __syncthreads();
        if ((wave & 1) != w) continue;
#pragma unroll
        for (int j = 0; j < TB; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                floatx4_t *p = reinterpret_cast<floatx4_t *>(s_h + (16 * j + i) * HP + cw + 16 * q + 4 * x);
                const floatx4_t v = {dh[j][0][x], dh[j][1][x], dh[j][2][x], dh[j][3][x]};
                *p = w == 0 ? v : *p + v;
            }
    }
    __syncthreads();
    for (int k = tid; k < a.rows * (kSmallCols / 4); k += 256) {
        const int t = k / (kSmallCols / 4), c = k % (kSmallCols / 4) * 4;
        if (d0 + c < a.cols4)
            *reinterpret_cast<floatx4_t *>(a.part + ((size_t)blockIdx.x * a.rows + t) * a.cols4 + d0 + c) =
                *reinterpret_cast<const floatx4_t *>(s_h + t * HP + c);
    }
}

template <class T>
void small_stat(const SmallStat &a, uint32_t grid, hipStream_t s) {
    const bool two = small_turn(a.rows, a.table) == 32;
    if (a.rows <= 16)
        k_small_stat<T, 1, 1><<<grid, 256, 0, s>>>(a);
    else if (a.rows <= 32)
        two ? k_small_stat<T, 2, 2><<<grid, 256, 0, s>>>(a) : k_small_stat<T, 2, 1><<<grid, 256, 0, s>>>(a);
    else if (two && a.rows <= 48)
        k_small_stat<T, 3, 2><<<grid, 256, 0, s>>>(a);
    else
        two ? k_small_stat<T, 4, 2><<<grid, 256, 0, s>>>(a) : k_small_stat<T, 4, 1><<<grid, 256, 0, s>>>(a);
}

template <class T>
void small_grad(const SmallGrad &a, uint32_t gx, hipStream_t s) {
    const dim3 grid(gx, (uint32_t)ceil_div(a.dim, kSmallCols));
#define SMALL_GRAD(TB)                                             \
    if (a.dim % 4)                                                 \
        k_small_grad<T, TB, true><<<grid, 256, 0, s>>>(a);         \
    else                                                           \
        k_small_grad<T, TB, false><<<grid, 256, 0, s>>>(a);
    if (a.rows <= 16) {
        SMALL_GRAD(1)
    } else if (a.rows <= 32) {
        SMALL_GRAD(2)
    } else {
        SMALL_GRAD(4)
    }
#undef SMALL_GRAD
}

}  // namespace
}  // namespace vh
