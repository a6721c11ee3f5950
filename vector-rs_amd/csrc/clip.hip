// clip.hip -- the norm of many arrays together, and their values scaled to a largest norm.
//
//   norm = sqrt(sum over all arrays of g^2),  c = min(1, max_norm / (norm + eps)),  out = c g
//
// Bound by memory: every value is read once for the norm and, where it is scaled, once more (the norm has to be known
// first) and written. Two kernels: the first leaves a sum for each workgroup, the second adds all of these up in each of
// its workgroups (16 KB at most, from the caches), which spares a launch between. Squares and sums are in 64 bits, where
// a square of any value is exact or nearly so: 32 bits would overflow from 1.8e19 on and lose everything below 1e-19.
// Sums are in a fixed order, so the norm does not depend on timing.
//
// The arrays' places go with the launch as kernel arguments, so nothing is copied to the device or kept there; more arrays
// than fit take more launches. A launch's values are cut into chunks of one vector a thread, an array beginning with
// a chunk of its own, and every workgroup takes a contiguous run of chunks, four vectors of a thread in flight.
//
// 456M values in bfloat16 (0.9 GB read twice, 0.9 written): 555 us, 4.9 TB/s; 594 with one vector in flight in the second kernel.
#include <algorithm>
#include <new>
#include <vector>

#include "train_common.h"

namespace vh {
namespace {

constexpr int kArrays = 112;     // of a launch: its arguments stay below 4 KB
constexpr int kChunk = 2048;     // values
constexpr int kParts = 2048;     // workgroups of all launches together, and one more for each launch

struct Array {
    const void *in;
    void *out;
    uint64_t count;
    uint32_t first;      // its first chunk
    uint16_t type, out_type;
};
struct Batch {
    Array a[kArrays];
    uint32_t arrays, chunks;
};
static_assert(sizeof(Batch) + 64 <= 4096, "kernel arguments");

// Calls f(array, first value, values) for the runs of this workgroup's chunks.
template <class F>
__device__ __forceinline__ void each_run(const Batch &b, const F &f) {
    uint32_t c = (uint32_t)((uint64_t)b.chunks * blockIdx.x / gridDim.x);
    const uint32_t end = (uint32_t)((uint64_t)b.chunks * (blockIdx.x + 1) / gridDim.x);
    uint32_t lo = 0, hi = b.arrays;  // the last array that begins at c or before
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (b.a[mid].first <= c)
            lo = mid;
        else
            hi = mid;
    }
    while (c < end) {
        const uint32_t next = lo + 1 < b.arrays ? min(end, b.a[lo + 1].first) : end;
        const uint64_t from = (uint64_t)(c - b.a[lo].first) * kChunk;
        const uint64_t to = min(b.a[lo].count, (uint64_t)(next - b.a[lo].first) * kChunk);
        f(b.a[lo], from, to - from);
        c = next;
        ++lo;
    }
}

// Vectors of 8 values, four of each thread in flight.
template <class T>
__device__ __forceinline__ void load8(float (&v)[8], const T *p) {
    const Pack<T, 8> x = load_any<8>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)x.v[e];
}

template <class T>
__device__ __forceinline__ double squares(const T *p, uint64_t n) {
    double s[4] = {};
    uint64_t i = threadIdx.x * 8;
    for (; i + 3 * 2048 + 8 <= n; i += 4 * 2048) {
        float v[4][8];
#pragma unroll
        for (int k = 0; k < 4; ++k) load8(v[k], p + i + k * 2048);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) s[k] = fma((double)v[k][e], (double)v[k][e], s[k]);
    }
    for (; i < n; i += 2048) {
        if (i + 8 <= n) {
            float v[8];
            load8(v, p + i);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[0] = fma((double)v[e], (double)v[e], s[0]);
        } else {
            for (uint64_t j = i; j < n; ++j) s[1] = fma((double)(float)p[j], (double)(float)p[j], s[1]);
        }
    }
    return (s[0] + s[1]) + (s[2] + s[3]);
}

// Sum over the workgroup, in every thread.
__device__ __forceinline__ double group_sum(double x, double *lds) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

__global__ __launch_bounds__(256) void k_squares(Batch b, double *part) {
    __shared__ double lds[4];
    double s = 0.;
    each_run(b, [&](const Array &a, uint64_t from, uint64_t n) {
        if (a.type == VHIP_DTYPE_F32)
            s += squares((const float *)a.in + from, n);
        else if (a.type == VHIP_DTYPE_F16)
            s += squares((const half_t *)a.in + from, n);
        else
            s += squares((const bf16_t *)a.in + from, n);
    });
    s = group_sum(s, lds);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

template <class T, class O>
__device__ __forceinline__ void scale(const T *p, O *o, uint64_t n, float c) {
    uint64_t i = threadIdx.x * 8;
    for (; i + 3 * 2048 + 8 <= n; i += 4 * 2048) {
        float v[4][8];
#pragma unroll
        for (int k = 0; k < 4; ++k) load8(v[k], p + i + k * 2048);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            Pack<O, 8> x;
#pragma unroll
            for (int e = 0; e < 8; ++e) x.v[e] = (O)(v[k][e] * c);
            store_any<8>(o + i + k * 2048, x);
        }
    }
    for (; i < n; i += 2048) {
        if (i + 8 <= n) {
            float v[8];
            load8(v, p + i);
            Pack<O, 8> x;
#pragma unroll
            for (int e = 0; e < 8; ++e) x.v[e] = (O)(v[e] * c);
            store_any<8>(o + i, x);
        } else {
            for (uint64_t j = i; j < n; ++j) o[j] = (O)((float)p[j] * c);
        }
    }
}
template <class T>
__device__ __forceinline__ void scale_to(const Array &a, uint64_t from, uint64_t n, float c) {
    const T *p = (const T *)a.in + from;
    if (a.out_type == VHIP_DTYPE_F32)
        scale(p, (float *)a.out + from, n, c);
    else if (a.out_type == VHIP_DTYPE_F16)
        scale(p, (half_t *)a.out + from, n, c);
    else
        scale(p, (bf16_t *)a.out + from, n, c);
}

__global__ __launch_bounds__(256) void k_scale(Batch b, const double *part, int parts, float max_norm, float eps, float *norm) {
    __shared__ double lds[4];
    double s = 0.;
    for (int i = threadIdx.x; i < parts; i += 256) s += part[i];
    const double n = sqrt(group_sum(s, lds));
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    // without the quotients that are none: 0 / 0 is within the limit, and an infinite norm gives zeros whatever the limit
    const double over = n + (double)eps;
    const float c = n != n ? NAN : n == INFINITY ? 0.f : over <= max_norm ? 1.f : (float)(max_norm / over);
    each_run(b, [&](const Array &a, uint64_t from, uint64_t count) {
        if (!a.out || (c == 1.f && a.out == a.in)) return;
        if (a.type == VHIP_DTYPE_F32)
            scale_to<float>(a, from, count, c);
        else if (a.type == VHIP_DTYPE_F16)
            scale_to<half_t>(a, from, count, c);
        else
            scale_to<bf16_t>(a, from, count, c);
    });
}

struct Range {
    uintptr_t begin, end;
    size_t of;
    bool out;
};

// Outputs overlap nothing but the input that they replace.
int check_ranges(const vhip_array *arrays, size_t count) {
    std::vector<Range> r;
    r.reserve(2 * count);
    for (size_t i = 0; i < count; ++i) {
        const vhip_array &a = arrays[i];
        if (!a.count) continue;
        const uintptr_t b = (uintptr_t)a.data, o = (uintptr_t)a.out;
        r.push_back({b, b + a.count * dtype_size(a.dtype), i, false});
        if (a.out) r.push_back({o, o + a.count * dtype_size(a.out_dtype), i, true});
    }
    std::sort(r.begin(), r.end(), [](const Range &x, const Range &y) { return x.begin < y.begin; });
    // the furthest end so far, of outputs and of inputs, and whose it is
    const Range *out = nullptr, *in = nullptr, *in2 = nullptr;  // in2: the furthest of another array than in
    for (const Range &x : r) {
        auto meets = [&](const Range *y) { return y && y->end > x.begin && !(y->of == x.of && y->begin == x.begin); };
        if (meets(out) || (x.out && (meets(in) || meets(in2))))
            return set_error(VHIP_ERR_INVALID_CONFIG, "an output overlaps another array");
        const Range *&far = x.out ? out : in;
        if (!far || x.end > far->end) {
            if (!x.out) in2 = in;
            far = &x;
        } else if (!x.out && (!in2 || x.end > in2->end)) {
            in2 = &x;
        }
    }
    return VHIP_OK;
}

int check_arrays(const vhip_array *arrays, size_t count, bool outputs) {
    if (count && !arrays) return set_error(VHIP_ERR_INVALID_CONFIG, "arrays are null");
    uint64_t chunks = 0;
    for (size_t i = 0; i < count; ++i) {
        const vhip_array &a = arrays[i];
        const void *out = outputs ? a.out : nullptr;  // the norm alone does not look at them
        if (!dtype_known(a.dtype) || (out && !dtype_known(a.out_dtype)))
            return set_error(VHIP_ERR_INVALID_CONFIG, "unknown element type of array " + std::to_string(i));
        if (a.count > ((size_t)1 << 40)) return set_error(VHIP_ERR_INVALID_CONFIG, "an array of more than 2^40 values");
        if (a.count && (!a.data || (outputs && !out))) return set_error(VHIP_ERR_INVALID_CONFIG, "array " + std::to_string(i) + " is null");
        if ((uintptr_t)a.data % dtype_size(a.dtype) || (out && (uintptr_t)out % dtype_size(a.out_dtype)))
            return set_error(VHIP_ERR_INVALID_CONFIG, "array " + std::to_string(i) + " is not aligned to its type");
        if (out == a.data && out && a.out_dtype != a.dtype)
            return set_error(VHIP_ERR_INVALID_CONFIG, "an array that is scaled in place keeps its type");
        chunks += (a.count + kChunk - 1) / kChunk;
    }
    if (chunks > 0x7fffffff) return set_error(VHIP_ERR_INVALID_CONFIG, "too many values");
    return outputs ? check_ranges(arrays, count) : VHIP_OK;
}

inline size_t launches_of(size_t count) { return (count + kArrays - 1) / kArrays; }

int run(int ordinal, const vhip_array *arrays, size_t count, bool outputs, float max_norm, float eps, float *norm, void *workspace,
        size_t workspace_bytes, hipStream_t s) {
    VH_CHECK(check_arrays(arrays, count, outputs));
    if (!norm && !outputs) return set_error(VHIP_ERR_INVALID_CONFIG, "norm is null");
    if (count && (!workspace || workspace_bytes < vhip_clip_gradients_workspace(count) || ((uintptr_t)workspace & 7)))
        return set_error(VHIP_ERR_INVALID_CONFIG, "the workspace is smaller than vhip_clip_gradients_workspace() or not aligned");
    std::vector<Batch> batches;
    uint64_t chunks = 0;
    for (size_t i = 0; i < count; ++i) {
        const vhip_array &a = arrays[i];
        if (!a.count) continue;
        if (batches.empty() || batches.back().arrays == kArrays) batches.push_back(Batch{});
        Batch &b = batches.back();
        b.a[b.arrays++] = {a.data, outputs ? a.out : nullptr, a.count, b.chunks, (uint16_t)a.dtype, (uint16_t)a.out_dtype};
        const uint32_t n = (uint32_t)((a.count + kChunk - 1) / kChunk);
        b.chunks += n;
        chunks += n;
    }
    CallDevice dev;
    VH_CHECK(dev.enter(ordinal));
    double *part = (double *)workspace;
    int parts = 0;
    auto groups = [&](const Batch &b) {
        const uint64_t n = chunks <= kParts ? b.chunks : (uint64_t)b.chunks * kParts / chunks + 1;
        return (uint32_t)(n < b.chunks ? n : b.chunks);
    };
    for (const Batch &b : batches) {
        const uint32_t n = groups(b);
        k_squares<<<n, 256, 0, s>>>(b, part + parts);
        parts += (int)n;
    }
    if (batches.empty()) batches.push_back(Batch{});  // the norm of nothing
    bool first = true;
    for (const Batch &b : batches) {
        if (!outputs && !first) break;
        k_scale<<<outputs && b.chunks ? groups(b) : 1, 256, 0, s>>>(outputs ? b : Batch{}, part, parts, max_norm, eps, first ? norm : nullptr);
        first = false;
    }
    return launch_status("gradient norm launch");
}

}  // namespace
}  // namespace vh

using namespace vh;

extern "C" {

size_t vhip_clip_gradients_workspace(size_t count) { return (kParts + launches_of(count)) * sizeof(double); }

int vhip_gradient_norm(int ordinal, const vhip_array *arrays, size_t count, float *norm, void *workspace, size_t workspace_bytes,
                       void *stream) {
    clear_error();
    try {
        return run(ordinal, arrays, count, false, 1.f, 0.f, norm, workspace, workspace_bytes, (hipStream_t)stream);
    } catch (const std::bad_alloc &) {
        return set_error(VHIP_ERR_DRIVER, "out of host memory");
    }
}

int vhip_clip_gradients(int ordinal, const vhip_array *arrays, size_t count, float max_norm, float eps, float *norm, void *workspace,
                        size_t workspace_bytes, void *stream) {
    clear_error();
    if (!(max_norm >= 0.f)) return set_error(VHIP_ERR_INVALID_CONFIG, "max_norm must be >= 0");
    if (!(eps >= 0.f)) return set_error(VHIP_ERR_INVALID_CONFIG, "eps must be >= 0");
    try {
        return run(ordinal, arrays, count, true, max_norm, eps, norm, workspace, workspace_bytes, (hipStream_t)stream);
    } catch (const std::bad_alloc &) {
        return set_error(VHIP_ERR_DRIVER, "out of host memory");
    }
}

}  // extern "C"
