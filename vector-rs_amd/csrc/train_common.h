// train_common.h -- what the training operators share: element types, wave reductions, the device of a
// call and the checks of its arguments.
#pragma once

#include "vh_runtime.h"

namespace vh {

typedef _Float16 half_t;
typedef __bf16 bf16_t;
typedef float floatx4_t __attribute__((ext_vector_type(4)));

inline bool dtype_known(int dtype) { return dtype == VHIP_DTYPE_F32 || dtype == VHIP_DTYPE_F16 || dtype == VHIP_DTYPE_BF16; }
inline size_t dtype_size(int dtype) { return dtype == VHIP_DTYPE_F32 ? 4 : 2; }
inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

template <class T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
    T v[N];
};

// N values from or to memory that is aligned to one of them: one access all the same, as global memory takes
// any alignment.
template <int N, class T>
__device__ __forceinline__ Pack<T, N> load_any(const T *p) {
    Pack<T, N> v;
    __builtin_memcpy(&v, p, sizeof v);
    return v;
}
template <int N, class T>
__device__ __forceinline__ void store_any(T *p, const Pack<T, N> &v) {
    __builtin_memcpy(p, &v, sizeof v);
}
// The same of a row's values from column c on, of which those past dim are zeros, or left alone.
template <int N, class T>
__device__ __forceinline__ Pack<T, N> load_row(const T *row, int c, int dim) {
    if (c + N <= dim) return load_any<N>(row + c);
    asm volatile("" ::: "memory");  // or the compiler makes single loads of both branches
    Pack<T, N> v;
#pragma unroll
    for (int e = 0; e < N; ++e) v.v[e] = c + e < dim ? row[c + e] : (T)0.f;
    return v;
}
template <int N, class T>
__device__ __forceinline__ void store_row(T *row, int c, int dim, const Pack<T, N> &v) {
    if (c + N <= dim) {
        store_any<N>(row + c, v);
    } else {
        asm volatile("" ::: "memory");
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (c + e < dim) row[c + e] = v.v[e];
    }
}

template <int W>
__device__ __forceinline__ float lane_sum(float x) {
#pragma unroll
    for (int o = 1; o < W; o <<= 1) x += __shfl_xor(x, o, 64);
    return x;
}

// The GPU of a training call for as long as the call lasts: these calls only enqueue work, so the
// caller's current device is put back when they return.  A device is looked at in full once per process.
struct CallDevice {
    int back = -1;
    int enter(int ordinal);
    ~CallDevice() {
        if (back >= 0) (void)hipSetDevice(back);
    }
};

// Threads of a 256-lane workgroup over rows of `chunks` items each: 2^log2 lanes a row.
inline int lanes_log2(size_t chunks) {
    int l = 0;
    while (l < 8 && ((size_t)1 << l) < chunks) ++l;
    return l;
}

// Calls f(first workgroup, workgroups) for the launches that `groups` workgroups of `threads` take: one has fewer than 2^32 threads.
template <class F>
inline void each_launch(int64_t groups, int threads, const F &f) {
    const int64_t most = 0xffffffffll / threads;
    for (int64_t first = 0; first < groups; first += most) f(first, (uint32_t)(groups - first < most ? groups - first : most));
}

// Status of the launches of a call so far.
inline int launch_status(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? VHIP_OK
                           : set_error(VHIP_ERR_DRIVER, std::string(what) + ": " + hipGetErrorString(e));
}

// Hands out the parts of a caller's workspace; with base null it only adds them up.
struct Carver {
    char *base = nullptr;
    size_t used = 0;
    template <class T>
    T *take(size_t count) {
        used = round_up(used, 256);
        T *p = base ? reinterpret_cast<T *>(base + used) : nullptr;
        used += count * sizeof(T);
        return p;
    }
};

}  // namespace vh
