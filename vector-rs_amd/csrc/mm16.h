// mm16.h -- tile product C = A B^T of 16-bit operands on the matrix cores, shared by the training operators.
//
// A is M x K, B is N x K, both row-major with K contiguous ("planes"): rows 16-byte aligned, K a multiple of
// 64.  Sums are held in 32 bits.  A 32-bit operand is carried as two float16 planes, x ~ hi + lo with
// hi = f16(x) and lo = f16(x - hi) (22 bits), and the product as three segments of one long K loop,
// hi hi + hi lo + lo hi; the dropped lo lo term is 2^-22 of the product.
//
// A workgroup computes a BM x BN tile, its waves MB x NB blocks of 16 x 16.  Operand tiles of 64 k come in
// by 16-byte global->LDS DMA into two buffers; a row's 128 bytes lie as eight 16-byte slots, slot s of row r
// holding chunk s ^ (r & 7), so the 16 rows that one fragment read touches spread over all banks (the DMA
// writes LDS in lane order, so the swizzle is in the addresses that the lanes read from).  The two halves of
// a tile's k are two sets of fragments: while one set is multiplied the other is read, and the next tile's
// DMA has the time of a whole tile's products to land.  Rows past M or N are clamped to the last row: what
// they give is in accumulators that the epilogue does not use.
#pragma once

#include "train_common.h"

namespace vh {

struct MmArgs {
    const void *a[2], *b[2];  // planes; [1] the low halves where nseg is 3
    size_t lda, ldb;          // elements; 2^23 at most
    size_t sa, sb;            // from one product of a batch to the next, elements
    int M, N;
    int ktiles;               // K / 64
    int nseg;                 // 1, or 3 for split operands
    int mt, nt;               // tiles along M and N
    int ksplit;               // parts of the K loop, each a workgroup of its own
    int batch;
    bool upper;               // only tiles on and above the diagonal (square and symmetric products)
};

constexpr int kMmK = 64;               // k of one stage
constexpr size_t kMmMaxLd = 1u << 23;  // a tile's byte offsets stay below 2^32
constexpr int kXcds = 8;

template <class T>
struct MmVec;
template <>
struct MmVec<half_t> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ floatx4_t mfma(v8 a, v8 b, floatx4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct MmVec<bf16_t> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ floatx4_t mfma(v8 a, v8 b, floatx4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

// Global->LDS DMA of 16 bytes per lane from base + off to LDS byte address m0_base + 16 x lane (see dma_lds16).
__device__ __forceinline__ void dma_lds16_at(const void *base, uint32_t off, uint32_t m0_base) {
    uint32_t sv;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(sv)
                 : "v"(off), "s"(base), "s"(m0_base)
                 : "memory");
}

// Position of this workgroup: workgroups go round the XCDs, so XCD x takes the tiles of the x-th eighth of
// the order, and the order runs down strips of 8 tiles of M before it moves along N: the 32 tiles an XCD
// works on share 8 + 4 operand tiles in its L2.
struct MmPlace {
    int tm, tn, part, batch;
};
__device__ __forceinline__ MmPlace mm_place(const MmArgs &g, uint32_t id, uint32_t total) {
    const uint32_t x = id % kXcds, k = id / kXcds, q = total / kXcds, r = total % kXcds;
    uint32_t t = x * q + (x < r ? x : r) + k;
    MmPlace p;
    const uint32_t tiles = g.upper ? (uint32_t)g.mt * (g.mt + 1) / 2 : (uint32_t)g.mt * g.nt;
    const uint32_t per = tiles * g.ksplit;
    p.batch = t / per;
    t -= p.batch * per;
    p.part = t / tiles;
    t -= p.part * tiles;
    if (g.upper) {
        int n = 0;
        while ((uint32_t)(n + 1) * (n + 2) / 2 <= t) ++n;
        p.tn = n;
        p.tm = t - (uint32_t)n * (n + 1) / 2;
        return p;
    }
    constexpr uint32_t H = 8;
    const uint32_t strip = t / (H * g.nt), first = strip * H;
    const uint32_t h = (uint32_t)g.mt - first < H ? (uint32_t)g.mt - first : H;
    t -= strip * H * g.nt;
    p.tm = first + t % h;
    p.tn = t / h;
    return p;
}

// Epi: void operator()(acc, m, n, place): the wave's MB x NB blocks, block (i, j) lane l element e being
// C[m + 16 i + 4 (l >> 4) + e][n + 16 j + (l & 15)].
template <class T, int WM, int WN, int MB, int NB, class Epi>
__global__ __launch_bounds__(WM *WN * 64) void k_mm(MmArgs g, Epi epi) {
    constexpr int NW = WM * WN, BM = WM * MB * 16, BN = WN * NB * 16;
    constexpr int IA = BM / 8 / NW, IB = BN / 8 / NW;  // DMAs of a wave: 8 rows each
    static_assert(IA * 8 * NW == BM && IB * 8 * NW == BN, "whole DMAs");
    typedef typename MmVec<T>::v8 v8;
    __shared__ __align__(1024) char lds[2 * (BM + BN) * 128];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % WM, wn = wave / WM;
    const MmPlace pl = mm_place(g, blockIdx.x, gridDim.x);
    const int m0 = pl.tm * BM, n0 = pl.tn * BN;

    // this part's stages: [s0, s1) of nseg * ktiles
    const int all = g.nseg * g.ktiles;
    const int s0 = (int)((long)all * pl.part / g.ksplit), s1 = (int)((long)all * (pl.part + 1) / g.ksplit);
    int seg = s0 / g.ktiles, kt = s0 % g.ktiles;

    uint32_t offa[IA], offb[IB];
    {
        const int r = lane >> 3, c = (lane & 7) ^ r;
#pragma unroll
        for (int i = 0; i < IA; ++i) {
            const int row = min(m0 + (wave * IA + i) * 8 + r, g.M - 1) - m0;
            offa[i] = (uint32_t)((size_t)row * g.lda * 2 + c * 16);
        }
#pragma unroll
        for (int i = 0; i < IB; ++i) {
            const int row = min(n0 + (wave * IB + i) * 8 + r, g.N - 1) - n0;
            offb[i] = (uint32_t)((size_t)row * g.ldb * 2 + c * 16);
        }
    }
    const size_t pa = ((size_t)m0 * g.lda + pl.batch * g.sa) * 2, pb = ((size_t)n0 * g.ldb + pl.batch * g.sb) * 2;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;

    auto issue = [&](int buf) {
        const char *ga = (const char *)g.a[seg == 2] + pa + (size_t)kt * (kMmK * 2);
        const char *gb = (const char *)g.b[seg == 1] + pb + (size_t)kt * (kMmK * 2);
        const uint32_t la = lds0 + buf * (BM + BN) * 128 + wave * IA * 1024;
        const uint32_t lb = lds0 + buf * (BM + BN) * 128 + BM * 128 + wave * IB * 1024;
#pragma unroll
        for (int i = 0; i < IA; ++i) dma_lds16_at(ga, offa[i], la + i * 1024);
#pragma unroll
        for (int i = 0; i < IB; ++i) dma_lds16_at(gb, offb[i], lb + i * 1024);
        if (++kt == g.ktiles) {
            kt = 0;
            ++seg;
        }
    };

    // fragment addresses: row l & 15 of a block, chunk (l >> 4) of its half
    const int fr = lane & 15, fc = lane >> 4;
    const int sw0 = ((fc) ^ (fr & 7)) * 16, sw1 = ((fc + 4) ^ (fr & 7)) * 16;
    const char *fa = lds + (wm * MB * 16 + fr) * 128, *fb = lds + (BM + wn * NB * 16 + fr) * 128;

    floatx4_t acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = floatx4_t{0.f, 0.f, 0.f, 0.f};

    v8 a0[MB], b0[NB], a1[MB], b1[NB];
    auto read = [&](v8(&a)[MB], v8(&b)[NB], int buf, int sw) {
#pragma unroll
        for (int j = 0; j < NB; ++j) b[j] = *(const v8 *)(fb + buf * (BM + BN) * 128 + j * 2048 + sw);
#pragma unroll
        for (int i = 0; i < MB; ++i) a[i] = *(const v8 *)(fa + buf * (BM + BN) * 128 + i * 2048 + sw);
    };
    auto multiply = [&](const v8(&a)[MB], const v8(&b)[NB]) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] = MmVec<T>::mfma(a[i], b[j], acc[i][j]);
    };

    if (s0 < s1) {
        const int n = s1 - s0;
        issue(0);
        if (n > 1) {
            issue(1);
            __builtin_amdgcn_s_waitcnt(VH_VMCNT(IA + IB));
        } else {
            __builtin_amdgcn_s_waitcnt(VH_VMCNT(0));
        }
        lds_barrier();
        read(a0, b0, 0, sw0);
        for (int s = 0; s < n; ++s) {
            const int buf = s & 1;
            read(a1, b1, buf, sw1);
            multiply(a0, b0);
            if (s + 1 < n) {
                // this wave's reads of the buffer are done (lds_barrier waits for them) and the next
                // tile has landed; after the barrier that holds for every wave
                __builtin_amdgcn_s_waitcnt(VH_VMCNT(0));
                lds_barrier();
                if (s + 2 < n) issue(buf);
                read(a0, b0, buf ^ 1, sw0);
            }
            multiply(a1, b1);
        }
    }
    epi(acc, m0 + wm * MB * 16, n0 + wn * NB * 16, pl);
}

template <class T, int WM, int WN, int MB, int NB, class Epi>
int mm_launch(MmArgs g, const Epi &epi, hipStream_t s) {
    g.mt = ceil_div(g.M, WM * MB * 16);
    g.nt = ceil_div(g.N, WN * NB * 16);
    const size_t tiles = g.upper ? (size_t)g.mt * (g.mt + 1) / 2 : (size_t)g.mt * g.nt;
    const size_t total = tiles * g.ksplit * g.batch;
    if (total > 0x7fffffff || g.lda > kMmMaxLd || g.ldb > kMmMaxLd)
        return set_error(VHIP_ERR_INVALID_CONFIG, "a product of the call has too many tiles");
    k_mm<T, WM, WN, MB, NB, Epi><<<dim3((uint32_t)total), dim3(WM * WN * 64), 0, s>>>(g, epi);
    return launch_status("product launch");
}

}  // namespace vh
