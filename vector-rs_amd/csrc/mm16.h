// mm16.h -- tile product C = A B^T of 16-bit operands on the matrix cores, shared by the training operators.
//
// A is M x K and B is N x K, each either with K contiguous, or ("across", a template flag) stored as K rows
// of its M or N values.  Rows are 16-byte aligned; K is a multiple of 64 where it is contiguous, and an
// operand across may have fewer rows: the missing ones are read as its last, for the other operand to
// multiply with zeros.  Sums are held in 32 bits.
// A 32-bit operand is carried in pairs of float16, x ~ hi + lo with hi = f16(x) and lo = f16(x - hi) (22 bits),
// and its product is hi hi + hi lo + lo hi; the dropped lo lo term is 2^-22 of the product.  A row of pairs
// lies as blocks of 32 hi and 32 lo, so that a stage of 64 halves holds both of 32 k and its fragments serve
// three products where a plain stage's serve two.
//
// A workgroup computes a BM x BN tile, its waves MB x NB blocks of 16 x 16.  Operand tiles of 64 k come in
// by 16-byte global->LDS DMA into two buffers; the two halves of a tile's k are two sets of fragments: while
// one set is multiplied the other is read, and the next tile's DMA has the time of a whole tile's products to
// land.  Rows past M or N are clamped to the last row: what they give is in accumulators that the epilogue
// does not use.  The DMA writes LDS in lane order, so a tile is swizzled by the addresses that lanes read:
//  * K contiguous: a row's 128 bytes are eight 16-byte slots, slot s of row r holding chunk s ^ (r & 7), so
//    the 16 rows of a fragment read spread over all banks;
//  * across: a row of k is BM / 8 slots, chunk s ^ 2 f(k), f from the bits of k that differ between the 16
//    rows of a read (two 4 x 16 blocks of the transposing LDS read make a lane's 8 values of k).
// Measured on 8192^3 in bfloat16: 256 x 256 tiles of 8 waves 1,260 TFLOP/s (1,120 to 1,280 with operands across),
// 128 x 128 of 4 waves 1,040, the library's product 1,326.  The matrix units are busy 64% of the time (131072 x
// 2048 x 4096); the rest is the barrier of each stage, where every wave issues its DMAs.
#pragma once

#include "train_common.h"

namespace vh {

// How the operands are stored, and what of them is multiplied.
enum MmMode {
    kPlain,  // 16-bit values
    kPairs,  // pairs: all three products, or (MmArgs::alo, blo) those of the low halves that are not empty
    kHigh,   // pairs: the high halves alone
};
// Where value c of a row of pairs has its high half, in halves; the low one is 32 further.
__host__ __device__ inline size_t pair_at(size_t c) { return (c >> 5) * 64 + (c & 31); }

struct MmArgs {
    const void *a, *b;
    size_t lda, ldb;          // 16-bit elements; 2^23 at most where K is contiguous
    size_t sa, sb;            // from one product of a batch to the next, 16-bit elements
    int M, N, K;              // K: rows where an operand is stored across
    bool alo, blo;            // kPairs: whether the low halves count
    int mt, nt;               // tiles along M and N
    int ksplit;               // parts of the K loop, each a workgroup of its own
    int batch;
    bool upper;               // only tiles on and above the diagonal (square and symmetric products)
    const uint32_t *only;     // null, or which tiles to compute: [tile of N][tile of M]
};

constexpr int kMmK = 64;               // k of one stage
constexpr size_t kMmMaxLd = 1u << 23;  // a tile's byte offsets stay below 2^32
constexpr int kXcds = 8;

template <class T>
struct MmVec;
template <>
struct MmVec<half_t> {
    typedef _Float16 v4 __attribute__((ext_vector_type(4)));
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ floatx4_t mfma(v8 a, v8 b, floatx4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct MmVec<bf16_t> {
    typedef __bf16 v4 __attribute__((ext_vector_type(4)));
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

// One operand's tile of BR rows (of M or N) by 64 halves of k in LDS: its DMAs and its fragments.
template <class T, MmMode MODE, bool ACROSS, int BR, int NW>
struct MmTile {
    static constexpr int I = BR / 8 / NW;           // DMAs of a wave
    static constexpr int CH = BR / 8;               // chunks of a k row where stored across
    static constexpr int kBytes = BR * 128;
    static constexpr int KS = MODE == kPairs ? 32 : 64;  // k of a stage
    static_assert(I * 8 * NW == BR && CH % 8 == 0, "whole DMAs, chunks by eights");
    typedef typename MmVec<T>::v4 v4;
    typedef typename MmVec<T>::v8 v8;
    uint32_t off[I];
    const char *base;
    size_t step;    // bytes from one stage to the next
    size_t ld2;
    int c_last, wave, lane;

    // byte of a row's chunk of 8 (high) values
    static __device__ __forceinline__ int chunk(int c) { return MODE == kPlain ? c * 16 : (c >> 2) * 128 + (c & 3) * 16; }
    // A fragment's read takes 32 bytes of each of 16 rows of k: 0..3 and, further on, every eighth.  What is
    // xored into their chunks puts them in other banks; rows of 384 bytes (24 chunks) alternate between halves
    // of the banks by themselves, and a chunk has to stay within its 8.
    static __device__ __forceinline__ int swizzle(int k) {
        if constexpr (CH % 16) return 2 * ((((k >> 1) & 1) << 1) | ((k >> 3) & 1));
        return 2 * ((k & 3) | (((k >> 3) & (CH >= 32 ? 3 : 1)) << 2));
    }
    // DMA i, across: its row of k, and the byte in that row.  In pairs the tile's rows from 32 on are low halves.
    __device__ __forceinline__ void spot(int i, int &k, int &at) const {
        const int n = (wave * I + i) * 64 + lane;
        k = n / CH;
        at = chunk(min((n % CH) ^ swizzle(k), c_last));
        if constexpr (MODE == kPairs) {
            at += k >= 32 ? 64 : 0;
            k &= 31;
        }
    }
    __device__ __forceinline__ void init(const void *p, size_t ld, int r0, int rows, size_t batch_off, int w, int l) {
        wave = w;
        lane = l;
        ld2 = ld * 2;
        if constexpr (ACROSS) {
            c_last = (rows - 1 - r0) / 8;
            step = ld2 * KS;
            base = (const char *)p + (batch_off + (size_t)r0 * (MODE == kPlain ? 1 : 2)) * 2;  // r0: a multiple of 32
#pragma unroll
            for (int i = 0; i < I; ++i) {
                int k, at;
                spot(i, k, at);
                off[i] = (uint32_t)(k * ld2 + at);
            }
        } else {
            step = MODE == kHigh ? 256 : 128;
            base = (const char *)p + (batch_off + (size_t)r0 * ld) * 2;
            const int r = l >> 3, c = (l & 7) ^ r;
            const int at = MODE == kHigh ? chunk(c) : c * 16;
#pragma unroll
            for (int i = 0; i < I; ++i) off[i] = (uint32_t)((size_t)(min(r0 + (w * I + i) * 8 + r, rows - 1) - r0) * ld2 + at);
        }
    }
    // DMA of stage kt to LDS address `to`; krows: rows of k from this stage on
    __device__ __forceinline__ void issue(int kt, int krows, uint32_t to) const {
        const char *g = base + kt * step;
        to += wave * I * 1024;
        if (ACROSS && krows < KS) {
#pragma unroll
            for (int i = 0; i < I; ++i) {
                int k, at;
                spot(i, k, at);
                dma_lds16_at(g, (uint32_t)(min(k, krows - 1) * ld2 + at), to + i * 1024);
            }
        } else {
#pragma unroll
            for (int i = 0; i < I; ++i) dma_lds16_at(g, off[i], to + i * 1024);
        }
    }
    // Fragments of N blocks from row r0 of the tile, half h of its k (in pairs: the high or the low halves).
    template <int N>
    static __device__ __forceinline__ void read(v8 (&f)[N], const char *tile, int r0, int h, int l) {
        const int i = l & 15, q = l >> 4;
        if constexpr (ACROSS) {
            typedef __attribute__((address_space(3))) v4 lds_v4;
            const int k = h * 32 + q * 8 + (i >> 2);
            const char *p = tile + k * (BR * 2) + (i & 1) * 8;
            const int s = swizzle(k);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int c = (((r0 >> 3) + 2 * n + ((i >> 1) & 1)) ^ s) * 16;
                const v4 x = read_tr((lds_v4 *)(p + c)), y = read_tr((lds_v4 *)(p + c + 4 * BR * 2));
                f[n] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
            }
        } else {
            const char *p = tile + (r0 + i) * 128 + ((q + 4 * h) ^ (i & 7)) * 16;
#pragma unroll
            for (int n = 0; n < N; ++n) f[n] = *(const v8 *)(p + n * 2048);
        }
    }
    static __device__ __forceinline__ v4 read_tr(__attribute__((address_space(3))) v4 *p) {
        typedef short s4 __attribute__((ext_vector_type(4)));
        return __builtin_bit_cast(v4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)p));
    }
};

// LDS of a wave for its epilogue, 16 KB.
constexpr int kEpiBytes = 16384;

// Values of a wave's blocks as whole rows: value(i, j, e) is element e of block (i, j) (see Epi), given once
// each; emit(n, m, pack) gets 16 bytes of row n (of N, within the wave's) from column m.  What 16 lanes hold
// of 16 rows goes through LDS, so that rows leave in pieces of up to 256 bytes.
template <class O, int MB, int NB, class Value, class Emit>
__device__ __forceinline__ void rows_through_lds(char *w, const Value &value, const Emit &emit) {
    constexpr int PER = 16 / (int)sizeof(O);  // values of a chunk
    constexpr int FIT = 16 / (int)sizeof(O);  // blocks in 256 bytes
    constexpr int BP = MB <= FIT ? MB : MB % FIT == 0 ? FIT : FIT - 1;  // blocks of a pass
    constexpr int NC = BP * (int)sizeof(O);                             // chunks of a row
    constexpr int XOR = NC == 12 ? 15 : NC - 1, PITCH = (XOR + 1) * 16;
    static_assert((NC & (NC - 1)) == 0 || NC == 12, "chunks");
    static_assert(NB * 16 * PITCH <= kEpiBytes && MB % BP == 0, "fits");
    int l = threadIdx.x & 63;
    // Large tiles have no registers left: the compiler would keep addresses in scratch from one call to the next
    // (Newton-Schulz steps of 4096 x 4096: 3740 us, made anew 3450).
    if constexpr (MB * NB > 16) asm volatile("" : "+v"(l));
    const int q = l >> 4;
#pragma unroll
    for (int p = 0; p < MB / BP; ++p) {
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int n = 16 * j + (l & 15);
#pragma unroll
            for (int i = 0; i < BP; ++i) {
                Pack<O, 4> v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v.v[e] = value(p * BP + i, j, e);
                const int at = (16 * i + 4 * q) * (int)sizeof(O);
                *reinterpret_cast<Pack<O, 4> *>(w + n * PITCH + (((at >> 4) ^ (n & XOR)) << 4) + (at & 15)) = v;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int k = 0; k < NB * 16 * NC / 64; ++k) {
            const int n = NC == 12 ? (k * 64 + l) / NC : k * (64 / NC) + l / NC, c = NC == 12 ? (k * 64 + l) % NC : l % NC;
            emit(n, p * BP * 16 + c * PER, *reinterpret_cast<const Pack<O, PER> *>(w + n * PITCH + ((c ^ (n & XOR)) << 4)));
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

// Epi: void operator()(acc, m, n, place, lds): the wave's MB x NB blocks, block (i, j) lane l element e being
// C[m + 16 i + 4 (l >> 4) + e][n + 16 j + (l & 15)]; lds: kEpiBytes of the wave's own.
template <class T, MmMode MODE, bool TA, bool TB, int WM, int WN, int MB, int NB, class Epi>
__global__ __launch_bounds__(WM *WN * 64) void k_mm(MmArgs g, Epi epi) {
    constexpr int NW = WM * WN, BM = WM * MB * 16, BN = WN * NB * 16, BUF = (BM + BN) * 128;
    typedef MmTile<T, MODE, TA, BM, NW> TileA;
    typedef MmTile<T, MODE, TB, BN, NW> TileB;
    typedef typename MmVec<T>::v8 v8;
    __shared__ __align__(1024) char lds[2 * BUF >= NW * kEpiBytes ? 2 * BUF : NW * kEpiBytes];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % WM, wn = wave / WM;
    const MmPlace pl = mm_place(g, blockIdx.x, gridDim.x);
    if (g.only && !g.only[(size_t)pl.tn * g.mt + pl.tm]) return;
    const int m0 = pl.tm * BM, n0 = pl.tn * BN;

    // this part's stages
    const int all = (g.K + TileA::KS - 1) / TileA::KS;
    const int s0 = (int)((long)all * pl.part / g.ksplit), n = (int)((long)all * (pl.part + 1) / g.ksplit) - s0;

    TileA ta;
    TileB tb;
    ta.init(g.a, g.lda, m0, g.M, pl.batch * g.sa, wave, lane);
    tb.init(g.b, g.ldb, n0, g.N, pl.batch * g.sb, wave, lane);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    auto issue = [&](int s) {
        const int kt = s0 + s, krows = g.K - kt * TileA::KS, buf = s & 1;
        ta.issue(kt, krows, lds0 + buf * BUF);
        tb.issue(kt, krows, lds0 + buf * BUF + TileA::kBytes);
    };

    floatx4_t acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = floatx4_t{0.f, 0.f, 0.f, 0.f};

    v8 a0[MB], b0[NB], a1[MB], b1[NB];
    auto read_a = [&](v8(&a)[MB], int buf, int h) {
        TileA::template read<MB>(a, lds + buf * BUF, wm * MB * 16, h, lane);
    };
    auto read_b = [&](v8(&b)[NB], int buf, int h) {
        TileB::template read<NB>(b, lds + buf * BUF + TileA::kBytes, wn * NB * 16, h, lane);
    };
    auto multiply = [&](const v8(&a)[MB], const v8(&b)[NB]) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] = MmVec<T>::mfma(a[i], b[j], acc[i][j]);
    };

    if (n > 0) {
        issue(0);
        if (n > 1) {
            issue(1);
            __builtin_amdgcn_s_waitcnt(VH_VMCNT(TileA::I + TileB::I));
        } else {
            __builtin_amdgcn_s_waitcnt(VH_VMCNT(0));
        }
        lds_barrier();
        read_b(b0, 0, 0);
        read_a(a0, 0, 0);
        // The last stage stands by itself: with a way round the barrier inside the loop the compiler would
        // have the second half's products wait for fragments that are read for the next stage.
        int s = 0;
        for (; s + 1 < n; ++s) {
            const int buf = s & 1;
            read_b(b1, buf, 1);
            read_a(a1, buf, 1);
            multiply(a0, b0);
            // this wave's reads of the buffer are done (lds_barrier waits for them) and the next tile has
            // landed; after the barrier that holds for every wave
            __builtin_amdgcn_s_waitcnt(VH_VMCNT(0));
            lds_barrier();
            if (s + 2 < n) issue(s + 2);
            if constexpr (MODE == kPairs) {
                if (g.blo) multiply(a0, b1);
                read_a(a0, buf ^ 1, 0);
                if (g.alo) multiply(a1, b0);
                read_b(b0, buf ^ 1, 0);
            } else {
                read_b(b0, buf ^ 1, 0);
                read_a(a0, buf ^ 1, 0);
                multiply(a1, b1);
            }
        }
        read_b(b1, s & 1, 1);
        read_a(a1, s & 1, 1);
        multiply(a0, b0);
        if constexpr (MODE == kPairs) {
            if (g.blo) multiply(a0, b1);
            if (g.alo) multiply(a1, b0);
        } else {
            multiply(a1, b1);
        }
    }
    lds_barrier();  // every wave's fragments are read: the buffers are the epilogue's
    epi(acc, m0 + wm * MB * 16, n0 + wn * NB * 16, pl, lds + wave * kEpiBytes);
}

template <class T, MmMode MODE, bool TA, bool TB, int WM, int WN, int MB, int NB, class Epi>
int mm_launch_tile(MmArgs g, const Epi &epi, hipStream_t s) {
    g.mt = ceil_div(g.M, WM * MB * 16);
    g.nt = ceil_div(g.N, WN * NB * 16);
    const size_t tiles = g.upper ? (size_t)g.mt * (g.mt + 1) / 2 : (size_t)g.mt * g.nt;
    const size_t total = tiles * g.ksplit * g.batch;
    if (total > 0x7fffffff || (!TA && g.lda > kMmMaxLd) || (!TB && g.ldb > kMmMaxLd))
        return set_error(VHIP_ERR_INVALID_CONFIG, "a product of the call has too many tiles");
    k_mm<T, MODE, TA, TB, WM, WN, MB, NB, Epi><<<dim3((uint32_t)total), dim3(WM * WN * 64), 0, s>>>(g, epi);
    return launch_status("product launch");
}

// Whether 256 x 256 tiles (8 waves, one workgroup a CU) beat 128 x 128 ones (4 waves, two a CU): whole rounds
// of workgroups times a tile's work; small tiles are given 1.4 times the time, which also stands for their
// reading each operand twice as often (4096 x 131072 x 1024: loss 955 us with large tiles, 1230 with small;
// 100 x 10000 x 128 with gradients: 65 and 46).
inline bool mm_big_tiles(size_t M, size_t N, size_t batch, bool upper = false) {
    auto tiles = [&](size_t b) {
        const size_t m = (M + b - 1) / b, n = (N + b - 1) / b;
        return (upper ? m * (m + 1) / 2 : m * n) * batch;
    };
    return ((tiles(256) + 255) / 256) * 4 * 10 <= ((tiles(128) + 511) / 512) * 2 * 14;
}

template <class T, MmMode MODE, bool TA, bool TB, class Epi>
int mm_launch(const MmArgs &g, bool big, const Epi &epi, hipStream_t s) {
    return big ? mm_launch_tile<T, MODE, TA, TB, 2, 4, 8, 4>(g, epi, s) : mm_launch_tile<T, MODE, TA, TB, 2, 2, 4, 4>(g, epi, s);
}

// The same for a product whose M may be a few hundred: tiles of 192 x 256 (8 waves) where they hold at least a
// ninth less padding (gradients of 1000 x 200003 x 300 in bfloat16: 873 us, 909 with 256 x 256).  A round of
// them counts as 33 against the 28 of small ones (4096 x 30000 x 384: 505 us, 537 with small tiles;
// 2048 x 40000 x 300: 351 and 341).
enum MmShape { k128x128, k256x256, k192x256 };

inline bool mm_narrow(size_t M) { return (M + 191) / 192 * 192 * 9 <= (M + 255) / 256 * 256 * 8; }

inline MmShape mm_shape(size_t M, size_t N, size_t batch) {
    if (!mm_narrow(M)) return mm_big_tiles(M, N, batch) ? k256x256 : k128x128;
    const size_t narrow = (M + 191) / 192 * ((N + 255) / 256) * batch, small = (M + 127) / 128 * ((N + 127) / 128) * batch;
    return (narrow + 255) / 256 * 33 <= (small + 511) / 512 * 28 ? k192x256 : k128x128;
}

template <class T, MmMode MODE, bool TA, bool TB, class Epi>
int mm_launch(const MmArgs &g, MmShape shape, const Epi &epi, hipStream_t s) {
    if (shape == k192x256) return mm_launch_tile<T, MODE, TA, TB, 2, 4, 6, 4>(g, epi, s);
    return mm_launch<T, MODE, TA, TB>(g, shape == k256x256, epi, s);
}

}  // namespace vh
