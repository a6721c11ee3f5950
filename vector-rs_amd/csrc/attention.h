// attention.h -- what the passes of attention over packed sequences share: which rows a workgroup has, tiles of
// rows in LDS, and products of them on the matrix cores.
//
// Rows.  A query row is a (token, head).  The heads of a group read the same keys and values, so a tile holds
// consecutive packed rows of one sequence and one key head, packed row r being token r / group, head r % group of the
// group: keys are read once for the whole group, and a single token of many heads still fills a tile.
//
// Products.  All are 32 x 32 blocks (32x32x16 of 16-bit values, 32x32x2 of 32-bit ones), whose result has column l % 32
// in lane l and, in its register i, row 8 (i / 4) + 4 (l / 32) + i % 4.  Scores are made transposed to what multiplies
// them next: with S^T = K Q^T a lane has one query row and 16 of a block's keys, so a softmax needs one exchange between
// the lanes' halves, its statistics are a lane's own scalars, and the values that a lane holds are the ones that it
// has to give as operand of O^T = V^T P^T: the order of keys in that product is free as long as both operands have
// the same, so the operand from LDS is read in the order in which registers hold the other (no data moves between
// lanes).
//
// Tiles in LDS are rows of DP values as chunks of 16 bytes, chunk c of row r at slot c ^ swz(r): both the reads of a
// chunk of 32 rows and the transposing reads (4 rows x 32 bytes to 16 lanes) then spread over all banks.
#pragma once

#include <climits>
#include <type_traits>

#include "mm16.h"

namespace vh {
namespace attn {

typedef float floatx16_t __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// ---- which rows --------------------------------------------------------------------------------

// Sequences in one array of `tokens` rows.  The rows before the first and after the last one count as two more
// sequences without a counterpart on the other side.  Offsets are device data: each is clamped to the array, so wrong
// ones give wrong rows and no access out of bounds.
struct Packed {
    const int64_t *offsets;
    int64_t tokens;
    int count;  // sequences
};

struct Span {
    int64_t begin;
    int len;
};

__device__ __forceinline__ int64_t packed_bound(const Packed &p, int s) {
    if (s <= 0) return 0;
    if (s > p.count + 1) return p.tokens;
    const int64_t v = p.offsets[s - 1];
    return v < 0 ? 0 : v > p.tokens ? p.tokens : v;
}
__device__ __forceinline__ Span packed_span(const Packed &p, int s) {
    const int64_t b = packed_bound(p, s), e = packed_bound(p, s + 1);
    return {b, e > b ? (int)(e - b) : 0};
}

// Workgroup `slot` of ceil-sized tiles of R rows (times `mult` for each token) without a list of them: sequence s has
// the slots from floor(begin_s mult / R) + s on, which are as many as it has tiles or one more.  Each wave finds its
// s by itself, 64 candidates a round.
template <int R>
__device__ __forceinline__ int64_t first_slot(const Packed &p, int s, int mult) {
    return packed_bound(p, s) * mult / R + s;
}
inline int64_t slot_count(int64_t tokens, int64_t sequences, int64_t mult, int64_t R) { return tokens * mult / R + sequences + 2; }

struct Place {
    int seq;   // 0 and count + 1: rows of no sequence
    int tile;  // of that sequence; may be past its last
};
template <int R>
__device__ __forceinline__ Place find_tile(const Packed &p, int mult, int64_t slot) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = p.count + 2;
    for (int step = (hi + 63) / 64;; step = (step + 63) / 64) {
        const int s = lo + lane * step;
        const uint64_t in = __ballot(s < hi && first_slot<R>(p, s, mult) <= slot);
        const int n = in ? __popcll(in) : 1;
        lo += (n - 1) * step;
        hi = hi < lo + step ? hi : lo + step;
        if (step == 1) break;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    const int64_t t = slot - first_slot<R>(p, lo, mult);
    return {lo, __builtin_amdgcn_readfirstlane((int)(t < 0 ? INT_MAX : t > INT_MAX ? INT_MAX : t))};
}

// r / group, quickly where group is a power of two.
struct Group {
    int size, shift;  // shift < 0: not a power of two
    __device__ __forceinline__ int token(int r) const { return shift >= 0 ? r >> shift : (int)((unsigned)r / (unsigned)size); }
};

// Rows of one array: element (t, h, c) at t * token + h * head + c.
struct Heads {
    char *data;
    size_t token, head;  // bytes
};

// ---- tiles in LDS ------------------------------------------------------------------------------

// A cycle serves 256 bytes: 16 rows' same chunk, or the 64 bytes of each of 4 rows from 4 a on that half a wave reads by
// transposing. Rows of 256 bytes give the 4 rows other quarters of the banks, and the 16 rows all sixteen chunks.
constexpr int swz_of(int row_bytes, int r) {
    return row_bytes % 256 == 0 ? ((r & 3) << 2) | ((r >> 2) & 3)
           : row_bytes % 128 == 0 ? (((r >> 1) & 1) << 2) | ((r >> 2) & 3)
                                  : (r >> 2) & 3;
}

// dma_lds16_at with a lane's whole address: heads may be further apart than 32 bits count.
__device__ __forceinline__ void dma_lds16_far(const void *p, uint32_t m0_base) {
    uint32_t sv;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(sv)
                 : "v"(p), "s"(m0_base)
                 : "memory");
}

// A lane's number that the compiler takes for new: what is computed from it stays inside the loop that asks for it, where
// it costs an instruction or two a tile and no register from one tile to the next.
__device__ __forceinline__ int anew(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// A tile of ROWS rows of DP values that NW waves load.
template <class T, int DP, int ROWS, int NW, bool DMA>
struct Tile {
    static constexpr int RB = DP * (int)sizeof(T), CH = RB / 16, N = (ROWS * CH + NW * 64 - 1) / (NW * 64);
    static constexpr int kBytes = ROWS * RB;
    static constexpr int VEC = 16 / (int)sizeof(T);
    // Where a row's chunks are a power of two, the rows of a thread's loads are STEP apart and its chunk is the same.
    static constexpr int STEP = NW * 64 / CH;
    static constexpr bool kWhole = N * NW * 64 == ROWS * CH;  // or the last load is some waves' only
    static constexpr bool kEven = kWhole && (CH & (CH - 1)) == 0 && STEP % 16 == 0;  // 16: the rows' swizzle
    static_assert(ROWS * CH % 64 == 0, "whole waves");
    static constexpr int swz(int r) { return swz_of(RB, r); }

    static __device__ __forceinline__ void spot(int i, int thread, int &row, int &chunk) {
        const int n = i * NW * 64 + thread;
        row = n / CH;
        chunk = (n % CH) ^ swz(row);
    }
    // Loads the tile to `to`: row r is at base + at(r) bytes (uniform base; 32 or 64 bits), of `dim` values.  By DMA rows are
    // whole chunks at 16-byte addresses, and lanes whose chunk is past the last stay out of it: what is there are the zeros
    // of clear_past, as infinities or NaN times the other operand's zeros would be NaN.  Otherwise values come one vector at a
    // time, zeros past dim.
    template <class At>
    static __device__ __forceinline__ void load(const char *base, const At &at, int dim, char *to) {
        const int thread = anew(threadIdx.x);
        const uint32_t lds = place(to);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            int r, c;
            spot(i, thread, r, c);
            one(base, at(r), c, dim, to, lds, i, thread);
        }
    }
    // Zeros in the chunks past the last of `rows` rows, tiles one behind the other.
    static __device__ __forceinline__ void clear_past(int dim, int rows, char *to) {
        if constexpr (DMA) {
            const int first = dim * (int)sizeof(T) / 16;
            if (first == CH) return;
            for (int r = threadIdx.x; r < rows; r += NW * 64)
                for (int c = first; c < CH; ++c) *(Pack<float, 4> *)(to + r * RB + (c ^ swz(r)) * 16) = Pack<float, 4>{};
        }
    }
    // load() where row r + STEP i is i `step` bytes after row r (kEven): one lane's offset for all loads.
    template <class At>
    static __device__ __forceinline__ void load_even(const char *base, const At &at, int64_t step, int dim, char *to) {
        const int thread = anew(threadIdx.x);
        const uint32_t lds = place(to);
        int r, c;
        spot(0, thread, r, c);
        const auto off = at(r);
#pragma unroll
        for (int i = 0; i < N; ++i) one(base + i * step, off, c, dim, to, lds, i, thread);
    }

   private:
    static __device__ __forceinline__ uint32_t place(char *to) {
        return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)to + (threadIdx.x >> 6) * 1024);
    }
    template <class Off>
    static __device__ __forceinline__ void one(const char *base, Off off, int c, int dim, char *to, uint32_t lds, int i, int thread) {
        if (!kWhole && i == N - 1 && (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) >= ROWS * CH / 64 - i * NW) return;
        if constexpr (DMA) {
            if (c >= dim * (int)sizeof(T) / 16) return;
            if constexpr (sizeof(Off) == 4)
                dma_lds16_at(base, off + (uint32_t)c * 16, lds + i * NW * 1024);
            else
                dma_lds16_far(base + off + c * 16, lds + i * NW * 1024);
        } else {
            const auto v = load_row<VEC>((const T *)(base + off), c * VEC, dim);
            *(Pack<T, VEC> *)(to + (i * NW * 64 + thread) * 16) = v;
        }
    }
};

// A tile of consecutive rows from row0 on, of which those past `last` are copies of it; rows `stride` bytes apart, less
// than 2^25.
template <class TILE, int ROWS>
__device__ __forceinline__ void load_rows(const char *base, int64_t stride, int row0, int last, int dim, char *to) {
    const char *p = base + row0 * stride;
    const uint32_t s = (uint32_t)stride;
    last -= row0;
    if (TILE::kEven && last >= ROWS - 1)
        TILE::load_even(p, [&](int r) { return (uint32_t)r * s; }, TILE::STEP * stride, dim, to);
    else
        TILE::load(p, [&](int r) { return (uint32_t)min(r, last) * s; }, dim, to);
}

// A tile of packed rows from row0 on, those past `last` copies of it; base is token 0 of the group's first head.
template <class TILE, int ROWS>
__device__ __forceinline__ void load_packed(const char *base, const Heads &x, const Group &g, int row0, int last, int dim, char *to) {
    const int tok0 = g.token(row0);
    const char *p = base + tok0 * (int64_t)x.token;
    if (TILE::kEven && last >= row0 + ROWS - 1 && g.shift >= 0 && TILE::STEP % g.size == 0) {
        // the group divides STEP and so row0, a multiple of ROWS: the tile begins with the group's first head
        TILE::load_even(p, [&](int r) { return (int64_t)(r >> g.shift) * (int64_t)x.token + (int64_t)(r & (g.size - 1)) * (int64_t)x.head; },
                        (int64_t)(TILE::STEP >> g.shift) * (int64_t)x.token, dim, to);
    } else {
        TILE::load(p, [&](int i) {
            const int r = min(row0 + i, last), token = g.token(r);
            return (int64_t)(token - tok0) * (int64_t)x.token + (int64_t)(r - token * g.size) * (int64_t)x.head;
        }, dim, to);
    }
}

// ---- fragments and products --------------------------------------------------------------------

template <class T>
struct Frag;  // 16 bytes of a row: operand of a step of 32 bytes of k, half a step from each half of the lanes
template <>
struct Frag<half_t> {
    typedef MmVec<half_t>::v8 type;
};
template <>
struct Frag<bf16_t> {
    typedef MmVec<bf16_t>::v8 type;
};
template <>
struct Frag<float> {
    typedef floatx4_t type;
};

__device__ __forceinline__ floatx16_t mma(MmVec<half_t>::v8 a, MmVec<half_t>::v8 b, floatx16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ floatx16_t mma(MmVec<bf16_t>::v8 a, MmVec<bf16_t>::v8 b, floatx16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ floatx16_t mma(floatx4_t a, floatx4_t b, floatx16_t c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ constexpr int row_of(int i) { return 8 * (i / 4) + i % 4; }  // plus 4 (lane / 32)

// Chunk 2 ks + lane / 32 of row r0 + lane % 32 (r0 a multiple of 32).
template <class T, int RB>
__device__ __forceinline__ typename Frag<T>::type rows_frag(const char *tile, int r0, int ks, int lane) {
    const int r = lane & 31, x = swz_of(RB, r) ^ (lane >> 5);
    return *(const typename Frag<T>::type *)(tile + r * RB + ((2 * ks) ^ x) * 16 + r0 * RB);
}

// Operand k (of kOps) of columns 32 dt .. 32 dt + 31 of the tile's rows r0 .. r0 + 31, the rows in the order in which a
// product's registers hold its rows (see to_operand).
template <class T>
constexpr int kOps = sizeof(T) == 2 ? 2 : 4;
template <class T, int RB>
__device__ __forceinline__ typename Frag<T>::type cols_frag(const char *tile, int r0, int dt, int k, int lane) {
    if constexpr (sizeof(T) == 2) {
        typedef typename MmVec<T>::v4 v4;
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s4 lds_s4;
        const int g = lane >> 4, i = lane & 15, r = 4 * (g >> 1) + (i >> 2);
        const int x = (2 * (g & 1) + ((i & 3) >> 1)) ^ swz_of(RB, r);
        const char *p = tile + r * RB + (i & 1) * 8 + (r0 + 16 * k) * RB;
        const v4 lo = __builtin_bit_cast(v4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(p + ((4 * dt) ^ x) * 16)));
        const v4 hi = __builtin_bit_cast(
            v4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(p + 8 * RB + ((4 * dt) ^ x ^ swz_of(RB, 8)) * 16)));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
        const int h = lane >> 5, x = ((lane & 31) >> 2) ^ swz_of(RB, 4 * h);
        const char *p = tile + (r0 + 4 * h) * RB + (lane & 3) * 4;
        floatx4_t f;
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = *(const float *)(p + row_of(4 * k + e) * RB + ((8 * dt) ^ x ^ swz_of(RB, row_of(4 * k + e))) * 16);
        return f;
    }
}

// sum[d] += A^T B for the DT blocks of columns of A, the tile's rows r0 .. r0 + 31; B as to_operand gives it.
template <class T, int RB, int DT>
__device__ __forceinline__ void mma_cols(const char *tile, int r0, const typename Frag<T>::type (&b)[kOps<T>], floatx16_t (&sum)[DT], int lane) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int k = 0; k < kOps<T>; ++k) sum[d] = mma(cols_frag<T, RB>(tile, r0, d, k, lane), b[k], sum[d]);
}
// The same of two operands, by the same reads.
template <class T, int RB, int DT>
__device__ __forceinline__ void mma_cols2(const char *tile, int r0, const typename Frag<T>::type (&b)[kOps<T>], floatx16_t (&sum)[DT],
                                          const typename Frag<T>::type (&b2)[kOps<T>], floatx16_t (&sum2)[DT], int lane) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int k = 0; k < kOps<T>; ++k) {
            const auto f = cols_frag<T, RB>(tile, r0, d, k, lane);
            sum[d] = mma(f, b[k], sum[d]);
            sum2[d] = mma(f, b2[k], sum2[d]);
        }
}
// What is not seen has weight 0, which an infinity or NaN still turns into NaN. The forward pass multiplies without a thought
// for that; only where its sums are not finite in the end, it does its work once more with this form of mma_cols for tiles
// that are not seen as a whole (seen(i): what register i of B belongs to): zeros in place of A's values that are not finite,
// and then infinities and NaN where one that is seen has them. What is finite keeps its bits.
template <class T, int RB, int DT, class Seen>
__device__ __forceinline__ void mma_cols_masked(const char *tile, int r0, const typename Frag<T>::type (&b)[kOps<T>], floatx16_t (&sum)[DT],
                                                int lane, const Seen &seen) {
    typedef typename Frag<T>::type frag;
    constexpr int E = 16 / kOps<T>;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
#pragma unroll
        for (int k = 0; k < kOps<T>; ++k) {
            frag f = cols_frag<T, RB>(tile, r0, d, k, lane);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (!(fabsf((float)f[e]) < INFINITY)) f[e] = (T)0.f;
            sum[d] = mma(f, b[k], sum[d]);
        }
#pragma unroll 1
        for (int c = 0; c < 3; ++c) {
            floatx16_t count = {};
#pragma unroll
            for (int k = 0; k < kOps<T>; ++k) {
                frag f = cols_frag<T, RB>(tile, r0, d, k, lane), m;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float x = (float)f[e];
                    f[e] = (T)((c == 0 ? x == INFINITY : c == 1 ? x == -INFINITY : x != x) ? 1.f : 0.f);
                    m[e] = (T)(seen(k * E + e) ? 1.f : 0.f);
                }
                count = mma(f, m, count);
            }
            const float value = c == 0 ? INFINITY : c == 1 ? -INFINITY : NAN;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (count[i] > 0.f) sum[d][i] += value;
        }
    }
}
// NaN where a sum is not finite, 0 otherwise.
template <int DT>
__device__ __forceinline__ float not_finite(const floatx16_t (&sum)[DT]) {
    float bad = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) bad = fmaf(sum[d][i], 0.f, bad);
    return bad;
}
// A B over KS steps, A the tile's rows r0 .. r0 + 31.
template <class T, int RB, int KS>
__device__ __forceinline__ floatx16_t mma_rows(const char *tile, int r0, const typename Frag<T>::type (&b)[KS], int lane) {
    floatx16_t sum = {};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) sum = mma(rows_frag<T, RB>(tile, r0, ks, lane), b[ks], sum);
    return sum;
}

// The 16 values of a block as that operand: two of 8 in 16 bits, four of 4 in 32.
template <class T>
__device__ __forceinline__ void to_operand(const floatx16_t &v, typename Frag<T>::type (&o)[kOps<T>]) {
    constexpr int E = 16 / kOps<T>;
#pragma unroll
    for (int k = 0; k < kOps<T>; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) o[k][e] = (T)v[k * E + e];
}

// c plus the sum of an operand's values.
__device__ __forceinline__ float operand_sum(const MmVec<bf16_t>::v8 &v, float c) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    const v2 one = {(bf16_t)1.f, (bf16_t)1.f};
#pragma unroll
    for (int e = 0; e < 8; e += 2) c = __builtin_amdgcn_fdot2_f32_bf16(v2{v[e], v[e + 1]}, one, c, false);
    return c;
}
__device__ __forceinline__ float operand_sum(const MmVec<half_t>::v8 &v, float c) {
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    const v2 one = {(half_t)1.f, (half_t)1.f};
#pragma unroll
    for (int e = 0; e < 8; e += 2) c = __builtin_amdgcn_fdot2(v2{v[e], v[e + 1]}, one, c, false);
    return c;
}

// Writes a lane's part of a transposed result: its row's values 32 dt + 8 (i / 4) + 4 (lane / 32) + i % 4.
template <class T, int DT, class F>
__device__ __forceinline__ void store_cols(T *row, const floatx16_t (&acc)[DT], int dim, int lane, const F &f) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int c = 32 * dt + 8 * b + 4 * (lane >> 5);
            Pack<T, 4> v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v.v[e] = (T)f(acc[dt][4 * b + e]);
            if (c < dim) store_row<4>(row, c, dim, v);
        }
}

// Both halves' values together, in every lane.
template <class F>
__device__ __forceinline__ float both_halves(float x, const F &f) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    return f(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float half_max(float x) {
    return both_halves(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float half_sum(float x) {
    return both_halves(x, [](float a, float b) { return a + b; });
}

// Float16 has too few powers of two for a row's ds = p (dp - delta): what a lane's row or key adds up is held in
// units of 2^-e, e as large as lets its largest |ds| so far stay below 2^15.  A value then loses what falls below
// 2^-39 of that largest one.  Other types need none of it.
template <class T>
struct Units {
    static constexpr bool kOn = std::is_same<T, half_t>::value;
    int e = 100;
    // ds (a lane's 16 values and those of its other half) in units, sums scaled anew where those got coarser
    template <int DT>
    __device__ __forceinline__ void to_units(floatx16_t &ds, floatx16_t (&sum)[DT], float &sum2) {
        if constexpr (kOn) {
            float t = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) t = fmaxf(t, fabsf(ds[i]));
            t = half_max(t);
            const int next = t > 0.f ? min(e, 15 - __builtin_amdgcn_frexp_expf(t)) : e;
            if (__any(next != e)) {
                const float f = ldexpf(1.f, next - e);
                e = next;
                sum2 *= f;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum[d][i] *= f;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) ds[i] = ldexpf(ds[i], e);
        }
    }
    __device__ __forceinline__ float back(float x) const {
        if constexpr (kOn) return ldexpf(x, -e);
        return x;
    }
};

// All DMAs of this wave have landed, and everyone is past what it read before.
__device__ __forceinline__ void tiles_ready() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// The DP values of a row as DP / 4 threads' vectors of 4; a workgroup has as many rows, or parts of one, as fit (96 columns:
// 10 of 24 threads, and 16 idle ones).
template <int DP>
constexpr int kRowsOf256 = 256 / (DP / 4);

// ---- host --------------------------------------------------------------------------------------

// Arguments that all passes check alike.
struct Shape {
    size_t tokens, key_tokens, heads, kv_heads, dim, sequences;
};
inline size_t padded(size_t dim) { return round_up(dim, 32); }
// Parts of what a workgroup walks along (the keys that rows see, the rows that see keys), each a workgroup of its own, where there
// are fewer than `enough` workgroups; none is shorter than `shortest` of an average sequence.  Lengths are on the device, so
// it goes by the sizes alone.
constexpr int kMaxSplits = 64;
inline int split_count(int64_t workgroups, size_t along, size_t sequences, int enough, int shortest) {
    const int64_t each = (int64_t)(along / (sequences ? sequences : 1)) / shortest;
    int64_t n = enough / (workgroups ? workgroups : 1);
    n = n < each ? n : each;
    return n < 1 ? 1 : n > kMaxSplits ? kMaxSplits : (int)n;
}
// Of the keys, for workgroups of `rows` rows: enough for two on each CU, and more, since sequences differ in length, as long as the parts'
// sums (32 bits, written and read) stay below a quarter of the keys and values that are read: with few rows they do.
inline int key_splits(int dtype, const Shape &s, int rows) {
    const int64_t wgs = slot_count(s.tokens, s.sequences, s.heads / s.kv_heads, rows) * s.kv_heads;
    const int fill = split_count(wgs, s.key_tokens, s.sequences, 512, 256);
    const int even = split_count(wgs, s.key_tokens, s.sequences, 4096, 256);
    const size_t cheap = s.tokens ? s.key_tokens * s.kv_heads * dtype_size(dtype) / (s.tokens * s.heads * 16) : 0;
    const int more = cheap < (size_t)even ? (int)cheap : even;
    return fill > more ? fill : more;
}
inline Group to_group(size_t heads, size_t kv_heads) {
    const int n = (int)(heads / kv_heads);
    return {n, (n & (n - 1)) ? -1 : __builtin_ctz(n)};
}
int check_shape(int dtype, const Shape &s, const int64_t *offsets, const int64_t *key_offsets, float scale);
int check_heads(const char *name, const vhip_heads *a, int dtype, size_t tokens, size_t heads, size_t dim);
// Whether rows can be loaded by 16-byte chunks.
bool whole_chunks(const vhip_heads *a, int dtype, size_t dim);
Heads to_heads(const vhip_heads *a, int dtype);

}  // namespace attn
}  // namespace vh
