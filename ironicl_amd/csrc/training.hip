// Attention for training, its backward pass, and dropout.
//
// With x_ij = scale log2(e) q_i.k_j over the keys that a query attends to:
//   r_i = ceil(max_j x_ij), s_i = sum_j 2^(x_ij - r_i), P_ij = 2^(x_ij - r_i) / s_i
//   out_i = w sum_j P_ij Z_ij v_j, Z_ij in {0, 1} the weights' dropout, w = 65,536 / (65,536 - dropped)
// and, from dout and delta_i = dout_i.out_i:
//   dS_ij = P_ij (w Z_ij dout_i.v_j - delta_i)
//   dv_j = w sum_i P_ij Z_ij dout_i, dk_j = scale sum_i dS_ij q_i, dq_i = scale sum_j dS_ij k_j.
// The reference r is a whole number: FP32 holds it exactly at any size, and what was summed under another
// reference comes to it by an exact power of two. (One FP32 logarithm r + log2 s in place of the two
// would put 2^-24 of itself into every weight of its row: 1e-5 at scores of 300.)
//
// Products run on the 16-bit matrix cores with FP32 sums: BF16 and FP16 operands as they are, FP32 ones as
// pairs of FP16 values, three products (pair8; half the matrix cores' work of six products of three BF16 parts,
// with which 512 queries over 50,000 keys took 293 us and their gradients 1,019). Pairs keep 2^-23 of a number of
// [2^-14, 2^15] and 2^-25 of a smaller one, so FP32 operands and weights come to that range by powers of two:
//   - a lane's own row (of q, or of k and v) by its own;
//   - a streamed tile's rows by one power each for the tile's keys and its values (or queries and dout), the
//     largest number's. Rows 2^14 smaller than the largest go in a turn of their own over the same tile, so
//     that every row keeps 2^-24 of itself at least, whatever stands beside it;
//   - weights and dS by a lane's power, raised as larger terms come, its sums with it: what is rounded is below
//     2^-38 of the sum's largest term. FP16 operands' weights and dS, single values, take that too.
// BF16 has FP32's exponents; weights and dS are rounded to its eight bits and take no power.
#include "common.hpp"

#include <algorithm>
#include <cmath>

// LLVM's intrinsic, for which this compiler has no builtin: `old` with `value` in the named lane.
extern "C" __device__ unsigned irx_writelane(unsigned value, unsigned lane, unsigned old) __asm("llvm.amdgcn.writelane.i32");

namespace irx {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int kTile = 64;   // rows of a streamed tile
constexpr float kLn2 = 0.69314718055994530942f;

constexpr int parts_of(int element) { return element == kTrainF32 ? 2 : 1; }
constexpr bool scaled(int element) { return element == kTrainF32; }   // operands come by powers of two
constexpr bool ranged(int element) { return element != kTrainBF16; }  // weights and dS do
template <int EL>
using V8 = std::conditional_t<EL == kTrainBF16, bf16x8, half8>;
constexpr int kTop = 15;     // scaled numbers are below 2^15
constexpr int kSpread = 14;  // rows of a turn: exponents within 14 of the largest

// ---- elements ----

// Eight adjacent numbers as they lie in memory.
template <int EL>
struct Raw {
    u32x4 w[EL == kTrainF32 ? 2 : 1];
};

template <int EL>
__device__ __forceinline__ Raw<EL> load8(const void *base, long long at) {
    Raw<EL> r;
    const u32x4 *p = reinterpret_cast<const u32x4 *>(static_cast<const char *>(base) + at * (EL == kTrainF32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < (EL == kTrainF32 ? 2 : 1); ++i) r.w[i] = p[i];
    return r;
}

template <int EL>
__device__ __forceinline__ void to_floats(const Raw<EL> &r, float *x) {
    if constexpr (EL == kTrainF32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(r.w[i / 4][i % 4]);
    } else if constexpr (EL == kTrainF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned w = r.w[0][i];
            const half2v h = __builtin_bit_cast(half2v, w);
            x[2 * i] = (float)h[0], x[2 * i + 1] = (float)h[1];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(r.w[0][i] << 16);
            x[2 * i + 1] = __uint_as_float(r.w[0][i] & 0xffff0000u);
        }
    }
}

// Two numbers rounded to BF16 (nearest, ties to even), the first in the lower half.
__device__ __forceinline__ unsigned bf16_pair(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

// A number as three BF16 parts, each the rounded rest of those before: 24 bits.
__device__ __forceinline__ u32x2 bf16_parts(float x) {
    const unsigned a = bf16_pair(x, 0.f);
    const float y = x - __uint_as_float(a << 16);
    const unsigned b = bf16_pair(y, 0.f);
    return {a | b << 16, bf16_pair(y - __uint_as_float(b << 16), 0.f)};
}

// Eight FP32 numbers, times a power of two where SCALED, as pairs of FP16 values, the second the rounded rest of the first:
// each rest one mixed multiplication and addition (with an opaque -1 in place of a subtraction), the first's conversion kept
// from being made again for it.
template <bool SCALED>
__device__ __forceinline__ void pairs8(const float *x, float scale, half8 (&out)[2]) {
    u32x4 h, l;
    float minus = -1.f;
    asm("" : "+s"(minus));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = x[2 * i], b = x[2 * i + 1];
        unsigned w = __builtin_bit_cast(unsigned, __builtin_convertvector((SCALED ? f32x2{a * scale, b * scale} : f32x2{a, b}), half2v));
        asm("" : "+v"(w));
        const half2v hi = __builtin_bit_cast(half2v, w);
        half2v lo;
        lo[0] = (_Float16)(SCALED ? __builtin_fmaf(a, scale, -(float)hi[0]) : __builtin_fmaf((float)hi[0], minus, a));
        lo[1] = (_Float16)(SCALED ? __builtin_fmaf(b, scale, -(float)hi[1]) : __builtin_fmaf((float)hi[1], minus, b));
        h[i] = w, l[i] = __builtin_bit_cast(unsigned, lo);
    }
    out[0] = __builtin_bit_cast(half8, h), out[1] = __builtin_bit_cast(half8, l);
}

// Eight numbers as an operand's parts.
template <int EL>
__device__ __forceinline__ void operand8(const float *x, V8<EL> (&out)[parts_of(EL)]) {
    if constexpr (EL == kTrainF32) {
        pairs8<false>(x, 1.f, out);
    } else {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (EL == kTrainF16)
                w[i] = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{x[2 * i], x[2 * i + 1]}), half2v));
            else
                w[i] = bf16_pair(x[2 * i], x[2 * i + 1]);
        }
        out[0] = __builtin_bit_cast(V8<EL>, w);
    }
}

// Eight numbers as they lie in memory, FP32 ones times `scale`.
template <int EL>
__device__ __forceinline__ void raw_operand(const Raw<EL> &r, float scale, V8<EL> (&out)[parts_of(EL)]) {
    if constexpr (EL == kTrainF32) {
        float x[8];
        to_floats<EL>(r, x);
        pairs8<true>(x, scale, out);
    } else {
        out[0] = __builtin_bit_cast(V8<EL>, r.w[0]);
    }
}

// The largest size of eight FP32 numbers.
__device__ __forceinline__ float largest8(const Raw<kTrainF32> &r) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(__uint_as_float(r.w[i / 4][i % 4])));
    return m;
}

// A number's exponent field, held to 16 (2^-111) so that the powers below are normal.
__device__ __forceinline__ int field_of(float m) { return max(16, (int)(__float_as_uint(m) >> 23 & 255)); }
// x times scale_of(f) is below 2^15 where x has the exponent field f; 2^down(f) takes it back.
__device__ __forceinline__ int down(int f) { return f - 126 - kTop; }
__device__ __forceinline__ float scale_of(int f) { return __uint_as_float((unsigned)(127 - down(f)) << 23); }

// Four numbers rounded to the element type and stored.
template <int EL>
__device__ __forceinline__ void store4(void *base, long long at, f32x4 x) {
    if constexpr (EL == kTrainF32) {
        *reinterpret_cast<f32x4 *>(static_cast<float *>(base) + at) = x;
    } else if constexpr (EL == kTrainF16) {
        const half2v a = __builtin_convertvector((f32x2{x[0], x[1]}), half2v);
        const half2v b = __builtin_convertvector((f32x2{x[2], x[3]}), half2v);
        *reinterpret_cast<u32x2 *>(static_cast<unsigned short *>(base) + at) =
            u32x2{__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b)};
    } else {
        *reinterpret_cast<u32x2 *>(static_cast<unsigned short *>(base) + at) =
            u32x2{bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3])};
    }
}

template <int EL>
__device__ __forceinline__ void store1(void *base, long long at, float x) {
    if constexpr (EL == kTrainF32)
        static_cast<float *>(base)[at] = x;
    else if constexpr (EL == kTrainF16)
        static_cast<_Float16 *>(base)[at] = (_Float16)x;
    else
        static_cast<unsigned short *>(base)[at] = (unsigned short)bf16_pair(x, 0.f);
}

template <int EL>
__device__ __forceinline__ f32x4 load4(const void *base, long long at) {
    if constexpr (EL == kTrainF32) {
        return *reinterpret_cast<const f32x4 *>(static_cast<const float *>(base) + at);
    } else {
        const u32x2 w = *reinterpret_cast<const u32x2 *>(static_cast<const unsigned short *>(base) + at);
        if constexpr (EL == kTrainF16) {
            const unsigned low = w[0], high = w[1];
            const half2v a = __builtin_bit_cast(half2v, low), b = __builtin_bit_cast(half2v, high);
            return f32x4{(float)a[0], (float)a[1], (float)b[0], (float)b[1]};
        } else {
            return f32x4{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u), __uint_as_float(w[1] << 16),
                         __uint_as_float(w[1] & 0xffff0000u)};
        }
    }
}

// ---- products ----

// acc += A B, of pairs the small terms first.
template <int EL>
__device__ __forceinline__ void mma(f32x16 &acc, const V8<EL> (&a)[parts_of(EL)], const V8<EL> (&b)[parts_of(EL)]) {
    if constexpr (EL == kTrainF32) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1], b[0], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[1], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[0], acc, 0, 0, 0);
    } else if constexpr (EL == kTrainF16) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[0], acc, 0, 0, 0);
    } else {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[0], acc, 0, 0, 0);
    }
}

// A tile in LDS: for each part a plane of 64 rows of 64 16-bit numbers, so that loads can go straight there. The 64 banks hold
// two rows; number d of row r lies in the row's 16 bytes (d / 8) ^ swizzle(r). Sixteen rows' 16 bytes of the same dims, as a
// rows operand takes them at once, meet no bank twice, and nor do four rows' 64 bytes, as a dims operand does.
template <int EL>
struct Tile {
    alignas(16) unsigned short p[parts_of(EL)][kTile * 64];
};
__device__ __forceinline__ int swizzle(int row) { return (row & 2) * 2 | (row >> 2 & 3); }
__device__ __forceinline__ int swizzled(int row, int chunk) { return row * 64 + 8 * (chunk ^ swizzle(row)); }

// Where a lane's operands of row 0 and dim 0 begin; a row is 64 on, dims 16 c (of rows) and 32 d (of dims) are exclusive ors.
struct Lanes {
    int rows, dims, dims8;  // dims8: eight rows on
    __device__ __forceinline__ explicit Lanes(int lane) {
        const int row = 4 * (lane >> 5) + (lane & 15) / 4, chunk = (lane & 16) / 8 + (lane & 3) / 2;
        rows = swizzled(lane & 31, lane >> 5);
        dims = swizzled(row, chunk) + 4 * (lane & 1);
        dims8 = swizzled(row + 8, chunk) + 4 * (lane & 1);
    }
};

// The A operand of rows `row0` .. + 31, dims 16 c .. + 15: lane (row l % 32, half h) holds dims 16 c + 8 h .. + 7.
template <int EL>
__device__ __forceinline__ void rows_operand(const Tile<EL> &t, int row0, int c, const Lanes &l, V8<EL> (&a)[parts_of(EL)]) {
    const int at = row0 * 64 + (l.rows ^ 16 * c);
#pragma unroll
    for (int p = 0; p < parts_of(EL); ++p) a[p] = __builtin_bit_cast(V8<EL>, *reinterpret_cast<const u32x4 *>(&t.p[p][at]));
}

// The A operand of dims 32 d .. + 31 over rows row0 .. + 15, for a B operand whose eight numbers in half h are those of rows
// 4 h .. + 3 and 8 + 4 h .. + 3: a product's result as it lies in a lane.
template <int EL>
__device__ __forceinline__ void dims_operand(const Tile<EL> &t, int row0, int d, const Lanes &l, V8<EL> (&a)[parts_of(EL)]) {
    typedef __attribute__((address_space(3))) s16x4 *lds4;
    const int at = row0 * 64 + (l.dims ^ 32 * d), at8 = row0 * 64 + (l.dims8 ^ 32 * d);
#pragma unroll
    for (int p = 0; p < parts_of(EL); ++p) {
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(&t.p[p][at]));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(&t.p[p][at8]));
        a[p] = __builtin_bit_cast(V8<EL>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
}

__device__ __forceinline__ float other_half(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// ---- random numbers ----

// Philox4x32 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) with seven rounds, the
// fewest that pass their whole test suite. FLIP: an exclusive or with every word, half of it in what the last round adds.
template <unsigned FLIP = 0>
__device__ __forceinline__ u32x4 philox(unsigned c0, unsigned c1, unsigned c2, unsigned c3, unsigned long long seed) {
    unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
#pragma unroll
    for (int round = 0; round < 7; ++round) {
        if (round == 6) k0 ^= FLIP, k1 ^= FLIP;
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = __builtin_amdgcn_bitop3_b32((unsigned)(b >> 32), c1, k0, 0x96);  // the three's exclusive or
        c1 = (unsigned)b;
        c2 = __builtin_amdgcn_bitop3_b32((unsigned)(a >> 32), c3, k1, 0x96);
        c3 = (unsigned)a;
        k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
    }
    return u32x4{c0, c1 ^ FLIP, c2, c3 ^ FLIP};
}

// Whether number j of a call's eight 16-bit ones is kept; `line` is dropped << 16.
__device__ __forceinline__ bool kept16(const u32x4 &w, int j, unsigned line) {
    return (j & 1 ? w[j >> 1] : w[j >> 1] << 16) >= line;
}

// Eight 16-bit numbers without those that a call drops. `z` holds its words with every value's highest bit flipped, so that
// two values at a time are compared as signed ones: a saturated difference's sign, over the half, is the mask (3.5
// instructions a pair, with comparisons and selections 5).
constexpr unsigned kFlip = 0x80008000u;
template <int EL>
__device__ __forceinline__ V8<EL> drop8(V8<EL> x, const u32x4 &z, unsigned line) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    u32x4 w = __builtin_bit_cast(u32x4, x);
    const s16x2 at = __builtin_bit_cast(s16x2, (line | line >> 16) ^ kFlip);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned values = z[i];
        const s16x2 below = __builtin_elementwise_sub_sat(__builtin_bit_cast(s16x2, values), at) >> 15;
        const unsigned lost = __builtin_bit_cast(unsigned, below);
        w[i] &= ~lost;
    }
    return __builtin_bit_cast(V8<EL>, w);
}

// ---- lengths and masks ----

__device__ __forceinline__ int length_of(const unsigned *lengths, int e, int rows) {
    return lengths ? (int)min(lengths[e], (unsigned)rows) : rows;
}

// Bit r: key 64 word + r is attended; `rows` is the estimator's length.
__device__ __forceinline__ unsigned long long attended(const unsigned long long *keep, int words, int e, int word, int rows) {
    const int left = rows - word * 64;
    if (left <= 0) return 0;
    unsigned long long m = keep ? keep[(long long)e * words + word] : ~0ull;
    if (left < 64) m &= (1ull << left) - 1;
    return m;
}

// Scores of keys row0 .. + 31 of a tile that are not attended become -inf.
__device__ __forceinline__ void leave_out(f32x16 &s, unsigned long long some, int row0, int half) {
    const unsigned bits = (unsigned)(some >> (row0 + 4 * half));
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = bits >> (8 * (i / 4) + i % 4) & 1 ? s[i] : -INFINITY;
}

struct Args {
    const void *q, *k, *v;
    long long qs[3], ks[3], vs[3];
    const unsigned *q_lengths, *lengths;
    const unsigned long long *keep;
    int heads, kv_heads, pairs, q_rows, rows, words;
    float scale, c;  // c = scale log2(e)
    const unsigned long long *seed;
    unsigned site, line;
    float w;
    // forward
    void *out;
    long long os[3];
    float *stats, *lse;
    // backward
    const void *dout;
    void *dq, *dk, *dv;
    long long gs[3], dqs[3], dks[3], dvs[3];
    f32x4 *record;
    // plans
    int q_tiles, q_splits, q_chunk;  // units of queries; a split's key tiles
    int k_tiles, k_splits, k_chunk;  // units of 128 keys; a split's query tiles
    int q_blocks;                    // workgroups on queries, before those on keys
    float *q_part, *k_part;
    int keys_last;  // 1: the keys' side walks further
};

__device__ __forceinline__ long long at(const long long *s, int e, int h, int row) {
    return e * s[0] + h * s[1] + (long long)row * s[2];
}

// x 2^by (x > 0), held to FP32's normal numbers: a factor of 0 or of infinity would make NaN of scores that are left out or 0.
// Where the power would be a smaller one, scores are below 2^-90. dP, of which any size counts, takes its power by itself.
__device__ __forceinline__ float times_power(float x, int by) {
    return fminf(fmaxf(__builtin_ldexpf(x, by), 0x1p-126f), 0x1p127f);
}

// The largest of eight adjacent lanes' values.
__device__ __forceinline__ float largest_of_8_lanes(float m) {
    auto step = [&](int moved) { m = fmaxf(m, __int_as_float(moved)); };
    step(__builtin_amdgcn_mov_dpp(__float_as_int(m), 0xB1, 15, 15, true));   // lane ^ 1
    step(__builtin_amdgcn_mov_dpp(__float_as_int(m), 0x4E, 15, 15, true));   // lane ^ 2
    step(__builtin_amdgcn_mov_dpp(__float_as_int(m), 0x141, 15, 15, true));  // lane ^ 7
    return m;
}

// 16-bit elements: a tile of rows row0 .. + 63 straight to LDS, a wave's instruction to eight rows. Rows past `rows` are read
// from the last.
template <int EL, int NT>
__device__ __forceinline__ void load_tile(Tile<EL> &t, const void *base, const long long *s, int e, int h, int row0, int rows) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < 512 / NT; ++i) {
        const int first = 8 * (wave + i * (NT / 64)), row = first + lane / 8;
        const long long place = at(s, e, h, min(row0 + row, rows - 1)) + 8 * ((lane & 7) ^ swizzle(row));
        const unsigned short *from = static_cast<const unsigned short *>(base) + place;
        __builtin_amdgcn_global_load_lds(from, (__attribute__((address_space(3))) void *)&t.p[0][first * 64], 16, 0, 0);
    }
}

// A wave's loads to LDS have arrived: vmcnt(0); expcnt and lgkmcnt left at their maxima (no wait). What other waves loaded has
// arrived after the barrier that follows.
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0F70); }

// Rows whose bit is not set become zeros, whatever they hold.
template <int EL, int NT>
__device__ __forceinline__ void clear_rows(Tile<EL> &t, unsigned long long some) {
#pragma unroll
    for (int i = 0; i < 512 / NT; ++i) {
        const int u = threadIdx.x + i * NT;
        if (!(some >> u / 8 & 1)) *reinterpret_cast<u32x4 *>(&t.p[0][8 * u]) = u32x4{0, 0, 0, 0};
    }
}

// FP32: a tile's numbers on their way to LDS. NT threads load 64 x 64, eight adjacent ones at a time.
template <int EL, int NT>
struct Staged {
    static constexpr int N = 512 / NT;
    Raw<EL> r[N];

    // Rows past `rows` are read from the last.
    __device__ __forceinline__ void load(const void *base, const long long *s, int e, int h, int row0, int rows) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = threadIdx.x + i * NT;
            r[i] = load8<EL>(base, at(s, e, h, min(row0 + u / 8, rows - 1)) + 8 * (u % 8));
        }
    }
    // FP32: rows times what stands for them in `factor`.
    __device__ __forceinline__ void times(const float (&factor)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) r[i].w[j / 4][j % 4] = __float_as_uint(__uint_as_float(r[i].w[j / 4][j % 4]) * factor[i]);
    }
    // FP32: every row's largest number's exponent field, 0 for zeros.
    __device__ __forceinline__ void fields(int *to) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = threadIdx.x + i * NT;
            const float m = largest_of_8_lanes(largest8(r[i]));
            if (u % 8 == 0) to[u / 8] = (int)(__float_as_uint(m) >> 23);
        }
    }
    // Rows whose bit is not set become zeros, whatever they hold.
    __device__ __forceinline__ void store(Tile<EL> &t, unsigned long long some, float scale) const {
        if (some == ~0ull)
            put<true>(t, some, scale);
        else
            put<false>(t, some, scale);
    }
    template <bool ALL>
    __device__ __forceinline__ void put(Tile<EL> &t, unsigned long long some, float scale) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = threadIdx.x + i * NT, row = u / 8;
            V8<EL> b[parts_of(EL)];
            raw_operand<EL>(r[i], scale, b);
            const bool in = ALL || (some >> row & 1);
#pragma unroll
            for (int p = 0; p < parts_of(EL); ++p) {
                u32x4 w = __builtin_bit_cast(u32x4, b[p]);
                if (!in) w = u32x4{0, 0, 0, 0};
                *reinterpret_cast<u32x4 *>(&t.p[p][swizzled(row, u % 8)]) = w;
            }
        }
    }
};

// A wave's largest value, in every lane. (Through LDS, as shuffles go, six steps cost a tile more than its softmax.)
__device__ __forceinline__ int wave_max_int(int v) {
    v = max(v, __builtin_amdgcn_mov_dpp(v, 0xB1, 15, 15, true));   // lane ^ 1
    v = max(v, __builtin_amdgcn_mov_dpp(v, 0x4E, 15, 15, true));   // lane ^ 2
    v = max(v, __builtin_amdgcn_mov_dpp(v, 0x141, 15, 15, true));  // lane ^ 7
    v = max(v, __builtin_amdgcn_mov_dpp(v, 0x140, 15, 15, true));  // lane ^ 15
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max((int)a[0], (int)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max((int)b[0], (int)b[1]);
}

// The rows of `todo` that a turn takes, and the exponent fields for x and y: those within 2^14 of the largest x (rows of
// zeros go with any), and of them those within 2^14 of the largest y. It takes one row at least.
struct Turn {
    unsigned long long some;
    int x, y;
};
__device__ __forceinline__ Turn turn_of(unsigned long long todo, const int *fx, const int *fy, int lane) {
    const bool mine = todo >> lane & 1;
    const int x = mine ? fx[lane] : 0, y = fy[lane];
    const int most_x = wave_max_int(x);
    bool in = mine && (x == 0 || x >= most_x - kSpread);
    const int most_y = wave_max_int(in ? y : 0);
    in = in && (y == 0 || y >= most_y - kSpread);
    return {__ballot(in), __builtin_amdgcn_readfirstlane(max(16, most_x)), __builtin_amdgcn_readfirstlane(max(16, most_y))};
}

// The B operand of a lane's own row: dims 16 c + 8 h .. + 7; zeros where !in. FP32: returns the row's exponent field.
template <int EL>
__device__ __forceinline__ int own_row(const void *base, long long row, bool in, int lane, V8<EL> (&b)[4][parts_of(EL)]) {
    Raw<EL> r[4] = {};
    if (in)
#pragma unroll
        for (int c = 0; c < 4; ++c) r[c] = load8<EL>(base, row + 16 * c + 8 * (lane >> 5));
    int field = 127;
    float scale = 1.f;
    if constexpr (scaled(EL)) {
        float m = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) m = fmaxf(m, largest8(r[c]));
        field = field_of(fmaxf(m, other_half(m)));
        scale = scale_of(field);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) raw_operand<EL>(r[c], scale, b[c]);
    return field;
}

// FP32 and FP16: weights or dS of 32 rows brought below 2^15 by a lane's power 2^-k, k raised where they need it, and what a
// lane has summed under the former one with it. `row`: the power that the streamed rows of the product came by.
__device__ __forceinline__ void bring(f32x16 &x, float most, int row, int &k, f32x16 (&sums)[2]) {
    if (__any(__builtin_ldexpf(most, row - k) >= 32768.f)) {
        // A factor of two to spare, so that a slightly larger term does not raise it again.
        const int raised = max(k, row + (int)(__float_as_uint(most) >> 23) - 126 - (kTop - 1));
        const int by = max(k - raised, -300);
#pragma unroll
        for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) sums[d][i] = __builtin_ldexpf(sums[d][i], by);
        k = raised;
    }
    const int by = row - k;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = __builtin_ldexpf(x[i], by);
}
constexpr int kNone = -1000;  // a lane's power before its first term

// ---- forward ----

// 32 WQ queries to a workgroup, 32 to a wave; keys and values pass through LDS in tiles of 64, and where WK is 2 a wave
// takes 32 of each. S^T = K Q^T leaves a query's scores in one lane (and its other half), in the order in which the next
// product takes them. FP32 tiles are loaded into registers while the last is worked on and become pairs on their way to LDS;
// 16-bit ones go straight to LDS, the next tile's while one's scores and softmax are worked on: the compiler, which cannot tell
// the two buffers apart, has the transposed reads of one wait for the loads to the other. (With two buffers and two barriers
// a tile in place of one, FP32's took as long.)
// 512 FP32 queries over 50,000 rows of 8 heads: 200 to 218 us, 250 TFLOP/s, the matrix cores 36% busy and the vector unit 55%;
// with two waves a SIMD they overlap little (a wave alone issues a vector instruction every seven cycles), and a third wave's
// registers are not there. (icl_attention_kernel, eight waves to a workgroup with products and softmax opposite each other,
// takes 165 for the same products.) 10,007 BF16 rows over themselves with dropout: 361 to 401 us, the vector unit 79% busy,
// half of it with random numbers.
constexpr int forward_waves(int element, int wq, int wk) {  // of a SIMD: what registers leave room for
    return element == kTrainF32 ? 2 : wq * wk;
}
template <int EL, int WQ, int WK, bool DROP>
__global__ __launch_bounds__(64 * WQ * WK, forward_waves(EL, WQ, WK)) void train_forward_kernel(const Args a) {
    constexpr int P = parts_of(EL), NT = 64 * WQ * WK, NS = 2 / WK;
    constexpr float TOP = ranged(EL) ? kTop - 1 : 0;  // weights are brought below 2^TOP
    __shared__ Tile<EL> tiles[scaled(EL) ? 1 : 2][2];  // 16-bit: the next tile's while one is worked on
    __shared__ int fields[2][scaled(EL) ? kTile : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wq = wave % WQ, wk = wave / WQ, half = lane >> 5;
    const unsigned unit = blockIdx.x / (unsigned)a.pairs;
    const int pair = blockIdx.x % (unsigned)a.pairs, tile = unit % (unsigned)a.q_tiles, split = unit / (unsigned)a.q_tiles;
    const int e = pair / a.heads, h = pair % a.heads, hk = h / (a.heads / a.kv_heads);
    const int q_len = length_of(a.q_lengths, e, a.q_rows), len = length_of(a.lengths, e, a.rows);
    if (tile * 32 * WQ >= q_len) return;
    const int query = tile * 32 * WQ + 32 * wq + (lane & 31);
    const bool mine = query < q_len;
    V8<EL> qb[4][P];
    const int q_down = down(own_row<EL>(a.q, at(a.qs, e, h, query), mine, lane, qb));

    // o holds sum 2^(x - k) v: with FP32 a value's tile comes by 2^-v_down, its weights by 2^v_down, and k follows the largest
    // of x + v_down, apart from the sum's reference r. With 16-bit elements k is r - TOP. FP32's sum is that of the same
    // weights, taken back to r, but where earlier values outweigh a tile's by so much (2^60) that weights of its order fall
    // out of FP32's range beside them: there it has exponentials of its own.
    f32x16 o[2] = {};
    float r = -INFINITY, k = -INFINITY, sum = 0.f;
    const unsigned long long seed = DROP ? *a.seed : 0;
    const int end = min((split + 1) * a.q_chunk, (int)((len + 63) / 64));
    auto next = [&](int t, unsigned long long &m) {
        for (m = 0; t < end && !(m = attended(a.keep, a.words, e, t, len)); ++t) {}
        return t;
    };
    const Lanes lanes(lane);
    // One turn: rows `some` of tile t, its keys by 2^-k_down and its values by 2^-v_down.
    auto work = [&](const Tile<EL> &kt, const Tile<EL> &vt, int t, unsigned long long some, int k_down, int v_down) {
        const float c = scaled(EL) ? times_power(a.c, k_down + q_down) : a.c;
        f32x16 s[NS] = {};
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int b = 0; b < NS; ++b) {
                V8<EL> x[P];
                rows_operand<EL>(kt, 32 * (WK == 1 ? b : wk), c, lanes, x);
                mma<EL>(s[b], x, qb[c]);
            }
        if (some != ~0ull)
#pragma unroll
            for (int b = 0; b < NS; ++b) leave_out(s[b], some, 32 * (WK == 1 ? b : wk), half);
        float top = -INFINITY;
#pragma unroll
        for (int b = 0; b < NS; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
        // A scale is positive: the largest score is that of the largest product.
        top = ceilf(fmaxf(top, other_half(top)) * c);
        const float upto = fmaxf(k, top + (float)v_down - TOP);
        if (__any(upto > k)) {
            const float f = k == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(k - upto);
            if constexpr (!scaled(EL)) sum *= f;
#pragma unroll
            for (int d = 0; d < 2; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= f;
            k = upto;
        }
        const float from = (float)v_down - (k == -INFINITY ? 0.f : k);
        float part = 0.f, own = 0.f;
        const float most = fmaxf(r, top), ref = most == -INFINITY ? 0.f : most;
        const bool apart = scaled(EL) && __any(-from - ref > 60.f);
        if (apart)
#pragma unroll
            for (int b = 0; b < NS; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) own += __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], c, -ref));
#pragma unroll
        for (int b = 0; b < NS; ++b) {
            const int sub = WK == 1 ? b : wk;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[b][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], c, from));
                part += s[b][i];
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) p[j] = s[b][8 * c + j];
                u32x4 z;
                if constexpr (DROP) z = philox<scaled(EL) ? 0 : kFlip>(2 * (4 * t + 2 * sub + c) + half, query, pair, a.site, seed);
                if constexpr (DROP && scaled(EL))
#pragma unroll
                    for (int j = 0; j < 8; ++j) p[j] = kept16(z, j, a.line) ? p[j] : 0.f;
                V8<EL> pb[P];
                operand8<EL>(p, pb);
                if constexpr (DROP && !scaled(EL)) pb[0] = drop8<EL>(pb[0], z, a.line);
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    V8<EL> x[P];
                    dims_operand<EL>(vt, 32 * sub + 16 * c, d, lanes, x);
                    mma<EL>(o[d], x, pb);
                }
            }
        }
        if constexpr (scaled(EL)) {
            const float here = apart ? own : part * __builtin_amdgcn_exp2f(-from - ref);
            sum = sum * (r == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(r - ref)) + here;
            r = most;
        } else {
            sum += part;
        }
    };
    unsigned long long todo, following = 0;
    int t = next(split * a.q_chunk, todo);
    if constexpr (scaled(EL)) {
        Staged<EL, NT> ks, vs;
        auto load = [&](int tile) {
            ks.load(a.k, a.ks, e, hk, tile * 64, len);
            vs.load(a.v, a.vs, e, hk, tile * 64, len);
        };
        if (t < end) load(t);
        bool fresh = true;
        while (t < end) {
            if (fresh) ks.fields(fields[0]), vs.fields(fields[1]);
            __syncthreads();
            const Turn turn = turn_of(todo, fields[0], fields[1], lane);
            ks.store(tiles[0][0], turn.some, scale_of(turn.x));
            vs.store(tiles[0][1], turn.some, scale_of(turn.y));
            __syncthreads();
            todo &= ~turn.some;
            const int at_tile = t;
            fresh = !todo;
            if (fresh) {
                t = next(t + 1, following);
                if (t < end) load(t);
                todo = following;
            }
            work(tiles[0][0], tiles[0][1], at_tile, turn.some, down(turn.x), down(turn.y));
        }
    } else {
        auto load = [&](int tile, int to) {
            load_tile<EL, NT>(tiles[to][0], a.k, a.ks, e, hk, tile * 64, len);
            load_tile<EL, NT>(tiles[to][1], a.v, a.vs, e, hk, tile * 64, len);
        };
        if (t < end) load(t, 0);
        for (int now = 0; t < end; now ^= 1) {
            wait_loads();
            __syncthreads();  // the tile has come, and the other is read
            if (todo != ~0ull) {
                clear_rows<EL, NT>(tiles[now][0], todo), clear_rows<EL, NT>(tiles[now][1], todo);
                __syncthreads();
            }
            const int n = next(t + 1, following);
            if (n < end) load(n, now ^ 1);
            work(tiles[now][0], tiles[now][1], t, todo, 0, 0);
            t = n, todo = following;
        }
    }
    sum += other_half(sum);
    if constexpr (scaled(EL)) {
        const int by = sum == 0.f ? 0 : (int)(k - r);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i / 16][i % 16] = __builtin_ldexpf(o[i / 16][i % 16], by);
    } else if constexpr (TOP != 0) {
        r = k + TOP, sum = __builtin_ldexpf(sum, (int)-TOP);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i / 16][i % 16] = __builtin_ldexpf(o[i / 16][i % 16], (int)-TOP);
    } else {
        r = k;
    }
    if constexpr (WK == 2) {
        // The second wave's half of the keys joins the first's.
        struct Half {
            float o[32][64], r[64], sum[64];
        };
        static_assert(WQ * sizeof(Half) <= sizeof(tiles));
        Half *join = reinterpret_cast<Half *>(tiles) + wq;
        __syncthreads();
        if (wk == 1) {
#pragma unroll
            for (int i = 0; i < 32; ++i) join->o[i][lane] = o[i / 16][i % 16];
            join->r[lane] = r, join->sum[lane] = sum;
        }
        __syncthreads();
        if (wk == 1) return;
        const float upto = fmaxf(r, join->r[lane]), ref = upto == -INFINITY ? 0.f : upto;
        const float f = __builtin_amdgcn_exp2f(r - ref), g = __builtin_amdgcn_exp2f(join->r[lane] - ref);
        r = upto, sum = sum * f + join->sum[lane] * g;
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i / 16][i % 16] = o[i / 16][i % 16] * f + join->o[i][lane] * g;
    }
    if (!mine) return;
    const long long row = (long long)pair * a.q_rows + query;
    if (a.q_splits > 1) {
        float *part = a.q_part + ((long long)split * a.pairs * a.q_rows + row) * 64;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const f32x16 &x = o[i / 4];
            const int j = 4 * (i % 4);
            *reinterpret_cast<f32x4 *>(part + 32 * (i / 4) + 2 * j + 4 * half) = f32x4{x[j], x[j + 1], x[j + 2], x[j + 3]};
        }
        if (!half) {
            float *m = a.q_part + (long long)a.q_splits * a.pairs * a.q_rows * 64 + ((long long)split * a.pairs * a.q_rows + row) * 2;
            *reinterpret_cast<f32x2 *>(m) = f32x2{r, sum};
        }
        return;
    }
    const float f = sum == 0.f ? 0.f : a.w / sum;
    const long long to = at(a.os, e, h, query);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const f32x16 &x = o[i / 4];
        const int j = 4 * (i % 4);
        store4<EL>(a.out, to + 32 * (i / 4) + 2 * j + 4 * half, f32x4{x[j] * f, x[j + 1] * f, x[j + 2] * f, x[j + 3] * f});
    }
    if (!half) {
        const float ref = r == -INFINITY ? 0.f : r;
        if (a.stats) *reinterpret_cast<f32x2 *>(a.stats + 2 * row) = f32x2{ref, sum};
        if (a.lse) a.lse[row] = kLn2 * (ref + __builtin_amdgcn_logf(sum));
    }
}

// One to eight rows (queries of the heads that share a key head) against their keys, for which the matrix cores' 32 columns
// stand empty and reading keys and values is all there is: FP32 sums, LK lanes to a key (16 bytes each), eight keys of one
// call of random numbers to a group of lanes, a wave's 64 keys (FP32: 32) in flight at once. One query of 8 FP32 heads over
// 50,000 rows: 31 us, 6.6 TB/s, and 5 for the joining of 32 splits.
template <int EL, int NQ, bool DROP>
__global__ __launch_bounds__(256) void train_rows_kernel(const Args a) {
    constexpr int D = EL == kTrainF32 ? 4 : 8, LK = 64 / D, GROUPS = 64 / LK;  // dims of a lane; groups of a wave
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane / LK, dim = D * (lane % LK);
    const int share = a.heads / a.kv_heads, owners = a.pairs / share;
    const int owner = blockIdx.x % (unsigned)owners, split = blockIdx.x / (unsigned)owners;
    const int e = owner / a.kv_heads, hk = owner % a.kv_heads;
    const int q_len = length_of(a.q_lengths, e, a.q_rows), len = length_of(a.lengths, e, a.rows);
    if (!q_len) return;
    auto place = [&](int n, int &h, int &query) {
        n = min(n, share * a.q_rows - 1);
        h = hk * share + n / a.q_rows, query = n % a.q_rows;
    };
    float q[NQ][D], o[NQ][D] = {}, r[NQ], sum[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        int h, query;
        place(n, h, query);
        r[n] = -INFINITY, sum[n] = 0.f;
#pragma unroll
        for (int j = 0; j < D; j += 4) {
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
            if (query < q_len) x = load4<EL>(a.q, at(a.qs, e, h, query) + dim + j);
#pragma unroll
            for (int i = 0; i < 4; ++i) q[n][j + i] = x[i];
        }
    }
    const unsigned long long seed = DROP ? *a.seed : 0;
    const int end = min((split + 1) * a.q_chunk, (int)((len + 63) / 64));
    for (int t = split * a.q_chunk + wave; t < end; t += 4) {
        const unsigned long long some = attended(a.keep, a.words, e, t, len);
        if (!some) continue;
#pragma unroll 1
        for (int first = 0; first < 64; first += 8 * GROUPS) {
            // The group's cell: keys 16 (cell / 2) + 4 (cell % 2) + 0..3 and 8..11 of the tile.
            const int cell = first / 8 + group, base = 16 * (cell / 2) + 4 * (cell % 2);
            u32x4 k[8], v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int row = min(t * 64 + base + 8 * (j / 4) + j % 4, len - 1);
                const int bytes = EL == kTrainF32 ? 4 : 2;
                k[j] = *reinterpret_cast<const u32x4 *>(static_cast<const char *>(a.k) + (at(a.ks, e, hk, row) + dim) * bytes);
                v[j] = *reinterpret_cast<const u32x4 *>(static_cast<const char *>(a.v) + (at(a.vs, e, hk, row) + dim) * bytes);
            }
            const unsigned bits = (unsigned)(some >> base);
            if (some != ~0ull)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!(bits >> (8 * (j / 4) + j % 4) & 1)) k[j] = v[j] = u32x4{0, 0, 0, 0};
            auto numbers = [](const u32x4 &w, float *x) {
                Raw<EL> raw;
                if constexpr (EL == kTrainF32) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
                } else {
                    raw.w[0] = w;
                    to_floats<EL>(raw, x);
                }
            };
            float x[NQ][8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float kk[D];
                numbers(k[j], kk);
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    float d = 0.f;
#pragma unroll
                    for (int i = 0; i < D; ++i) d = __builtin_fmaf(q[n][i], kk[i], d);
                    auto step = [&](int moved) { d += __int_as_float(moved); };
                    step(__builtin_amdgcn_mov_dpp(__float_as_int(d), 0xB1, 15, 15, true));
                    step(__builtin_amdgcn_mov_dpp(__float_as_int(d), 0x4E, 15, 15, true));
                    step(__builtin_amdgcn_mov_dpp(__float_as_int(d), 0x141, 15, 15, true));
                    if constexpr (LK == 16) step(__builtin_amdgcn_mov_dpp(__float_as_int(d), 0x140, 15, 15, true));
                    x[n][j] = d;
                }
            }
            if (some != ~0ull)
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[n][j] = bits >> (8 * (j / 4) + j % 4) & 1 ? x[n][j] : -INFINITY;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                float top = x[n][0];
#pragma unroll
                for (int j = 1; j < 8; ++j) top = fmaxf(top, x[n][j]);
                // A scale is positive: the largest score is that of the largest product.
                const float upto = fmaxf(r[n], ceilf(top * a.c));
                if (__any(upto > r[n])) {
                    const float f = r[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(r[n] - upto);
                    sum[n] *= f;
#pragma unroll
                    for (int i = 0; i < D; ++i) o[n][i] *= f;
                    r[n] = upto;
                }
                const float ref = r[n] == -INFINITY ? 0.f : r[n];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    x[n][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[n][j], a.c, -ref));
                    sum[n] += x[n][j];
                }
                if constexpr (DROP) {
                    int h, query;
                    place(n, h, query);
                    const u32x4 z = philox(8 * t + cell, query, e * a.heads + h, a.site, seed);
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[n][j] = kept16(z, j, a.line) ? x[n][j] : 0.f;
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float vv[D];
                numbers(v[j], vv);
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int i = 0; i < D; ++i) o[n][i] = __builtin_fmaf(x[n][j], vv[i], o[n][i]);
            }
        }
    }
    // The groups of the workgroup's waves: each leaves its sums, and a wave joins a row's.
    __shared__ float left_o[NQ][4 * GROUPS][64], left_r[NQ][4 * GROUPS], left_sum[NQ][4 * GROUPS];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int i = 0; i < D; ++i) left_o[n][wave * GROUPS + group][dim + i] = o[n][i];
        if (lane % LK == 0) left_r[n][wave * GROUPS + group] = r[n], left_sum[n][wave * GROUPS + group] = sum[n];
    }
    __syncthreads();
#pragma unroll 1
    for (int n = wave; n < min(NQ, share * a.q_rows); n += 4) {
        int h, query;
        place(n, h, query);
        if (query >= q_len) continue;
        float top = -INFINITY, total = 0.f, out = 0.f;
#pragma unroll
        for (int g = 0; g < 4 * GROUPS; ++g) top = fmaxf(top, left_r[n][g]);
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int g = 0; g < 4 * GROUPS; ++g) {
            const float f = __builtin_amdgcn_exp2f(left_r[n][g] - ref);
            total += left_sum[n][g] * f;
            out += left_o[n][g][lane] * f;
        }
        const long long row = (long long)(e * a.heads + h) * a.q_rows + query;
        if (a.q_splits > 1) {
            a.q_part[((long long)split * a.pairs * a.q_rows + row) * 64 + lane] = out;
            float *m = a.q_part + (long long)a.q_splits * a.pairs * a.q_rows * 64 + ((long long)split * a.pairs * a.q_rows + row) * 2;
            if (!lane) *reinterpret_cast<f32x2 *>(m) = f32x2{top, total};
            continue;
        }
        store1<EL>(a.out, at(a.os, e, h, query) + lane, total == 0.f ? 0.f : out * (a.w / total));
        if (!lane) {
            if (a.stats) *reinterpret_cast<f32x2 *>(a.stats + 2 * row) = f32x2{ref, total};
            if (a.lse) a.lse[row] = kLn2 * (ref + __builtin_amdgcn_logf(total));
        }
    }
}

// Joins the splits of a query: sixteen lanes to a row's numbers, and W groups of them to its splits (one group after another
// waits for memory each time: 64 splits of 8 rows took 27 us by one group and 5 by sixteen).
template <int EL, int W>
__global__ __launch_bounds__(256) void train_merge_kernel(const Args a) {
    const long long rows = (long long)a.pairs * a.q_rows;
    const int lane = threadIdx.x & 15, group = threadIdx.x / 16 % W;
    const long long row = (long long)blockIdx.x * (16 / W) + threadIdx.x / (16 * W);
    __shared__ float joined[W > 1 ? 16 : 1][16][4];
    bool some = row < rows;  // fewer than 2^27 of them
    const int pair = some ? (int)((unsigned)row / (unsigned)a.q_rows) : 0, e = pair / a.heads;
    const int query = some ? (int)((unsigned)row % (unsigned)a.q_rows) : 0;
    some = some && query < length_of(a.q_lengths, e, a.q_rows);
    const float *m = a.q_part + (long long)a.q_splits * rows * 64;
    float r = -INFINITY, ref = 0.f, sum = 0.f;
    f32x4 o = {};
    if (some) {
        // Every group takes every split's statistics: the same reference and sum in all.
        for (int s = lane; s < a.q_splits; s += 16) r = fmaxf(r, m[(s * rows + row) * 2]);
#pragma unroll
        for (int i = 8; i; i >>= 1) r = fmaxf(r, __shfl_xor(r, i, 16));
        ref = r == -INFINITY ? 0.f : r;
        for (int s = lane; s < a.q_splits; s += 16) {
            const f32x2 x = *reinterpret_cast<const f32x2 *>(m + (s * rows + row) * 2);
            sum += x[1] * __builtin_amdgcn_exp2f(x[0] - ref);
        }
#pragma unroll
        for (int i = 8; i; i >>= 1) sum += __shfl_xor(sum, i, 16);
#pragma unroll 4
        for (int s = group; s < a.q_splits; s += W) {
            const float f = __builtin_amdgcn_exp2f(m[(s * rows + row) * 2] - ref);
            o += *reinterpret_cast<const f32x4 *>(a.q_part + (s * rows + row) * 64 + 4 * lane) * f;
        }
    }
    if constexpr (W > 1) {
        *reinterpret_cast<f32x4 *>(joined[threadIdx.x / 16][lane]) = o;
        __syncthreads();
        if (group) return;
#pragma unroll
        for (int i = 1; i < W; ++i) o += *reinterpret_cast<const f32x4 *>(joined[threadIdx.x / 16 + i][lane]);
    }
    if (!some) return;
    const float f = sum == 0.f ? 0.f : a.w / sum;
    store4<EL>(a.out, at(a.os, e, pair % a.heads, query) + 4 * lane, o * f);
    if (!lane) {
        if (a.stats) *reinterpret_cast<f32x2 *>(a.stats + 2 * row) = f32x2{ref, sum};
        if (a.lse) a.lse[row] = kLn2 * (ref + __builtin_amdgcn_logf(sum));
    }
}

// ---- backward ----

// The two sides of the backward pass are workgroups of one launch, which fill its end for each other (two launches: 988 us
// in place of 858 for 10,007 BF16 rows). Both compute the scores and dP: seven products in place of five. Five would take
// either atomic additions to dq, whose order changes results, or dq's part of every 128 keys through memory, written and
// read (10,007 rows: 1.6 GB each way, 0.6 ms; the two products take 0.2).
// 10,007 BF16 rows: 771 to 814 us, 630 TFLOP/s counted as five products, 880 as seven; the matrix cores 44% busy, the vector
// unit 55%. 512 FP32 queries over 50,000 rows: 613 to 667 us, 205 (three FP16 products each: 860 as seven); 38% and 53%. Two
// masked tables of 12,345 rows, FP16 with dropout: 197 to 265; 15% and 50%. Four tables of 1,024 FP32 rows with dropout: 139
// to 148; 26% and 47%, with 104 bytes a lane spilled.

// What the backward pass needs of each query: {r, 1 / s, delta, log2 s}; r is +inf (all weights 0) for one that attends to
// nothing or lies past the length. Sixteen lanes to a row.
template <int EL>
__global__ __launch_bounds__(256) void train_record_kernel(const Args a) {
    const long long rows = (long long)a.pairs * a.q_rows;
    const long long row = (long long)blockIdx.x * 16 + threadIdx.x / 16;
    if (row >= rows) return;
    const int pair = (int)(row / a.q_rows), query = (int)(row % a.q_rows), lane = threadIdx.x & 15;
    const int e = pair / a.heads, h = pair % a.heads;
    f32x4 record = {INFINITY, 0.f, 0.f, 0.f};
    const f32x2 x = *reinterpret_cast<const f32x2 *>(a.stats + 2 * row);
    if (query < length_of(a.q_lengths, e, a.q_rows) && x[1] != 0.f) {
        const f32x4 o = load4<EL>(a.out, at(a.os, e, h, query) + 4 * lane);
        const f32x4 g = load4<EL>(a.dout, at(a.gs, e, h, query) + 4 * lane);
        float d = o[0] * g[0] + o[1] * g[1] + o[2] * g[2] + o[3] * g[3];
#pragma unroll
        for (int i = 8; i; i >>= 1) d += __shfl_xor(d, i, 16);
        record = f32x4{x[0], 1.f / x[1], d, __builtin_amdgcn_logf(x[1])};
    }
    if (!lane) a.record[row] = record;
}

template <int EL>
struct Streamed {
    static constexpr int N = scaled(EL) ? 1 : 2;
    Tile<EL> x[N], y[N];
    alignas(16) float r[N][kTile], delta[N][kTile];
    alignas(16) float logs[scaled(EL) ? 1 : N][kTile];  // 16-bit: log2 s
    alignas(16) u32x4 more[N][scaled(EL) ? 1 : kTile];  // 16-bit: what each row's scores and dP take besides
    float coming[scaled(EL) ? kTile : 1];               // the next tile's r
    int fields[2][scaled(EL) ? kTile : 1];  // and exponents
};

// The gradient of 32 queries a wave: S^T = K Q^T, V dout^T, then K^T dS, over a split's key tiles.
template <int EL, bool DROP>
__device__ __forceinline__ void queries_backward(const Args &a, Streamed<EL> &lds, unsigned block) {
    constexpr int P = parts_of(EL);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const unsigned unit = block / (unsigned)a.pairs;
    const int pair = block % (unsigned)a.pairs, tile = unit % (unsigned)a.q_tiles, split = unit / (unsigned)a.q_tiles;
    const int e = pair / a.heads, h = pair % a.heads, hk = h / (a.heads / a.kv_heads);
    const int q_len = length_of(a.q_lengths, e, a.q_rows), len = length_of(a.lengths, e, a.rows);
    if (tile * 128 >= q_len) return;
    const int query = tile * 128 + 32 * wave + (lane & 31);
    const bool mine = query < q_len;
    const long long row = (long long)pair * a.q_rows + query;
    f32x4 record = {INFINITY, 0.f, 0.f, 0.f};
    if (mine) record = a.record[row];
    const bool some_row = record[0] != INFINITY;
    V8<EL> qb[4][P], gb[4][P];
    const int q_down = down(own_row<EL>(a.q, at(a.qs, e, h, query), some_row, lane, qb));
    const int g_down = down(own_row<EL>(a.dout, at(a.gs, e, h, query), some_row, lane, gb));

    f32x16 o[2] = {};
    int power = kNone;
    const unsigned long long seed = DROP ? *a.seed : 0;
    const int end = min((split + 1) * a.q_chunk, (int)((len + 63) / 64));
    auto next = [&](int t, unsigned long long &m) {
        for (m = 0; t < end && !(m = attended(a.keep, a.words, e, t, len)); ++t) {}
        return t;
    };
    const Lanes lanes(lane);
    // A wave without a query has nothing to do but load (8 FP32 queries over 50,000 rows: 178 us where it worked on, 166).
    const bool idle = __builtin_amdgcn_readfirstlane(tile * 128 + 32 * wave) >= q_len;
    auto work = [&](const Tile<EL> &kt, const Tile<EL> &vt, int t, unsigned long long some, int k_down, int v_down) {
        if (idle) return;
        const float c = scaled(EL) ? times_power(a.c, k_down + q_down) : a.c;
#pragma unroll 1
        for (int b = 0; b < 2; ++b) {
            if (!(unsigned)(some >> 32 * b)) continue;
            f32x16 s = {}, dp = {};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                V8<EL> x[P];
                rows_operand<EL>(kt, 32 * b, c, lanes, x);
                mma<EL>(s, x, qb[c]);
                rows_operand<EL>(vt, 32 * b, c, lanes, x);
                mma<EL>(dp, x, gb[c]);
            }
            if constexpr (scaled(EL))
#pragma unroll
                for (int i = 0; i < 16; ++i) dp[i] = __builtin_ldexpf(dp[i], v_down + g_down);
            if (some != ~0ull) leave_out(s, some, 32 * b, half);
            float most = 0.f;
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) {
                u32x4 z;
                if constexpr (DROP) z = philox(2 * (4 * t + 2 * b + cc) + half, query, pair, a.site, seed);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int i = 8 * cc + j;
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -record[0]));
                    if constexpr (DROP || scaled(EL))
                        s[i] = p * __builtin_fmaf(!DROP || kept16(z, j, a.line) ? dp[i] : 0.f, a.w, -record[2]);
                    else
                        s[i] = p * (dp[i] - record[2]);
                    if constexpr (ranged(EL)) most = fmaxf(most, fabsf(s[i]));
                }
            }
            if constexpr (ranged(EL)) bring(s, fmaxf(most, other_half(most)), k_down, power, o);
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) {
                float ds[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) ds[j] = s[8 * cc + j];
                V8<EL> db[P];
                operand8<EL>(ds, db);
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    V8<EL> x[P];
                    dims_operand<EL>(kt, 32 * b + 16 * cc, d, lanes, x);
                    mma<EL>(o[d], x, db);
                }
            }
        }
    };
    unsigned long long todo, following = 0;
    int t = next(split * a.q_chunk, todo);
    if constexpr (scaled(EL)) {
        Staged<EL, 256> ks, vs;
        auto load = [&](int tile) {
            ks.load(a.k, a.ks, e, hk, tile * 64, len);
            vs.load(a.v, a.vs, e, hk, tile * 64, len);
        };
        if (t < end) load(t);
        bool fresh = true;
        while (t < end) {
            if (fresh) ks.fields(lds.fields[0]), vs.fields(lds.fields[1]);
            __syncthreads();
            const Turn turn = turn_of(todo, lds.fields[0], lds.fields[1], lane);
            ks.store(lds.x[0], turn.some, scale_of(turn.x));
            vs.store(lds.y[0], turn.some, scale_of(turn.y));
            __syncthreads();
            todo &= ~turn.some;
            const int at_tile = t;
            fresh = !todo;
            if (fresh) {
                t = next(t + 1, following);
                if (t < end) load(t);
                todo = following;
            }
            work(lds.x[0], lds.y[0], at_tile, turn.some, down(turn.x), down(turn.y));
        }
    } else {
        auto load = [&](int tile, int to) {
            load_tile<EL, 256>(lds.x[to], a.k, a.ks, e, hk, tile * 64, len);
            load_tile<EL, 256>(lds.y[to], a.v, a.vs, e, hk, tile * 64, len);
        };
        if (t < end) load(t, 0);
        for (int now = 0; t < end; now ^= 1) {
            wait_loads();
            __syncthreads();  // the tile has come, and the other is read
            if (todo != ~0ull) {
                clear_rows<EL, 256>(lds.x[now], todo), clear_rows<EL, 256>(lds.y[now], todo);
                __syncthreads();
            }
            const int n = next(t + 1, following);
            if (n < end) load(n, now ^ 1);
            work(lds.x[now], lds.y[now], t, todo, 0, 0);
            t = n, todo = following;
        }
    }
    if (!mine) return;
    const float f = a.scale * record[1];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const f32x16 &x = o[i / 4];
        const int j = 4 * (i % 4), dim = 32 * (i / 4) + 2 * j + 4 * half;
        f32x4 y = {x[j], x[j + 1], x[j + 2], x[j + 3]};
#pragma unroll
        for (int n = 0; n < 4; ++n) y[n] = ranged(EL) ? __builtin_ldexpf(y[n] * f, power) : y[n] * f;
        if (a.q_splits > 1)
            *reinterpret_cast<f32x4 *>(a.q_part + ((long long)split * a.pairs * a.q_rows + row) * 64 + dim) = y;
        else
            store4<EL>(a.dq, at(a.dqs, e, h, query) + dim, y);
    }
}

// Lane l (and l + 32) of the result: bit i of key l's word is whether query i of a wave's 32 keeps its weight of that key.
// Each lane draws its query's numbers as the other passes do; a comparison's bits over the wave are then a key's word.
__device__ __forceinline__ unsigned kept_words(unsigned cell, int query, int pair, unsigned site, unsigned line,
                                               unsigned long long seed, int half) {
    unsigned mine = 0;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const u32x4 z = philox(cell + 2 * c + half, query, pair, site, seed);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const unsigned long long word = __ballot(kept16(z, j, line));
            const int key = 16 * c + 8 * (j / 4) + j % 4;  // of the lower half's cell; the upper half's is 4 further
            mine = irx_writelane((unsigned)word, key, mine);
            mine = irx_writelane((unsigned)(word >> 32), key + 4, mine);
        }
    }
    const auto r = __builtin_amdgcn_permlane32_swap(mine, mine, false, false);
    return half ? r[0] : mine;
}

constexpr float kNear = 128.f;  // references up to here stand as one number with their sums' logarithms (keys_backward)

// The gradients of 32 keys a wave: S = Q K^T, dout V^T, then dout^T P and Q^T dS, over a split's query tiles of every head
// that shares the keys.
template <int EL, bool DROP>
__device__ __forceinline__ void keys_backward(const Args &a, Streamed<EL> &lds, unsigned block) {
    constexpr int P = parts_of(EL);
    typedef Staged<EL, 256> Rows;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int group = a.heads / a.kv_heads, owners = a.pairs / group;
    const unsigned unit = block / (unsigned)owners;
    const int owner = block % (unsigned)owners, tile = unit % (unsigned)a.k_tiles, split = unit / (unsigned)a.k_tiles;
    const int e = owner / a.kv_heads, hk = owner % a.kv_heads;
    const int q_len = length_of(a.q_lengths, e, a.q_rows), len = length_of(a.lengths, e, a.rows);
    if (tile * 128 >= len) return;
    const int key = tile * 128 + 32 * wave + (lane & 31);
    const unsigned long long here[2] = {attended(a.keep, a.words, e, 2 * tile, len), attended(a.keep, a.words, e, 2 * tile + 1, len)};
    const bool in = here[wave / 2] >> (32 * (wave & 1) + (lane & 31)) & 1;
    V8<EL> kb[4][P], vb[4][P];
    const int k_down = down(own_row<EL>(a.k, at(a.ks, e, hk, key), in, lane, kb));
    const int v_down = down(own_row<EL>(a.v, at(a.vs, e, hk, key), in, lane, vb));

    f32x16 dk[2] = {}, dv[2] = {};
    int dk_power = kNone, dv_power = kNone;
    const unsigned long long seed = DROP ? *a.seed : 0;
    // Query tiles that hold a query, of all heads of the group in turn.
    const int q_tiles = (q_len + kTile - 1) / kTile;
    const int end = here[0] | here[1] ? min((split + 1) * a.k_chunk, group * q_tiles) : 0;
    int u = split * a.k_chunk;
    const Lanes lanes(lane);
    // One turn: queries of the tile at row0 of head h. FP32's r and delta stand beside them. With 16-bit elements one more
    // product of BF16 parts adds -(r + log2 s) / c to the scores (24 bits of it) and, without dropout, -delta to dP: read from
    // LDS for every element, the three take as much of its time as the tiles' operands. Where a reference is past kNear,
    // 2^-24 of it, several times over, would show beside the weights' own rounding (2^-11 for FP16): such a tile's are read,
    // r taken from the score in one multiplication and addition and log2 s after it (for every tile so: the gradients of 10,007
    // BF16 rows 902 us in place of 806).
    bf16x8 ones[2] = {};
    if (!half)
#pragma unroll
        for (int n = 0; n < 3; ++n) ones[0][n] = ones[1][3 + n] = (__bf16)1.f;
    auto work = [&](const Tile<EL> &qt, const Tile<EL> &gt, const float *r, const float *logs, const u32x4 *more, const float *delta,
                    int h, int row0, unsigned long long some, bool near, int q_down, int g_down) {
        const float c = scaled(EL) ? times_power(a.c, q_down + k_down) : near ? a.c : 1.f;
#pragma unroll 1
        for (int b = 0; b < 2; ++b) {
            if (!(unsigned)(some >> 32 * b)) continue;  // 24 FP32 queries over 50,000 rows, dropout: 223 us without, 214
            f32x16 s = {}, dp = {};
            if constexpr (!scaled(EL)) {
                const bf16x8 x = __builtin_bit_cast(bf16x8, more[32 * b + (lane & 31)]);
                if (near) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, ones[0], s, 0, 0, 0);
                if constexpr (!DROP) dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, ones[1], dp, 0, 0, 0);
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                V8<EL> x[P];
                rows_operand<EL>(qt, 32 * b, n, lanes, x);
                mma<EL>(s, x, kb[n]);
                rows_operand<EL>(gt, 32 * b, n, lanes, x);
                mma<EL>(dp, x, vb[n]);
            }
            if (!scaled(EL) && !near)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const int q = 32 * b + 2 * i + 4 * half;
                    const f32x4 ref = *reinterpret_cast<const f32x4 *>(r + q), log = *reinterpret_cast<const f32x4 *>(logs + q);
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[i + j] = __builtin_fmaf(s[i + j], a.c, -ref[j]) - log[j];
                    __builtin_amdgcn_sched_barrier(0);  // all sixteen's at once cost registers: spills, and 839 us in place of 806
                }
            // The power by itself: as part of w it would have to stay a normal number, for which dout of 2^-100 is too small. (Only
            // where some lane needs it so: 512 FP32 queries over 50,000 rows 631 us in place of 636, but registers spill with
            // dropout, and four tables of 1,024 rows take 149 in place of 137.)
            if constexpr (scaled(EL))
#pragma unroll
                for (int i = 0; i < 16; ++i) dp[i] = __builtin_ldexpf(dp[i], g_down + v_down);
            unsigned kept = ~0u;
            if constexpr (DROP)
                kept = kept_words(16 * tile + 4 * wave, row0 + 32 * b + (lane & 31), e * a.heads + h, a.site, a.line, seed, half) >>
                       (4 * half);
            float most_p = 0.f, most_ds = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int q = 32 * b + 8 * (i / 4) + 4 * half + i % 4;
                const float p = __builtin_amdgcn_exp2f(scaled(EL) ? __builtin_fmaf(s[i], c, -r[q]) : s[i] * c);
                s[i] = p;
                if constexpr (DROP && scaled(EL)) {
                    const bool z = kept >> (8 * (i / 4) + i % 4) & 1;
                    dp[i] = z ? dp[i] : 0.f;
                    s[i] = z ? p : 0.f;
                } else if constexpr (DROP) {
                    // A bit as a mask of the whole number: an instruction less; FP32's kernel has no registers left for it (195 us
                    // in place of 163 for the gradients of four tables of 1,024 rows).
                    const int z = __builtin_amdgcn_sbfe((int)kept, 8 * (i / 4) + i % 4, 1);
                    dp[i] = __int_as_float(__float_as_int(dp[i]) & z);
                    s[i] = __int_as_float(__float_as_int(p) & z);
                }
                if constexpr (DROP || scaled(EL))
                    dp[i] = p * __builtin_fmaf(dp[i], a.w, -delta[q]);
                else
                    dp[i] *= p;
                if constexpr (ranged(EL)) most_p = fmaxf(most_p, s[i]), most_ds = fmaxf(most_ds, fabsf(dp[i]));
            }
            if constexpr (ranged(EL)) {
                bring(s, fmaxf(most_p, other_half(most_p)), g_down, dv_power, dv);
                bring(dp, fmaxf(most_ds, other_half(most_ds)), q_down, dk_power, dk);
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                float p[8], ds[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) p[j] = s[8 * n + j], ds[j] = dp[8 * n + j];
                V8<EL> x[P], pb[P];
                operand8<EL>(p, pb);
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    dims_operand<EL>(gt, 32 * b + 16 * n, d, lanes, x);
                    mma<EL>(dv[d], x, pb);
                }
                operand8<EL>(ds, pb);
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    dims_operand<EL>(qt, 32 * b + 16 * n, d, lanes, x);
                    mma<EL>(dk[d], x, pb);
                }
            }
        }
    };
    auto record = [&](int i, int row) {
        const int h = hk * group + i / q_tiles, query = i % q_tiles * kTile + row;
        f32x4 x = {INFINITY, 0.f, 0.f, 0.f};
        if (query < q_len) x = a.record[(long long)(e * a.heads + h) * a.q_rows + query];
        return x;
    };
    if constexpr (scaled(EL)) {
        Rows qs, gs;
        float r[Rows::N], inv[Rows::N], delta[Rows::N];
        auto load = [&](int i) {
            const int h = hk * group + i / q_tiles, row0 = i % q_tiles * kTile;
            qs.load(a.q, a.qs, e, h, row0, q_len);
            gs.load(a.dout, a.gs, e, h, row0, q_len);
#pragma unroll
            for (int n = 0; n < Rows::N; ++n) {
                const f32x4 x = record(i, threadIdx.x / 8 + 32 * n);
                r[n] = x[0], inv[n] = x[1], delta[n] = x[2];
            }
        };
        if (u < end) load(u);
        unsigned long long todo = 0;
        while (u < end) {
            const int h = hk * group + u / q_tiles, row0 = u % q_tiles * kTile;
            const bool fresh = !todo;
            if (fresh) {
                gs.times(inv);  // 1 / s goes with dout, whose parts are made here
                qs.fields(lds.fields[0]), gs.fields(lds.fields[1]);
                if (threadIdx.x % 8 == 0)
#pragma unroll
                    for (int n = 0; n < Rows::N; ++n) lds.coming[threadIdx.x / 8 + 32 * n] = r[n];
            }
            __syncthreads();
            if (fresh) todo = __ballot(lds.coming[lane] != INFINITY);
            const Turn turn = turn_of(todo, lds.fields[0], lds.fields[1], lane);
            qs.store(lds.x[0], turn.some, scale_of(turn.x));
            gs.store(lds.y[0], turn.some, scale_of(turn.y));
            if (threadIdx.x % 8 == 0)
#pragma unroll
                for (int n = 0; n < Rows::N; ++n) {
                    const int row = threadIdx.x / 8 + 32 * n;
                    lds.r[0][row] = turn.some >> row & 1 ? r[n] : INFINITY;
                    lds.delta[0][row] = delta[n] * inv[n];
                }
            __syncthreads();
            todo &= ~turn.some;
            if (!todo) {
                ++u;
                if (u < end) load(u);
            }
            work(lds.x[0], lds.y[0], lds.r[0], nullptr, nullptr, lds.delta[0], h, row0, turn.some, true, down(turn.x), down(turn.y));
        }
    } else {
        const float inverse = -1.f / a.c;
        f32x4 coming = {};
        auto load = [&](int i, int to) {
            const int h = hk * group + i / q_tiles, row0 = i % q_tiles * kTile;
            load_tile<EL, 256>(lds.x[to], a.q, a.qs, e, h, row0, q_len);
            load_tile<EL, 256>(lds.y[to], a.dout, a.gs, e, h, row0, q_len);
            if (threadIdx.x < kTile) coming = record(i, threadIdx.x);
        };
        if (u < end) load(u, 0);
        for (int now = 0; u < end; ++u, now ^= 1) {
            if (threadIdx.x < kTile) {
                lds.r[now][threadIdx.x] = coming[0];
                lds.delta[now][threadIdx.x] = coming[2];
                lds.logs[now][threadIdx.x] = coming[3];
                // A row without weights has a score that leaves none.
                const bool none = coming[0] == INFINITY;
                const u32x2 x = bf16_parts(none ? -0x1p120f : (coming[0] + coming[3]) * inverse), y = bf16_parts(-coming[2]);
                lds.more[now][threadIdx.x] = u32x4{x[0], x[1] | y[0] << 16, y[0] >> 16 | y[1] << 16, 0};
            }
            wait_loads();
            __syncthreads();  // the tile has come, and the other is read
            const float of_lane = lds.r[now][lane];
            const unsigned long long some = __ballot(of_lane != INFINITY);
            const bool near = !__any(of_lane != INFINITY && !(fabsf(of_lane) <= kNear));
            if (some != ~0ull) {
                clear_rows<EL, 256>(lds.x[now], some), clear_rows<EL, 256>(lds.y[now], some);
                __syncthreads();
            }
            if (u + 1 < end) load(u + 1, now ^ 1);
            work(lds.x[now], lds.y[now], lds.r[now], lds.logs[now], lds.more[now], lds.delta[now], hk * group + u / q_tiles,
                 u % q_tiles * kTile, some, near, 0, 0);
        }
    }
    if (key >= len) return;
    // A key that is not attended to has no gradient, whatever its lane summed.
    const long long row = (long long)owner * a.rows + key, plane = (long long)owners * a.rows * 64;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const f32x16 &x = dk[i / 4], &y = dv[i / 4];
        const int j = 4 * (i % 4), dim = 32 * (i / 4) + 2 * j + 4 * half;
        f32x4 gk = {x[j], x[j + 1], x[j + 2], x[j + 3]}, gv = {y[j], y[j + 1], y[j + 2], y[j + 3]};
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            gk[n] = ranged(EL) ? __builtin_ldexpf(gk[n] * a.scale, dk_power) : gk[n] * a.scale;
            gv[n] = ranged(EL) ? __builtin_ldexpf(gv[n] * a.w, dv_power) : gv[n] * a.w;
        }
        if (!in) gk = gv = f32x4{0.f, 0.f, 0.f, 0.f};
        if (a.k_splits > 1) {
            float *part = a.k_part + 2 * split * plane + row * 64 + dim;
            *reinterpret_cast<f32x4 *>(part) = gk;
            *reinterpret_cast<f32x4 *>(part + plane) = gv;
        } else {
            store4<EL>(a.dk, at(a.dks, e, hk, key) + dim, gk);
            store4<EL>(a.dv, at(a.dvs, e, hk, key) + dim, gv);
        }
    }
}

template <int EL, bool DROP>
__global__ __launch_bounds__(256, EL == kTrainF32 || DROP ? 2 : 3) void train_backward_kernel(const Args a) {
    __shared__ Streamed<EL> lds;
    // The side that walks further goes ahead of the other where both have instructions to issue.
    if ((blockIdx.x < (unsigned)a.q_blocks) != a.keys_last) __builtin_amdgcn_s_setprio(1);
    if (blockIdx.x < (unsigned)a.q_blocks)
        queries_backward<EL, DROP>(a, lds, blockIdx.x);
    else
        keys_backward<EL, DROP>(a, lds, blockIdx.x - a.q_blocks);
}

// Sums the splits' parts, in order, so that results hang on nothing else. Rows of dq, then of dk, then of dv; sixteen lanes to a row.
template <int EL>
__global__ __launch_bounds__(256) void train_sum_kernel(const Args a) {
    const long long q_rows = a.q_splits > 1 ? (long long)a.pairs * a.q_rows : 0;
    const long long k_rows = a.k_splits > 1 ? (long long)(a.pairs / (a.heads / a.kv_heads)) * a.rows : 0;
    long long row = (long long)blockIdx.x * 16 + threadIdx.x / 16;
    const int lane = threadIdx.x & 15;
    const float *part;
    long long step;
    int splits;
    void *to;
    long long offset;
    if (row < q_rows) {
        const int pair = (int)(row / a.q_rows), query = (int)(row % a.q_rows), e = pair / a.heads;
        if (query >= length_of(a.q_lengths, e, a.q_rows)) return;
        part = a.q_part + row * 64, step = q_rows * 64, splits = a.q_splits;
        to = a.dq, offset = at(a.dqs, e, pair % a.heads, query);
    } else {
        row -= q_rows;
        if (row >= 2 * k_rows) return;
        const bool values = row >= k_rows;
        if (values) row -= k_rows;
        const int owner = (int)(row / a.rows), key = (int)(row % a.rows), e = owner / a.kv_heads, hk = owner % a.kv_heads;
        if (key >= length_of(a.lengths, e, a.rows)) return;
        part = a.k_part + (values ? k_rows * 64 : 0) + row * 64, step = 2 * k_rows * 64, splits = a.k_splits;
        to = values ? a.dv : a.dk, offset = values ? at(a.dvs, e, hk, key) : at(a.dks, e, hk, key);
    }
    f32x4 sum = {};
    for (int s = 0; s < splits; ++s) sum += *reinterpret_cast<const f32x4 *>(part + s * step + 4 * lane);
    store4<EL>(to, offset + 4 * lane, sum);
}

// ---- dropout ----

struct DropArgs {
    const void *x, *residual;
    void *out;
    long long xs, rs, os;
    long long groups;  // of eight columns, in all
    int per_row, width;
    const unsigned long long *seed;
    unsigned site, line;
    float w;
};

// Eight adjacent numbers of a row, one call of random numbers, to a thread; bound by memory: 200,000 x 1,024 FP32 numbers 278
// us, 5.9 TB/s.
template <int EL>
__global__ __launch_bounds__(256) void train_dropout_kernel(const DropArgs a) {
    const long long g = (long long)blockIdx.x * 256 + threadIdx.x;
    if (g >= a.groups) return;
    const unsigned row = (unsigned)g / (unsigned)a.per_row, col = (unsigned)g % (unsigned)a.per_row;
    const int left = min(8, a.width - 8 * (int)col);
    const long long xi = row * a.xs + 8ll * col, ri = row * a.rs + 8ll * col, oi = row * a.os + 8ll * col;
    float x[8], y[8] = {};
    typedef std::conditional_t<EL == kTrainF32, float, std::conditional_t<EL == kTrainF16, _Float16, __bf16>> T;
    if (left == 8) {
        to_floats<EL>(load8<EL>(a.x, xi), x);
        if (a.residual) to_floats<EL>(load8<EL>(a.residual, ri), y);
    } else {
        for (int j = 0; j < 8; ++j) {
            x[j] = j < left ? (float)static_cast<const T *>(a.x)[xi + j] : 0.f;
            if (a.residual && j < left) y[j] = (float)static_cast<const T *>(a.residual)[ri + j];
        }
    }
    if (a.line) {
        const u32x4 z = philox(col, row, ~0u, a.site, *a.seed);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = kept16(z, j, a.line) ? x[j] : 0.f;
    }
    // One rounding to FP32; without a residual zeros keep their signs.
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = a.residual ? __builtin_fmaf(x[j], a.w, y[j]) : x[j] * a.w;
    if (left == 8) {
        store4<EL>(a.out, oi, f32x4{x[0], x[1], x[2], x[3]});
        store4<EL>(a.out, oi + 4, f32x4{x[4], x[5], x[6], x[7]});
    } else {
        for (int j = 0; j < left; ++j) static_cast<T *>(a.out)[oi + j] = (T)x[j];
    }
}

// ---- plans ----

struct Plan {
    int q_tiles, q_splits, q_chunk, k_tiles, k_splits, k_chunk;
    int q_unit;  // queries of a workgroup
    size_t record, q_part, k_part;  // bytes
    double blocks;
};

int splits_of(double length, double target, long long tiles) {
    return (int)std::min<long long>(std::max(1ll, std::llround(length / target)), std::min(tiles, 128ll));
}

// Splits of `units` 128-query units over `words` key tiles: as many as take the least time, of those with which the launch is
// 1, 2, .. 16 workgroups to a compute unit. A workgroup's tile takes so many us beside 0, 1, .. others on its compute unit,
// and so does the last, partly filled round (10,007 FP32 queries over as many rows in 1 / 2 / 3 / 4 / 5 splits: 883, 748, 774,
// 746, 781 us; 1,024 over 1,024: 49, 33, 29, 26, 26, in 16 splits 41; four tables of 1,024 BF16 rows: 24, 31, 32, 33, 33). Joining
// writes and reads every split's sums. Where only the device knows how much there is to do, the sum of two times: as if every
// workgroup had everything, and as if half of them had nothing (512 FP32 queries over four masked tables of 20,000 rows: 260 us
// by the first alone, 234 so; of twelve masked shapes 3% and 6% from the best on average).
int splits_of_rounds(double units, int words, double rows, bool single, bool uneven, int compute_units) {
    static constexpr double kTileUs[2][4] = {{1.0, 1.6, 2.1, 2.7}, {2.45, 3.83, 0.0, 0.0}};
    const int most = single ? 2 : 4;
    const double *us = kTileUs[single];
    double best = INFINITY;
    int splits = 1;
    for (int m = 0, last = 0; m <= 16; ++m) {
        const int s = std::min((int)std::max(m * compute_units / units, 1.0), std::min(words, 128));
        if (s == last) continue;
        last = s;
        const double tiles = (words + s - 1) / s;
        double time = 0.0;
        for (const double full : {1.0, 0.5}) {
            const double blocks = full * units * s / compute_units, rounds = std::floor(blocks / most);
            const int left = (int)std::ceil(blocks - most * rounds);
            time += tiles * (rounds * us[most - 1] + (left ? us[left - 1] : 0.0));
            if (s > 1) time += 2.5 + full * rows * s * 528 / 6e6;
            if (!uneven) break;
        }
        if (time < best) best = time, splits = s;
    }
    return splits;
}

// What a compute unit takes for `first` workgroups that each take a and then `second` of b (the last of either may be a part
// of one), `most` of them at once, where us[0], us[1], .. pass for a unit of that with none, one, .. beside it.
double us_of_workgroups(double first, double a, double second, double b, int most, const double *us) {
    double left[3], time = 0.0;
    for (int n = 0;;) {
        for (; n < most && (first > 0.0 || second > 0.0); ++n) {
            double &of = first > 0.0 ? first : second;
            left[n] = (&of == &first ? a : b) * std::min(of, 1.0);
            of -= 1.0;
        }
        if (!n) return time;
        const double least = *std::min_element(left, left + n);
        time += least * us[n - 1];
        int kept = 0;
        for (int i = 0; i < n; ++i)
            if (left[i] - least > 1e-9) left[kept++] = left[i] - least;
        n = kept;
    }
}

// What a tile of keys costs 128 queries and a tile of queries 128 keys, and a workgroup's start.
constexpr double kQueriesCost = 3.0, kKeysCost = 5.5, kStartCost = 1.2;

// The backward pass' splits: as many as take the least time, of those with which the launch has 1, 2, 3 or 4 workgroups of as
// many products to a compute unit; more only where that saves a fortieth. The costs are fitted to 64 shapes with ten choices
// each, of which these are 1% from the best on average and 9% at most (in us, with as many as let no workgroup walk further than
// half a compute unit's share, and these: 3,000 FP32 queries over as many rows 272 and 244, 5,000 FP16 with dropout 421 and 337,
// four tables of 300 FP16 rows 29 and 23). Where only the device knows how much there is to do, as if half the workgroups had
// nothing, the others everything (for ten masked shapes 5% from the best on average and 16% at most; with a third of a share as
// the longest walk 14% and 37%: four tables of 1,024 FP32 rows with dropout 154 us, so 143, of BF16 rows without 61 and 47).
void backward_splits(Plan &p, double pairs, double owners, int words, int q_words, const TrainShape &s, int element, bool uneven,
                     bool drop, int compute_units) {
    static constexpr double kUs[2][2][3] = {{{0.39, 0.52, 0.87}, {0.74, 1.0, 0.0}}, {{1.05, 1.43, 0.0}, {1.85, 2.5, 0.0}}};
    const bool single = element == kTrainF32;
    const int most = single || drop ? 2 : 3;
    const double *us = kUs[single][drop], q_units = pairs * p.q_tiles, k_units = owners * p.k_tiles;
    const double all = 3.0 * q_units * words + 4.0 * k_units * q_words;  // products
    double best = INFINITY;
    const double full = uneven ? 0.5 : 1.0;
    const int last = uneven ? 8 : 4;
    // Where there are many workgroups anyway, no one walks further than half a compute unit's share.
    const bool many = q_units + k_units > 20.0 * compute_units;
    for (int m = many ? last / 2 : 0; m <= last; ++m) {
        const double share = m ? all / (m * compute_units) : INFINITY;
        const int q_chunk = (int)ceil_div(words, splits_of(3.0 * words, share, words));
        const int k_chunk = (int)ceil_div(q_words, splits_of(4.0 * q_words, share, q_words));
        const int q_splits = (int)ceil_div(words, q_chunk), k_splits = (int)ceil_div(q_words, k_chunk);
        const double q_blocks = full * q_units * q_splits / compute_units, k_blocks = full * k_units * k_splits / compute_units;
        const double blocks = q_blocks + k_blocks;
        if (many) {
            p.q_splits = q_splits, p.k_splits = k_splits;
            break;
        }
        const double q_cost = kQueriesCost * q_chunk + kStartCost, k_cost = kKeysCost * k_chunk + kStartCost;
        // The compute unit with the most to do has as many as it can of those that take longer; the others level out where they
        // are many.
        const double longer = std::ceil(k_cost >= q_cost ? k_blocks : q_blocks), rest = std::max(blocks - longer, 0.0);
        const double others = rest > 2.0 ? rest : std::ceil(rest);
        const double q_jobs = k_cost >= q_cost ? others : longer, k_jobs = k_cost >= q_cost ? longer : others;
        double sums = q_splits > 1 ? pairs * s.q_rows * q_splits * 512.0 : 0.0;
        if (k_splits > 1) sums += owners * s.rows * k_splits * 1024.0;
        double time = us_of_workgroups(q_jobs, q_cost, k_jobs, k_cost, most, us);
        if (sums > 0.0) time += 3.0 + full * sums / 4.3e6;
        if (time < 0.978 * best) best = time, p.q_splits = q_splits, p.k_splits = k_splits;
    }
}

// `uneven`: estimators' lengths or masks are given, which only the device knows. `drop`: weights are dropped.
Plan plan(const TrainShape &s, int element, bool backward, bool uneven, bool drop, int compute_units) {
    Plan p{};
    const long long pairs = (long long)s.estimators * s.heads, owners = (long long)s.estimators * s.kv_heads;
    const long long words = (s.rows + 63) / 64, q_words = (s.q_rows + 63) / 64, group = s.heads / s.kv_heads;
    p.q_unit = backward || s.q_rows > 64 ? 128 : s.q_rows > 32 ? 64 : 32;
    // Workgroups that a launch should have at once: what registers leave room for on the compute units (with two of 128 threads
    // on each, 32 FP32 queries over 50,000 rows took 59 us in place of 47).
    const double slots = (element == kTrainF32 && p.q_unit > 32 ? 2.0 : 4.0) * compute_units;
    // Few rows go one key at a time where that is faster. In us, so and by the matrix cores, over 50,000 rows: 8 FP32 heads
    // of 1 / 2 / 4 / 8 queries 37.9 / 40.1 / 42.8 / 53.1 and 44.6 / 45.4 / 45.2 / 45.8; 8 over 2 key heads, of 1 / 2 queries
    // 21.0 / 27.6 and 45; 8 BF16 heads of 1 / 2 / 4 queries 24.4 / 27.0 / 30.1 and 26.1 / 26.3 / 26.8, over 2 key heads, of 1
    // query 16.7 and 26.3. Over 1,000: 8 FP32 heads of 1 / 2 / 4 / 8 queries 7.7 / 8.9 / 10.8 / 14.8 and 10.0 to 10.3, over 2
    // key heads, of 2 queries 14.2 and 10.1; BF16, of 1 query 9.9 and 7.9.
    const long long few = group * s.q_rows;
    const bool shared = group > 1 && s.rows >= 8192, single = element == kTrainF32;
    if (!backward && (few == 1 || (few <= 4 && (single || shared)) || (few <= 8 && single && shared))) p.q_unit = (int)few;
    p.q_tiles = (int)ceil_div(s.q_rows, p.q_unit);
    p.k_tiles = (int)ceil_div(s.rows, 128);
    if (backward) {
        backward_splits(p, (double)pairs, (double)owners, (int)words, (int)(group * q_words), s, element, uneven, drop,
                        compute_units);
    } else if (p.q_unit <= 8) {
        // A wave takes a tile at a time.
        p.q_splits = splits_of((double)words, std::max((double)owners * words / compute_units, 4.0), words);
        p.k_splits = 1;
    } else {
        p.q_splits = p.q_unit == 128
                         ? splits_of_rounds((double)pairs * p.q_tiles, (int)words, (double)pairs * s.q_rows, single, uneven, compute_units)
                         : splits_of((double)words, std::max(pairs * p.q_tiles * words / slots, 1.0), words);
        p.k_splits = 1;
    }
    p.q_chunk = (int)ceil_div(words, p.q_splits);
    p.q_splits = (int)ceil_div(words, p.q_chunk);
    p.k_chunk = (int)ceil_div(group * q_words, p.k_splits);
    p.k_splits = (int)ceil_div(group * q_words, p.k_chunk);
    const size_t rows = (size_t)pairs * s.q_rows;
    p.record = backward ? rows * 16 : 0;
    p.q_part = p.q_splits > 1 ? (size_t)p.q_splits * rows * (backward ? 256 : 264) : 0;
    p.k_part = p.k_splits > 1 ? (size_t)p.k_splits * owners * s.rows * 512 : 0;
    p.blocks = (double)(p.q_unit <= 8 ? owners : pairs * p.q_tiles) * p.q_splits;
    if (backward) p.blocks += (double)owners * p.k_tiles * p.k_splits;
    return p;
}

size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }

Args common(const TrainInputs &a, const Plan &p) {
    Args k{};
    const TrainShape &s = a.shape;
    k.q = a.q, k.k = a.k, k.v = a.v;
    std::copy_n(a.qs, 3, k.qs), std::copy_n(a.ks, 3, k.ks), std::copy_n(a.vs, 3, k.vs);
    k.q_lengths = a.q_lengths, k.lengths = a.lengths, k.keep = a.keep;
    k.heads = s.heads, k.kv_heads = s.kv_heads, k.pairs = s.estimators * s.heads, k.q_rows = s.q_rows, k.rows = s.rows;
    k.words = (int)ceil_div(s.rows, 64);
    k.scale = a.scale, k.c = a.scale * kLog2e;
    k.seed = a.drop.seed, k.site = a.drop.site, k.line = a.drop.dropped << 16;
    k.w = 65536.f / (float)(65536u - a.drop.dropped);
    k.q_tiles = p.q_tiles, k.q_splits = p.q_splits, k.q_chunk = p.q_chunk;
    k.k_tiles = p.k_tiles, k.k_splits = p.k_splits, k.k_chunk = p.k_chunk;
    return k;
}

template <int EL>
void forward(const TrainInputs &a, const TrainForward &f, const Plan &p, hipStream_t stream) {
    Args k = common(a, p);
    k.out = f.out, k.stats = f.stats, k.lse = f.lse, k.q_part = static_cast<float *>(f.workspace);
    std::copy_n(f.os, 3, k.os);
    const dim3 grid((unsigned)p.blocks);
    {
        KernelTimer timer(kFamIcl, stream, 256.0 * k.pairs * k.q_rows * k.rows, 0.0);
        auto launch = [&]<bool DROP>() {
            if (p.q_unit == 1)
                hipLaunchKernelGGL((train_rows_kernel<EL, 1, DROP>), grid, dim3(256), 0, stream, k);
            else if (p.q_unit == 2)
                hipLaunchKernelGGL((train_rows_kernel<EL, 2, DROP>), grid, dim3(256), 0, stream, k);
            else if (p.q_unit <= 4)
                hipLaunchKernelGGL((train_rows_kernel<EL, 4, DROP>), grid, dim3(256), 0, stream, k);
            else if (EL == kTrainF32 && p.q_unit <= 8)
                hipLaunchKernelGGL((train_rows_kernel<kTrainF32, 8, DROP>), grid, dim3(256), 0, stream, k);
            else if (p.q_unit == 32)
                hipLaunchKernelGGL((train_forward_kernel<EL, 1, 2, DROP>), grid, dim3(128), 0, stream, k);
            else if (p.q_unit == 64)
                hipLaunchKernelGGL((train_forward_kernel<EL, 2, 2, DROP>), grid, dim3(256), 0, stream, k);
            else
                hipLaunchKernelGGL((train_forward_kernel<EL, 4, 1, DROP>), grid, dim3(256), 0, stream, k);
        };
        if (k.line)
            launch.template operator()<true>();
        else
            launch.template operator()<false>();
        IRX_HIP(hipGetLastError());
    }
    if (p.q_splits > 1) {
        KernelTimer timer(kFamIclMerge, stream, 0.0, (double)p.q_part);
        // A group of sixteen lanes to two splits or so: one after another they wait for memory each time.
        const size_t rows = (size_t)k.pairs * k.q_rows;
        if (p.q_splits > 8)
            hipLaunchKernelGGL((train_merge_kernel<EL, 16>), dim3((unsigned)rows), dim3(256), 0, stream, k);
        else if (p.q_splits > 4)
            hipLaunchKernelGGL((train_merge_kernel<EL, 4>), dim3(ceil_div(rows, 4)), dim3(256), 0, stream, k);
        else
            hipLaunchKernelGGL((train_merge_kernel<EL, 1>), dim3(ceil_div(rows, 16)), dim3(256), 0, stream, k);
        IRX_HIP(hipGetLastError());
    }
}

template <int EL>
void backward(const TrainInputs &a, const TrainBackward &b, const Plan &p, hipStream_t stream) {
    Args k = common(a, p);
    k.out = const_cast<void *>(b.out), k.stats = const_cast<float *>(b.stats), k.dout = b.dout;
    k.dq = b.dq, k.dk = b.dk, k.dv = b.dv;
    std::copy_n(b.os, 3, k.os), std::copy_n(b.gs, 3, k.gs);
    std::copy_n(b.dqs, 3, k.dqs), std::copy_n(b.dks, 3, k.dks), std::copy_n(b.dvs, 3, k.dvs);
    char *space = static_cast<char *>(b.workspace);
    k.record = reinterpret_cast<f32x4 *>(space);
    k.q_part = reinterpret_cast<float *>(space + round16(p.record));
    k.k_part = reinterpret_cast<float *>(space + round16(p.record) + round16(p.q_part));
    const size_t rows = (size_t)k.pairs * k.q_rows, owned = (size_t)a.shape.estimators * a.shape.kv_heads * k.rows;
    {
        KernelTimer timer(kFamGlue, stream, 0.0, rows * (EL == kTrainF32 ? 512.0 : 256.0));
        hipLaunchKernelGGL(train_record_kernel<EL>, dim3(ceil_div(rows, 16)), dim3(256), 0, stream, k);
        IRX_HIP(hipGetLastError());
    }
    k.keys_last = kKeysCost * p.k_chunk > kQueriesCost * p.q_chunk;
    k.q_blocks = b.dq ? (int)((size_t)k.pairs * p.q_tiles * p.q_splits) : 0;
    const size_t k_blocks = b.dk ? (size_t)a.shape.estimators * a.shape.kv_heads * p.k_tiles * p.k_splits : 0;
    {
        KernelTimer timer(kFamIcl, stream, 640.0 * rows * k.rows, 0.0);
        const dim3 grid((unsigned)(k.q_blocks + k_blocks));
        if (k.line)
            hipLaunchKernelGGL((train_backward_kernel<EL, true>), grid, dim3(256), 0, stream, k);
        else
            hipLaunchKernelGGL((train_backward_kernel<EL, false>), grid, dim3(256), 0, stream, k);
        IRX_HIP(hipGetLastError());
    }
    if (!b.dq) k.q_splits = 1;
    if (!b.dk) k.k_splits = 1;
    const size_t sums = (k.q_splits > 1 ? rows : 0) + (k.k_splits > 1 ? 2 * owned : 0);
    if (sums) {
        KernelTimer timer(kFamIclMerge, stream, 0.0, (double)(p.q_part + p.k_part));
        hipLaunchKernelGGL(train_sum_kernel<EL>, dim3(ceil_div(sums, 16)), dim3(256), 0, stream, k);
        IRX_HIP(hipGetLastError());
    }
}

}  // namespace

bool train_needs(const TrainShape &s, int element, bool backward, int compute_units, size_t *workspace) {
    // 256 work-items to a workgroup, less than 2^32 in a launch.
    *workspace = 0;
    if ((double)s.estimators * std::max((double)s.heads * s.q_rows, 2.0 * s.kv_heads * s.rows) >= 134217728.0) return false;
    // The workspace serves every plan of the shape: with lengths or masks and without, with dropout and without.
    for (int i = 0; i < (backward ? 4 : 2); ++i) {
        const Plan p = plan(s, element, backward, i & 1, i & 2, compute_units);
        if (p.blocks >= 16777216.0) return false;
        *workspace = std::max(*workspace, round16(p.record) + round16(p.q_part) + round16(p.k_part));
    }
    return true;
}

void train_attention(const TrainInputs &a, const TrainForward &f, int compute_units, hipStream_t stream) {
    const Plan p = plan(a.shape, a.element, false, a.q_lengths || a.lengths || a.keep, false, compute_units);
    if (a.element == kTrainF32)
        forward<kTrainF32>(a, f, p, stream);
    else if (a.element == kTrainF16)
        forward<kTrainF16>(a, f, p, stream);
    else
        forward<kTrainBF16>(a, f, p, stream);
}

void train_backward(const TrainInputs &a, const TrainBackward &b, int compute_units, hipStream_t stream) {
    const Plan p = plan(a.shape, a.element, true, a.q_lengths || a.lengths || a.keep, a.drop.dropped, compute_units);
    if (a.element == kTrainF32)
        backward<kTrainF32>(a, b, p, stream);
    else if (a.element == kTrainF16)
        backward<kTrainF16>(a, b, p, stream);
    else
        backward<kTrainBF16>(a, b, p, stream);
}

void train_dropout(const TrainRows &a, hipStream_t stream) {
    DropArgs k{};
    k.x = a.x, k.residual = a.residual, k.out = a.out, k.xs = a.xs, k.rs = a.rs, k.os = a.os;
    k.width = (int)a.width, k.per_row = (int)ceil_div(a.width, 8), k.groups = (long long)a.rows * k.per_row;
    k.seed = a.drop.seed, k.site = a.drop.site, k.line = a.drop.dropped << 16;
    k.w = 65536.f / (float)(65536u - a.drop.dropped);
    const dim3 grid(ceil_div((size_t)k.groups, 256));
    KernelTimer timer(kFamGlue, stream, 0.0, (double)a.rows * a.width * (a.element == kTrainF32 ? 4 : 2) * (a.residual ? 3 : 2));
    if (a.element == kTrainF32)
        hipLaunchKernelGGL(train_dropout_kernel<kTrainF32>, grid, dim3(256), 0, stream, k);
    else if (a.element == kTrainF16)
        hipLaunchKernelGGL(train_dropout_kernel<kTrainF16>, grid, dim3(256), 0, stream, k);
    else
        hipLaunchKernelGGL(train_dropout_kernel<kTrainBF16>, grid, dim3(256), 0, stream, k);
    IRX_HIP(hipGetLastError());
}

}  // namespace irx
