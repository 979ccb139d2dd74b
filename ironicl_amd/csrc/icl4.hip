// The 4-bit ICL cache: its writer and reader, the attention over it, and the
// choice of blocks for attention over a part of it.
//
// A cache holds keys and values of 64-wide heads, [pairs, rows, 64] with pair
// = estimator * heads + head, as E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and
// their negatives) times powers of two 2^e: one e per key and 32 dims, one per
// value dim and 32 rows, the smallest with max |x| <= 6 * 2^e, held to -13..13.
// Every held number is then exact in FP16 (2^-14 at least, 49,152 at most, or
// zero), so the FP16 matrix cores take it without another rounding. Rows go in
// blocks of 64, each 4,352 contiguous bytes in the order in which the
// 16x16x32 products read them:
//   0     keys' codes [s 2][g 4][a 2][i 8][b 2][8 bytes]: row 32 s + 16 a +
//         8 b + i, dims 16 g .. +15, the lower dim in the lower nibble
//   2048  values' codes [s 2][t 2][h 2][i 16][d 4][b 2][2 bytes]: dim 16 d + i,
//         rows 32 s + 16 t + 8 b + 4 h .. +3, the lower row in the lower nibble
//   4096  keys' e + 127, bytes [32 dims 2][a 2][i 8][s 2][b 2]
//   4224  values' e + 127, bytes [i 16][s 2][d 4]
// Lane 16 g + (8 a + i) of a wave finds its operands of rows 32 s .. +31 in 16
// contiguous bytes of keys and 16 of values (g = 2 t + h).
// After the blocks of every pair come their bounds, int8 [pairs, blocks, low
// and high, 64], and the bounds' scales, FP32 [pairs, 64] (powers of two).
#include "common.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace irx {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int kBlock = kIcl4Block;            // rows of a block
constexpr int kBlockBytes = kIcl4BlockBytes;  // bytes of one pair's block
constexpr int kValuesAt = 2048, kKeyExpsAt = 4096, kValueExpsAt = 4224;

// The exponent byte I of a word as the scale of a conversion, which reads
// nothing but the scale's exponent bits: the bits beside them are left in.
template <int I>
__device__ __forceinline__ float scale_byte(unsigned word) {
    return __uint_as_float(I == 0 ? word << 23 : I == 1 ? word << 15 : I == 2 ? word << 7 : word >> 1);
}

// Eight E2M1 codes times `scale` (a power of two) as FP16, exactly.
__device__ __forceinline__ half8 codes8(unsigned word, float scale) {
    const half2v a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, 0);
    const half2v b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, 1);
    const half2v c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, 2);
    const half2v d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, 3);
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Rows that estimator e's queries may attend to.
__device__ __forceinline__ int rows_of(const unsigned *lengths, int e, int rows) {
    return lengths ? (int)min(lengths[e], (unsigned)rows) : rows;
}

// Bit r: row 64 block + r is attended.
__device__ __forceinline__ unsigned long long block_mask(const unsigned long long *keep, int e, int blocks, int block,
                                                         int rows) {
    const int left = rows - block * kBlock;
    if (left <= 0) return 0;
    unsigned long long m = keep ? keep[(long long)e * blocks + block] : ~0ull;
    if (left < kBlock) m &= (1ull << left) - 1;
    return m;
}

// Whole division of 0 <= n < 2^31 by a constant of the launch: with 2^(l - 1) < d
// <= 2^l and m = floor(2^(31 + l) / d) + 1, n m / 2^(31 + l) is past n / d by less
// than 1 / d. (A division by a variable is some 25 scalar instructions, before
// a workgroup's first load.)
struct Division {
    unsigned d, m, shift;
};
Division division(long long d) {
    unsigned l = 0;
    while ((1ll << l) < d) ++l;
    return {(unsigned)d, (unsigned)((1ull << (31 + l)) / (unsigned long long)d + 1), 31 + l};
}
__device__ __forceinline__ unsigned divide(unsigned n, const Division &by) {
    return (unsigned)(((unsigned long long)n * by.m) >> by.shift);
}

// ---- writing ----

// The smallest e with m <= 6 * 2^e, held to -13..13 (m finite).
__device__ __forceinline__ int code_exponent(float m) {
    if (m == 0.f) return -13;
    const unsigned bits = __float_as_uint(m);
    // m = f * 2^x with f in [0.5, 1); subnormal m ends at -13 whatever x is.
    const int x = (int)(bits >> 23) - 126;
    return min(13, max(-13, (bits & 0x7fffffu) <= 0x400000u ? x - 3 : x - 2));
}

// Eight numbers as E2M1 codes of x / 2^e: to nearest, ties to the even code, saturated.
__device__ __forceinline__ unsigned coded8(const float *x, float scale) {
    unsigned w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
}

// The smallest x >= -20 with m <= 127 * 2^x (m a held key's size).
__device__ __forceinline__ int unit_exponent(float m) {
    if (m == 0.f) return -20;
    const unsigned bits = __float_as_uint(m);
    const int x = (int)(bits >> 23) - 126;  // m = f 2^x, f in [0.5, 1); f <= 127/128?
    return (bits & 0x7fffffu) <= 0x7e0000u ? x - 7 : x - 6;
}

struct StoreArgs {
    const void *k, *v;
    long long k_est, k_head, k_row, v_est, v_head, v_row;
    const unsigned *lengths;
    int heads, pairs, rows, blocks;
    unsigned char *tiles;
    signed char *bounds;
    float *scales;
    unsigned *nonfinite;
};

// The value of the lane eight, or sixteen, away (lane ^ 8 and lane ^ 16).
__device__ __forceinline__ unsigned other_eight(unsigned x) {
    return __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, true);
}
__device__ __forceinline__ float rows_max(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// Lane ^ N of a row of 16, N a power of two below 16.
template <int N>
__device__ __forceinline__ unsigned row_xor(unsigned x) {
    if constexpr (N == 1) return __builtin_amdgcn_update_dpp(0, x, 0xb1, 0xf, 0xf, true);  // 1, 0, 3, 2
    if constexpr (N == 2) return __builtin_amdgcn_update_dpp(0, x, 0x4e, 0xf, 0xf, true);  // 2, 3, 0, 1
    if constexpr (N == 4) {  // the halves of each eight swapped: mirrored, then each four mirrored
        const unsigned m = __builtin_amdgcn_update_dpp(0, x, 0x141, 0xf, 0xf, true);
        return __builtin_amdgcn_update_dpp(0, m, 0x1b, 0xf, 0xf, true);
    }
    if constexpr (N == 8) return other_eight(x);
}
typedef short short2v __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned pk_max(unsigned a, unsigned b) {  // of positive FP16 pairs
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(short2v, a), __builtin_bit_cast(short2v, b)));
}

__device__ __forceinline__ void load16(const float *src, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x4 v = *reinterpret_cast<const f32x4 *>(src + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * i + j] = v[j];
    }
}
__device__ __forceinline__ void load16(const _Float16 *src, float *x) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const half8 v = *reinterpret_cast<const half8 *>(src + 8 * i);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[8 * i + j] = (float)v[j];
    }
}

// The largest magnitude; numbers that are not finite become 0 and are counted.
template <int N>
__device__ __forceinline__ float finite_peak(float *x, unsigned &bad) {
    constexpr float kLargest = 3.4028235e38f;
    float m = 0.f;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        m = fmaxf(m, fmaxf(fabsf(x[i]), fabsf(x[i + 1])));  // a NaN beside a number is passed over
        odd |= __builtin_isunordered(x[i], x[i + 1]);
    }
    if (odd || m > kLargest) {
        m = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (!(fabsf(x[i]) <= kLargest)) x[i] = 0.f, ++bad;
            m = fmaxf(m, fabsf(x[i]));
        }
    }
    return m;
}

// One workgroup per (block, pair): codes and exponents, and the exponents that
// the block's own bounds would take (icl4_units_kernel takes the largest of a
// pair's; by atomics into one word per dim the kernel took 97 instead of 52 us
// at 50,000 rows). Bound by its reads: every load of the block is issued first,
// and the codes are the conversion instructions' own. The block is put together
// in LDS and written in whole lines: from registers, in words of several waves
// each, 50,000 rows took 315 us. 8 heads x 50,000 FP32 rows, 232 MB: 57 us, 4.1
// TB/s (a large copy: 4.9); whole 256-byte rows to a load, or two blocks to a
// workgroup, the second's loads beneath the first's work, are no quicker. 2 x 8 x
// 12,345 FP16 rows 13.4 us, 4.8 TB/s. Keys: wave 2 s + b, lane (g, 8 a + i) takes dims
// 16 g .. of row 32 s + 16 a + 8 b + i. Values: wave d, lane 8 (4 s + 2 t + b) + i
// takes dims 16 d + 2 i and + 1 of rows 32 s + 16 t + 8 b .. +7.
template <typename T>
__global__ __launch_bounds__(256) void icl4_encode_kernel(StoreArgs p) {
    typedef T T2 __attribute__((ext_vector_type(2)));
    __shared__ unsigned peaks[4][32];
    __shared__ __attribute__((aligned(16))) unsigned char out[kBlockBytes];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, i16 = lane & 15;
    const int block = (int)(blockIdx.x % (unsigned)p.blocks), pair = (int)(blockIdx.x / (unsigned)p.blocks);
    const int e = pair / p.heads, head = pair - e * p.heads;
    const int left = rows_of(p.lengths, e, p.rows) - block * kBlock;  // rows of the block inside the length
    const int key_row = 32 * (wave >> 1) + 16 * (i16 >> 3) + 8 * (wave & 1) + (i16 & 7);
    const int value_row = 8 * (lane >> 3), value_dim = 16 * wave + 2 * (lane & 7);
    float x[16];
    T2 v[8];
    {
        const long long row0 = (long long)block * kBlock;
        const T *k = static_cast<const T *>(p.k) + e * p.k_est + head * p.k_head + (row0 + key_row) * p.k_row + 16 * g;
        const T *vs = static_cast<const T *>(p.v) + e * p.v_est + head * p.v_head + (row0 + value_row) * p.v_row + value_dim;
        if (left >= kBlock) {
            load16(k, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const T2 *>(vs + i * p.v_row);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = 0.f;
            if (key_row < left) load16(k, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] = T2{(T)0.f, (T)0.f};
                if (value_row + i < left) v[i] = *reinterpret_cast<const T2 *>(vs + i * p.v_row);
            }
        }
    }
    unsigned bad = 0;
    {
        const float m = finite_peak<16>(x, bad);
        const int ex = code_exponent(rows_max(m));  // lanes of dims 32 u and + 16
        const float scale = pow2(ex);
        const u32x2 w = {coded8(x, scale), coded8(x + 8, scale)};
        const int s = wave >> 1, b = wave & 1;
        *reinterpret_cast<u32x2 *>(out + s * 1024 + lane * 16 + b * 8) = w;
        if (!(g & 1)) out[kKeyExpsAt + ((g >> 1) * 16 + i16) * 4 + 2 * s + b] = (unsigned char)(ex + 127);
        // Largest held |key| of each dim over the wave's rows, FP16 pairs, exact: in three steps a lane hands half of its
        // pairs to another, so that lanes 2 i and 2 i + 1 of a row of 16 end with pair i.
        u32x4 held[2];
        held[0] = __builtin_bit_cast(u32x4, codes8(w[0], scale)), held[1] = __builtin_bit_cast(u32x4, codes8(w[1], scale));
        unsigned y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = held[i >> 2][i & 3] & 0x7fff7fffu;
        auto step = [&](auto lanes, int keep, bool upper) {
            constexpr int N = decltype(lanes)::value;
#pragma unroll
            for (int i = 0; i < keep; ++i) {
                const unsigned give = upper ? y[i] : y[i + keep], own = upper ? y[i + keep] : y[i];
                y[i] = pk_max(own, row_xor<N>(give));
            }
        };
        step(std::integral_constant<int, 8>{}, 4, i16 & 8);
        step(std::integral_constant<int, 4>{}, 2, i16 & 4);
        step(std::integral_constant<int, 2>{}, 1, i16 & 2);
        y[0] = pk_max(y[0], row_xor<1>(y[0]));
        if (!(i16 & 1)) peaks[wave][8 * g + (i16 >> 1)] = y[0];
    }
    __syncthreads();
    if (tid < 32) {
        const unsigned m = pk_max(pk_max(peaks[0][tid], peaks[1][tid]), pk_max(peaks[2][tid], peaks[3][tid]));
        // The block's own exponents (plus 64, as bytes), where its bounds will stand.
        const half2v both = __builtin_bit_cast(half2v, m);
        const int x0 = unit_exponent((float)both[0]) + 64, x1 = unit_exponent((float)both[1]) + 64;
        reinterpret_cast<unsigned short *>(p.bounds + ((long long)pair * p.blocks + block) * 128)[tid] =
            (unsigned short)(x0 | x1 << 8);
    }
    {
        float m[2], y[2][8];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[c][i] = (float)v[i][c];
            m[c] = finite_peak<8>(y[c], bad);
            // The 32 rows of a group: lanes ^ 8 and ^ 16.
            m[c] = fmaxf(m[c], __uint_as_float(other_eight(__float_as_uint(m[c]))));
            m[c] = rows_max(m[c]);
        }
        const int s = lane >> 5, t = (lane >> 4) & 1, b = (lane >> 3) & 1;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int i = 2 * (lane & 7) + c, ex = code_exponent(m[c]);
            const unsigned w = coded8(y[c], pow2(ex));  // rows 4 h + j of h = 0 in the low half
            // The lane of b = 0 writes the word of h = 0, that of b = 1 the other.
            const unsigned far = other_eight(w);
            const unsigned word = b ? (far >> 16) | (w & 0xffff0000u) : (w & 0xffffu) | (far << 16);
            *reinterpret_cast<unsigned *>(out + kValuesAt + s * 1024 + (16 * (2 * t + b) + i) * 16 + wave * 4) = word;
            if (!(lane & 24)) out[kValueExpsAt + i * 8 + s * 4 + wave] = (unsigned char)(ex + 127);
        }
    }
    __syncthreads();
    u32x4 *to = reinterpret_cast<u32x4 *>(p.tiles + ((long long)pair * p.blocks + block) * kBlockBytes);
    to[tid] = reinterpret_cast<const u32x4 *>(out)[tid];
    if (tid < kBlockBytes / 16 - 256) to[256 + tid] = reinterpret_cast<const u32x4 *>(out)[256 + tid];
    if (bad && p.nonfinite) atomicAdd(p.nonfinite, bad);
}

// A pair's units: the largest of its blocks' exponents, 16 dims to a workgroup.
// Latency: 4.8 us for 782 blocks.
__global__ __launch_bounds__(1024) void icl4_units_kernel(StoreArgs p) {
    __shared__ unsigned part[16][8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, pair = blockIdx.x >> 2, g = blockIdx.x & 3;
    const signed char *src = p.bounds + (long long)pair * p.blocks * 128 + 16 * g;
    unsigned m[8];  // bytes 0 and 2, then 1 and 3, of the four words
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] = 0u;
    for (int t = tid; t < p.blocks; t += 1024) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(src + (long long)t * 128);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            m[2 * i] = pk_max(m[2 * i], w[i] & 0xff00ffu);
            m[2 * i + 1] = pk_max(m[2 * i + 1], w[i] >> 8 & 0xff00ffu);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) m[i] = pk_max(m[i], (unsigned)__shfl_xor((int)m[i], off, 64));
        if (lane == 0) part[wave][i] = m[i];
    }
    __syncthreads();
    if (tid >= 16) return;
    const int i = 2 * (tid >> 2) + (tid & 1), shift = 16 * ((tid >> 1) & 1);
    int x = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) x = max(x, (int)(part[w][i] >> shift & 0xffffu));
    p.scales[pair * 64 + 16 * g + tid] = pow2(x - 64);
}

__device__ __forceinline__ unsigned pk_least(unsigned a, unsigned b) {
    return __builtin_bit_cast(unsigned, __builtin_elementwise_min(__builtin_bit_cast(half2v, a), __builtin_bit_cast(half2v, b)));
}
__device__ __forceinline__ unsigned pk_most(unsigned a, unsigned b) {
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(half2v, a), __builtin_bit_cast(half2v, b)));
}

// Bounds of a block by one wave, from the codes as FP16 pairs (exact): lane
// (g, i16) holds dims 16 g .. +15 of four rows; in four steps each lane hands
// half of its dims to another and keeps the least and most of the rest, so
// that lane i16 ends with dim 16 g + i16's. `inv`: of the lane's dim, 1 / unit
// (a power of two: exact).
__device__ __forceinline__ void block_bounds(const StoreArgs &p, int pair, int block, int lane, float inv) {
    const int g = lane >> 4, i16 = lane & 15;
    const long long at = (long long)pair * p.blocks + block;
    const int left = rows_of(p.lengths, pair / p.heads, p.rows) - block * kBlock;
    const unsigned char *in = p.tiles + at * kBlockBytes;
    const unsigned exps = *reinterpret_cast<const unsigned *>(in + kKeyExpsAt + ((g >> 1) * 16 + i16) * 4);
    unsigned lo[8], hi[8];  // dims 2 i, 2 i + 1
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = 0x7c007c00u, hi[i] = 0xfc00fc00u;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(in + s * 1024 + lane * 16);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int r = 32 * s + 16 * (i16 >> 3) + 8 * b + (i16 & 7);
            const float scale = __uint_as_float(((exps >> (8 * (2 * s + b))) & 0xffu) << 23);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const u32x4 y = __builtin_bit_cast(u32x4, codes8(w[2 * b + c], scale));
                if (r < left)
#pragma unroll
                    for (int i = 0; i < 4; ++i) lo[4 * c + i] = pk_least(lo[4 * c + i], y[i]), hi[4 * c + i] = pk_most(hi[4 * c + i], y[i]);
            }
        }
    }
    // Bits 3, 2 and 1 of the lane pick the pair of dims, bit 0 the dim of the pair.
    auto step = [&](auto lanes, int keep, bool upper) {
        constexpr int N = decltype(lanes)::value;
#pragma unroll
        for (int i = 0; i < keep; ++i) {
            const unsigned give_lo = upper ? lo[i] : lo[i + keep], give_hi = upper ? hi[i] : hi[i + keep];
            const unsigned own_lo = upper ? lo[i + keep] : lo[i], own_hi = upper ? hi[i + keep] : hi[i];
            lo[i] = pk_least(own_lo, row_xor<N>(give_lo)), hi[i] = pk_most(own_hi, row_xor<N>(give_hi));
        }
    };
    step(std::integral_constant<int, 8>{}, 4, i16 & 8);
    step(std::integral_constant<int, 4>{}, 2, i16 & 4);
    step(std::integral_constant<int, 2>{}, 1, i16 & 2);
    const unsigned low2 = pk_least(lo[0], row_xor<1>(lo[0])), high2 = pk_most(hi[0], row_xor<1>(hi[0]));
    const float low = (float)__builtin_bit_cast(half2v, low2)[i16 & 1], high = (float)__builtin_bit_cast(half2v, high2)[i16 & 1];
    p.bounds[at * 128 + lane] = left > 0 ? (signed char)floorf(low * inv) : (signed char)0;
    p.bounds[at * 128 + 64 + lane] = left > 0 ? (signed char)ceilf(high * inv) : (signed char)0;
}

// One block to a wave. Reads the keys' codes, which the encoder has left in the
// caches: 7.0 us for 8 x 782 blocks.
__global__ __launch_bounds__(256) void icl4_bounds_kernel(StoreArgs p) {
    const int lane = threadIdx.x & 63;
    const long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= (long long)p.pairs * p.blocks) return;
    const int pair = (int)(at / p.blocks);
    block_bounds(p, pair, (int)(at - (long long)pair * p.blocks), lane, 1.0f / p.scales[pair * 64 + lane]);
}

// Units and bounds of a pair of at most 32 blocks by one workgroup: a thread to
// four dims of a block's exponents, then a wave to every sixteenth block. A store
// and its reading back, 8 heads: 1,024 rows 13.2 against 15.0 us in two launches
// (25.4 against 28.2 called one by one), 2,048 17.0 and 16.4 (25.5 and 28.2), 240
// pairs of 2,000 133 and 143; 4,096 27.6 and 21.8, one workgroup being slow to
// read so much.
constexpr int kSmallBlocks = 32;
__global__ __launch_bounds__(1024) void icl4_small_bounds_kernel(StoreArgs p) {
    __shared__ unsigned part[16][16][2];
    __shared__ float units[64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, pair = blockIdx.x, t = tid >> 4;
    unsigned w = 0u;
    if (t < p.blocks) w = *reinterpret_cast<const unsigned *>(p.bounds + ((long long)pair * p.blocks + t) * 128 + 4 * (tid & 15));
    unsigned m[2] = {w & 0xff00ffu, w >> 8 & 0xff00ffu};  // bytes 0 and 2, then 1 and 3
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        m[i] = pk_max(m[i], (unsigned)__shfl_xor((int)m[i], 16, 64));
        m[i] = pk_max(m[i], (unsigned)__shfl_xor((int)m[i], 32, 64));
        if (lane < 16) part[wave][lane][i] = m[i];
    }
    __syncthreads();
    if (tid < 64) {
        int x = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) x = max(x, (int)(part[i][tid >> 2][tid & 1] >> (8 * (tid & 2)) & 0xffffu));
        units[tid] = p.scales[pair * 64 + tid] = pow2(x - 64);
    }
    __syncthreads();
    for (int block = wave; block < p.blocks; block += 16) block_bounds(p, pair, block, lane, 1.0f / units[lane]);
}

struct ReadArgs {
    void *k, *v;
    long long k_est, k_head, k_row, v_est, v_head, v_row;
    const unsigned *lengths;
    int heads, pairs, rows, blocks;
    const unsigned char *tiles;
    const signed char *bounds;
    const float *scales;
    float *bounds_out;
};

// The encoder's lanes and rows, the other way. Bound by its writes: 8 heads x
// 50,000 FP32 rows, 232 MB, 45 us, 5.1 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void icl4_decode_kernel(ReadArgs p) {
    typedef T T2 __attribute__((ext_vector_type(2)));
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, i16 = lane & 15;
    const int block = (int)(blockIdx.x % (unsigned)p.blocks), pair = (int)(blockIdx.x / (unsigned)p.blocks);
    const int e = pair / p.heads, head = pair - e * p.heads;
    const int left = rows_of(p.lengths, e, p.rows) - block * kBlock;
    const long long at = (long long)pair * p.blocks + block, row0 = (long long)block * kBlock;
    const unsigned char *in = p.tiles + at * kBlockBytes;
    if (p.k) {
        const int s = wave >> 1, b = wave & 1, r = 32 * s + 16 * (i16 >> 3) + 8 * b + (i16 & 7);
        const u32x2 w = *reinterpret_cast<const u32x2 *>(in + s * 1024 + lane * 16 + b * 8);
        const float scale = pow2((int)in[kKeyExpsAt + ((g >> 1) * 16 + i16) * 4 + 2 * s + b] - 127);
        if (r < left) {
            T *dst = static_cast<T *>(p.k) + e * p.k_est + head * p.k_head + (row0 + r) * p.k_row + 16 * g;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const half8 y = codes8(w[c], scale);
                if constexpr (sizeof(T) == 2) {
                    *reinterpret_cast<half8 *>(dst + 8 * c) = y;
                } else {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        *reinterpret_cast<f32x4 *>(dst + 8 * c + 4 * i) =
                            f32x4{(float)y[4 * i], (float)y[4 * i + 1], (float)y[4 * i + 2], (float)y[4 * i + 3]};
                }
            }
        }
    }
    if (p.v) {
        const int s = lane >> 5, t = (lane >> 4) & 1, b = (lane >> 3) & 1, r = 8 * (lane >> 3);
        half8 y[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int i = 2 * (lane & 7) + c;
            unsigned w = 0u;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const unsigned both = *reinterpret_cast<const unsigned *>(in + kValuesAt + s * 1024 +
                                                                          (16 * (2 * t + h) + i) * 16 + wave * 4);
                w |= (b ? both >> 16 : both & 0xffffu) << (16 * h);
            }
            y[c] = codes8(w, pow2((int)in[kValueExpsAt + i * 8 + s * 4 + wave] - 127));
        }
        T *dst = static_cast<T *>(p.v) + e * p.v_est + head * p.v_head + (row0 + r) * p.v_row + 16 * wave + 2 * (lane & 7);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (r + i < left) *reinterpret_cast<T2 *>(dst + i * p.v_row) = T2{(T)y[0][i], (T)y[1][i]};
    }
    if (p.bounds_out && tid < 128)
        p.bounds_out[at * 128 + tid] = (float)p.bounds[at * 128 + tid] * p.scales[pair * 64 + (tid & 63)];
}

// ---- choosing blocks ----

struct SelectArgs {
    const void *q;
    long long q_est, q_head, q_row;
    const unsigned *lengths;
    const unsigned long long *keep;
    int heads, pairs, q_rows, rows, blocks;
    const signed char *bounds;
    const float *scales;
    int n;
    int *out;
    int *scores;            // [pair rows, padded]
    long long padded;       // blocks rounded up to 64
    int pair0, row0, rows_here;  // this launch's pairs and queries: scores row (pair - pair0) * rows_here + row - row0
    int qtiles, chunks, chunk;   // chunk: blocks of one wave
};

constexpr int kNoScore = -(1 << 30);
typedef int i32x4 __attribute__((ext_vector_type(4)));

// The smallest f >= -100 with m <= 127 * 2^f.
__device__ __forceinline__ int code_power(float m) {
    const unsigned bits = __float_as_uint(m);
    const int x = (int)(bits >> 23) - 126;  // zero and subnormal m end at -100
    return min(122, max(-100, (bits & 0x7fffffu) <= 0x7e0000u ? x - 7 : x - 6));  // 122: the largest finite m's
}

// A query's codes as operands: lane (g, i16) dims 16 g .. of query i16,
// positive and negative parts as bytes.
struct QueryCodes {
    i32x4 pos, neg;
};
template <typename T>
__device__ __forceinline__ QueryCodes query_codes(const SelectArgs &p, int pair, int row, int g) {
    const int e = pair / p.heads, head = pair - e * p.heads;
    const T *src = static_cast<const T *>(p.q) + e * p.q_est + head * p.q_head + row * p.q_row + 16 * g;
    float x[16];
    load16(src, x);
    float m = 0.f;
    float unit[16];
    load16(p.scales + pair * 64 + 16 * g, unit);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        x[i] *= unit[i];
        m = fmaxf(m, fabsf(x[i]));
    }
    m = fmaxf(m, __shfl_xor(m, 16, 64));
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    const float inv = pow2(-code_power(m));
    QueryCodes c;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        unsigned a = 0u, b = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int v = (int)rintf(fminf(fmaxf(x[4 * w + i] * inv, -127.f), 127.f));
            a |= (unsigned)max(v, 0) << (8 * i);
            b |= ((unsigned)min(v, 0) & 0xffu) << (8 * i);
        }
        c.pos[w] = (int)a, c.neg[w] = (int)b;
    }
    return c;
}

// The bounds of blocks b .. +15 as operands (`bounds`: the pair's, at dims 16
// g); past the last block it stands in.
__device__ __forceinline__ void load_bounds(const signed char *bounds, int b, int blocks, int i16, i32x4 &low, i32x4 &high) {
    const signed char *src = bounds + (long long)min(b + i16, blocks - 1) * 128;
    low = *reinterpret_cast<const i32x4 *>(src), high = *reinterpret_cast<const i32x4 *>(src + 64);
}
// Scores of 16 queries against them: per sign one 16x16x64 product of whole
// numbers, lower bounds by the codes' negative parts, upper bounds by the
// positive ones. Register r: block b + 4 g + r of query i16.
__device__ __forceinline__ i32x4 block_scores(const i32x4 &low, const i32x4 &high, const QueryCodes &c) {
    i32x4 s = {0, 0, 0, 0};
    s = __builtin_amdgcn_mfma_i32_16x16x64_i8(low, c.neg, s, 0, 0, 0);
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(high, c.pos, s, 0, 0, 0);
}

// Scores of 16 queries against `chunk` blocks per wave: one query, 8 heads, 3,125
// blocks (3.2 MB of bounds) 3.8 us, most of it a workgroup's start and one trip to memory.
template <typename T>
__global__ __launch_bounds__(256) void icl4_scores_kernel(SelectArgs p) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, i16 = lane & 15;
    unsigned id = blockIdx.x;
    const int part = (int)(id % (unsigned)p.chunks);
    id /= (unsigned)p.chunks;
    const int qt = (int)(id % (unsigned)p.qtiles), pair = p.pair0 + (int)(id / (unsigned)p.qtiles);
    const int b0 = (part * 4 + wave) * p.chunk;
    if (b0 >= p.blocks) return;
    const int here = 16 * qt + i16;
    const QueryCodes c = query_codes<T>(p, pair, p.row0 + min(here, p.rows_here - 1), g);
    const signed char *bounds = p.bounds + (long long)pair * p.blocks * 128 + 16 * g;
    int *out = p.scores + ((long long)(pair - p.pair0) * p.rows_here + here) * p.padded + 4 * g;
    const int end = min(p.blocks, b0 + p.chunk);
    for (int b = b0; b < end; b += 16) {
        i32x4 low, high;
        load_bounds(bounds, b, p.blocks, i16, low, high);
        const i32x4 s = block_scores(low, high, c);
        // Blocks past the last lie in the row's padding.
        if (here < p.rows_here) *reinterpret_cast<i32x4 *>(out + b) = s;
    }
}

// Sums, and largest, over a wave, in every lane: quads, eights and rows of 16
// by DPP, then the rows.
template <class Op>
__device__ __forceinline__ int wave_join(int x, Op op) {
    x = op(x, (int)row_xor<1>(x));
    x = op(x, (int)row_xor<2>(x));
    x = op(x, (int)__builtin_amdgcn_update_dpp(0, x, 0x141, 0xf, 0xf, true));  // mirrored eights
    x = op(x, (int)__builtin_amdgcn_update_dpp(0, x, 0x140, 0xf, 0xf, true));  // mirrored rows
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = op((int)r[0], (int)r[1]);
    const auto h = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return op((int)h[0], (int)h[1]);
}

// Scores b .. +3 of a query, those of blocks without an attended row replaced.
__device__ __forceinline__ i32x4 attended_scores(const SelectArgs &p, const int *scores, int e, int rows, int b) {
    i32x4 s = *reinterpret_cast<const i32x4 *>(scores + b);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = rows > (b + i) * kBlock ? s[i] : kNoScore;
    if (p.keep) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // Past the length, and past the last block, the score is gone already.
            const unsigned long long word = p.keep[(long long)e * p.blocks + min(b + i, p.blocks - 1)];
            const int past = kBlock - (rows - (b + i) * kBlock);  // of the block's rows
            s[i] = word << min(max(past, 0), kBlock - 1) ? s[i] : kNoScore;
        }
    }
    return s;
}

// The n best of one query's scores by one wave with every score in a register
// (up to 1,024): bisection between the least and the largest for a value
// that exactly n scores reach, or else the n-th largest. Lane l holds blocks
// 256 i + 4 l + j of GROUPS 256s.
constexpr int kWavePicks = 960;  // sixteen queries' scores in 64 KB of LDS
template <int GROUPS>
__device__ __forceinline__ void pick_by_wave(const SelectArgs &p, const int *scores, const unsigned *attended, int *out) {
    const int lane = threadIdx.x & 63, padded = (int)p.padded;
    i32x4 held[GROUPS];
    int least = 1 << 30, most = kNoScore, total = 0;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
        const int b = 256 * i + 4 * lane;
        held[i] = *reinterpret_cast<const i32x4 *>(scores + min(b, padded - 4));
        const unsigned some = attended[64 * i + lane];  // a byte to a block, 0 past the last
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            held[i][j] = some >> (8 * j) & 0xffu ? held[i][j] : kNoScore;
            most = max(most, held[i][j]);
            least = held[i][j] == kNoScore ? least : min(least, held[i][j]);
            total += __popcll(__ballot(held[i][j] != kNoScore));
        }
    }
    least = __builtin_amdgcn_readfirstlane(wave_join(least, [](int a, int b) { return min(a, b); }));
    most = __builtin_amdgcn_readfirstlane(wave_join(most, [](int a, int b) { return max(a, b); }));
    // More than n scores reach lo, fewer lo + gap.
    int lo = least, gap = most + 1 - least;
    bool exact = total <= p.n;
    if (exact) lo = kNoScore;  // every candidate lies above
    while (!exact && gap > 1) {
        const int cut = lo + (gap >> 1);
        int c = 0;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) c += __popcll(__ballot(held[i][j] >= cut));
        exact = c == p.n;
        if (exact)
            lo = cut - 1;  // the scores above are the n best
        else if (c > p.n)
            gap -= cut - lo, lo = cut;
        else
            gap = cut - lo;
    }
    // Scores above lo and, where no value parts n of them, the first at it that there is room for, in order.
    int all = 0;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) all += __popcll(__ballot(held[i][j] > lo));
    const int room = exact ? 0 : p.n - all;
    const unsigned long long below = (1ull << lane) - 1;
    int before_above = 0, before_equal = 0;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
        if (256 * i >= padded) break;
        int a = before_above, q = before_equal;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned long long va = __ballot(held[i][j] > lo), ve = room > 0 ? __ballot(held[i][j] == lo) : 0ull;
            a += __popcll(va & below), q += __popcll(ve & below);
            before_above += __popcll(va), before_equal += __popcll(ve);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool above = held[i][j] > lo, equal = room > 0 && held[i][j] == lo;
            if (above || (equal && q < room)) out[a + min(q, room)] = 256 * i + 4 * lane + j;
            a += above, q += equal;
        }
    }
    for (int i = min(total, p.n) + lane; i < p.n; i += 64) out[i] = -1;
}

// Sum over the lanes up to this one.
__device__ __forceinline__ int wave_prefix(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // one lane up in each row of 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row 0's last to row 1, 2's to 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row 1's last to rows 2 and 3
    return x;
}

// The n best of one query's scores by a workgroup, for any number of blocks:
// the n-th largest by a histogram of 1,024 steps of 2^sh over the scores'
// range, then over the step that holds it, until a step ends at exactly n or is
// one value wide (two rounds as a rule). Bisection by the sixteen waves took
// 1,550 cycles a step and 11 steps for 3,125 scores; this takes 6.6 us for 8 of
// them, its barriers one after another. Scores stand in `held`, LDS (STAGED) or
// where they are.
constexpr int kPickWaves = 8;
constexpr int kStagedPicks = 12288;  // scores that fit a workgroup's LDS beside the histogram
template <bool STAGED>
__global__ __launch_bounds__(kPickWaves * 64) void icl4_pick_kernel(SelectArgs p) {
    constexpr int THREADS = kPickWaves * 64, BINS = 2 * THREADS;
    extern __shared__ __attribute__((aligned(16))) int staged[];
    __shared__ int bins[BINS];  // from the highest down
    __shared__ int joint[5][kPickWaves];
    __shared__ int found[3];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int at = (int)(blockIdx.x / (unsigned)p.rows_here);
    const int pair = p.pair0 + at, row = p.row0 + (int)(blockIdx.x - (unsigned)at * p.rows_here);
    const int e = pair / p.heads, rows = rows_of(p.lengths, e, p.rows), padded = (int)p.padded;
    int *scores = p.scores + (long long)blockIdx.x * p.padded;
    int *held = STAGED ? staged : scores;
    int *out = p.out + ((long long)pair * p.q_rows + row) * p.n;
    int total = 0, least = 1 << 30, most = kNoScore;
    for (int b = 4 * tid; b < padded; b += 4 * THREADS) {
        const i32x4 s = attended_scores(p, scores, e, rows, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            total += s[j] != kNoScore;
            most = max(most, s[j]);
            least = s[j] == kNoScore ? least : min(least, s[j]);
        }
        *reinterpret_cast<i32x4 *>(held + b) = s;
    }
    const auto add = [](int a, int b) { return a + b; };
    total = wave_join(total, add);
    least = wave_join(least, [](int a, int b) { return min(a, b); });
    most = wave_join(most, [](int a, int b) { return max(a, b); });
    if (lane == 0) joint[0][wave] = total, joint[1][wave] = least, joint[2][wave] = most;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < kPickWaves; ++w)
        total += joint[0][w], least = min(least, joint[1][w]), most = max(most, joint[2][w]);
    int lo = kNoScore, room = 0;  // chosen: the scores above lo and `room` of those at it
    if (total > p.n) {
        int base = __builtin_amdgcn_readfirstlane(least), sh = 0, above = 0, limit = BINS;
        const int range = __builtin_amdgcn_readfirstlane(most) - base;
        while (range >> sh >= BINS) ++sh;
        for (;;) {
            bins[tid] = 0, bins[tid + THREADS] = 0;
            __syncthreads();
            for (int b = 4 * tid; b < padded; b += 4 * THREADS) {
                const i32x4 s = *reinterpret_cast<const i32x4 *>(held + b);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned bin = (unsigned)(s[j] - base) >> sh;
                    if (bin < (unsigned)limit) atomicAdd(&bins[BINS - 1 - bin], 1);
                }
            }
            __syncthreads();
            const int c0 = bins[2 * tid], c1 = bins[2 * tid + 1];
            int upto = wave_prefix(c0 + c1);
            if (lane == 63) joint[0][wave] = upto;
            __syncthreads();
            upto += above;
#pragma unroll
            for (int w = 0; w < kPickWaves; ++w) upto += w < wave ? joint[0][w] : 0;
            // The step where the count from the top reaches n: its thread tells the others.
            const int to0 = upto - c1, before = to0 - c0;
            if (before < p.n && upto >= p.n) {
                const bool first = to0 >= p.n;
                found[0] = BINS - 1 - (2 * tid + (first ? 0 : 1));
                found[1] = first ? before : to0;
                found[2] = first ? to0 : upto;
            }
            __syncthreads();
            const int bin = found[0];
            above = found[1];
            lo = base + (bin << sh);
            if (found[2] == p.n) {
                --lo;  // the whole step is chosen
                break;
            }
            if (sh == 0) {
                room = p.n - above;
                break;
            }
            // The step's 2^sh values alone: what lies above it is counted already.
            static_assert(BINS == 1024, "a step's values fit the next histogram");
            base = lo;
            limit = 1 << min(sh, 10);
            sh = max(0, sh - 10);
        }
    }
    // In order: each wave a contiguous share.
    const int share = (padded / 64 + kPickWaves - 1) / kPickWaves * 64;
    const int first = wave * share, end = min(padded, first + share);
    int more = 0, equal = 0;
    for (int b = first + lane; b < end; b += 64) more += held[b] > lo, equal += held[b] == lo;
    more = wave_join(more, add), equal = wave_join(equal, add);
    if (lane == 0) joint[3][wave] = more, joint[4][wave] = equal;
    __syncthreads();
    int before_more = 0, before_equal = 0;
#pragma unroll
    for (int w = 0; w < kPickWaves; ++w)
        before_more += w < wave ? joint[3][w] : 0, before_equal += w < wave ? joint[4][w] : 0;
    const unsigned long long below = (1ull << lane) - 1;
    for (int b = first + lane; b < end; b += 64) {
        const int s = held[b];
        const unsigned long long va = __ballot(s > lo), ve = __ballot(s == lo);
        const int a = before_more + __popcll(va & below), q = before_equal + __popcll(ve & below);
        if (s > lo || (s == lo && q < room)) out[a + min(q, room)] = b;
        before_more += __popcll(va), before_equal += __popcll(ve);
    }
    for (int i = min(total, p.n) + tid; i < p.n; i += THREADS) out[i] = -1;
}

// Scores and choice in one launch, no scores in memory, up to 960 blocks:
// sixteen queries to a workgroup, scored together, then each chosen for by a
// wave of its own. Every load is issued first; each wave makes one query's
// codes (the sixteen by every wave cost more than the scores). 512 queries x 8
// heads x 782 blocks 15.1 us (8.7 and 20.0 in two launches with the scores in
// memory); 154 x 8 of 193 blocks 7.7, most of it latency.
constexpr int kChooseWaves = 16;
template <typename T, int GROUPS>
__global__ __launch_bounds__(kChooseWaves * 64) void icl4_choose_kernel(SelectArgs p) {
    extern __shared__ __attribute__((aligned(16))) int staged[];  // [queries][padded + 4]
    __shared__ __attribute__((aligned(16))) unsigned char attended[kChooseWaves * 64];
    __shared__ __attribute__((aligned(16))) signed char codes[2][kChooseWaves][64 + 16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, i16 = lane & 15;
    const int qt = blockIdx.x, head = blockIdx.y, e = blockIdx.z, pair = e * p.heads + head;
    const int rows = rows_of(p.lengths, e, p.rows), row = min(16 * qt + wave, p.q_rows - 1);
    const float x0 = (float)static_cast<const T *>(p.q)[e * p.q_est + head * p.q_head + row * p.q_row + lane];
    const float unit = p.scales[pair * 64 + lane];
    const signed char *bounds = p.bounds + (long long)pair * p.blocks * 128 + 16 * g;
    const int stride = (int)p.padded + 4;  // four banks on from one query to the next
    // At most GROUPS steps of sixteen blocks to a wave.
    constexpr int STEP = 16 * kChooseWaves;
    i32x4 low[GROUPS], high[GROUPS];
#pragma unroll
    for (int u = 0; u < GROUPS; ++u) load_bounds(bounds, 16 * wave + u * STEP, p.blocks, i16, low[u], high[u]);
    const int mine = threadIdx.x;  // a thread to a block
    const unsigned long long word = p.keep ? p.keep[(long long)e * p.blocks + min(mine, p.blocks - 1)] : ~0ull;
    {
        const float x = x0 * unit;
        const float inv = pow2(-code_power(wave_max(fabsf(x))));
        const int c = (int)rintf(fminf(fmaxf(x * inv, -127.f), 127.f));
        codes[0][wave][lane] = (signed char)max(c, 0), codes[1][wave][lane] = (signed char)min(c, 0);
    }
    const int left = rows - mine * kBlock;
    attended[mine] = mine < p.blocks && left > 0 && word << max(0, kBlock - left) != 0;
    __syncthreads();
    const QueryCodes c = {*reinterpret_cast<const i32x4 *>(&codes[0][i16][16 * g]),
                          *reinterpret_cast<const i32x4 *>(&codes[1][i16][16 * g])};
#pragma unroll
    for (int u = 0; u < GROUPS; ++u) {
        const int b = 16 * wave + u * STEP;
        const i32x4 s = block_scores(low[u], high[u], c);
        // Only queries that there are have a row.
        if (b < p.padded && 16 * qt + i16 < p.q_rows)
            *reinterpret_cast<i32x4 *>(staged + i16 * stride + b + 4 * g) = s;
    }
    __syncthreads();
    const int query = 16 * qt + wave;
    if (query < p.q_rows)
        pick_by_wave<GROUPS>(p, staged + wave * stride, reinterpret_cast<const unsigned *>(attended),
                             p.out + ((long long)pair * p.q_rows + query) * p.n);
}

// ---- attention ----

struct AttendArgs {
    const void *q;
    long long q_est, q_head, q_row;
    void *o;
    long long o_est, o_head, o_row;
    float *lse;
    const unsigned char *tiles;
    const float *units;  // [pairs, 64], of the cache
    const unsigned *lengths;
    const unsigned long long *keep;
    const int *list;  // [pairs, q_rows, n] or null
    int n;
    int heads, pairs, q_rows, rows, blocks;
    float scale;
    // Outputs [splits, part_rows, 64], then [splits, part_rows, 2]: their softmax's reference (log2) and the sum of weights
    // against it. Apart, not as one logarithm: next to a reference of 2^20 that would keep a sum to three bits.
    float *partial;
    int splits, per_split;  // blocks (or listed places) of a split
    int qtiles, count, per_xcd;
    Division by_qtiles, by_splits, by_queries, by_heads;
    int whole, unit_rows;  // units that are not split; rows of a split unit (0: partials of every row)
    Division by_rest;      // units that are
    long long part_rows;   // rows of a split's partials
};

constexpr float kLn2 = 0.69314718055994530942f;
// Weights are held against a reference below the largest so far, so that FP16's
// smallest step, 2^-24, is small beside the largest weight: 2^-32 of it where a
// reference is cheap to raise. The wide kernels raise theirs when weights pass
// 2^15 or so, which costs them most of a block's work: with 2^5 (FP16) and 2^6
// (FP32) 1.2 and 1.7 times in a wave's 40 blocks of 10,007 rows, with 2^8 4.9
// times; a weight is then off by at most 2^-30 and 2^-31 of the largest.
// FP16 queries' weights over every block are rounded once to FP16, a choice: their
// outputs are off by 2.8e-4 (2-norm; 8 x 200,000 x 2 by 2.2e-4), where the rounding
// of the output alone leaves 2.1e-4 and pairs would too, but take 342 us instead
// of 242 at 10,007 x 10,007, 84 instead of 70 at 777 x 12,345 x 2 masked, 54.4
// instead of 50.3 at 8 x 200,000 x 2. Over listed blocks pairs cost 1%.
constexpr float kHeadroom = 8.0f, kWideHeadroom16 = 5.0f, kWideHeadroom32 = 6.0f;

// A product that is rounded by itself, whatever is added to it.
__device__ __forceinline__ float product(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}

// The reference of weights whose largest score is `top`: `headroom` below it, or
// `top` itself where FP32's step there is so large that more than 15 lie between
// (a weight must not pass FP16's 65,504).
__device__ __forceinline__ float reference(float top, float headroom) {
    const float r = top - headroom;
    return top - r > 15.0f ? top : r;
}

// The smallest e with |m| < 2^e of a finite m, subnormal or not (0 and infinity: 0).
__device__ __forceinline__ int binade(float m) { return __builtin_amdgcn_frexp_expf(m); }

// What a product of 2^-e q and k is multiplied by for its score times log2 e.
__device__ __forceinline__ float factor(const AttendArgs &p, int e) { return __builtin_ldexpf(p.scale, e) * kLog2e; }

// The writer of one query's output: dims d .. +3.
template <typename T>
__device__ __forceinline__ void store_out(const AttendArgs &p, int e, int head, int row, int d, f32x4 v) {
    T *dst = static_cast<T *>(p.o) + e * p.o_est + head * p.o_head + row * p.o_row + d;
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<f32x4 *>(dst) = v;
    } else {
        typedef _Float16 half4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<half4 *>(dst) = __builtin_convertvector(v, half4);
    }
}

// The same of a split's row `at` of all splits' (`all` rows each).
__device__ __forceinline__ void store_part(const AttendArgs &p, long long all, long long at, int d, f32x4 v, float reference,
                                           float sum) {
    *reinterpret_cast<f32x4 *>(p.partial + at * 64 + d) = v;
    if (d == 0) *reinterpret_cast<f32x2 *>(p.partial + p.splits * all * 64 + 2 * at) = f32x2{reference, sum};
}

constexpr int kWaves = 4;

// One workgroup per (16 queries, pair, split): wave w takes every fourth block
// of the split. FP32 queries and probabilities are pairs of FP16 values, two
// products each. Bound by its reads of the cache: 8 FP16 queries x 16 pairs x
// 200,000 rows, 218 MB, 41 us, 5.3 TB/s; with a block's loads all issued before
// its work, and none beside it, 47.
template <typename T, bool SPLIT>
__global__ __launch_bounds__(kWaves * 64) void icl4_rows_kernel(AttendArgs p) {
    constexpr bool PAIRS = sizeof(T) == 4;
    __shared__ __attribute__((aligned(16))) float red_o[kWaves][16 * 68];
    static_assert(__alignof__(red_o) >= alignof(f32x4), "read and written in fours");
    __shared__ float red_m[kWaves][16], red_l[kWaves][16];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, i16 = lane & 15;
    const unsigned tile = SPLIT ? divide(blockIdx.x, p.by_splits) : blockIdx.x;
    const int split = SPLIT ? (int)(blockIdx.x - tile * p.by_splits.d) : 0;
    const int pair = (int)divide(tile, p.by_qtiles), qt = (int)(tile - pair * p.by_qtiles.d);
    const int e = (int)divide(pair, p.by_heads), head = pair - e * p.heads;
    const int rows = rows_of(p.lengths, e, p.rows);
    const int qrow = min(16 * qt + i16, p.q_rows - 1);
    // The first block's operands, beneath the queries' setup; then a block's keys are loaded as soon as the one before
    // has its scores, its values once that one has its output.
    const unsigned char *tiles = p.tiles + (long long)pair * p.blocks * kBlockBytes;
    const int end = min(p.blocks, (split + 1) * p.per_split);
    const unsigned chunk_at = 16u * lane, ke_at = kKeyExpsAt + ((g >> 1) * 16 + i16) * 4, ve_at = kValueExpsAt + i16 * 8;
    u32x4 kw[2], vw[2];
    unsigned ke;
    u32x2 ve;
    auto load_keys = [&](const unsigned char *in) {
        kw[0] = *reinterpret_cast<const u32x4 *>(in + chunk_at);
        kw[1] = *reinterpret_cast<const u32x4 *>(in + 1024 + chunk_at);
        ke = *reinterpret_cast<const unsigned *>(in + ke_at);
    };
    auto load_values = [&](const unsigned char *in) {
        vw[0] = *reinterpret_cast<const u32x4 *>(in + kValuesAt + chunk_at);
        vw[1] = *reinterpret_cast<const u32x4 *>(in + kValuesAt + 1024 + chunk_at);
        ve = *reinterpret_cast<const u32x2 *>(in + ve_at);
    };
    auto find = [&](int &at, unsigned long long &mask) {
        for (; at < end; at += kWaves) {
            mask = block_mask(p.keep, e, p.blocks, at, rows);
            if (mask) return true;
        }
        return false;
    };
    unsigned long long next_mask = 0;
    int at = split * p.per_split + wave;
    bool more = find(at, next_mask);
    if (more) load_keys(tiles + (long long)at * kBlockBytes), load_values(tiles + (long long)at * kBlockBytes);
    half8 qh[2], ql[2];
    float c;
    {
        const T *src = static_cast<const T *>(p.q) + e * p.q_est + head * p.q_head + (long long)qrow * p.q_row + 16 * g;
        if constexpr (PAIRS) {
            float x[16];
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 v = *reinterpret_cast<const f32x4 *>(src + 4 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[4 * i + j] = v[j], m = fmaxf(m, fabsf(v[j]));
            }
            m = fmaxf(m, __shfl_xor(m, 16, 64));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            const int ex = pair_exponent(m);
            const float up = pow2(ex);
            c = factor(p, -ex);
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] *= up;
            pair8(x, qh[0], ql[0]);
            pair8(x + 8, qh[1], ql[1]);
        } else {
            c = factor(p, 0);
            qh[0] = *reinterpret_cast<const half8 *>(src);
            qh[1] = *reinterpret_cast<const half8 *>(src + 8);
        }
    }
    f32x4 o[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;  // m_run: the largest score less the headroom
    while (more) {
        const unsigned long long mask = next_mask;
        at += kWaves;
        more = find(at, next_mask);
        const unsigned char *next = tiles + (long long)at * kBlockBytes;
        f32x4 s[4];
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
            const unsigned w[2] = {kw[kb >> 1][2 * (kb & 1)], kw[kb >> 1][2 * (kb & 1) + 1]};
            const float scale = kb == 0 ? scale_byte<0>(ke) : kb == 1 ? scale_byte<1>(ke) : kb == 2 ? scale_byte<2>(ke) : scale_byte<3>(ke);
            s[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const half8 a = codes8(w[m], scale);
                if constexpr (PAIRS) s[kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[m], s[kb], 0, 0, 0);
                s[kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[m], s[kb], 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) s[kb][r] = product(s[kb][r], c);
        }
        if (more) load_keys(next);
        // Register r of s[2 s + b]: row 32 s + 16 (g / 2) + 8 b + 4 (g % 2) + r.
        if (mask != ~0ull) {
            const unsigned long long mine = mask >> (16 * (g >> 1) + 4 * (g & 1));
#pragma unroll
            for (int kb = 0; kb < 4; ++kb)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (!((mine >> (32 * (kb >> 1) + 8 * (kb & 1) + r)) & 1)) s[kb][r] = -INFINITY;
        }
        float mt = s[0][0];
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r) mt = fmaxf(mt, s[kb][r]);
        mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
        mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
        const float m_new = fmaxf(m_run, reference(mt, kHeadroom));  // finite: the block has an attended row
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        l_run *= alpha;
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] *= alpha;
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = __builtin_amdgcn_exp2f(s[2 * st + (i >> 2)][i & 3] - m_new);
                l_run += x[i];
            }
            half8 ph, pl;
            if constexpr (PAIRS) {
                pair8(x, ph, pl);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) ph[i] = (_Float16)x[i];
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const float scale = d == 0 ? scale_byte<0>(ve[st]) : d == 1 ? scale_byte<1>(ve[st]) : d == 2 ? scale_byte<2>(ve[st]) : scale_byte<3>(ve[st]);
                const half8 a = codes8(vw[st][d], scale);
                if constexpr (PAIRS) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl, o[d], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph, o[d], 0, 0, 0);
            }
        }
        if (more) load_values(next);
    }
    // The waves' parts: lane (g, i16) holds dims 16 d + 4 g + r of query i16.
    l_run += __shfl_xor(l_run, 16, 64);
    l_run += __shfl_xor(l_run, 32, 64);
    if (g == 0) red_m[wave][i16] = m_run, red_l[wave][i16] = l_run;
#pragma unroll
    for (int d = 0; d < 4; ++d) *reinterpret_cast<f32x4 *>(&red_o[wave][i16 * 68 + 16 * d + 4 * g]) = o[d];
    __syncthreads();
    const int qi = threadIdx.x >> 4, d = 4 * (threadIdx.x & 15);
    const int out_row = 16 * qt + qi;
    if (out_row >= p.q_rows) return;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, red_m[w][qi]);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float den = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        // Nothing attended: every part is zero. (A query that is not finite gives NaN.)
        const float a = mx > -INFINITY ? __builtin_amdgcn_exp2f(red_m[w][qi] - mx) : 1.0f;
        acc += a * *reinterpret_cast<const f32x4 *>(&red_o[w][qi * 68 + d]);
        den += a * red_l[w][qi];
    }
    if (den != 0.f) acc *= 1.0f / den;
    if constexpr (SPLIT) {
        const long long all = (long long)p.pairs * p.q_rows;
        store_part(p, all, split * all + (long long)pair * p.q_rows + out_row, d, acc, mx, den);
    } else {
        store_out<T>(p, e, head, out_row, d, acc);
        // -inf where nothing is attended.
        if (p.lse && d == 0) p.lse[(long long)pair * p.q_rows + out_row] = (mx + log2f(den)) * kLn2;
    }
}

typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr int kWideStride = 68;  // floats of one query's row in LDS

// Larger of, or sum of, a lane's value and lane ^ 32's.
__device__ __forceinline__ float halves_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x6 __attribute__((ext_vector_type(6)));
typedef float f32x32 __attribute__((ext_vector_type(32)));

// 32 numbers as PARTS operands in E2M3 (multiples of 1/8 below 2, of 1/4 below
// 4): x = p0 + p1 / 2^4 + p2 / 2^9 + ..., the largest of a row scaled into [2,
// 4), each part the nearest to what is left: the first is off by at most 1/8,
// the next, in a unit 2^-4 and then 2^-5 as large, by at most 1/16. What four
// leave is at most 2^-18, 2^-19 of the row's largest, what five leave 2^-24 of
// it. (FP16 numbers down to 2^-8 of the largest are whole multiples of the last
// one's step, 2^-17: exact.) Fixed steps are coarse for a row whose largest
// number, times small keys, does not make its scores: see kMoreParts. The
// exponent bytes of parts 0 to 3 and of part 4; `even` and `odd` become what is
// left.
constexpr int kPartExps = 127 | (127 - 4) << 8 | (127 - 9) << 16 | (127 - 14) << 24, kPartExps4 = 127 - 19;
template <int PARTS>
__device__ __forceinline__ void query_parts(f32x16 &even, f32x16 &odd, u32x6 (&parts)[PARTS]) {
    float unit = 1.0f;
#pragma unroll
    for (int n = 0; n < PARTS; ++n) {
        parts[n] = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, unit);
        const f32x32 held = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(parts[n], unit);
#pragma unroll
        for (int i = 0; i < 16; ++i) even[i] -= held[2 * i], odd[i] -= held[2 * i + 1];
        unit *= n == 0 ? 0.0625f : 0.03125f;
    }
}

// Parts that a query takes beyond the kernel's own, as many as it needs, from
// LDS: while what is left of its numbers, times the largest keys that the cache's
// units allow, may move a score (times log2 e) by more than 2^-14 and more than
// 2^-21 of the sum of its terms' sizes. Nine parts hold every FP16 row exactly
// (2^-38 of [2, 4) is its last bit), ten an FP32 one to 2^-49 of its largest.
// Queries that need none multiply zeros in their neighbours' extra parts, which
// changes no bit of theirs. Normal queries take none. With one number of 200, 2,000
// or 30,000 beside normal ones, on keys of zero, in every query: 10,007 x 10,007
// FP16 258 us without it and 273, 278 and 291 with, off by 2.8e-4 each; 512 x
// 50,000 FP32 106 and 119, 125 and 123, off by 1.0e-6 at most. (Four parts alone are
// off by 2e-2 at 30,000, and five by 6e-4.)
constexpr int kMoreParts = 5;
constexpr float kScoreLeft = 0x1p-14f, kScoreShare = 0x1p-21f;

// 32 NJ queries per workgroup, every fourth block of its share to a wave. A wave
// reads its blocks straight into registers: 4 bits a number are few enough that
// neither LDS nor a barrier stands between the cache and the products. Scores
// are scaled 32x32x64 products of the E2M1 keys as they lie in the cache by the
// queries' E2M3 parts (33 cycles for what two 32x32x16 ones take 66 for, and no
// conversion of keys, 7.4 cycles a pair of numbers); values are converted to
// FP16 and multiplied by FP16 weights (FP32: pairs). What bounds it is the vector
// unit: per 64 x 64 scores 64 exponentials (9.3 cycles), 64 multiply-adds, 32
// conversions of values and 32 of weights, and the sums: at 10,007 FP16 queries
// and rows it is busy for 62% of the time, the matrix cores for 36%, one or the
// other for 85% (three or two waves to a SIMD hide the rest no further). 8 heads:
// 512 FP32 queries x 50,000 rows 102 us with the merge, 514 TFLOP/s (a pair's two
// products counted once); 10,007 x 10,007 FP16 239, 859.
// Lane (r = lane % 32, h = lane / 32), r = 16 s + 8 a + i:
//   S^T, b = 0, 1: A = rows 32 s + 16 a + 8 b + i, dims 32 h ..; B = query r, the same dims;
//     result register 8 s + 4 a + j is row 32 s + 16 a + 8 b + 4 h + j, query r;
//   O^T, D = 0, 1, step (s, a): A = dim 32 x + 16 D + i (r = 16 x + i), rows 32 s + 16 a + 8 b
//     + 4 h + j; B = those weights, where they are; result register 8 x + 4 y + j is
//     dim 32 x + 16 D + 8 y + 4 h + j, query r.
// Workgroups 0 .. whole - 1 take every block for a (query tile, pair) and write
// its output; the later ones take a split each of the units left over.
template <typename T, int NJ>
__global__ __launch_bounds__(kWaves * 64, NJ == 1 ? 3 : 2) void icl4_wide_kernel(AttendArgs p) {
    constexpr bool PAIRS = sizeof(T) == 4;
    constexpr int PARTS = PAIRS ? 5 : 4;
    __shared__ __attribute__((aligned(16))) float red_o[kWaves][32 * NJ * kWideStride];
    static_assert(__alignof__(red_o) >= alignof(f32x4), "read and written in fours");
    __shared__ float red_m[kWaves][32 * NJ], red_l[kWaves][32 * NJ];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int h = lane >> 5, r32 = lane & 31, i16 = lane & 15, x16 = (lane >> 4) & 1;
    // Workgroups of one XCD take consecutive query tiles of one pair (or share of its blocks), read into one L2.
    const bool tail = blockIdx.x >= (unsigned)p.whole;
    const unsigned bid = tail ? blockIdx.x - p.whole : blockIdx.x, per_xcd = tail ? p.per_xcd : p.whole >> 3;
    const unsigned id = (bid & 7u) * per_xcd + (bid >> 3);
    if (tail && id >= (unsigned)p.count) return;
    // A tail's order is pair, split, query tile, as far as its units go: unit = whole + id % rest.
    const int split = tail ? (int)divide(id, p.by_rest) : 0;
    const int unit = tail ? p.whole + (int)(id - split * p.by_rest.d) : (int)id;
    const int pair = (int)divide(unit, p.by_qtiles), qt = unit - pair * p.by_qtiles.d;
    const int e = (int)divide(pair, p.by_heads), head = pair - e * p.heads;
    const int rows = rows_of(p.lengths, e, p.rows);
    const unsigned char *tiles = p.tiles + (long long)pair * p.blocks * kBlockBytes;
    const unsigned k_at = x16 * 1024 + (32 * h + i16) * 16, v_at = kValuesAt + (16 * h + i16) * 16 + 8 * x16;
    const unsigned ke_at = kKeyExpsAt + (16 * h + i16) * 4, ve_at = kValueExpsAt + i16 * 8;
    u32x2 kw[2][2], vw[4];
    unsigned ke;
    u32x2 ve;
    auto load_keys = [&](const unsigned char *in) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int n = 0; n < 2; ++n) kw[b][n] = *reinterpret_cast<const u32x2 *>(in + k_at + 256 * n + 8 * b);
        ke = *reinterpret_cast<const unsigned *>(in + ke_at);
    };
    auto load_values = [&](const unsigned char *in) {
#pragma unroll
        for (int t = 0; t < 4; ++t) vw[t] = *reinterpret_cast<const u32x2 *>(in + v_at + 512 * t);
        ve = *reinterpret_cast<const u32x2 *>(in + ve_at);
    };
    const int end = tail ? min(p.blocks, (split + 1) * p.per_split) : p.blocks;
    auto find = [&](int &at, unsigned long long &mask) {
        for (; at < end; at += kWaves) {
            mask = block_mask(p.keep, e, p.blocks, at, rows);
            if (mask) return true;
        }
        return false;
    };
    unsigned long long mask = 0;
    int at = split * p.per_split + wave;
    bool more = find(at, mask);
    if (more) load_keys(tiles + (long long)at * kBlockBytes), load_values(tiles + (long long)at * kBlockBytes);
    u32x6 parts[NJ][PARTS];
    float c[NJ];
    int more_parts[NJ];
    static_assert(kMoreParts * 6 * 64 <= 32 * kWideStride, "a wave's outputs have room for them");
    bool far = false;
    float units[32];  // of the lane's dims of keys
    load16(p.units + pair * 64 + 32 * h, units);
    load16(p.units + pair * 64 + 32 * h + 16, units + 16);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        const int row = min(32 * (NJ * qt + j) + r32, p.q_rows - 1);
        const T *src = static_cast<const T *>(p.q) + e * p.q_est + head * p.q_head + (long long)row * p.q_row + 32 * h;
        float x[32];
        load16(src, x);
        load16(src + 16, x + 16);
        float m = 0.f, nan = 0.f, reach = 0.f;
        f32x16 even, odd;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            even[i] = x[2 * i], odd[i] = x[2 * i + 1];
            m = fmaxf(m, fmaxf(fabsf(even[i]), fabsf(odd[i])));
            nan = fmaf(odd[i], 0.f, fmaf(even[i], 0.f, nan));
        }
        // The largest into [2, 4).
        const int ex = binade(halves_max(m)) - 2;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            even[i] = __builtin_ldexpf(even[i], -ex), odd[i] = __builtin_ldexpf(odd[i], -ex);
            reach = fmaf(fabsf(even[i]), units[2 * i], fmaf(fabsf(odd[i]), units[2 * i + 1], reach));
        }
        query_parts<PARTS>(even, odd, parts[j]);
        // A query that is not finite makes NaN of its own scores alone. The factor is normal, for -inf, a masked score,
        // times 0 is no score; one that is less makes nothing of any score either way (they are below 2^25).
        c[j] = fmaxf(factor(p, ex), 1.17549435e-38f) + halves_sum(nan);
        // Scores that may reach 2^22 (no key's size passes 127 units) are products rounded by themselves, against which
        // a reference can be held; weights take the others as they are multiplied. The factor waits in LDS, a lane's own.
        const float most = halves_sum(reach) * (127.0f * c[j]);
        const bool is_far = !(most < 4194304.0f);
        more_parts[j] = 0;
        float step = PAIRS ? 0x1p-24f : 0x1p-19f;
        for (;;) {
            float left = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                asm volatile("" ::: "memory");  // read again, four at a time: held, they would cost the loop registers
                const f32x4 u = *reinterpret_cast<const f32x4 *>(p.units + pair * 64 + 32 * h + 4 * i);
                left = fmaf(fabsf(even[2 * i]), u[0], fmaf(fabsf(odd[2 * i]), u[1], left));
                left = fmaf(fabsf(even[2 * i + 1]), u[2], fmaf(fabsf(odd[2 * i + 1]), u[3], left));
            }
            // (Of a query that is not finite: no.)
            const bool needs = halves_sum(left) * (127.0f * c[j]) > fmaxf(kScoreLeft, most * kScoreShare);
            if (!__any(needs)) break;
#pragma unroll
            for (int i = 0; i < 16; ++i) even[i] = needs ? even[i] : 0.f, odd[i] = needs ? odd[i] : 0.f;
            const u32x6 part = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, step);
            u32x2 *to = reinterpret_cast<u32x2 *>(&red_o[wave][32 * kWideStride * j]) + 192 * more_parts[j] + lane;
#pragma unroll
            for (int i = 0; i < 3; ++i) to[64 * i] = u32x2{part[2 * i], part[2 * i + 1]};
            if (++more_parts[j] == kMoreParts) break;
            const f32x32 held = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(part, step);
#pragma unroll
            for (int i = 0; i < 16; ++i) even[i] -= held[2 * i], odd[i] -= held[2 * i + 1];
            step *= 0.03125f;
        }
        (h ? red_m : red_l)[wave][32 * j + r32] = is_far ? c[j] : 1.0f;
        c[j] = is_far ? 1.0f : c[j];
        far = far || __any(is_far);
    }
    // The products take exponents from vector registers only.
    int part_exps = kPartExps, part_exps4 = kPartExps4, one_exp = 127, most_exp = 254;
    asm volatile("" : "+v"(part_exps), "+v"(part_exps4), "+v"(one_exp), "+v"(most_exp));
    f32x16 o[NJ][2];
    float ref[NJ], l_run[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        ref[j] = -INFINITY, l_run[j] = 0.f;
#pragma unroll
        for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[j][d][r] = 0.f;
    }
    // A block's keys are loaded as soon as the one before has its scores, its values once that one has its output.
    while (more) {
        const unsigned long long now = mask;
        at += kWaves;
        more = find(at, mask);
        const unsigned char *next = tiles + (long long)at * kBlockBytes;
        f32x16 s[NJ][2];
        {
            const int ks = (int)(ke >> (16 * x16));
            const i32x8 a[2] = {{(int)kw[0][0][0], (int)kw[0][0][1], (int)kw[0][1][0], (int)kw[0][1][1], 0, 0, 0, 0},
                                {(int)kw[1][0][0], (int)kw[1][0][1], (int)kw[1][1][0], (int)kw[1][1][1], 0, 0, 0, 0}};
            // Formats 4 (E2M1) and 2 (E2M3); bytes b and n of the exponents.
#define IRX_PART(j, b, n, exps, byte)                                                                                    \
    s[j][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a[b],                                                      \
                                                              (i32x8{(int)parts[j][n][0], (int)parts[j][n][1],           \
                                                                     (int)parts[j][n][2], (int)parts[j][n][3],           \
                                                                     (int)parts[j][n][4], (int)parts[j][n][5], 0, 0}),   \
                                                              s[j][b], 4, 2, b, ks, byte, exps)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[j][b][r] = 0.f;
                if constexpr (PAIRS) {
                    IRX_PART(j, 0, 4, part_exps4, 0);
                    IRX_PART(j, 1, 4, part_exps4, 0);
                }
                IRX_PART(j, 0, 3, part_exps, 3);
                IRX_PART(j, 1, 3, part_exps, 3);
                IRX_PART(j, 0, 2, part_exps, 2);
                IRX_PART(j, 1, 2, part_exps, 2);
                IRX_PART(j, 0, 1, part_exps, 1);
                IRX_PART(j, 1, 1, part_exps, 1);
                IRX_PART(j, 0, 0, part_exps, 0);
                IRX_PART(j, 1, 0, part_exps, 0);
            }
#undef IRX_PART
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                // Last, so that the others begin at 0 without registers that hold it (before them: 252 us instead of 241
                // for 10,007 x 10,007 FP16 queries that take none).
                for (int n = 0; n < more_parts[j]; ++n) {
                    const u32x2 *from = reinterpret_cast<const u32x2 *>(&red_o[wave][32 * kWideStride * j]) + 192 * n + lane;
                    const u32x2 part[3] = {from[0], from[64], from[128]};
                    const i32x8 x = {(int)part[0][0], (int)part[0][1], (int)part[1][0], (int)part[1][1],
                                     (int)part[2][0], (int)part[2][1], 0, 0};
                    const int exps = 127 - (5 * (PARTS + n) - 1);
                    s[j][0] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a[0], x, s[j][0], 4, 2, 0, ks, 0, exps);
                    s[j][1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a[1], x, s[j][1], 4, 2, 1, ks, 0, exps);
                }
        }
        if (now != ~0ull) {
            // Rows that are not attended: one more product, of -6 * 2^127 in their first term by 1, makes -inf of
            // their scores.
            const unsigned bits = x16 ? (unsigned)(now >> 32) : (unsigned)now;
            const int r = r32 & 15, first = r + (r & 8);  // 16 a + i
            const i32x8 one = {h ? 0 : 8, 0, 0, 0, 0, 0, 0, 0};
            const i32x8 a0 = {h || (bits >> first & 1) ? 0 : 15, 0, 0, 0, 0, 0, 0, 0};
            const i32x8 a1 = {h || (bits >> (first + 8) & 1) ? 0 : 15, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                s[j][0] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a0, one, s[j][0], 4, 2, 0, most_exp, 0, one_exp);
                s[j][1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a1, one, s[j][1], 4, 2, 0, most_exp, 0, one_exp);
            }
        }
        if (far) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const float f = (h ? red_m : red_l)[wave][32 * j + r32];
#pragma unroll
                for (int r = 0; r < 16; ++r) s[j][0][r] = product(s[j][0][r], f), s[j][1][r] = product(s[j][1][r], f);
            }
        }
        if (more) load_keys(next);
        half8 ph[NJ][4], pl[PAIRS ? NJ : 1][4];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            // The query's weights against its reference, and the lane's sum of them.
            auto weigh = [&] {
                float l = 0.f;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    float x[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        x[i] = __builtin_amdgcn_exp2f(fmaf(s[j][i >> 2][4 * t + (i & 3)], c[j], -ref[j]));
                        l += x[i];
                    }
                    if constexpr (PAIRS)
                        pair8(x, ph[j][t], pl[j][t]);
                    else
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const half2v w = __builtin_convertvector((f32x2{x[2 * i], x[2 * i + 1]}), half2v);
                            ph[j][t][2 * i] = w[0], ph[j][t][2 * i + 1] = w[1];
                        }
                }
                return l;
            };
            auto largest = [&] {
                float mt = s[j][0][0];
#pragma unroll
                for (int r = 0; r < 16; ++r) mt = fmaxf(mt, fmaxf(s[j][0][r], s[j][1][r]));
                return mt;
            };
            // Raises the reference of the queries of which `past` says so, each by its own scores alone, whatever the
            // others of its wave do.
            auto raise = [&](bool past, float mt) {
                const bool fits = halves_max(past ? 1.f : 0.f) == 0.f;
                const float top = product(halves_max(mt), c[j]);
                const float ref_new = fits ? ref[j] : fmaxf(ref[j], reference(top, PAIRS ? kWideHeadroom32 : kWideHeadroom16));
                const float alpha = __builtin_amdgcn_exp2f(ref[j] - ref_new);
                ref[j] = ref_new;
                l_run[j] *= alpha;
#pragma unroll
                for (int d = 0; d < 2; ++d) o[j][d] *= alpha;
            };
            // A weight must not pass FP16. FP16 weights leave registers for the scores, so the sum of the weights, at
            // most 2^15, tells; FP32's pairs take their place, so the largest score is looked for first.
            float l;
            if constexpr (PAIRS) {
                const float mt = largest();
                const bool past = !(fmaf(mt, c[j], -ref[j]) <= 15.0f);
                if (__any(past)) raise(past, mt);
                l = weigh();
            } else {
                l = weigh();
                const bool past = !(l <= 32768.0f);
                if (__any(past)) {
                    raise(past, largest());
                    l = weigh();
                }
            }
            l_run[j] += l;
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {  // t = 2 s + a
            const unsigned v = ve[t >> 1] >> (16 * x16);
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                const half8 a = codes8(vw[t][d], d ? scale_byte<1>(v) : scale_byte<0>(v));
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    if constexpr (PAIRS) o[j][d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl[j][t], o[j][d], 0, 0, 0);
                    o[j][d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[j][t], o[j][d], 0, 0, 0);
                }
            }
        }
        if (more) load_values(next);
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        const int q = 32 * j + r32;
        const float l = halves_sum(l_run[j]);
        if (h == 0) red_m[wave][q] = ref[j], red_l[wave][q] = l;
#pragma unroll
        for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int a = 0; a < 4; ++a)
                *reinterpret_cast<f32x4 *>(&red_o[wave][q * kWideStride + 32 * (a >> 1) + 16 * d + 8 * (a & 1) + 4 * h]) =
                    f32x4{o[j][d][4 * a], o[j][d][4 * a + 1], o[j][d][4 * a + 2], o[j][d][4 * a + 3]};
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2 * NJ; ++i) {
        const int q = 16 * i + (threadIdx.x >> 4), d = 4 * (threadIdx.x & 15), row = 32 * NJ * qt + q;
        if (row >= p.q_rows) continue;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, red_m[w][q]);
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        float den = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float a = mx > -INFINITY ? __builtin_amdgcn_exp2f(red_m[w][q] - mx) : 1.0f;
            acc += a * *reinterpret_cast<const f32x4 *>(&red_o[w][q * kWideStride + d]);
            den += a * red_l[w][q];
        }
        if (den != 0.f) acc *= 1.0f / den;
        if (tail && p.splits > 1) {
            const long long all = (long long)p.by_rest.d * (32 * NJ);
            store_part(p, all, split * all + (long long)(unit - p.whole) * (32 * NJ) + q, d, acc, mx, den);
        } else {
            store_out<T>(p, e, head, row, d, acc);
            if (p.lse && d == 0) p.lse[(long long)pair * p.q_rows + row] = (mx + log2f(den)) * kLn2;
        }
    }
}

// Four consecutive lanes' neighbour: lane ^ 1.
__device__ __forceinline__ float next_lane(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0xb1, 0xf, 0xf, true));
}

// Lane N of each row of 16, in all of the row's lanes.
template <int N>
__device__ __forceinline__ unsigned row_lane(unsigned x) {
    return __builtin_amdgcn_update_dpp(0, x, 0x150 + N, 0xf, 0xf, true);
}

// One query per workgroup, its blocks (listed, or all) in turn over the waves.
//
// Scores come from the codes as they lie in the cache: 16x16x128 products of the
// query, in whole numbers, by E2M1 rows with their exponents, which take no
// conversion. The query, scaled by a power of two to 31-bit integers, is eight
// digits to the base 16 (the first signed), exact in E4M3. Row 4 n + r of the
// query's operand holds digits 2 r (times 16) and 2 r + 1: the 128 terms are the
// 64 dims by the two; terms 32 g .. +15 are dims 16 g .. by the first, the next 16
// the same dims by the second, so a lane's 16 dims of a key stand twice. The
// exponent of row 4 n + r is that of its digits in the product of the n-th 16
// rows of the block and 2^-127 in the others, so that the four products add up
// in one accumulator: lane (g, i16) ends with the four digit pairs of the i16-th
// row of the g-th sixteen, and adds them. The softmax so costs one exponential
// per row. (With keys converted to FP16 and every column the query, a block
// took 190 vector instructions instead of 100.) Weights go through LDS to where
// the second product wants them, as high FP16 parts in even and low ones in odd
// columns: pairs cost FP16 queries next to nothing here (512 of 32 blocks of 782,
// choice included, 54.0 us, 53.5 with one part). One FP32 query, 8 heads x 50,000 rows (27 MB) 9.0 us, latency:
// a third of it before a block is there. 4,096 queries x 32 listed blocks, 570 MB
// through the L2s, 40 us, 14.3 TB/s, one wave to a query (vector unit 57% busy,
// matrix cores 33%, one or the other 75%); 8 queries x 64 listed blocks 8.8 us in
// sixteen.
template <typename T, bool LISTED, bool SPLIT, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 4) void icl4_one_kernel(AttendArgs p) {
    __shared__ __attribute__((aligned(16))) float red_o[WAVES][64];
    static_assert(__alignof__(red_o) >= alignof(f32x4), "read and written in fours");
    __shared__ float red_m[WAVES], red_l[WAVES];
    __shared__ __attribute__((aligned(16))) _Float16 shared_weights[WAVES][2][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int g = lane >> 4, i16 = lane & 15;
    // Workgroups of one XCD (every eighth) take consecutive queries of a pair, whose blocks then share its L2.
    const unsigned id = (blockIdx.x & 7u) * (unsigned)p.per_xcd + (blockIdx.x >> 3);
    if (id >= (unsigned)p.count) return;
    const int pq = SPLIT ? (int)divide(id, p.by_splits) : (int)id, split = SPLIT ? (int)(id - pq * p.by_splits.d) : 0;
    const int pair = (int)divide(pq, p.by_queries), row = pq - pair * p.q_rows;
    const int e = (int)divide(pair, p.by_heads), head = pair - e * p.heads;
    const int rows = rows_of(p.lengths, e, p.rows);
    _Float16 *weights = shared_weights[wave][0];
    i32x8 digits;
    float c;
    {
        // Terms 16 g .. and 64 + 16 g .. stand in lane (g, .): dims 16 (g / 2) .. and 32 more, digit 2 (i16 % 4) + g % 2.
        // Every fourth lane of a row makes a part: dims 4 (i16 / 4) .. +3 of both.
        const T *src = static_cast<const T *>(p.q) + e * p.q_est + head * p.q_head + (long long)row * p.q_row +
                       16 * (g >> 1) + 4 * (i16 >> 2);
        typedef T T4 __attribute__((ext_vector_type(4)));
        const T4 v[2] = {*reinterpret_cast<const T4 *>(src), *reinterpret_cast<const T4 *>(src + 32)};
        float x[8];
        float m = 0.f;
        bool finite = true;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = (float)v[i >> 2][i & 3];
            m = fmaxf(m, fabsf(x[i]));
            finite = finite && fabsf(x[i]) <= 3.4028235e38f;
        }
        m = fmaxf(m, __uint_as_float(row_xor<4>(__float_as_uint(m))));
        m = fmaxf(m, __uint_as_float(row_xor<8>(__float_as_uint(m))));
        m = halves_max(m);
        // The largest into [2^29, 2^30).
        const int ex = 30 - binade(m);
        c = __all(finite) ? factor(p, -ex) : NAN;
        const int digit = 2 * (i16 & 3) + (g & 1), sh = 28 - 4 * digit;
        const float first = g & 1 ? 1.0f : 16.0f;
        unsigned *words = reinterpret_cast<unsigned *>(weights);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int whole = (int)fminf(fmaxf(rintf(__builtin_ldexpf(x[4 * n + i], ex)), -1073741824.f), 1073741824.f);
                y[i] = (float)(digit ? (whole >> sh) & 15 : whole >> 28) * first;
            }
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
            w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
            words[(4 * g + (i16 & 3)) * 4 + (i16 >> 2)] = (unsigned)w;
            __builtin_amdgcn_wave_barrier();  // the wave's own LDS operations run in order
            const u32x4 all = *reinterpret_cast<const u32x4 *>(words + (4 * g + (i16 & 3)) * 4);
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < 4; ++i) digits[4 * n + i] = (int)all[i];
        }
    }
    // Exponent bytes of row i16 in the products of the four sixteens: 16^(6 - 2 (i16 % 4)) in its own.
    const int digit_exps = (127 + 24 - 8 * (i16 & 3)) << (8 * (i16 >> 2));
    f32x4 o[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float ref = -INFINITY, l_run = 0.f;
    const unsigned char *tiles = p.tiles + (long long)pair * p.blocks * kBlockBytes;
    const int *list = LISTED ? p.list + (long long)pq * p.n : nullptr;
    const int places = LISTED ? p.n : p.blocks;
    const int end = min(places, (split + 1) * p.per_split);
    // The lane's row of a block, and its weight's place: [step s][lanes g = 2 t + h][4 b + j].
    const int mine = 32 * (g >> 1) + 16 * (i16 >> 3) + 8 * (g & 1) + (i16 & 7);
    _Float16 *give = weights + 32 * (g >> 1) + 8 * (i16 >> 2) + 4 * (g & 1) + (i16 & 3);
    const _Float16 *get = weights + 64 * (i16 & 1) + 8 * g;
    const unsigned chunk_at = 16u * lane, ke_at = kKeyExpsAt + ((g >> 1) * 16 + i16) * 4, ve_at = kValueExpsAt + i16 * 8;

    u32x4 kw[2], vw[2];
    unsigned ke;
    u32x2 ve;
    auto load_keys = [&](const unsigned char *in) {
        kw[0] = *reinterpret_cast<const u32x4 *>(in + chunk_at);
        kw[1] = *reinterpret_cast<const u32x4 *>(in + 1024 + chunk_at);
        ke = *reinterpret_cast<const unsigned *>(in + ke_at);
    };
    auto load_values = [&](const unsigned char *in) {
        vw[0] = *reinterpret_cast<const u32x4 *>(in + kValuesAt + chunk_at);
        vw[1] = *reinterpret_cast<const u32x4 *>(in + kValuesAt + 1024 + chunk_at);
        ve = *reinterpret_cast<const u32x2 *>(in + ve_at);
    };
    // 64 of the wave's places at a time, one to a lane. A block's keys are loaded as soon as the one before has its
    // scores, its values once that one has its output.
    for (int at0 = split * p.per_split + wave; at0 < end; at0 += 64 * WAVES) {
        int block = at0 + WAVES * lane;
        unsigned long long mask = 0;
        if (block < end) {
            if (LISTED) block = list[block];
            if ((unsigned)block < (unsigned)p.blocks) mask = block_mask(p.keep, e, p.blocks, block, rows);
        }
        unsigned long long live = __ballot(mask != 0);
        if (!live) continue;
        const unsigned long long whole = __ballot(mask == ~0ull);
        const int low = (int)(unsigned)mask, high = (int)(unsigned)(mask >> 32);
        int i = __builtin_ctzll(live);
        const unsigned char *in = tiles + (long long)__builtin_amdgcn_readlane(block, i) * kBlockBytes;
        load_keys(in);
        load_values(in);
        for (;;) {
            const int now = i;
            live &= live - 1;
            if (live) {
                i = __builtin_ctzll(live);
                in = tiles + (long long)__builtin_amdgcn_readlane(block, i) * kBlockBytes;
            }
            f32x4 s = {0.f, 0.f, 0.f, 0.f};
            // Formats 0 (E4M3) and 4 (E2M1); the exponents are byte n of their words.
#define IRX_SCORES(n)                                                                                                       \
    {                                                                                                                       \
        const int w0 = (int)kw[n / 2][2 * (n % 2)], w1 = (int)kw[n / 2][2 * (n % 2) + 1];                                   \
        s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(digits, (i32x8{w0, w1, w0, w1, 0, 0, 0, 0}), s, 0, 4, n,       \
                                                             digit_exps, n, (int)ke);                                       \
    }
            IRX_SCORES(0)
            IRX_SCORES(1)
            IRX_SCORES(2)
            IRX_SCORES(3)
#undef IRX_SCORES
            if (live) load_keys(in);
            float x = product((s[0] + s[1]) + (s[2] + s[3]), c);
            if (!(whole >> now & 1)) {
                const unsigned long long m = (unsigned long long)(unsigned)__builtin_amdgcn_readlane(high, now) << 32 |
                                             (unsigned)__builtin_amdgcn_readlane(low, now);
                if (!((m >> mine) & 1)) x = -INFINITY;
            }
            float weight = __builtin_amdgcn_exp2f(x - ref);
            if (__any(!(weight <= 32768.0f))) {
                const float ref_new = fmaxf(ref, reference(wave_max(x), kHeadroom));
                const float alpha = __builtin_amdgcn_exp2f(ref - ref_new);
                l_run *= alpha;
#pragma unroll
                for (int d = 0; d < 4; ++d) o[d] *= alpha;
                ref = ref_new;
                weight = __builtin_amdgcn_exp2f(x - ref);
            }
            l_run += weight;
            const _Float16 hi = (_Float16)weight;
            give[0] = hi;
            give[64] = (_Float16)(weight - (float)hi);
            __builtin_amdgcn_wave_barrier();  // the wave's own LDS operations run in order
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                const half8 w = *reinterpret_cast<const half8 *>(get + 32 * st);
                o[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(vw[st][0], scale_byte<0>(ve[st])), w, o[0], 0, 0, 0);
                o[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(vw[st][1], scale_byte<1>(ve[st])), w, o[1], 0, 0, 0);
                o[2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(vw[st][2], scale_byte<2>(ve[st])), w, o[2], 0, 0, 0);
                o[3] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(vw[st][3], scale_byte<3>(ve[st])), w, o[3], 0, 0, 0);
            }
            if (!live) break;
            load_values(in);
        }
    }
    // Register r of o[d]: dim 16 d + 4 g + r, in every column (pair of columns).
    l_run = wave_sum(l_run);
    if (lane == 0) red_m[wave] = ref, red_l[wave] = l_run;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        f32x4 v = o[d];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += next_lane(v[r]);
        if (i16 == 0) *reinterpret_cast<f32x4 *>(&red_o[wave][16 * d + 4 * g]) = v;
    }
    __syncthreads();
    if (threadIdx.x >= 16) return;
    const int d = 4 * threadIdx.x;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) mx = fmaxf(mx, red_m[w]);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float den = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const float a = mx > -INFINITY ? __builtin_amdgcn_exp2f(red_m[w] - mx) : 1.0f;
        acc += a * *reinterpret_cast<const f32x4 *>(&red_o[w][d]);
        den += a * red_l[w];
    }
    if (den != 0.f) acc *= 1.0f / den;
    if constexpr (SPLIT) {
        const long long all = (long long)p.pairs * p.q_rows;
        store_part(p, all, split * all + pq, d, acc, mx, den);
    } else {
        store_out<T>(p, e, head, row, d, acc);
        if (p.lse && d == 0) p.lse[pq] = (mx + log2f(den)) * kLn2;
    }
}

// Splits' outputs weighted by their sums. 16 lanes of four dims each take a
// (pair, query) and every GROUPS-th split; a workgroup holds 16 / GROUPS rows.
// 3.4 to 5 us, the latency of one trip to memory and of a launch.
template <typename T, int GROUPS>
__global__ __launch_bounds__(256) void icl4_merge_kernel(AttendArgs p) {
    __shared__ __attribute__((aligned(16))) float sums[GROUPS > 1 ? 16 * 66 : 1];
    static_assert(__alignof__(sums) >= alignof(f32x2), "read and written in pairs");
    const long long all = p.part_rows;
    const int tid = threadIdx.x, slot = tid >> 4, group = slot % GROUPS, d = 4 * (tid & 15);
    const long long mine = (long long)blockIdx.x * (16 / GROUPS) + slot / GROUPS;
    const long long at_row = min(mine, all - 1);
    const float *sum_of = p.partial + p.splits * all * 64 + 2 * at_row;  // reference and sum
    const float *part = p.partial + at_row * 64 + d;
    // Eight splits' loads at once; slots past the last read it again and weigh nothing.
    float ref = -INFINITY, den = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = group; s0 < p.splits; s0 += 8 * GROUPS) {
        f32x2 l[8];
        f32x4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int s = s0 + i * GROUPS, at = min(s, p.splits - 1);
            l[i] = *reinterpret_cast<const f32x2 *>(sum_of + 2 * at * all);
            v[i] = *reinterpret_cast<const f32x4 *>(part + at * all * 64);
            if (s >= p.splits) l[i] = f32x2{-INFINITY, 0.f}, v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        float top = ref;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, l[i][0]);
        const float base = top > -INFINITY ? top : 0.f;
        const float a = __builtin_amdgcn_exp2f(ref - base);
        acc *= a, den *= a;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float w = __builtin_amdgcn_exp2f(l[i][0] - base) * l[i][1];
            acc += w * v[i];
            den += w;
        }
        ref = top;
    }
    if constexpr (GROUPS > 1) {
        *reinterpret_cast<f32x2 *>(&sums[slot * 66 + d]) = f32x2{acc[0], acc[1]};
        *reinterpret_cast<f32x2 *>(&sums[slot * 66 + d + 2]) = f32x2{acc[2], acc[3]};
        if (d == 0) sums[slot * 66 + 64] = ref, sums[slot * 66 + 65] = den;
        __syncthreads();
        if (group) return;
        float top = ref;
#pragma unroll
        for (int i = 1; i < GROUPS; ++i) top = fmaxf(top, sums[(slot + i) * 66 + 64]);
        const float base = top > -INFINITY ? top : 0.f;
        acc = f32x4{0.f, 0.f, 0.f, 0.f}, den = 0.f;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            const float *of = sums + (slot + i) * 66;
            const float a = __builtin_amdgcn_exp2f(of[64] - base);
            acc += a * f32x4{of[d], of[d + 1], of[d + 2], of[d + 3]};
            den += a * of[65];
        }
        ref = top;
    }
    if (mine >= all) return;
    int pair, row;
    if (p.unit_rows) {
        // A unit's rows, some past the last query.
        const unsigned of = (unsigned)mine, shift = p.unit_rows == 64 ? 6 : 5;
        const int unit = p.whole + (int)(of >> shift);
        pair = (int)divide(unit, p.by_qtiles);
        row = (unit - pair * (int)p.by_qtiles.d) * p.unit_rows + (int)(of & (p.unit_rows - 1u));
        if (row >= p.q_rows) return;
    } else {
        pair = (int)divide((unsigned)mine, p.by_queries), row = (int)mine - pair * p.q_rows;
    }
    if (den != 0.f) acc *= 1.0f / den;
    const int e = (int)divide(pair, p.by_heads);
    store_out<T>(p, e, pair - e * p.heads, row, d, acc);
    // Nothing attended: log 0.
    if (p.lse && d == 0)
        p.lse[(long long)pair * p.q_rows + row] = ((ref > -INFINITY ? ref : 0.f) + log2f(den)) * kLn2;
}

struct Plan {
    int queries;  // of a workgroup: 1, 16, 32 or 64
    int waves;    // of a workgroup of one query: 1, 4 or 16
    int qtiles, splits, per_split;
    long long rows;       // (pair, query) rows
    long long whole;      // 32 or 64 queries: units (query tile, pair) that are not split
    long long rest;       // and those that are
    long long part_rows;  // rows of a split's partials
};

// Queries up to which FP32 attention over every block takes a workgroup per query
// (1 x 200,000 rows x 8 heads 22.1 us against 27.0 with 16 to a workgroup, 2
// 25.9 against 27.4, 3 36.4 against 27.1; FP16, which takes one product where
// FP32 takes two, 48.5 against 46.2 at 1 x 200,000 x 16).
constexpr int kOneQueries = 2;
// Up to 16, FP32 or FP16, take the 16-query form in splits: 16 x 50,000 x 8 14.5
// against 19.1 us in the wide one. (32 queries as two such tiles 18.9 against
// 20.6, but 73.6 against 57.5 at 200,000 x 16; 33 x 1,024 x 16 7.2 against 8.9,
// with a second launch.)
constexpr int kRowQueries = 16;
// Blocks, four to a tile, that they take without splits and a merge: 1 x 1,024
// rows 5.4 against 6.7 us, 16 x 1,024 6.8 against 6.9; 16 x 2,000 10.4 against 7.0.
constexpr int kWholeTiles = 4;
// Queries per compute unit from which a query with listed blocks takes one wave,
// up to the 64 blocks that its lanes hold at once (4,096 queries of 8 blocks 28.5
// against 33.8 us with four waves, of 32 52.0 against 55.2, of 64 85.7 against
// 87.0; of 128 151 against 148; 2,048 of 32 blocks 39.4 against 38.0).
constexpr int kManyQueries = 16;
// Waves that take a query's listed blocks unsplit where queries are few.
constexpr int kManyWaves = 16;

// About two workgroups per compute unit, at least four blocks to a split (one to
// a wave). Listed blocks of queries that do not fill the compute units: a
// compute unit reads a block in about 1/16 us whatever its waves, so sixteen
// waves to a query and no merge where its busiest unit has at most 64 blocks (4
// us, a merge with its launch) more than in splits of four waves: 8 queries of
// 64 blocks of 3,125 17.7 against 16.2 us in a graph and two launches against
// one, of 256 30.0 against 17.9; 256 of 256 34.9 against 43.3, 304 of 256 53.8
// against 46.9. Attention over every block: above 16 queries a workgroup takes
// 32, three to a compute unit (168 registers), or 64, two (256): FP16 queries 64
// where that makes a whole round of workgroups (10,007 queries x 10,007 rows 237
// against 248 us; 777 x 12,345 x 2 estimators, 208 workgroups, 70.3 against
// 68.2), FP32 ones, whose pairs do not fit 256 registers beside 64 queries'
// scores, never (512 x 50,000 111 against 106.6 us).
Plan plan_attend(const Icl4Shape &s, bool half, int q_rows, int n_blocks, int compute_units) {
    Plan pl{};
    const int places = n_blocks ? n_blocks : s.blocks();
    const bool full = half && (long long)s.pairs() * ceil_div(q_rows, 64) >= 2LL * compute_units;
    pl.queries = n_blocks || (!half && q_rows <= kOneQueries) ? 1 : q_rows <= kRowQueries ? 16 : full ? 64 : 32;
    pl.qtiles = (int)ceil_div(q_rows, pl.queries);
    pl.rows = pl.part_rows = (long long)s.pairs() * q_rows;
    pl.waves = kWaves;
    const long long base = (long long)s.pairs() * pl.qtiles;
    const long long slots = (pl.queries == 32 ? 3LL : 2LL) * compute_units, tiles = ceil_div(places, kWaves);
    long long splits = 1;
    if (pl.queries <= 16) {
        if (n_blocks || tiles > kWholeTiles) splits = std::min(std::max(1LL, (slots + base - 1) / base), tiles);
        if (n_blocks && base >= (long long)kManyQueries * compute_units && n_blocks <= 64) {
            pl.waves = 1;
        } else if (n_blocks && splits > 1) {
            const auto of_unit = [&](long long workgroups) { return (workgroups + compute_units - 1) / compute_units; };
            const long long share = (tiles + splits - 1) / splits * kWaves;
            if (of_unit(base) * n_blocks <= of_unit(base * splits) * share + 64) pl.waves = kManyWaves, splits = 1;
        }
    } else {
        // Whole rounds of workgroups take every block; the units left over are split where that is quicker.
        // Microseconds: a workgroup's start and end, each round of its waves' blocks with one, two or three
        // workgroups on a compute unit, the merge with its launch. (16 units of 16 blocks, 33 queries: 15.1 us unsplit,
        // 18.0 in four; 400 units of 193 blocks, FP16 and masked, 63.2 unsplit, 77.0, 67.9 and 73.9 in two to four;
        // 128 of 782 blocks, FP32, 252, 132, 121, 102, 114, 101 and, in eight, 103.)
        static const double round32[2][3] = {{1.3, 1.85, 2.65}, {1.05, 1.2, 1.75}}, round64[2] = {1.6, 2.2};
        const auto round = [&](long long groups) {  // of up to `slots` workgroups
            const int k = (int)((groups + compute_units - 1) / compute_units) - 1;
            return pl.queries == 32 ? round32[half][k] : round64[k];
        };
        pl.whole = base / slots * slots / 8 * 8, pl.rest = base - pl.whole;
        double best = 1e30;
        for (long long n = 1; pl.rest && n <= std::min(tiles, std::max(8LL, 2 * slots / pl.rest)); ++n) {
            const long long rounds = pl.rest * n / slots, last = pl.rest * n - rounds * slots;
            const double share = (double)((tiles + n - 1) / n);
            double cost = (double)rounds * (6.0 + round(slots) * share) + (last ? 6.0 + round(last) * share : 0.0);
            if (n > 1) cost += 7.0 + (double)pl.rest * pl.queries * (double)n * (520.0 / 4e6);
            if (cost < best) best = cost, splits = n;
        }
        pl.part_rows = pl.rest * pl.queries;
    }
    pl.per_split = (int)((tiles + splits - 1) / splits) * kWaves;
    pl.splits = (int)ceil_div(places, pl.per_split);
    return pl;
}

// How blocks are chosen: in one launch up to 512 blocks, and up to 960 where 16
// queries to a workgroup come to 128 workgroups (512 blocks, 256 queries 15.8 us
// in one launch, with attention over 16 of them, 14.3 in two, 1,024 19.5 and
// 20.6; 782 blocks, 512 queries 21.8 and 17.5, 1,024 24.4 and 22.3, 2,048 30.4
// and 33.0: few workgroups are slow to read so many bounds); else scores first,
// then choices, in turns of at most 64 MiB of scores (or one query's): whole
// pairs, or a part of one pair's queries. (One launch with a workgroup to a
// query took 24 us for 8 queries of 3,125 blocks, a compute unit alone being
// slow to read 400 KB, where scores and choice apart take 3.8 and 6.5.)
struct SelectPlan {
    bool fused;
    long long padded;
    int pairs, rows;  // of a turn
};
SelectPlan plan_select(const Icl4Shape &s, int q_rows) {
    SelectPlan t{};
    t.padded = (s.blocks() + 63) / 64 * 64;
    t.fused = s.blocks() <= 512 || (s.blocks() <= kWavePicks && (long long)s.pairs() * ceil_div(q_rows, 16) >= 128);
    if (t.fused) return t;
    const long long most = std::max<long long>(1, (16LL << 20) / t.padded);  // queries of a turn
    t.rows = (int)std::min<long long>(q_rows, most);
    t.pairs = t.rows < q_rows ? 1 : (int)std::min<long long>(s.pairs(), std::max<long long>(1, most / q_rows));
    return t;
}

struct Parts {
    unsigned char *tiles;
    signed char *bounds;
    float *scales;
};
Parts parts(const void *cache, const Icl4Shape &s) {
    unsigned char *p = static_cast<unsigned char *>(const_cast<void *>(cache));
    const size_t blocks = (size_t)s.pairs() * s.blocks();
    return {p, reinterpret_cast<signed char *>(p + blocks * kBlockBytes),
            reinterpret_cast<float *>(p + blocks * (kBlockBytes + 128))};
}

// FP16 queries never ask for it.
template <typename T>
void launch_one_over_all(bool split, dim3 grid, dim3 wg, hipStream_t stream, const AttendArgs &p) {
    if constexpr (sizeof(T) == 4) {
        if (split)
            hipLaunchKernelGGL((icl4_one_kernel<T, false, true, kWaves>), grid, wg, 0, stream, p);
        else
            hipLaunchKernelGGL((icl4_one_kernel<T, false, false, kWaves>), grid, wg, 0, stream, p);
    }
}

template <typename T>
void attend(const Icl4Queries &a, const Icl4Attend &b, hipStream_t stream) {
    const Icl4Shape &s = a.shape;
    const Plan pl = plan_attend(s, a.half, a.q_rows, b.list ? b.n : 0, a.compute_units);
    AttendArgs p{};
    p.q = a.q, p.q_est = a.q_strides[0], p.q_head = a.q_strides[1], p.q_row = a.q_strides[2];
    p.o = b.out, p.o_est = b.o_strides[0], p.o_head = b.o_strides[1], p.o_row = b.o_strides[2];
    p.lse = b.lse, p.tiles = parts(a.cache, s).tiles, p.units = parts(a.cache, s).scales, p.lengths = a.lengths, p.keep = a.keep;
    p.list = b.list, p.n = b.n, p.heads = s.heads, p.pairs = s.pairs(), p.q_rows = a.q_rows, p.rows = s.rows;
    p.blocks = s.blocks(), p.scale = b.scale, p.partial = static_cast<float *>(b.workspace);
    p.splits = pl.splits, p.per_split = pl.per_split, p.qtiles = pl.qtiles;
    const bool wide = pl.queries > 16;
    const long long count = (wide ? pl.rest : (long long)pl.qtiles * s.pairs()) * pl.splits;
    p.count = (int)count, p.per_xcd = (int)ceil_div((size_t)count, 8);
    p.by_qtiles = division(pl.qtiles), p.by_splits = division(pl.splits), p.by_queries = division(a.q_rows);
    p.by_heads = division(s.heads), p.by_rest = division(std::max(1LL, pl.rest));
    p.whole = (int)pl.whole, p.unit_rows = wide ? pl.queries : 0, p.part_rows = pl.part_rows;
    const dim3 grid((unsigned)(pl.queries == 16 ? count : pl.whole + 8LL * p.per_xcd)), wg(kWaves * 64);
    {
        const long long tiles = b.list ? (long long)pl.rows * b.n : (long long)s.pairs() * s.blocks();
        const double work = 256.0 * kBlock * (b.list ? (double)tiles : (double)tiles * a.q_rows);
        KernelTimer timer(kFamIcl, stream, work, (double)tiles * kBlockBytes + 2.0 * sizeof(T) * 64 * pl.rows);
        const bool split = pl.splits > 1;
        if (b.list && pl.waves == kManyWaves)
            hipLaunchKernelGGL((icl4_one_kernel<T, true, false, kManyWaves>), grid, dim3(kManyWaves * 64), 0, stream, p);
        else if (b.list && pl.waves == 1)
            hipLaunchKernelGGL((icl4_one_kernel<T, true, false, 1>), grid, dim3(64), 0, stream, p);
        else if (b.list && split)
            hipLaunchKernelGGL((icl4_one_kernel<T, true, true, kWaves>), grid, wg, 0, stream, p);
        else if (b.list)
            hipLaunchKernelGGL((icl4_one_kernel<T, true, false, kWaves>), grid, wg, 0, stream, p);
        else if (pl.queries == 1)
            launch_one_over_all<T>(split, grid, wg, stream, p);
        else if (pl.queries == 16 && split)
            hipLaunchKernelGGL((icl4_rows_kernel<T, true>), grid, wg, 0, stream, p);
        else if (pl.queries == 16)
            hipLaunchKernelGGL((icl4_rows_kernel<T, false>), grid, wg, 0, stream, p);
        else if (pl.queries == 32)
            hipLaunchKernelGGL((icl4_wide_kernel<T, 1>), grid, wg, 0, stream, p);
        else if constexpr (sizeof(T) == 2)
            hipLaunchKernelGGL((icl4_wide_kernel<T, 2>), grid, wg, 0, stream, p);
        IRX_HIP(hipGetLastError());
    }
    if (pl.splits > 1) {
        KernelTimer timer(kFamIclMerge, stream, 0.0, 4.0 * pl.part_rows * (66.0 * pl.splits + 64.0));
        // A lane's splits come eight at a time: more groups where there are more splits (one group for 49 splits of 8
        // rows 4 us more than sixteen, for 32 of 128 rows 2.3 more than four).
        if (pl.splits <= 8)
            hipLaunchKernelGGL((icl4_merge_kernel<T, 1>), dim3(ceil_div((size_t)pl.part_rows, 16)), dim3(256), 0, stream, p);
        else if (pl.splits <= 32)
            hipLaunchKernelGGL((icl4_merge_kernel<T, 4>), dim3(ceil_div((size_t)pl.part_rows, 4)), dim3(256), 0, stream, p);
        else
            hipLaunchKernelGGL((icl4_merge_kernel<T, 16>), dim3((unsigned)pl.part_rows), dim3(256), 0, stream, p);
        IRX_HIP(hipGetLastError());
    }
}

}  // namespace

size_t icl4_bytes(const Icl4Shape &s) {
    return (size_t)s.pairs() * ((size_t)s.blocks() * (kBlockBytes + 128) + 64 * sizeof(float));
}

size_t icl4_attend_workspace(const Icl4Shape &s, bool half, int q_rows, int n_blocks, int compute_units) {
    const Plan pl = plan_attend(s, half, q_rows, n_blocks, compute_units);
    return pl.splits > 1 ? (size_t)pl.splits * (size_t)pl.part_rows * 66 * sizeof(float) : 0;
}

size_t icl4_select_workspace(const Icl4Shape &s, int q_rows) {
    const SelectPlan t = plan_select(s, q_rows);
    return t.fused ? 0 : (size_t)t.pairs * t.rows * t.padded * sizeof(int);
}

bool icl4_select_fits(const Icl4Shape &s, int q_rows) {
    return (double)s.pairs() * ceil_div(q_rows, 16) * (kChooseWaves * 64) < 4294967296.0;
}

bool icl4_grid_fits(const Icl4Shape &s, bool half, int q_rows, int n_blocks, int compute_units) {
    const Plan pl = plan_attend(s, half, q_rows, n_blocks, compute_units);
    const double units = pl.queries > 16 ? (double)pl.whole + (double)pl.rest * pl.splits : (double)pl.splits * pl.qtiles * s.pairs();
    return (units + 8) * pl.waves * 64 < 4294967296.0 && (double)pl.part_rows < 2147483648.0;
}

void icl4_encode(const Icl4Rows &a, void *cache, unsigned *nonfinite, hipStream_t stream) {
    const Icl4Shape &s = a.shape;
    const Parts c = parts(cache, s);
    StoreArgs p{};
    p.k = a.k, p.v = a.v, p.k_est = a.k_strides[0], p.k_head = a.k_strides[1], p.k_row = a.k_strides[2];
    p.v_est = a.v_strides[0], p.v_head = a.v_strides[1], p.v_row = a.v_strides[2];
    p.lengths = a.lengths, p.heads = s.heads, p.pairs = s.pairs(), p.rows = s.rows, p.blocks = s.blocks();
    p.tiles = c.tiles, p.bounds = c.bounds, p.scales = c.scales, p.nonfinite = nonfinite;
    const long long blocks = (long long)s.pairs() * s.blocks();
    KernelTimer timer(kFamGlue, stream, 0.0, 2.0 * s.pairs() * s.rows * 64 * (a.half ? 2 : 4) + (double)icl4_bytes(s));
    if (a.half)
        hipLaunchKernelGGL(icl4_encode_kernel<_Float16>, dim3((unsigned)blocks), dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL(icl4_encode_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, stream, p);
    IRX_HIP(hipGetLastError());
    if (s.blocks() <= kSmallBlocks) {
        hipLaunchKernelGGL(icl4_small_bounds_kernel, dim3(s.pairs()), dim3(1024), 0, stream, p);
        IRX_HIP(hipGetLastError());
        return;
    }
    hipLaunchKernelGGL(icl4_units_kernel, dim3(4 * s.pairs()), dim3(1024), 0, stream, p);
    IRX_HIP(hipGetLastError());
    hipLaunchKernelGGL(icl4_bounds_kernel, dim3(ceil_div((size_t)blocks, 4)), dim3(256), 0, stream, p);
    IRX_HIP(hipGetLastError());
}

void icl4_decode(const Icl4Rows &a, const void *cache, float *bounds, hipStream_t stream) {
    const Icl4Shape &s = a.shape;
    const Parts c = parts(cache, s);
    ReadArgs p{};
    p.k = a.k, p.v = a.v, p.k_est = a.k_strides[0], p.k_head = a.k_strides[1], p.k_row = a.k_strides[2];
    p.v_est = a.v_strides[0], p.v_head = a.v_strides[1], p.v_row = a.v_strides[2];
    p.lengths = a.lengths, p.heads = s.heads, p.pairs = s.pairs(), p.rows = s.rows, p.blocks = s.blocks();
    p.tiles = c.tiles, p.bounds = c.bounds, p.scales = c.scales, p.bounds_out = bounds;
    const long long blocks = (long long)s.pairs() * s.blocks();
    KernelTimer timer(kFamGlue, stream, 0.0, 2.0 * s.pairs() * s.rows * 64 * (a.half ? 2 : 4) + (double)icl4_bytes(s));
    if (a.half)
        hipLaunchKernelGGL(icl4_decode_kernel<_Float16>, dim3((unsigned)blocks), dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL(icl4_decode_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, stream, p);
    IRX_HIP(hipGetLastError());
}

template <typename T>
void choose(const Icl4Queries &a, int n, int *out, void *workspace, hipStream_t stream) {
    const Icl4Shape &s = a.shape;
    const Parts c = parts(a.cache, s);
    SelectArgs p{};
    p.q = a.q, p.q_est = a.q_strides[0], p.q_head = a.q_strides[1], p.q_row = a.q_strides[2];
    p.lengths = a.lengths, p.keep = a.keep, p.heads = s.heads, p.pairs = s.pairs(), p.q_rows = a.q_rows;
    p.rows = s.rows, p.blocks = s.blocks(), p.bounds = c.bounds, p.scales = c.scales, p.n = n, p.out = out;
    p.scores = static_cast<int *>(workspace);
    const SelectPlan t = plan_select(s, a.q_rows);
    p.padded = t.padded;
    KernelTimer timer(kFamIcl, stream, 256.0 * p.pairs * p.q_rows * p.blocks, 128.0 * p.pairs * p.blocks);
    const dim3 wg(kPickWaves * 64);
    if (t.fused) {
        const dim3 grid(ceil_div(p.q_rows, 16), (unsigned)s.heads, (unsigned)s.estimators), many(kChooseWaves * 64);
        const unsigned lds = (unsigned)(std::min(16, p.q_rows) * (t.padded + 4) * sizeof(int));
        if (t.padded <= 256)
            hipLaunchKernelGGL((icl4_choose_kernel<T, 1>), grid, many, lds, stream, p);
        else if (t.padded <= 512)
            hipLaunchKernelGGL((icl4_choose_kernel<T, 2>), grid, many, lds, stream, p);
        else
            hipLaunchKernelGGL((icl4_choose_kernel<T, 4>), grid, many, lds, stream, p);
        IRX_HIP(hipGetLastError());
        return;
    }
    for (p.pair0 = 0; p.pair0 < p.pairs; p.pair0 += t.pairs)
        for (p.row0 = 0; p.row0 < p.q_rows; p.row0 += t.rows) {
            const int pairs = std::min(t.pairs, p.pairs - p.pair0);
            p.rows_here = std::min(t.rows, p.q_rows - p.row0);
            p.qtiles = (int)ceil_div(p.rows_here, 16);
            // A wave takes 16 to 256 blocks: fewer where that leaves compute units idle (1 x 3,125 x 8: 16 each 3 us less
            // than 256; 512 x 3,125 x 8 19 us more).
            const long long tiles = (long long)pairs * p.qtiles;
            p.chunk = 256;
            while (p.chunk > 16 && tiles * ceil_div(p.blocks, 4 * p.chunk) < 2LL * a.compute_units) p.chunk /= 2;
            p.chunks = (int)ceil_div(p.blocks, 4 * p.chunk);
            const dim3 grid((unsigned)(tiles * p.chunks)), rows((unsigned)(pairs * p.rows_here));
            hipLaunchKernelGGL(icl4_scores_kernel<T>, grid, dim3(256), 0, stream, p);
            IRX_HIP(hipGetLastError());
            if (p.blocks <= kStagedPicks)
                hipLaunchKernelGGL(icl4_pick_kernel<true>, rows, wg, (unsigned)p.padded * sizeof(int), stream, p);
            else
                hipLaunchKernelGGL(icl4_pick_kernel<false>, rows, wg, 0, stream, p);
            IRX_HIP(hipGetLastError());
        }
}

void icl4_select(const Icl4Queries &a, int n, int *out, void *workspace, hipStream_t stream) {
    if (a.half)
        choose<_Float16>(a, n, out, workspace, stream);
    else
        choose<float>(a, n, out, workspace, stream);
}

void icl4_attend(const Icl4Queries &a, const Icl4Attend &b, hipStream_t stream) {
    if (a.half)
        attend<_Float16>(a, b, stream);
    else
        attend<float>(a, b, stream);
}

}  // namespace irx
