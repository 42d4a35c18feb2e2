// mlq_imma.cuh -- quantized products on the int8 matrix instructions, shared
// by the experts' products and the linear with an epilogue (sm_100a).
//
// The mathematics.  A weight block is d * c (+ m) with integer codes c, so
// the sum over one 32-value block is d * sum_i c_i x_i (+ m * sum_i x_i).
// Activations are carried as 24-bit block fixed point: for each 32-value
// block of a row of x a power of two s with
//     x_i = s * (65536 hi_i + 256 mid_i + lo_i),   hi, mid, lo in [-128, 127],
// rounded once (|error| <= s / 2 <= 2^-23 max|x_block|, at most one bit more
// than the rounding of fp32 itself).  The codes meet the three digits in
// m16n8k32 int8 matrix instructions -- one instruction covers exactly one
// block of 16 weight rows, and every integer sum in it is exact -- and are
// folded once per block in fp32 with d * s.
//
// Why this form: weights are read once and need no conversion (q8_0 codes are
// the operand, q4 codes take 3 instructions per 8 weights), so a warp issues
// ~30 instructions per 512 weights and the kernel is bound by HBM for up to
// ~8 rows of x per matrix.  The instruction runs at 1 per 2.2 cycles and SM
// here (1.05 POP/s measured).
#pragma once

#include <limits.h>

#include "mlq_device.cuh"
#include "mlq_kernels.h"

namespace mlq {

constexpr int kDigitBytes = 96;    // one sliced block: 3 digits x 32 values
constexpr int kChunkBlocks = 8;    // blocks of one K step of a warp
constexpr int kImmaWarps = 8;      // warps of a CTA
constexpr int kSegTokens = 32;     // rows of x (tokens) of a segment at most

__host__ __device__ inline int padded_blocks(int bpr) { return (bpr + kChunkBlocks - 1) / kChunkBlocks * kChunkBlocks; }

// A group of rows of x that meet the same matrix of a stack.
struct Segment {
    int expert;  // matrix of the stack
    int start;   // first position in the expert-sorted list of pairs
    int count;   // 1..kSegTokens
    int pad;
};

// Element of a block at position l (0..31) of the matrix instruction's K
// axis: l = 16 h + 4 t + j is byte j of operand register h of the lanes
// t mod 4.  The order follows from reading a block as aligned 32-bit words;
// q8_0 and q4_0 blocks are 2 mod 4 bytes long, so even and odd blocks differ.
__device__ __forceinline__ int imma_element(int fmt, int odd, int l) {
    const int h = l >> 4, t = (l >> 2) & 3, j = l & 3;
    if (fmt == kQ8_0) {
        if (odd) return l;
        if (h == 0) return 2 + 4 * t + j;
        return t < 3 ? 18 + 4 * t + j : (j < 2 ? j : 28 + j);
    }
    if (fmt == kQ4_0 && !odd) return 16 * h + (t < 3 ? 2 + 4 * t + j : (j < 2 ? j : 12 + j));
    return l;
}

// Slices one block: lane l holds the value at K position l.  Writes 96
// digit bytes, the scale s and the block's sum.  A block with a value that
// is not finite gets the scale NaN: every output that reads it is NaN.
__device__ __forceinline__ void slice_block(float v, uint8_t* dig, float* scale, float* sum, int lane) {
    float amax = fabsf(v);
    const bool bad = !(amax <= 3.402823466e38f);
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const bool any_bad = __any_sync(0xffffffffu, bad);
    const int eb = (int)(__float_as_uint(amax) >> 23) & 0xff;
    int sf = 276 - eb;  // exponent field of 2^(22 - floor(log2 amax))
    if (sf > 253) sf = 253;
    if (amax * __uint_as_float((uint32_t)sf << 23) > 8355711.0f) --sf;  // 127 * 65793: three digits hold it
    int q = any_bad ? 0 : __float2int_rn(v * __uint_as_float((uint32_t)sf << 23));
    const int d0 = (int)(int8_t)(q & 0xff);
    const int q1 = (q - d0) >> 8;
    const int d1 = (int)(int8_t)(q1 & 0xff);
    const int d2 = (q1 - d1) >> 8;
    const int j = lane & 3;
    uint32_t w2 = (uint32_t)(d2 & 0xff) << (8 * j), w1 = (uint32_t)(d1 & 0xff) << (8 * j),
             w0 = (uint32_t)(d0 & 0xff) << (8 * j);
    for (int o = 1; o <= 2; o <<= 1) {
        w2 |= __shfl_xor_sync(0xffffffffu, w2, o);
        w1 |= __shfl_xor_sync(0xffffffffu, w1, o);
        w0 |= __shfl_xor_sync(0xffffffffu, w0, o);
    }
    const int h = lane >> 4, t = (lane >> 2) & 3;
    if (j < 3)  // lane j of each four stores digit j (0: hi, 1: mid, 2: lo)
        *reinterpret_cast<uint32_t*>(dig + j * 32 + t * 8 + h * 4) = j == 0 ? w2 : (j == 1 ? w1 : w0);
    const int s = __reduce_add_sync(0xffffffffu, q);  // |s| < 2^28
    if (lane == 0) {
        const float inv = any_bad ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)(254 - sf) << 23);
        *scale = inv;
        *sum = (float)s * inv;
    }
}

__device__ __forceinline__ void imma_s8(int (&c)[4], const uint32_t (&a)[4], uint2 b) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "r"(0));
}

// Facts of a warp's weight slot (16 rows x 8 blocks in shared memory).
// Aligned rows come by 2-D TMA boxes; the row pitch is 4 mod 8 words, so the
// 8 rows x 4 words that a warp reads at a time touch 32 banks (q4_1 takes two
// boxes of 4 blocks for that).  Other rows come by 16-byte copies of the
// aligned window around each row, in a pitch with the same property.
template <int F, bool ALN>
struct Slot;
template <>
struct Slot<kQ8_0, true> {
    static constexpr int kBoxes = 1, kBoxBytes = 272, kBytes = 16 * 272;
};
template <>
struct Slot<kQ4_0, true> {
    static constexpr int kBoxes = 1, kBoxBytes = 144, kBytes = 16 * 144;
};
template <>
struct Slot<kQ4_1, true> {
    static constexpr int kBoxes = 2, kBoxBytes = 80, kBytes = 2 * 16 * 80;
};
template <>
struct Slot<kQ8_0, false> {
    static constexpr int kPitch = 304, kBytes = 16 * 304;
};
template <>
struct Slot<kQ4_0, false> {
    static constexpr int kPitch = 176, kBytes = 16 * 176;
};
template <>
struct Slot<kQ4_1, false> {
    static constexpr int kPitch = 176, kBytes = 16 * 176;
};

__host__ __device__ constexpr int chunk_bytes(int f) { return kChunkBlocks * block_bytes(f); }

// Four bytes at any byte address of shared memory.
__device__ __forceinline__ uint32_t lds_any(uint32_t a) {
    const uint32_t lo = lds_u32(a & ~3u), hi = lds_u32((a & ~3u) + 4);
    return __funnelshift_r(lo, hi, 8 * (a & 3));
}

template <bool ALN>
__device__ __forceinline__ uint32_t lds_word(uint32_t a) {
    if (ALN) return lds_u32(a);
    return lds_any(a);
}

// One block of 16 weight rows as the matrix instruction's A operand, with
// the rows' scales (rows g and g + 8 of lane 4 g + t).
struct BlockA {
    uint32_t a[4];
    float d[2], m[2];
};

// q4 codes as signed bytes 16 * (c - 8): one shift and two masks for 8 codes.
__device__ __forceinline__ void nibbles(uint32_t v, uint32_t& lo, uint32_t& hi) {
    lo = ((v << 4) & 0xf0f0f0f0u) ^ 0x80808080u;
    hi = (v & 0xf0f0f0f0u) ^ 0x80808080u;
}

// Blocks 2p and 2p + 1 of the slot rows at r0 (row g) and r1 (row g + 8).
template <int F, bool ALN>
__device__ __forceinline__ void load_pair(uint32_t r0, uint32_t r1, int p, int t, BlockA& even, BlockA& odd) {
    const uint32_t r[2] = {r0, r1};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (F == kQ8_0) {
            const uint32_t b = r[i] + 68 * p;
            const uint32_t w0 = lds_word<ALN>(b), w8 = lds_word<ALN>(b + 32);
            even.a[i] = lds_word<ALN>(b + 4 + 4 * t);
            const uint32_t e1 = lds_word<ALN>(b + 20 + 4 * t);
            even.a[2 + i] = t == 3 ? __byte_perm(w0, w8, 0x5432) : e1;
            odd.a[i] = lds_word<ALN>(b + 36 + 4 * t);
            odd.a[2 + i] = lds_word<ALN>(b + 52 + 4 * t);
            even.d[i] = half_bits_to_float(w0 & 0xffffu);
            odd.d[i] = half_bits_to_float(w8 >> 16);
        } else if (F == kQ4_0) {
            const uint32_t b = r[i] + 36 * p;
            const uint32_t w0 = lds_word<ALN>(b), w4 = lds_word<ALN>(b + 16);
            const uint32_t e = lds_word<ALN>(b + 4 + 4 * t);
            nibbles(t == 3 ? __byte_perm(w0, w4, 0x5432) : e, even.a[i], even.a[2 + i]);
            nibbles(lds_word<ALN>(b + 20 + 4 * t), odd.a[i], odd.a[2 + i]);
            even.d[i] = half_bits_to_float(w0 & 0xffffu);
            odd.d[i] = half_bits_to_float(w4 >> 16);
        } else {
            // aligned: blocks 0..3 in the first box, 4..7 in the second
            const uint32_t b = ALN ? r[i] + (p >> 1) * (16 * 80) + (p & 1) * 40 : r[i] + 40 * p;
            const uint32_t w0 = lds_word<ALN>(b), w5 = lds_word<ALN>(b + 20);
            nibbles(lds_word<ALN>(b + 4 + 4 * t), even.a[i], even.a[2 + i]);
            nibbles(lds_word<ALN>(b + 24 + 4 * t), odd.a[i], odd.a[2 + i]);
            even.d[i] = half_bits_to_float(w0 & 0xffffu);
            even.m[i] = fmaf(8.0f, even.d[i], half_bits_to_float(w0 >> 16));  // d c + m = d (c - 8) + (m + 8 d)
            odd.d[i] = half_bits_to_float(w5 & 0xffffu);
            odd.m[i] = fmaf(8.0f, odd.d[i], half_bits_to_float(w5 >> 16));
        }
    }
}

}  // namespace mlq
