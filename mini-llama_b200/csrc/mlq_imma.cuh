// mlq_imma.cuh -- quantized products on the matrix instructions: the
// arithmetic that the experts' products and the linear with an epilogue share (sm_100a).
//
// The mathematics.  A weight block is d * c (+ m) with integer codes c, so
// the sum over one 32-value block is d * sum_i c_i x_i (+ m * sum_i x_i).
// c_i is exact in 8 bits, and x is cut into pieces:
//
// * few rows of x (segments of up to 4): 4 signed base-256 digits of x_i / s, s a power of two
//   per 32-value block of a row (31-bit fixed point, error <= 2^-31
//   max|x_block|; below 2^-96 a fixed step of 2^-126).  The codes meet the digits in m16n8k32 int8 matrix
//   instructions: one covers exactly one block of 16 weight rows, its 8 columns are
//   the digits of 2 rows of x, every integer sum is exact, and one fp32 fold per
//   block (its sum rounded to fp32) applies d and the block's scale of x.  fp32 sums go over
//   8 blocks, then over those.  q8_0 codes are
//   the operand as they are.  q4 codes are bytes 16 c (a mask for the high
//   nibbles, a shift and a mask for the low ones): unsigned in q4_1, in q4_0 signed 16 (c - 8),
//   which is the same byte with its highest bit changed, so that a weight of 0 adds
//   exactly nothing however large its x is.  q4_1's two parts, d sum(c x) and m sum(x), cancel
//   each other where a weight is near 0, so the sums of x's digits are integers too and meet
//   the other part in fused steps that round only what is left (FewRows::step).
// * more rows: x_i / s = hi + lo in fp16 (error <= 2^-22 |x_i|, s a power of
//   two per 64 values of a row), and d c too (exact: at most 19 bits; q4_1's
//   d c + m to 22 bits), with a power of two per 64 values of a weight row.  tcgen05
//   products hi hi + hi lo + lo hi, 64 values of K at a time into a sum that both
//   scales then bring into an fp32 one: a product of 22 bits on both sides at 3
//   fp16 instructions, and the chain of roundings in the tensor core is short.
//
// Both are bound by HBM, past a launch's start and end, while an expert has few rows.  The int8 instruction
// runs at one per 2.2 cycles and SM here (1.05 POP/s measured).
#pragma once

#include <limits.h>

#include "mlq_device.cuh"
#include "mlq_kernels.h"

namespace mlq {

constexpr int kSlicedBytes = 128;  // one sliced block of x: 4 digits of 32 values
constexpr int kChunkBlocks = 8;    // blocks of one K step of a warp
constexpr int kImmaWarps = 8;      // warps of a CTA that compute
constexpr int kSegTokens = 128;    // rows of x of a segment at most
constexpr int kFewRows = 4;        // rows of x that go by digits

__host__ __device__ inline int padded_blocks(int bpr) { return (bpr + kChunkBlocks - 1) / kChunkBlocks * kChunkBlocks; }

// A group of rows of x that meet the same matrix of a stack.
struct Segment {
    int expert;  // matrix of the stack
    int start;   // first position in the expert-sorted list of pairs
    int count;   // 1..kSegTokens
    int pad;
};

// Element of a block at position l = 16 h + 4 t + j: byte j of the h-th word
// of codes that the lanes t mod 4 read (q4: h = 0 the low nibbles, 1 the high).
// The order follows from reading a block as aligned 32-bit words; q8_0 and
// q4_0 blocks are 2 mod 4 bytes long, so even and odd blocks differ.
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

// Element of a block at position p of the fp16 operands (many rows): the order
// in which a block's codes are turned to fp16 pairs (mlq_imma_many.cuh).
__device__ __forceinline__ int tile_element(int fmt, int p) {
    if (fmt == kQ8_0) return p;
    return (p >> 3) * 4 + ((p >> 2) & 1) + 2 * (p & 1) + 8 * (p & 2);
}

// A sliced row of x is a sequence of records, one per K step: 8 blocks of
// digits, their scales and, for q4_1, their sums of digits (block_sums).  One bulk
// copy brings a record to shared memory.
__host__ __device__ constexpr int record_bytes(int fmt) { return kChunkBlocks * (kSlicedBytes + (fmt == kQ4_1 ? 20 : 4)); }
constexpr int kRecordScales = kChunkBlocks * kSlicedBytes, kRecordSums = kRecordScales + kChunkBlocks * 4;

// Where block b of a record has its digits (see slice_digits).
__host__ __device__ constexpr int digit_block(int b) { return (b / 2) * 2 * kSlicedBytes + (b & 1) * 8; }

// And its sums of digits, for digits 3, 2 or 1, 0 (odd): two floats, of the
// higher digit and of the lower one, in the unit of a sum of codes 16 c with
// digits.  Two blocks share 32 bytes, [odd][block of the pair].
__host__ __device__ constexpr int block_sums(int b, int odd) { return kRecordSums + (b / 2) * 32 + odd * 16 + (b & 1) * 8; }

// The power of two 2^k whose product with amax is in (limit / 2, limit], as
// bits; top: floor(log2 limit).  Clamped so that 2^-k is a normal number.
__device__ __forceinline__ uint32_t block_scale(float amax, int top, float limit) {
    const int eb = (int)(__float_as_uint(amax) >> 23) & 0xff;
    int sf = 254 + top - eb;  // exponent field of 2^(top - floor(log2 amax))
    if (sf > 253) sf = 253;
    if (amax * __uint_as_float((uint32_t)sf << 23) > limit) --sf;
    return (uint32_t)sf << 23;
}

__device__ __forceinline__ float inverse_scale(uint32_t scale) { return __uint_as_float((254u << 23) - scale); }

// Largest magnitude of a block (lanes hold its values); NaN if one is not finite.
__device__ __forceinline__ float block_amax(float v) {
    float amax = fabsf(v);
    const bool bad = __any_sync(0xffffffffu, !(amax <= 3.402823466e38f));
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    return bad ? __uint_as_float(0x7fc00000u) : amax;
}

// Slices a block into digits: lane l holds the value at imma_element l.  Two
// blocks share 256 bytes, [digit][t][block of the pair][word h].  A block with a
// value that is not finite gets the scale NaN: every output that reads it is NaN.
// row: the row's first record, of format fmt; b: the block.
__device__ __forceinline__ void slice_digits(float x, int fmt, uint8_t* row, int b, int lane) {
    row += (size_t)(b / kChunkBlocks) * record_bytes(fmt);
    b %= kChunkBlocks;
    const float amax = block_amax(x);
    const bool bad = !(amax == amax);
    const uint32_t s = block_scale(bad ? 0.0f : amax, 30, 2139062016.0f);  // below 127 * 16843009: four digits hold it
    const int q = bad ? 0 : __float2int_rn(x * __uint_as_float(s));
    const int d0 = (int)(int8_t)(q & 0xff);
    const int q1 = (q - d0) >> 8;
    const int d1 = (int)(int8_t)(q1 & 0xff);
    const int q2 = (q1 - d1) >> 8;
    const int d2 = (int)(int8_t)(q2 & 0xff);
    const int d3 = (q2 - d2) >> 8;
    // 4x4 byte transpose among the 4 lanes of a word: lane j stores digit j (0: the highest) of all four
    const int j = lane & 3;
    const uint32_t w = (uint32_t)(d3 & 0xff) | (uint32_t)(d2 & 0xff) << 8 | (uint32_t)(d1 & 0xff) << 16 |
                       (uint32_t)(d0 & 0xff) << 24;
    uint32_t out = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t from = __shfl_sync(0xffffffffu, w, (lane & ~3) + k);
        out |= ((from >> (8 * j)) & 0xffu) << (8 * k);
    }
    const int h = lane >> 4, t = (lane >> 2) & 3;
    *reinterpret_cast<uint32_t*>(row + digit_block(b) + j * 64 + t * 16 + h * 4) = out;
    if (lane == 0) reinterpret_cast<float*>(row + kRecordScales)[b] = bad ? __uint_as_float(0x7fc00000u) : inverse_scale(s);
    if (fmt == kQ4_1) {
        // |sum of 32 digits| <= 4096: two sums in a word
        const int high = __reduce_add_sync(0xffffffffu, d3 * 65536 + d2), low = __reduce_add_sync(0xffffffffu, d1 * 65536 + d0);
        if (lane < 2) {
            const int both = lane == 0 ? high : low, second = (int)(int16_t)(both & 0xffff), first = (both - second) >> 16;
            float* at = reinterpret_cast<float*>(row + block_sums(b, lane));
            at[0] = (float)first * 4096.0f, at[1] = (float)second * 16.0f;
        }
    }
}

// 64 values (positions 2 lane and 2 lane + 1) as fp16 hi and lo with one
// power-of-two scale.
struct Sliced64 {
    __half2 hi, lo;
    float scale;
    // to: 64 hi, then 64 lo
    __device__ __forceinline__ void store(uint8_t* to, float* to_scale, int lane) const {
        reinterpret_cast<__half2*>(to)[lane] = hi;
        reinterpret_cast<__half2*>(to + 128)[lane] = lo;
        if (lane == 0) *to_scale = scale;
    }
};

__device__ __forceinline__ Sliced64 slice_64(float v0, float v1) {
    const float most = fmaxf(fabsf(v0), fabsf(v1));
    const float m = block_amax(v0 == v0 && v1 == v1 ? most : __uint_as_float(0x7fc00000u));
    const bool bad = !(m == m);
    const uint32_t s = block_scale(bad ? 0.0f : m, 14, 32767.0f);
    const float q0 = bad ? 0.0f : v0 * __uint_as_float(s), q1 = bad ? 0.0f : v1 * __uint_as_float(s);
    Sliced64 r;
    r.hi = __floats2half2_rn(q0, q1);
    const float2 h = __half22float2(r.hi);
    r.lo = __floats2half2_rn(q0 - h.x, q1 - h.y);
    r.scale = bad ? __uint_as_float(0x7fc00000u) : inverse_scale(s);
    return r;
}

// D = A B for 16 rows x 32 codes, signed or unsigned (q4_1), and digits.
template <int F>
__device__ __forceinline__ void imma(int (&c)[4], const uint32_t (&a)[4], uint2 b) {
    if constexpr (F != kQ4_1)
        asm volatile(
            "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "r"(0));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "r"(0));
}

// Facts of a warp's weight slot (16 rows x 8 blocks in shared memory).
// Aligned rows come by 2-D TMA boxes; the row pitch is 4 mod 8 words, so the
// 8 rows x 4 words that a warp reads at a time touch 32 banks (q4_1 takes two
// boxes of 4 blocks for that).  Other rows come one by one, as the 16-byte
// aligned pieces (cp.async) of the window around each, in a pitch with the same property.
template <int F, bool ALN>
struct Slot;
template <>
struct Slot<kQ8_0, true> {
    static constexpr int kBoxes = 1, kPitch = 272, kBytes = 16 * 272;
};
template <>
struct Slot<kQ4_0, true> {
    static constexpr int kBoxes = 1, kPitch = 144, kBytes = 16 * 144;
};
template <>
struct Slot<kQ4_1, true> {
    static constexpr int kBoxes = 2, kPitch = 80, kBytes = 2 * 16 * 80;
};
template <>
struct Slot<kQ8_0, false> {
    static constexpr int kBoxes = 1, kPitch = 304, kBytes = 16 * 304;
};
template <>
struct Slot<kQ4_0, false> {
    static constexpr int kBoxes = 1, kPitch = 176, kBytes = 16 * 176;
};
template <>
struct Slot<kQ4_1, false> {
    static constexpr int kBoxes = 1, kPitch = 176, kBytes = 16 * 176;
};

__host__ __device__ constexpr int chunk_bytes(int f) { return kChunkBlocks * block_bytes(f); }

// The word OFF bytes after `a` in shared memory; a is 4-byte aligned where ALN.
template <bool ALN, int OFF>
__device__ __forceinline__ uint32_t lds_word(uint32_t a) {
    uint32_t lo;
    if constexpr (ALN) {
        asm volatile("ld.shared.u32 %0, [%1+%2];" : "=r"(lo) : "r"(a), "n"(OFF));
        return lo;
    } else {
        uint32_t hi;
        const uint32_t w = a & ~3u;
        asm volatile("ld.shared.u32 %0, [%1+%2];" : "=r"(lo) : "r"(w), "n"(OFF));
        asm volatile("ld.shared.u32 %0, [%1+%2];" : "=r"(hi) : "r"(w), "n"(OFF + 4));
        return __funnelshift_r(lo, hi, 8 * (a & 3));
    }
}

template <int OFF>
__device__ __forceinline__ uint4 lds_u4_at(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4+%5];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(a), "n"(OFF));
    return v;
}

template <int OFF>
__device__ __forceinline__ float lds_f1_at(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1+%2];" : "=f"(v) : "r"(a), "n"(OFF));
    return v;
}

template <int OFF>
__device__ __forceinline__ float4 lds_f4_at(uint32_t a) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4+%5];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(a), "n"(OFF));
    return v;
}

template <int OFF>
__device__ __forceinline__ float2 lds_f2_at(uint32_t a) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0,%1}, [%2+%3];" : "=f"(v.x), "=f"(v.y) : "r"(a), "n"(OFF));
    return v;
}

__device__ __forceinline__ float low_half(uint32_t w) {
    return __low2float(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float high_half(uint32_t w) {
    return __high2float(*reinterpret_cast<const __half2*>(&w));
}

// One block of 16 weight rows (rows g and g + 8 of lane 4 g + t): the lane's
// words of codes (q4: one word per row) and the rows' scales.
struct RawA {
    uint32_t w[2][2];  // [row][word]
    float d[2], m[2];
};

// Where a lane finds its rows' blocks: rows g and g + 8 of its slot.
struct RowBase {
    uint32_t row[2];   // the row
    uint32_t word[2];  // the row + 4 t
    uint32_t pick;     // byte selection: lanes t = 3 join a word from two (q8_0 and q4_0 even blocks)
};

__device__ __forceinline__ RowBase row_base(uint32_t r0, uint32_t r1, int t) {
    return RowBase{{r0, r1}, {r0 + 4 * t, r1 + 4 * t}, t == 3 ? 0x5432u : 0x7654u};
}

// Blocks 2 P and 2 P + 1 of the lane's rows.
template <int F, bool ALN, int P>
__device__ __forceinline__ void load_pair(const RowBase& r, RawA& even, RawA& odd) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (F == kQ8_0) {
            constexpr int b = 68 * P;
            const uint32_t w0 = lds_word<ALN, b>(r.row[i]), w8 = lds_word<ALN, b + 32>(r.row[i]);
            even.w[i][0] = lds_word<ALN, b + 4>(r.word[i]);
            // the last word: bytes of words 0 and 8 (what lane 3 has loaded), the others theirs
            even.w[i][1] = __byte_perm(w0, lds_word<ALN, b + 20>(r.word[i]), r.pick);
            odd.w[i][0] = lds_word<ALN, b + 36>(r.word[i]);
            odd.w[i][1] = lds_word<ALN, b + 52>(r.word[i]);
            even.d[i] = low_half(w0);
            odd.d[i] = high_half(w8);
        } else if constexpr (F == kQ4_0) {
            constexpr int b = 36 * P;
            const uint32_t w0 = lds_word<ALN, b>(r.row[i]), w4 = lds_word<ALN, b + 16>(r.row[i]);
            even.w[i][0] = __byte_perm(w0, lds_word<ALN, b + 4>(r.word[i]), r.pick);
            odd.w[i][0] = lds_word<ALN, b + 20>(r.word[i]);
            even.d[i] = low_half(w0);
            odd.d[i] = high_half(w4);
        } else {
            // aligned: blocks 0..3 in the first box, 4..7 in the second
            constexpr int b = ALN ? (P >> 1) * (16 * 80) + (P & 1) * 40 : 40 * P;
            const uint32_t w0 = lds_word<ALN, b>(r.row[i]), w5 = lds_word<ALN, b + 20>(r.row[i]);
            even.w[i][0] = lds_word<ALN, b + 4>(r.word[i]);
            odd.w[i][0] = lds_word<ALN, b + 24>(r.word[i]);
            even.d[i] = low_half(w0);
            even.m[i] = high_half(w0);
            odd.d[i] = low_half(w5);
            odd.m[i] = high_half(w5);
        }
    }
}

// The A operand of the int8 instruction.
template <int F>
__device__ __forceinline__ void int8_operand(const RawA& r, uint32_t (&a)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        constexpr uint32_t sign = F == kQ4_0 ? 0x80808080u : 0u;
        a[i] = F == kQ8_0 ? r.w[i][0] : (r.w[i][0] << 4 & 0xf0f0f0f0u) ^ sign;
        a[2 + i] = F == kQ8_0 ? r.w[i][1] : (r.w[i][0] & 0xf0f0f0f0u) ^ sign;
    }
}

}  // namespace mlq
