// Microscaled 4-bit floating point: tensor scale, packing, unpacking (formats and layout: include/vrb.h).
//
// All three are bound by HBM: packing reads 2 or 4 bytes an element and writes 0.5 + 1/16 (NVFP4) or 0.5 + 1/32
// (MXFP4), unpacking the reverse.  A thread owns 16 consecutive elements of a row: 32 bytes of bf16 in, 8 bytes of codes
// out, so a warp reads 1 KB and writes 256 bytes, both contiguous; the scale bytes of the four blocks that share a
// word of the scale tile are collected by shuffles and leave as one 4-byte store.
//
// Rounding is that of the real quotients a / (6 g) -> e4m3 and x / (g s) -> e2m1.  The fast form multiplies by an F32
// quotient (its 2 ulp and three roundings: relative error < 2^-21) and converts the product moved up and down by kGuard = 2^-20:
// where both give one code it is the right one.  Where they differ a rounding border t lies between.  With s g = hi + lo in F32
// (one product and one multiply-add, exact) |x| - t hi is exact next to the border and a multiply-add with -t lo rounds to the
// sign that decides; 0 is the tie.
//   bf16: one element decides for its block.  Elements next to borders have x / t within 2^-19 of s g, and two such quotients of
//   8-bit by 3-bit significands are equal or 2^-11 apart; so all of them are on the same side, and the block takes the codes of
//   the product moved up, or down, or, on a tie, the form below.  (bf16 data meets the borders of NVFP4 to within 2^-24 all the
//   time: the tensor scale is amax / (2^7 3 7), whose factors the scales 9, 12, 14 and 15 eighths share.)
//   F32: the eight elements are done again (refined8): a residual step gives the quotient y to within an F32 step, so y is on t's
//   right side unless it is t itself; then the sign above moves it off the border.
// 13824 x 5120 bf16 took 99 us with a search in double, and 51 to 76, by amax, with refined8 for both types.
#include "vrb_fp4.cuh"

namespace vrb {
namespace {

constexpr int kThreads = 256;
constexpr float kGuard = 9.5367431640625e-7f;   // 2^-20

// codes of 8 values, element 0 in the lowest nibble (e2m1: to nearest, ties to even, saturating)
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
__device__ __forceinline__ uint32_t e4m3_bits(float v) {   // to nearest, ties to even, saturating at 448
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(v));
    return r & 0xffu;
}
// value of a finite non-negative e4m3 code: 3 mantissa bits, bias 7
__device__ __forceinline__ float e4m3_value(uint32_t code) {
    const uint32_t e = code >> 3, m = code & 7u;
    return e ? __uint_as_float(((e + 120u) << 23) | (m << 20)) : static_cast<float>(m) * 0.001953125f;   // 2^-9
}
// Scale byte of an NVFP4 block with largest magnitude a: RN_e4m3(min(a / (6 g), 448))
__device__ __noinline__ uint32_t nv_scale_exact(float a, float g) {
    // the quotient in double keeps its side of every border: borders have 5 significant bits, 6 g has 27, so the quotient
    // is either on one or at least 2^-31 away
    const double q = static_cast<double>(a) / (6.0 * static_cast<double>(g));
    if (!(q < 448.0)) return 126u;
    uint32_t code = e4m3_bits(static_cast<float>(q));
    for (uint32_t c = code > 0 ? code - 1 : 0; c <= code && c < 126u; ++c) {   // border between c and c + 1
        const double border = 0.5 * (static_cast<double>(e4m3_value(c)) + static_cast<double>(e4m3_value(c + 1)));
        if (q < border || (q == border && (c & 1u) == 0u)) return c;
    }
    return code < 126u ? code + 1u : 126u;
}
// the border above the magnitude of an e2m1 code: .25 .75 1.25 1.75 2.5 3.5 5, in quarters a byte each
__device__ __forceinline__ float e2m1_border(uint32_t magnitude) {
    return 0.25f * static_cast<float>(__byte_perm(0x07050301u, 0x00140e0au, magnitude) & 0xffu);
}
// one element in double, for tensor scales outside the range of the F32 form
__device__ __noinline__ uint32_t e2m1_exact(float x, double unit) {
    const uint32_t sign = __float_as_uint(x) >> 31 << 3;
    const double a = fabs(static_cast<double>(x));
    uint32_t code = 0;
    for (; code < 7u; ++code) {
        const double border = 0.25 * static_cast<double>(0x140e0a0705030100ull >> (8u * code + 8u) & 0xffu) * unit;   // .25 .75 1.25 1.75 2.5 3.5 5
        if (a < border || (a == border && (code & 1u) == 0u)) break;
    }
    return sign | code;
}

template <typename T> struct Elements;
template <> struct Elements<uint16_t> {
    static constexpr int kChunk = 8;     // elements of a 16-byte chunk
    static constexpr int kWords = 8;     // words of 16 elements
    __device__ static __forceinline__ float value(uint16_t h) { return bf16_bits_to_float(h); }
};
template <> struct Elements<float> {
    static constexpr int kChunk = 4;
    static constexpr int kWords = 16;
    __device__ static __forceinline__ float value(float f) { return f; }
};

// The words of elements [column, column + 16) of a row of k, zero past the end.  VEC: rows of whole 16-byte chunks on 16-byte boundaries.  Otherwise the 16 elements are cut out of the aligned
// chunks around them by a shift of whole words and, bf16, of half a word; at the tensor's ends element by element.
template <typename T, bool VEC>
__device__ __forceinline__ void load16(const T* x, int64_t count, const T* at, int64_t column, int64_t k, uint32_t (&w)[Elements<T>::kWords]) {
    constexpr int W = Elements<T>::kWords;
    const int live = k - column < 16 ? static_cast<int>(k - column) : 16;
    if constexpr (VEC) {
        constexpr int C = Elements<T>::kChunk;
#pragma unroll
        for (int c = 0; c < 16 / C; ++c) {
            uint4 q = make_uint4(0, 0, 0, 0);
            if (c * C < live) q = __ldcs(reinterpret_cast<const uint4*>(at + c * C));
            w[4 * c] = q.x; w[4 * c + 1] = q.y; w[4 * c + 2] = q.z; w[4 * c + 3] = q.w;
        }
    } else {
        const uintptr_t address = reinterpret_cast<uintptr_t>(at), low = address & ~uintptr_t{15};
        if (low >= reinterpret_cast<uintptr_t>(x) && low + (W + 4) * 4 <= reinterpret_cast<uintptr_t>(x + count)) {
            uint32_t c[W + 4];
#pragma unroll
            for (int i = 0; i < W / 4 + 1; ++i) {
                const uint4 q = *reinterpret_cast<const uint4*>(low + i * 16);
                c[4 * i] = q.x; c[4 * i + 1] = q.y; c[4 * i + 2] = q.z; c[4 * i + 3] = q.w;
            }
            const unsigned shift = static_cast<unsigned>(address & 15u);
            if (shift & 8u)
#pragma unroll
                for (int i = 0; i < W + 2; ++i) c[i] = c[i + 2];
            if (shift & 4u)
#pragma unroll
                for (int i = 0; i < W + 1; ++i) c[i] = c[i + 1];
            const unsigned bits = (shift & 2u) * 8u;   // 0 for F32
#pragma unroll
            for (int i = 0; i < W; ++i) w[i] = sizeof(T) == 4 ? c[i] : __funnelshift_r(c[i], c[i + 1], bits);
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) w[i] = 0u;
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (i < live) w[i] = __float_as_uint(at[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (i < live) w[i / 2] |= static_cast<uint32_t>(at[i]) << (i % 2 * 16);
            }
        }
        if (live < 16) {   // what follows the row's end belongs to the next row
#pragma unroll
            for (int i = 0; i < W; ++i) {
                if constexpr (sizeof(T) == 4) w[i] = i < live ? w[i] : 0u;
                else w[i] = 2 * i + 1 < live ? w[i] : 2 * i < live ? w[i] & 0xffffu : 0u;
            }
        }
    }
}
// The elements as F32, and the bits of the largest magnitude (a NaN's are above every other's)
template <typename T>
__device__ __forceinline__ uint32_t values16(const uint32_t (&w)[Elements<T>::kWords], float (&v)[16]) {
    constexpr int W = Elements<T>::kWords;
    uint32_t top;
    if constexpr (sizeof(T) == 2) {
        top = w[0] & 0x7fff7fffu;
#pragma unroll
        for (int i = 1; i < W; ++i) top = __vmaxu2(top, w[i] & 0x7fff7fffu);
        top = max(top << 16, top & 0xffff0000u);
#pragma unroll
        for (int i = 0; i < W; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    } else {
        top = 0u;
#pragma unroll
        for (int i = 0; i < W; ++i) { v[i] = __uint_as_float(w[i]); top = max(top, w[i] & 0x7fffffffu); }
    }
    return top;
}
// v[i] of eight registers
__device__ __forceinline__ float pick8(const float* v, int i) {
    const float a = i & 1 ? v[1] : v[0], b = i & 1 ? v[3] : v[2], c = i & 1 ? v[5] : v[4], d = i & 1 ? v[7] : v[6];
    const float ab = i & 2 ? b : a, cd = i & 2 ? d : c;
    return i & 4 ? cd : ab;
}
// y / (hi + lo) of eight values to within an F32 step, moved off a value of three significant bits (the borders among them) to the
// side the exact quotient lies on; r ~ 1 / hi
__device__ __forceinline__ void refined8(const float* v, float hi, float lo, float r, float (&y)[8]) {
    const unsigned long long nh = pack_f32x2(-hi, -hi), nl = pack_f32x2(-lo, -lo), rr = pack_f32x2(r, r);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const unsigned long long x = pack_f32x2(v[i], v[i + 1]);
        unsigned long long q = mul_f32x2(x, rr);
        q = fma_f32x2(fma_f32x2(q, nl, fma_f32x2(q, nh, x)), rr, q);
        const unsigned long long rest = fma_f32x2(q, nl, fma_f32x2(q, nh, x));
        float q0, q1, e0, e1;
        unpack_f32x2(q, q0, q1);
        unpack_f32x2(rest, e0, e1);
        auto move = [](float a, float e, float of) {
            const int bits = __float_as_int(a) | (__float_as_int(of) & 0x80000000), step = ((__float_as_int(e) ^ bits) >> 31) | 1;   // -1: the quotient is nearer to 0
            return __int_as_float((bits & 0x1fffff) == 0 && e != 0.0f ? bits + step : bits);
        };
        y[i] = move(q0, e0, v[i]);           // the sign of -0 is lost on the way
        y[i + 1] = move(q1, e1, v[i + 1]);
    }
}
__device__ __forceinline__ void scale8(const float* v, float r, float (&y)[8]) {
    const unsigned long long rr = pack_f32x2(r, r);
#pragma unroll
    for (int i = 0; i < 8; i += 2) unpack_f32x2(mul_f32x2(pack_f32x2(v[i], v[i + 1]), rr), y[i], y[i + 1]);
}

struct PackGeom {
    int64_t rows, k, row_bytes;
    int64_t segments;      // 16-element segments of a padded row (whole scale tiles)
    int64_t padded_rows;   // multiple of 128
    int64_t tile_row;      // bytes of a row of scale tiles
};

// LANES threads share a word of the scale tile (a segment of 16 elements each); 1: a thread takes all of a word's segments in
// turn, for rows so short that most segments of a word are padding.
template <typename T, int FORMAT, bool VEC, int LANES>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 4 : 3) fp4_quantize_kernel(const T* __restrict__ x, const float* tensor_scale, uint8_t* __restrict__ codes,
                                                               uint8_t* __restrict__ scales, PackGeom p) {
    constexpr int kPerWord = FORMAT == VRB_NVFP4 ? 4 : 8;      // segments of a scale word
    constexpr int kSerial = LANES == 1 ? kPerWord : 1;
    pdl_wait();
    const float g = FORMAT == VRB_NVFP4 && tensor_scale ? *tensor_scale : 1.0f;
    // 2^-100 .. 2^100: the F32 form neither overflows nor loses bits below the normal range
    const bool fast = g >= 7.888609052210118e-31f && g <= 1.2676506002282294e30f;
    const float g6 = __fmul_rn(6.0f, g);
    const int64_t units = p.segments / kSerial;                // of a row
    const int64_t total = p.rows * units, stride = static_cast<int64_t>(gridDim.x) * kThreads;
    int64_t u = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    const int64_t d_row = stride / units, d_unit = stride - d_row * units;
    int64_t row = u / units, unit = u - row * units;
    const int lane = threadIdx.x & 31;
    const int64_t count = p.rows * p.k;
    auto fetch = [&](int64_t r, int64_t column, uint32_t (&w)[Elements<T>::kWords]) {
        if (column < p.k) load16<T, VEC>(x, count, x + r * p.k + column, column, p.k, w);
        else
#pragma unroll
            for (int i = 0; i < Elements<T>::kWords; ++i) w[i] = 0u;
    };
    uint32_t ahead[Elements<T>::kWords];
    if constexpr (LANES > 1)
        if (u < total) fetch(row, unit * 16, ahead);
    // total and stride are multiples of the lanes that share a scale word, so those stay together
    for (; u < total; u += stride) {
        const int64_t warp_left = total - (u - lane);
        const unsigned group = warp_left >= 32 ? 0xffffffffu : (1u << warp_left) - 1u;   // lanes that hold a unit
        int64_t next_row = row + d_row, next_unit = unit + d_unit;
        if (next_unit >= units) { next_unit -= units; ++next_row; }
        uint32_t word = 0u, carried = 0u;
        // a short row's segments past its codes have nothing to write but the zero scales that `carried` begins with
        const int parts = LANES > 1 ? 1 : static_cast<int>(p.row_bytes / 8 < kSerial ? p.row_bytes / 8 : kSerial);
#pragma unroll 1
        for (int part = 0; part < parts; ++part) {
            const int64_t segment = unit * kSerial + part, column = segment * 16;
            float v[16];
            uint32_t top;
            if constexpr (LANES > 1) {   // the next unit's elements are on their way while this one's are packed
                top = values16<T>(ahead, v);
                if (u + stride < total) fetch(next_row, next_unit * 16, ahead);
            } else {
                uint32_t w[Elements<T>::kWords];
                fetch(row, column, w);
                top = values16<T>(w, v);
            }
            const bool live = column < p.k;
            uint32_t byte = 0u, word0 = 0u, word1 = 0u;
            if constexpr (FORMAT == VRB_NVFP4) {
                const float a = __uint_as_float(top);
                if (top >= 0x7f800000u || !(g <= 3.402823466e38f)) {
                    byte = live ? 0x7fu : 0u;
                } else if (top != 0u && g != 0.0f) {
                    const float q = __fdividef(a, g6);
                    byte = e4m3_bits(q * (1.0f - kGuard));
                    if (!fast) {
                        byte = nv_scale_exact(a, g);
                    } else if (byte != e4m3_bits(q * (1.0f + kGuard))) {   // next to a border: as for the elements, 6 g = g6 + its rest
                        const float border = 0.5f * (e4m3_value(byte) + e4m3_value(byte + 1u));
                        const float d = __fmaf_rn(-border, __fmaf_rn(6.0f, g, -g6), __fmaf_rn(-border, g6, a));
                        byte += d > 0.0f || (d == 0.0f && (byte & 1u) != 0u) ? 1u : 0u;
                    }
                }
                if (byte != 0u && byte != 0x7fu) {
                    const float s = e4m3_value(byte), hi = __fmul_rn(s, g), lo = __fmaf_rn(s, g, -hi);
                    const float r = __fdividef(1.0f, hi);
                    float y[8];
                    scale8(v, r * (1.0f - kGuard), y);
                    word0 = e2m1x8(y);
                    scale8(v + 8, r * (1.0f - kGuard), y);
                    word1 = e2m1x8(y);
                    scale8(v, r * (1.0f + kGuard), y);
                    const uint32_t above0 = e2m1x8(y);
                    scale8(v + 8, r * (1.0f + kGuard), y);
                    const uint32_t above1 = e2m1x8(y);
                    if (!fast) {
                        const double step = static_cast<double>(s) * static_cast<double>(g);
                        word0 = word1 = 0u;
#pragma unroll 1
                        for (int i = 0; i < 8; ++i) {
                            word0 |= e2m1_exact(pick8(v, i), step) << (4 * i);
                            word1 |= e2m1_exact(pick8(v + 8, i), step) << (4 * i);
                        }
                    } else if (word0 != above0 || word1 != above1) {
                        bool refine = true;
                        if constexpr (sizeof(T) == 2) {
                            const bool first = word0 != above0;
                            const uint32_t below = first ? word0 : word1;
                            const int i = (__ffs(static_cast<int>(below ^ (first ? above0 : above1))) - 1) >> 2;
                            const float a = fabsf(first ? pick8(v, i) : pick8(v + 8, i)), t = e2m1_border(below >> (4 * i) & 7u);
                            const float d = __fmaf_rn(-t, lo, __fmaf_rn(-t, hi, a));
                            if (d > 0.0f) { word0 = above0; word1 = above1; }
                            refine = d == 0.0f;
                        }
                        if (refine) {
                            refined8(v, hi, lo, r, y);
                            word0 = e2m1x8(y);
                            refined8(v + 8, hi, lo, r, y);
                            word1 = e2m1x8(y);
                        }
                    }
                }
            } else {
                // the block's two halves: neighbouring lanes, or this thread's last and next segment
                if constexpr (LANES > 1) {
                    top = max(top, __shfl_xor_sync(group, top, 1));
                } else {
                    uint32_t w[Elements<T>::kWords];
                    float other[16];
                    fetch(row, column ^ 16, w);
                    top = max(top, values16<T>(w, other));
                }
                if (top >= 0x7f800000u) {
                    byte = 0xffu;
                } else {
                    const int e = static_cast<int>(top >> 23) - 2;   // biased exponent of 2^(floor(log2 a) - 2)
                    byte = e > 0 ? static_cast<uint32_t>(e) : 0u;
                    const float r = __uint_as_float((254u - byte) << 23);   // 2^(127 - byte): the product is exact or far below the first border
                    float y[8];
                    scale8(v, r, y);
                    word0 = e2m1x8(y);
                    scale8(v + 8, r, y);
                    word1 = e2m1x8(y);
                }
            }
            if (segment * 8 < p.row_bytes)
                *reinterpret_cast<uint2*>(codes + row * p.row_bytes + segment * 8) = make_uint2(word0, word1);
            constexpr int kPerBlock = FORMAT == VRB_NVFP4 ? 1 : 2;   // segments of a block
            const bool in_block = FORMAT == VRB_NVFP4 ? column < p.k : (segment & ~int64_t{1}) * 16 < p.k;
            word = in_block ? byte : 0u;
            if constexpr (LANES > 1) {
                word |= __shfl_xor_sync(group, word, kPerBlock) << 8;
                word |= __shfl_xor_sync(group, word, 2 * kPerBlock) << 16;
            } else {
                carried |= word << (part / kPerBlock * 8);
            }
        }
        if (LANES == 1 || (unit & (kPerWord - 1)) == 0) {
            const int64_t word_index = LANES == 1 ? unit : unit / kPerWord;
            const int64_t at = (row >> 7) * p.tile_row + word_index * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4;
            *reinterpret_cast<uint32_t*>(scales + at) = LANES == 1 ? carried : word;
        }
        row = next_row;
        unit = next_unit;
    }
    // the scales of the rows that fill the last tile up
    const int64_t words = p.tile_row / 512, filling = (p.padded_rows - p.rows) * words;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < filling; i += stride) {
        const int64_t r = p.rows + i / words;
        *reinterpret_cast<uint32_t*>(scales + (r >> 7) * p.tile_row + i % words * 512 + (r & 31) * 16 + ((r & 127) >> 5) * 4) = 0u;
    }
}

// the two F32 values of a byte of codes
__device__ __forceinline__ void e2m1x2_values(uint32_t byte, float& lo, float& hi) {
    uint32_t h;
    asm("{\n\t.reg .b8 b;\n\t.reg .b16 w;\n\tcvt.u16.u32 w, %1;\n\tmov.b16 {b, _}, w;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(h) : "r"(byte));
    asm("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, u;\n\t}" : "=f"(lo), "=f"(hi) : "r"(h));
}

// A thread writes 16 elements that begin on a 16-byte boundary of the result.  Rows of whole chunks (VEC): one segment.
// Otherwise a row that begins `phase` elements past a boundary is cut into windows of columns [16 w - phase, 16 w - phase + 16):
// the codes of two segments joined by a shift and up to two scales; windows over a row's ends go element by element.
template <int FORMAT>
__device__ __forceinline__ float scale_of(const uint8_t* scales, const PackGeom& p, int64_t row, int64_t segment) {
    const int64_t block = FORMAT == VRB_NVFP4 ? segment : segment >> 1;
    const uint32_t byte = scales[(row >> 7) * p.tile_row + (block >> 2) * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4 + (block & 3)];
    if constexpr (FORMAT == VRB_NVFP4) return byte == 0x7fu ? __uint_as_float(0x7fffffffu) : e4m3_value(byte);
    else return byte == 0xffu ? __uint_as_float(0x7fffffffu) : __uint_as_float(byte ? byte << 23 : 0x00400000u);
}
template <typename T, int FORMAT, bool VEC>
__global__ void __launch_bounds__(kThreads) fp4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                 const float* tensor_scale, T* __restrict__ out, PackGeom p) {
    constexpr int kPhases = Elements<T>::kChunk;
    pdl_wait();
    const float g = FORMAT == VRB_NVFP4 && tensor_scale ? *tensor_scale : 1.0f;
    const int64_t windows = VEC ? (p.k + 15) / 16 : (p.k + kPhases - 1 + 15) / 16;
    const int64_t total = p.rows * windows, stride = static_cast<int64_t>(gridDim.x) * kThreads;
    int64_t u = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    const int64_t d_row = stride / windows, d_window = stride - d_row * windows;
    int64_t row = u / windows, window = u - row * windows;
    const int offset = static_cast<int>(reinterpret_cast<uintptr_t>(out) % 16 / sizeof(T));
    for (; u < total; u += stride) {
        const int phase = VEC ? 0 : static_cast<int>(static_cast<uint64_t>(row * p.k + offset) & (kPhases - 1));
        const int64_t column = window * 16 - phase;
        if (VEC || column < p.k) {
            const uint8_t* row_codes = codes + row * p.row_bytes;
            const int64_t last = (p.k - 1) / 16;               // segments of the row that hold elements
            uint64_t bits = 0;
            float s_lo = 0.0f, s_hi = 0.0f;                    // of the elements before and from `phase` on
            if (window <= last) {
                bits = __ldcs(reinterpret_cast<const unsigned long long*>(row_codes + window * 8));
                s_hi = scale_of<FORMAT>(scales, p, row, window);
            }
            if constexpr (!VEC) {
                if (phase > 0) {
                    bits <<= 4 * phase;
                    if (window > 0) {
                        bits |= *reinterpret_cast<const unsigned long long*>(row_codes + (window - 1) * 8) >> (64 - 4 * phase);
                        s_lo = scale_of<FORMAT>(scales, p, row, window - 1);
                    }
                }
            }
            float v[16];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                e2m1x2_values(static_cast<uint32_t>(bits >> (8 * i)) & 0xffu, v[2 * i], v[2 * i + 1]);
                const float s0 = !VEC && 2 * i < phase ? s_lo : s_hi, s1 = !VEC && 2 * i + 1 < phase ? s_lo : s_hi;
                v[2 * i] = __fmul_rn(__fmul_rn(v[2 * i], s0), g);
                v[2 * i + 1] = __fmul_rn(__fmul_rn(v[2 * i + 1], s1), g);
            }
            const int64_t at = row * p.k + column;
            if (VEC || (column >= 0 && column + 16 <= p.k)) {
                if constexpr (sizeof(T) == 2) {
                    store16_bf16(out, at, v);
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float y[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) y[i] = v[h * 8 + i];
                        store8(out, VRB_F32, at + h * 8, y);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (column + i >= 0 && column + i < p.k) {
                        if constexpr (sizeof(T) == 2) out[at + i] = static_cast<uint16_t>(float_to_bf16_bits(v[i]));
                        else out[at + i] = v[i];
                    }
            }
        }
        row += d_row;
        window += d_window;
        if (window >= windows) { window -= windows; ++row; }
    }
}

// Short rows in bf16, whose windows would be all ends: a thread writes one 16-byte chunk of the result, over as many rows as it spans.
template <int FORMAT>
__global__ void __launch_bounds__(kThreads) fp4_dequantize_short_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                       const float* tensor_scale, uint16_t* __restrict__ out, PackGeom p, int head) {
    constexpr int C = 8;
    pdl_wait();
    const float g = FORMAT == VRB_NVFP4 && tensor_scale ? *tensor_scale : 1.0f;
    const int64_t count = p.rows * p.k, chunks = (count - head + C - 1) / C + (head > 0 ? 1 : 0);
    const int k = static_cast<int>(p.k);
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; u < chunks; u += static_cast<int64_t>(gridDim.x) * kThreads) {
        const int64_t first = u * C - (head > 0 ? C - head : 0);   // the first chunk may begin before the result
        const int64_t begin = first > 0 ? first : 0;
        int64_t row = begin / k;
        int column = static_cast<int>(begin - row * k);
        float v[C], s = 0.0f;
        bool fresh = true;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            v[i] = 0.0f;
            const int64_t at = first + i;
            if (at >= 0 && at < count) {
                if (fresh || (column & (FORMAT == VRB_NVFP4 ? 15 : 31)) == 0) s = scale_of<FORMAT>(scales, p, row, column >> 4);
                fresh = false;
                float lo, hi;
                e2m1x2_values(codes[row * p.row_bytes + (column >> 1)], lo, hi);
                v[i] = __fmul_rn(__fmul_rn(column & 1 ? hi : lo, s), g);
                if (++column == k) { column = 0; ++row; fresh = true; }
            }
        }
        if (first >= 0 && first + C <= count) {
            *reinterpret_cast<uint4*>(out + first) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
        } else {
#pragma unroll
            for (int i = 0; i < C; ++i)
                if (first + i >= 0 && first + i < count) out[first + i] = static_cast<uint16_t>(float_to_bf16_bits(v[i]));
        }
    }
}

__global__ void fp4_scale_clear_kernel(float* tensor_scale) {
    pdl_wait();
    *tensor_scale = 0.0f;
}
// Division by 2688 is monotonic, so the maximum of the quotients is the quotient of the maximum; bit patterns of
// non-negative values order as integers, and a NaN's is above them all.  The maximum does not depend on the order.
template <typename T>
__global__ void __launch_bounds__(kThreads) fp4_tensor_scale_kernel(const T* __restrict__ x, int64_t count, int64_t head, float* tensor_scale) {
    pdl_wait();
    constexpr int C = Elements<T>::kChunk;
    const int64_t tid = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, stride = static_cast<int64_t>(gridDim.x) * kThreads;
    uint32_t top = 0;
    auto take = [&](T e) { top = max(top, __float_as_uint(Elements<T>::value(e)) & 0x7fffffffu); };
    if (tid < head) take(x[tid]);
    const T* body = x + head;
    const int64_t chunks = (count - head) / C;
    for (int64_t i = tid; i < chunks; i += 8 * stride) {
        uint4 w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j * stride < chunks) w[j] = *reinterpret_cast<const uint4*>(body + (i + j * stride) * C);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j * stride < chunks) {
                if constexpr (sizeof(T) == 2) {
                    const uint32_t two = __vmaxu2(__vmaxu2(w[j].x & 0x7fff7fffu, w[j].y & 0x7fff7fffu), __vmaxu2(w[j].z & 0x7fff7fffu, w[j].w & 0x7fff7fffu));
                    top = max(top, max(two << 16, two & 0xffff0000u));
                } else {
                    top = max(top, max(max(w[j].x & 0x7fffffffu, w[j].y & 0x7fffffffu), max(w[j].z & 0x7fffffffu, w[j].w & 0x7fffffffu)));
                }
            }
    }
    if (tid < count - head - chunks * C) take(body[chunks * C + tid]);
    top = __reduce_max_sync(0xffffffffu, top);
    __shared__ uint32_t tops[kThreads / 32];
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / 32; ++w) top = max(top, tops[w]);
        const uint32_t scale = __float_as_uint(__fdiv_rn(__uint_as_float(top), 2688.0f));
        atomicMax(reinterpret_cast<unsigned*>(tensor_scale), scale & 0x7fffffffu);
    }
}

int make_pack(PackGeom& p, int format, int64_t rows, int64_t k, const char* what) {
    VRB_REQUIRE(format == VRB_NVFP4 || format == VRB_MXFP4, VRB_ERR_INVALID, "%s: unknown 4-bit format %d", what, format);
    VRB_REQUIRE(rows > 0 && k > 0 && rows <= (int64_t{1} << 40) / k, VRB_ERR_INVALID, "%s: rows and k must be positive and rows * k at most 2^40", what);
    p.rows = rows; p.k = k; p.row_bytes = fp4_row_bytes(k);
    const int64_t tiles = fp4_block_tiles(format, k);
    p.segments = tiles * 4 * fp4_block(format) / 16;
    p.padded_rows = (rows + 127) / 128 * 128;
    p.tile_row = tiles * 512;
    return VRB_OK;
}

}  // namespace
}  // namespace vrb

using namespace vrb;

extern "C" int64_t vrb_fp4_row_bytes(int64_t k) { return k > 0 ? fp4_row_bytes(k) : 0; }
extern "C" size_t vrb_fp4_scale_bytes(int format, int64_t rows, int64_t k) {
    if (rows <= 0 || k <= 0 || (format != VRB_NVFP4 && format != VRB_MXFP4)) return 0;
    return static_cast<size_t>((rows + 127) / 128 * fp4_block_tiles(format, k) * 512);
}

extern "C" int vrb_fp4_tensor_scale(const void* x, int dtype, int64_t count, float* tensor_scale, vrb_stream stream) {
    VRB_REQUIRE(x && tensor_scale, VRB_ERR_INVALID, "fp4_tensor_scale: null tensor");
    VRB_REQUIRE(is_float_dtype(dtype), VRB_ERR_UNSUPPORTED, "fp4_tensor_scale: dtype must be F32 or BF16");
    VRB_REQUIRE(count > 0 && reinterpret_cast<uintptr_t>(x) % dtype_bytes(dtype) == 0 && (reinterpret_cast<uintptr_t>(tensor_scale) & 3u) == 0,
                VRB_ERR_INVALID, "fp4_tensor_scale: count must be positive and the tensors aligned to their elements");
    cudaStream_t s = as_stream(stream);
    launch_overlapped(fp4_scale_clear_kernel, dim3(1), dim3(1), 0, s, tensor_scale);
    if (int rc = after_launch("fp4_tensor_scale")) return rc;
    const int64_t element = static_cast<int64_t>(dtype_bytes(dtype));
    int64_t head = (16 - static_cast<int64_t>(reinterpret_cast<uintptr_t>(x) & 15u)) % 16 / element;
    if (head > count) head = count;
    const int grid = grid_for((count / (16 / element) + kThreads * 8 - 1) / (kThreads * 8), 4);
    if (dtype == VRB_BF16) launch_overlapped(fp4_tensor_scale_kernel<uint16_t>, dim3(grid), dim3(kThreads), 0, s, static_cast<const uint16_t*>(x), count, head, tensor_scale);
    else launch_overlapped(fp4_tensor_scale_kernel<float>, dim3(grid), dim3(kThreads), 0, s, static_cast<const float*>(x), count, head, tensor_scale);
    return after_launch("fp4_tensor_scale");
}

extern "C" int vrb_fp4_quantize(int format, const void* x, int dtype, const float* tensor_scale, void* codes, void* scales,
                                int64_t rows, int64_t k, vrb_stream stream) {
    VRB_REQUIRE(x && codes && scales, VRB_ERR_INVALID, "fp4_quantize: null tensor");
    VRB_REQUIRE(is_float_dtype(dtype), VRB_ERR_UNSUPPORTED, "fp4_quantize: dtype must be F32 or BF16");
    PackGeom p;
    if (int rc = make_pack(p, format, rows, k, "fp4_quantize")) return rc;
    VRB_REQUIRE(format == VRB_NVFP4 || !tensor_scale, VRB_ERR_INVALID, "fp4_quantize: MXFP4 has no tensor scale");
    VRB_REQUIRE(aligned16(codes) && aligned16(scales), VRB_ERR_INVALID, "fp4_quantize: codes and scales must be 16-byte aligned");
    VRB_REQUIRE(aligned_to(x, dtype_bytes(dtype)) && aligned_to(tensor_scale, 4), VRB_ERR_INVALID, "fp4_quantize: tensors must be aligned to their elements");
    // a thread to a scale word where the rows have one and at most half of its segments hold elements
    const bool serial = p.tile_row == 512 && k <= p.segments * 16 / 2;
    const int64_t units = rows * (serial ? 1 : p.segments), filling = (p.padded_rows - rows) * (p.tile_row / 512);
    const dim3 grid(static_cast<unsigned>(grid_for((units + filling + kThreads - 1) / kThreads, 8)));
    const bool vec = aligned16(x) && k % (16 / static_cast<int64_t>(dtype_bytes(dtype))) == 0;
    cudaStream_t s = as_stream(stream);
#define VRB_PACK(T, F, V, L) launch_overlapped(fp4_quantize_kernel<T, F, V, L>, grid, dim3(kThreads), 0, s, static_cast<const T*>(x), tensor_scale, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), p)
#define VRB_PACK_F(T, F, L) do { if (serial) VRB_PACK(T, F, false, 1); else if (vec) VRB_PACK(T, F, true, L); else VRB_PACK(T, F, false, L); } while (0)
#define VRB_PACK_T(T) do { if (format == VRB_NVFP4) VRB_PACK_F(T, VRB_NVFP4, 4); else VRB_PACK_F(T, VRB_MXFP4, 8); } while (0)
    if (dtype == VRB_BF16) VRB_PACK_T(uint16_t); else VRB_PACK_T(float);
#undef VRB_PACK_T
#undef VRB_PACK_F
#undef VRB_PACK
    return after_launch("fp4_quantize");
}

extern "C" int vrb_fp4_dequantize(int format, const void* codes, const void* scales, const float* tensor_scale, void* out,
                                  int out_dtype, int64_t rows, int64_t k, vrb_stream stream) {
    VRB_REQUIRE(codes && scales && out, VRB_ERR_INVALID, "fp4_dequantize: null tensor");
    VRB_REQUIRE(is_float_dtype(out_dtype), VRB_ERR_UNSUPPORTED, "fp4_dequantize: out dtype must be F32 or BF16");
    PackGeom p;
    if (int rc = make_pack(p, format, rows, k, "fp4_dequantize")) return rc;
    VRB_REQUIRE(format == VRB_NVFP4 || !tensor_scale, VRB_ERR_INVALID, "fp4_dequantize: MXFP4 has no tensor scale");
    VRB_REQUIRE(aligned16(codes) && aligned16(scales), VRB_ERR_INVALID, "fp4_dequantize: codes and scales must be 16-byte aligned");
    VRB_REQUIRE(aligned_to(out, dtype_bytes(out_dtype)) && aligned_to(tensor_scale, 4), VRB_ERR_INVALID, "fp4_dequantize: tensors must be aligned to their elements");
    const int64_t units = rows * ((k + 15) / 16 + 1);
    const dim3 grid(static_cast<unsigned>(grid_for((units + kThreads - 1) / kThreads, 8)));
    const bool vec = aligned16(out) && k % 16 == 0;
    cudaStream_t s = as_stream(stream);
    if (!vec && k < 64 && out_dtype == VRB_BF16) {   // 4000000 rows of 17: 195 us, 365 in windows; F32 stores by the element cost less (9000000 of 5: 142, 97)
        const int head = static_cast<int>((16 - reinterpret_cast<uintptr_t>(out) % 16) % 16) / 2;
        const dim3 blocks(static_cast<unsigned>(grid_for((rows * k / 8 + 2 + kThreads - 1) / kThreads, 8)));
#define VRB_SHORT(F) launch_overlapped(fp4_dequantize_short_kernel<F>, blocks, dim3(kThreads), 0, s, static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), tensor_scale, static_cast<uint16_t*>(out), p, head)
        if (format == VRB_NVFP4) VRB_SHORT(VRB_NVFP4); else VRB_SHORT(VRB_MXFP4);
#undef VRB_SHORT
        return after_launch("fp4_dequantize");
    }
#define VRB_UNPACK(T, F, V) launch_overlapped(fp4_dequantize_kernel<T, F, V>, grid, dim3(kThreads), 0, s, static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), tensor_scale, static_cast<T*>(out), p)
#define VRB_UNPACK_T(T) do { if (format == VRB_NVFP4) { if (vec) VRB_UNPACK(T, VRB_NVFP4, true); else VRB_UNPACK(T, VRB_NVFP4, false); } \
                             else { if (vec) VRB_UNPACK(T, VRB_MXFP4, true); else VRB_UNPACK(T, VRB_MXFP4, false); } } while (0)
    if (out_dtype == VRB_BF16) VRB_UNPACK_T(uint16_t); else VRB_UNPACK_T(float);
#undef VRB_UNPACK_T
#undef VRB_UNPACK
    return after_launch("fp4_dequantize");
}
