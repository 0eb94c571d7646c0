// Microscaled 4-bit floating point: tensor scale, packing, unpacking (formats and layout: include/vrb.h).
//
// All three are bound by HBM: packing reads 2 or 4 bytes an element and writes 0.5 + 1/16 (NVFP4) or 0.5 + 1/32
// (MXFP4), unpacking the reverse.  A thread owns 16 consecutive elements of a row: 32 bytes of bf16 in, 8 bytes of codes
// out, so a warp reads 1 KB and writes 256 bytes, both contiguous; the scale bytes of the four blocks that share a
// word of the scale tile are collected by shuffles and leave as one 4-byte store.
//
// Rounding is that of the real quotients a / (6 g) -> e4m3 and x / (g s) -> e2m1.  The fast form multiplies by an F32
// reciprocal (three roundings, relative error < 2^-22) and converts the product moved up and down by kGuard = 2^-21:
// where both give one code it is the right one.  Where they differ a rounding border lies between, and the sign of
// |x| - border * s * g, exact in double (at most 31 significant bits against 24), decides; 0 is the tie.
#include "vrb_fp4.cuh"

namespace vrb {
namespace {

constexpr int kThreads = 256;
constexpr float kGuard = 4.76837158203125e-7f;   // 2^-21

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
// 2 * magnitude of an e2m1 code: 0 1 2 3 4 6 8 12
__device__ __forceinline__ int e2m1_twice(uint32_t code) {
    const uint32_t m = code & 7u;
    return m < 4u ? static_cast<int>(m) : static_cast<int>((2u + (m & 1u)) << (m / 2u - 1u));
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
// one element, exactly: |x| against the borders times s g
__device__ __noinline__ uint32_t e2m1_exact(float x, double unit) {
    const uint32_t sign = __float_as_uint(x) >> 31 << 3;
    const double a = fabs(static_cast<double>(x));
    uint32_t code = 0;
    for (; code < 7u; ++code) {
        const double border = 0.25 * static_cast<double>(e2m1_twice(code) + e2m1_twice(code + 1u)) * unit;
        if (a < border || (a == border && (code & 1u) == 0u)) break;
    }
    return sign | code;
}

template <typename T> struct Elements;
template <> struct Elements<uint16_t> {
    static constexpr int kChunk = 8;     // elements of a 16-byte chunk
    __device__ static __forceinline__ float value(uint16_t h) { return bf16_bits_to_float(h); }
};
template <> struct Elements<float> {
    static constexpr int kChunk = 4;
    __device__ static __forceinline__ float value(float f) { return f; }
};

// elements [column, column + 16) of a row of k, zero past the end
template <typename T, bool VEC>
__device__ __forceinline__ void load16(const T* row, int64_t column, int64_t k, float (&v)[16]) {
    if constexpr (VEC) {
        constexpr int C = Elements<T>::kChunk;
#pragma unroll
        for (int c = 0; c < 16 / C; ++c) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (column + c * C < k) w = __ldcs(reinterpret_cast<const uint4*>(row + column + c * C));
            T e[C];
            *reinterpret_cast<uint4*>(e) = w;
#pragma unroll
            for (int i = 0; i < C; ++i) v[c * C + i] = Elements<T>::value(e[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = column + i < k ? Elements<T>::value(row[column + i]) : 0.0f;
    }
}

struct PackGeom {
    int64_t rows, k, row_bytes;
    int64_t segments;      // 16-element segments of a padded row (whole scale tiles)
    int64_t padded_rows;   // multiple of 128
    int64_t tile_row;      // bytes of a row of scale tiles
};

template <typename T, int FORMAT, bool VEC>
__global__ void __launch_bounds__(kThreads) fp4_quantize_kernel(const T* __restrict__ x, const float* tensor_scale, uint8_t* __restrict__ codes,
                                                               uint8_t* __restrict__ scales, PackGeom p) {
    pdl_wait();
    const float g = FORMAT == VRB_NVFP4 && tensor_scale ? *tensor_scale : 1.0f;
    // 2^-100 .. 2^100: the F32 form neither overflows nor loses bits below the normal range
    const bool fast = g >= 7.888609052210118e-31f && g <= 1.2676506002282294e30f;
    const int64_t total = p.padded_rows * p.segments, stride = static_cast<int64_t>(gridDim.x) * kThreads;
    int64_t u = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    const int64_t d_row = stride / p.segments, d_segment = stride - d_row * p.segments;
    int64_t row = u / p.segments, segment = u - row * p.segments;
    const int lane = threadIdx.x & 31;
    // total and stride are multiples of the 4 or 8 segments that share a scale word, so those lanes stay together
    for (; u < total; u += stride) {
        const int64_t warp_left = total - (u - lane);
        const unsigned group = warp_left >= 32 ? 0xffffffffu : (1u << warp_left) - 1u;   // lanes that hold a segment
        const int64_t column = segment * 16;
        float v[16];
        const bool live = row < p.rows && column < p.k;
        if (live) load16<T, VEC>(x + row * p.k, column, p.k, v);
        else
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = 0.0f;
        uint32_t top = 0;   // bits of the largest magnitude; a NaN is above everything
#pragma unroll
        for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
        if constexpr (FORMAT == VRB_MXFP4) top = max(top, __shfl_xor_sync(group, top, 1));
        uint32_t byte, word0 = 0, word1 = 0;
        if constexpr (FORMAT == VRB_NVFP4) {
            const float a = __uint_as_float(top);
            if (top >= 0x7f800000u || !(g <= 3.402823466e38f)) {
                byte = 0x7fu;
            } else if (top == 0u || g == 0.0f) {
                byte = 0u;
            } else {
                const float q = __fdiv_rn(a, __fmul_rn(6.0f, g));
                const uint32_t lo = e4m3_bits(q * (1.0f - kGuard)), hi = e4m3_bits(q * (1.0f + kGuard));
                byte = fast && lo == hi ? lo : nv_scale_exact(a, g);
            }
            if (byte != 0u && byte != 0x7fu) {
                const float s = e4m3_value(byte);
                const double unit = static_cast<double>(s) * static_cast<double>(g);
                const float r = __fdiv_rn(1.0f, __fmul_rn(s, g)), r_lo = r * (1.0f - kGuard), r_hi = r * (1.0f + kGuard);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float lo[8], hi[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) { lo[i] = v[h * 8 + i] * r_lo; hi[i] = v[h * 8 + i] * r_hi; }
                    uint32_t w = e2m1x8(lo);
                    if (!fast || w != e2m1x8(hi)) {
                        w = 0;
#pragma unroll
                        for (int i = 0; i < 8; ++i) w |= e2m1_exact(v[h * 8 + i], unit) << (4 * i);
                    }
                    (h ? word1 : word0) = w;
                }
            }
        } else {
            if (top >= 0x7f800000u) {
                byte = 0xffu;
            } else {
                const int e = static_cast<int>(top >> 23) - 2;   // biased exponent of 2^(floor(log2 a) - 2)
                byte = e > 0 ? static_cast<uint32_t>(e) : 0u;
                const float r = __uint_as_float((254u - byte) << 23);   // 2^(127 - byte): the product is exact or far below the first border
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float q[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) q[i] = v[h * 8 + i] * r;
                    (h ? word1 : word0) = e2m1x8(q);
                }
            }
            if (top == 0u) byte = 0u;
        }
        if (row < p.rows && segment * 8 < p.row_bytes)
            *reinterpret_cast<uint2*>(codes + row * p.row_bytes + segment * 8) = make_uint2(word0, word1);
        // four consecutive blocks make a word of the scale tile
        constexpr int kLanes = FORMAT == VRB_NVFP4 ? 1 : 2;   // lanes of a block
        const bool in_block = FORMAT == VRB_NVFP4 ? column < p.k : (segment & ~int64_t{1}) * 16 < p.k;
        uint32_t word = row < p.rows && in_block ? byte : 0u;
        word |= __shfl_xor_sync(group, word, kLanes) << 8;
        word |= __shfl_xor_sync(group, word, 2 * kLanes) << 16;
        if ((segment & (4 * kLanes - 1)) == 0) {
            const int64_t at = (row >> 7) * p.tile_row + segment / (4 * kLanes) * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4;
            *reinterpret_cast<uint32_t*>(scales + at) = word;
        }
        row += d_row;
        segment += d_segment;
        if (segment >= p.segments) { segment -= p.segments; ++row; }
    }
}

// the two F32 values of a byte of codes
__device__ __forceinline__ void e2m1x2_values(uint32_t byte, float& lo, float& hi) {
    uint32_t h;
    asm("{\n\t.reg .b8 b;\n\t.reg .b16 w;\n\tcvt.u16.u32 w, %1;\n\tmov.b16 {b, _}, w;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(h) : "r"(byte));
    asm("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, u;\n\t}" : "=f"(lo), "=f"(hi) : "r"(h));
}

template <typename T, int FORMAT, bool VEC>
__global__ void __launch_bounds__(kThreads) fp4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                 const float* tensor_scale, T* __restrict__ out, PackGeom p) {
    pdl_wait();
    const float g = FORMAT == VRB_NVFP4 && tensor_scale ? *tensor_scale : 1.0f;
    const int64_t segments = (p.k + 15) / 16;
    const int64_t total = p.rows * segments, stride = static_cast<int64_t>(gridDim.x) * kThreads;
    int64_t u = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    const int64_t d_row = stride / segments, d_segment = stride - d_row * segments;
    int64_t row = u / segments, segment = u - row * segments;
    for (; u < total; u += stride) {
        const uint2 w = __ldcs(reinterpret_cast<const uint2*>(codes + row * p.row_bytes + segment * 8));
        const int64_t block = FORMAT == VRB_NVFP4 ? segment : segment >> 1;
        const uint32_t byte = scales[(row >> 7) * p.tile_row + (block >> 2) * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4 + (block & 3)];
        float s;
        if constexpr (FORMAT == VRB_NVFP4) s = byte == 0x7fu ? __uint_as_float(0x7fffffffu) : e4m3_value(byte);
        else s = byte == 0xffu ? __uint_as_float(0x7fffffffu) : __uint_as_float(byte ? byte << 23 : 0x00400000u);
        float v[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            e2m1x2_values(((i < 4 ? w.x : w.y) >> (8 * (i & 3))) & 0xffu, v[2 * i], v[2 * i + 1]);
            v[2 * i] = __fmul_rn(__fmul_rn(v[2 * i], s), g);
            v[2 * i + 1] = __fmul_rn(__fmul_rn(v[2 * i + 1], s), g);
        }
        T* o = out + row * p.k + segment * 16;
        if constexpr (VEC) {   // k % 16 == 0
            if constexpr (sizeof(T) == 2) {
                store16_bf16(out, row * p.k + segment * 16, v);
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float y[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = v[h * 8 + i];
                    store8(out, VRB_F32, row * p.k + segment * 16 + h * 8, y);
                }
            }
        } else {
            const int n = static_cast<int>(p.k - segment * 16 < 16 ? p.k - segment * 16 : 16);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i < n) {
                    if constexpr (sizeof(T) == 2) o[i] = static_cast<uint16_t>(float_to_bf16_bits(v[i]));
                    else o[i] = v[i];
                }
        }
        row += d_row;
        segment += d_segment;
        if (segment >= segments) { segment -= segments; ++row; }
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
    for (int64_t i = tid; i < chunks; i += 4 * stride) {
        uint4 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j * stride < chunks) w[j] = *reinterpret_cast<const uint4*>(body + (i + j * stride) * C);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j * stride < chunks) {
                T e[C];
                *reinterpret_cast<uint4*>(e) = w[j];
#pragma unroll
                for (int k = 0; k < C; ++k) take(e[k]);
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
    const int grid = grid_for((count / (16 / element) + kThreads * 4 - 1) / (kThreads * 4), 8);
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
    const int64_t units = p.padded_rows * p.segments;
    const dim3 grid(static_cast<unsigned>(grid_for((units + kThreads - 1) / kThreads, 8)));
    const bool vec = aligned16(x) && k % (16 / static_cast<int64_t>(dtype_bytes(dtype))) == 0;
    cudaStream_t s = as_stream(stream);
#define VRB_PACK(T, F, V) launch_overlapped(fp4_quantize_kernel<T, F, V>, grid, dim3(kThreads), 0, s, static_cast<const T*>(x), tensor_scale, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), p)
#define VRB_PACK_T(T) do { if (format == VRB_NVFP4) { if (vec) VRB_PACK(T, VRB_NVFP4, true); else VRB_PACK(T, VRB_NVFP4, false); } \
                           else { if (vec) VRB_PACK(T, VRB_MXFP4, true); else VRB_PACK(T, VRB_MXFP4, false); } } while (0)
    if (dtype == VRB_BF16) VRB_PACK_T(uint16_t); else VRB_PACK_T(float);
#undef VRB_PACK_T
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
    const int64_t units = rows * ((k + 15) / 16);
    const dim3 grid(static_cast<unsigned>(grid_for((units + kThreads - 1) / kThreads, 8)));
    const bool vec = aligned16(out) && k % 16 == 0;
    cudaStream_t s = as_stream(stream);
#define VRB_UNPACK(T, F, V) launch_overlapped(fp4_dequantize_kernel<T, F, V>, grid, dim3(kThreads), 0, s, static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), tensor_scale, static_cast<T*>(out), p)
#define VRB_UNPACK_T(T) do { if (format == VRB_NVFP4) { if (vec) VRB_UNPACK(T, VRB_NVFP4, true); else VRB_UNPACK(T, VRB_NVFP4, false); } \
                             else { if (vec) VRB_UNPACK(T, VRB_MXFP4, true); else VRB_UNPACK(T, VRB_MXFP4, false); } } while (0)
    if (out_dtype == VRB_BF16) VRB_UNPACK_T(uint16_t); else VRB_UNPACK_T(float);
#undef VRB_UNPACK_T
#undef VRB_UNPACK
    return after_launch("fp4_dequantize");
}
