// The linear over packed 4-bit operands: out[m, n] = act(ga gb sum_k a[m, k] b[n, k] + bias[n]).
//
// The tensor core multiplies e2m1 elements 64 to an instruction and applies the block scales itself; they have to lie in
// tensor memory, a 32-bit word of four scales per row and column, which is the order of the packed scale tiles (one
// 32 x 128-bit copy per 128 rows x 4 blocks).  Persistent CTAs of 128 x 128 output tiles, six warps:
//   warp 0      copies 256 elements of k at a time into a ring of kStages buffers: codes by tensor map (128-byte swizzle,
//               zeros outside the operand), scale tiles as plain bulk copies
//   warp 1      copies the scale tiles on into tensor memory and issues the products (one thread); a buffer's scale
//               columns are its own, so the buffer's barrier also guards them
//   warps 2-5   read one accumulator out of tensor memory while the other is being filled, apply scale, bias and
//               activation and write rows
// Every wait is bounded: one that runs out sets a flag that the host can read and ends the CTA.
#include <cuda.h>

#include "vrb_fp4.cuh"
#include "vrb_tma.cuh"

namespace vrb {
namespace {

constexpr int kThreads = 192;
constexpr int kTile = 128;                 // rows of a, and of b, of an output tile
constexpr int kStageBytes = 128;           // bytes of codes per row and stage: 256 elements
constexpr int kStageElements = 256;
constexpr int kStages = 6;
constexpr int kCodeBytes = kTile * kStageBytes;
constexpr int kScaleBytes = 2048;          // NVFP4: 4 tiles of 512 bytes a stage; MXFP4 uses half
constexpr int kBufferBytes = 2 * kCodeBytes + 2 * kScaleBytes;
constexpr int kSharedBytes = kStages * kBufferBytes + 1024;   // + alignment of the swizzled tiles
constexpr int kColumns = 512;              // tensor memory columns: two accumulators, then 32 scale columns a stage
constexpr int kScaleColumn = 2 * kTile;
constexpr int kBand = 16;                  // row tiles that share a sweep over the columns (L2 reuse)
constexpr unsigned long long kWaitNs = 2000000000ull;

__device__ int g_fp4_wait_gave_up = 0;

struct LinearArgs {
    const uint8_t* a_scales;
    const uint8_t* b_scales;
    const float* a_scale;      // tensor scales or nullptr
    const float* b_scale;
    const void* bias;
    void* out;
    int64_t m, n;
    int64_t k;
    int64_t block_tiles;       // scale tiles along k
    int bias_dt, out_dt, activation;
    int vector_out;            // rows of out start on 16-byte boundaries
};

struct Control {
    uint64_t full[kStages], empty[kStages], done[2], drained[2];
    uint32_t tensor_base;
    volatile int abort;
};

__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ bool wait_barrier(uint64_t* barrier, unsigned parity, Control* control) {
    const unsigned address = shared_address(barrier);
    unsigned long long start = 0;
    for (unsigned tries = 0;; ++tries) {
        unsigned done;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(done) : "r"(address), "r"(parity) : "memory");
        if (done) return true;
        if ((tries & 63u) == 63u) {
            if (control->abort) return false;
            const unsigned long long t = now_ns();
            if (start == 0) start = t;
            else if (t - start > kWaitNs) {
                control->abort = 1;
                g_fp4_wait_gave_up = 1;
                return false;
            }
        }
    }
}
__device__ __forceinline__ void arrive(uint64_t* barrier) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(shared_address(barrier)) : "memory");
}
__device__ __forceinline__ void tma_load_2d(unsigned dst, const CUtensorMap* map, int x, int y, uint64_t* barrier) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(shared_address(barrier))
                 : "memory");
}
__device__ __forceinline__ void bulk_load(unsigned dst, const void* src, unsigned bytes, uint64_t* barrier) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
                 "r"(shared_address(barrier))
                 : "memory");
}

// Shared-memory operand descriptors (start address, offsets in units of 16 bytes; bit 46: descriptor version).
// Codes: rows of 128 bytes under the 128-byte swizzle, 8 rows = 1024 bytes apart.  Scale tile: 32 rows of 16 bytes, 8 rows
// = 128 bytes apart, no swizzle.
__device__ __forceinline__ uint64_t code_descriptor(unsigned address) {
    return static_cast<uint64_t>((address & 0x3ffffu) >> 4) | (uint64_t{1} << 16) | (uint64_t{64} << 32) | (uint64_t{1} << 46) | (uint64_t{2} << 61);
}
__device__ __forceinline__ uint64_t scale_descriptor(unsigned address) {
    return static_cast<uint64_t>((address & 0x3ffffu) >> 4) | (uint64_t{8} << 16) | (uint64_t{8} << 32) | (uint64_t{1} << 46);
}
// bits 4-5 / 29-30: which byte pair of the scale word (MXFP4), 7-9 and 10-12: e2m1, 17-22: N / 8, 23: e8m0 scales,
// 24-28: M / 16
template <int FORMAT>
__device__ __forceinline__ constexpr uint32_t instruction_descriptor(int m, int n) {
    return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (FORMAT == VRB_MXFP4 ? 1u << 23 : 0u) | (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ void copy_scales(uint32_t column, uint64_t descriptor) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(column), "l"(descriptor) : "memory");
}
template <int FORMAT>
__device__ __forceinline__ void multiply(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, uint32_t sa, uint32_t sb, bool add) {
    if constexpr (FORMAT == VRB_NVFP4)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                     "r"(instruction), "r"(sa), "r"(sb), "r"(add ? 1u : 0u)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                     "r"(instruction), "r"(sa), "r"(sb), "r"(add ? 1u : 0u)
                     : "memory");
}
__device__ __forceinline__ void commit(uint64_t* barrier) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(shared_address(barrier)) : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// 32 columns of this warp's 32 lanes
__device__ __forceinline__ void read_accumulator(uint32_t address, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
        "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(address));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// The tile of a linear index: bands of kBand row tiles, row tiles innermost, so that the CTAs at work share operand rows
__device__ __forceinline__ void tile_of(int64_t index, int64_t row_tiles, int64_t column_tiles, int64_t& row_tile, int64_t& column_tile) {
    const int64_t band = index / (kBand * column_tiles), first = band * kBand;
    const int64_t height = row_tiles - first < kBand ? row_tiles - first : kBand;
    const int64_t within = index - band * kBand * column_tiles;
    column_tile = within / height;
    row_tile = first + within - column_tile * height;
}

// SiLU and GELU-tanh through one exponential and one reciprocal: relative error below 2^-20, far under the bf16 step
__device__ __forceinline__ float linear_activation(float y, int kind) {
    if (kind == VRB_NO_ACTIVATION) return y;
    if (kind == VRB_SILU) return __fdividef(y, 1.0f + __expf(-y));
    if (kind == VRB_GELU_TANH) {
        const float u = 0.7978845608028654f * (y + 0.044715f * y * y * y);
        return __fdividef(y, 1.0f + __expf(-2.0f * u));
    }
    return activation_value(kind, y);
}

// 32 consecutive columns of a row of the result
__device__ __forceinline__ void write_columns(const LinearArgs& p, int64_t row, int64_t column, float alpha, float (&v)[32]) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        float b = 0.0f;
        if (p.bias && column + i < p.n) b = load1(p.bias, p.bias_dt, column + i);
        v[i] = linear_activation(fmaf(v[i], alpha, b), p.activation);
    }
    const int64_t at = row * p.n + column;
    if (p.vector_out && p.out_dt == VRB_BF16) {
#pragma unroll
        for (int i = 0; i < 32; i += 8)
            if (column + i < p.n) {
                uint4 w;
                w.x = pack_bf16x2(v[i], v[i + 1]); w.y = pack_bf16x2(v[i + 2], v[i + 3]);
                w.z = pack_bf16x2(v[i + 4], v[i + 5]); w.w = pack_bf16x2(v[i + 6], v[i + 7]);
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at + i) = w;
            }
    } else if (p.vector_out) {
#pragma unroll
        for (int i = 0; i < 32; i += 4)
            if (column + i < p.n) *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (column + i < p.n) store1(p.out, p.out_dt, at + i, v[i]);
    }
}

template <int FORMAT>
__global__ void __launch_bounds__(kThreads, 1) fp4_linear_kernel(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map, const LinearArgs p) {
    extern __shared__ uint8_t dynamic_shared[];
    __shared__ Control control;
    const unsigned buffers = (shared_address(dynamic_shared) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kPerTile = FORMAT == VRB_NVFP4 ? 64 : 128;        // elements of k of a scale tile
    constexpr int kTilesPerStage = kStageElements / kPerTile;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) { mbarrier_init(&control.full[s], 1); mbarrier_init(&control.empty[s], 1); }
        for (int i = 0; i < 2; ++i) { mbarrier_init(&control.done[i], 1); mbarrier_init(&control.drained[i], 4); }
        control.abort = 0;
        mbarrier_init_fence();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_address(&control.tensor_base)), "r"(kColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t base = control.tensor_base;
    pdl_wait();

    const int64_t row_tiles = (p.m + kTile - 1) / kTile, column_tiles = (p.n + kTile - 1) / kTile, tiles = row_tiles * column_tiles;
    const int stages = static_cast<int>((p.k + kStageElements - 1) / kStageElements);

    if (warp == 0) {
        if (lane == 0) {
            int slot = 0;
            unsigned phase = 0;
            bool ok = true;
            for (int64_t t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
                int64_t row_tile, column_tile;
                tile_of(t, row_tiles, column_tiles, row_tile, column_tile);
                for (int stage = 0; stage < stages; ++stage) {
                    if (!wait_barrier(&control.empty[slot], phase ^ 1u, &control)) { ok = false; break; }
                    const unsigned buffer = buffers + slot * kBufferBytes;
                    const int64_t first_tile = static_cast<int64_t>(stage) * kTilesPerStage;
                    const int64_t left = p.block_tiles - first_tile;
                    const unsigned scale_bytes = static_cast<unsigned>(left < kTilesPerStage ? left : kTilesPerStage) * 512u;
                    mbarrier_expect_bytes(&control.full[slot], 2 * kCodeBytes + 2 * scale_bytes);
                    tma_load_2d(buffer, &a_map, stage * kStageBytes, static_cast<int>(row_tile * kTile), &control.full[slot]);
                    tma_load_2d(buffer + kCodeBytes, &b_map, stage * kStageBytes, static_cast<int>(column_tile * kTile), &control.full[slot]);
                    bulk_load(buffer + 2 * kCodeBytes, p.a_scales + (row_tile * p.block_tiles + first_tile) * 512, scale_bytes, &control.full[slot]);
                    bulk_load(buffer + 2 * kCodeBytes + kScaleBytes, p.b_scales + (column_tile * p.block_tiles + first_tile) * 512, scale_bytes, &control.full[slot]);
                    if (++slot == kStages) { slot = 0; phase ^= 1u; }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t instruction = instruction_descriptor<FORMAT>(kTile, kTile);
            int slot = 0, accumulator = 0;
            unsigned phase = 0, drained_phase = 1;
            bool ok = true;
            for (int64_t t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
                if (!wait_barrier(&control.drained[accumulator], drained_phase, &control)) break;
                fence_after();
                const uint32_t d = base + accumulator * kTile;
                for (int stage = 0; stage < stages; ++stage) {
                    if (!wait_barrier(&control.full[slot], phase, &control)) { ok = false; break; }
                    fence_after();
                    const unsigned buffer = buffers + slot * kBufferBytes;
                    const uint32_t sa = base + kScaleColumn + slot * 32, sb = sa + 16;
                    const int64_t left = p.k - static_cast<int64_t>(stage) * kStageElements;
                    const int steps = static_cast<int>(left < kStageElements ? (left + 63) / 64 : 4);
#pragma unroll
                    for (int i = 0; i < kTilesPerStage; ++i)
                        if (i * kPerTile < steps * 64) {
                            copy_scales(sa + i * 4, scale_descriptor(buffer + 2 * kCodeBytes + i * 512));
                            copy_scales(sb + i * 4, scale_descriptor(buffer + 2 * kCodeBytes + kScaleBytes + i * 512));
                        }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (i < steps) {
                            const int word = i * 64 / kPerTile;
                            const uint32_t half = FORMAT == VRB_MXFP4 ? static_cast<uint32_t>(i & 1) * 2u : 0u;
                            multiply<FORMAT>(d, code_descriptor(buffer + i * 32), code_descriptor(buffer + kCodeBytes + i * 32),
                                             instruction | (half << 4) | (half << 29), sa + word * 4, sb + word * 4, stage > 0 || i > 0);
                        }
                    commit(&control.empty[slot]);
                    if (++slot == kStages) { slot = 0; phase ^= 1u; }
                }
                if (!ok) break;
                commit(&control.done[accumulator]);
                accumulator ^= 1;
                if (accumulator == 0) drained_phase ^= 1u;
            }
        }
    } else {
        const int quarter = warp & 3;      // the 32 tensor-memory lanes this warp may read
        const float alpha = (p.a_scale ? *p.a_scale : 1.0f) * (p.b_scale ? *p.b_scale : 1.0f);
        int accumulator = 0;
        unsigned phase = 0;
        for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
            int64_t row_tile, column_tile;
            tile_of(t, row_tiles, column_tiles, row_tile, column_tile);
            const bool arrived = wait_barrier(&control.done[accumulator], phase, &control);
            if (!__all_sync(0xffffffffu, arrived)) break;
            fence_after();
            const int64_t row = row_tile * kTile + quarter * 32 + lane;
#pragma unroll 1
            for (int c = 0; c < kTile; c += 32) {
                float v[32];
                read_accumulator(base + accumulator * kTile + c + (static_cast<uint32_t>(quarter * 32) << 16), v);
                const int64_t column = column_tile * kTile + c;
                if (row < p.m && column < p.n) write_columns(p, row, column, alpha, v);
                __syncwarp();
            }
            fence_before();
            __syncwarp();
            if (lane == 0) arrive(&control.drained[accumulator]);
            accumulator ^= 1;
            if (accumulator == 0) phase ^= 1u;
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (control.abort) {   // let copies and products in flight end before their memory goes
        const unsigned long long start = now_ns();
        for (int i = 0; i < 100000 && now_ns() - start < 20000000ull; ++i) __nanosleep(1000);
    }
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(kColumns));
}

// Codes as a two-dimensional map of bytes: box_rows rows of 128 bytes, 128-byte swizzle, zeros outside
bool encode_codes(CUtensorMap* map, const void* codes, int64_t rows, int64_t row_bytes, int box_rows) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    const Encode encode = reinterpret_cast<Encode>(tensor_map_encoder());
    if (!encode) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(row_bytes), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_bytes)};
    const cuuint32_t box[2] = {kStageBytes, static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t steps[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int FORMAT>
int launch_linear(const CUtensorMap& a, const CUtensorMap& b, const LinearArgs& p, cudaStream_t s) {
    static_assert(kSharedBytes + sizeof(Control) <= 227 * 1024, "ring does not fit shared memory");
    const cudaError_t e = cudaFuncSetAttribute(fp4_linear_kernel<FORMAT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedBytes);
    VRB_REQUIRE(e == cudaSuccess, VRB_ERR_CUDA, "CUDA error: %s (fp4_linear)", cudaGetErrorString(e));
    const int64_t tiles = ((p.m + kTile - 1) / kTile) * ((p.n + kTile - 1) / kTile);
    launch_overlapped(fp4_linear_kernel<FORMAT>, dim3(static_cast<unsigned>(grid_for(tiles, 1))), dim3(kThreads), kSharedBytes, s, a, b, p);
    return after_launch("fp4_linear");
}

}  // namespace

cudaError_t fp4_wait_failures(int* failures) { return cudaMemcpyFromSymbol(failures, g_fp4_wait_gave_up, sizeof(int)); }

}  // namespace vrb

using namespace vrb;

extern "C" int vrb_fp4_linear(int format, const void* a_codes, const void* a_scales, const float* a_tensor_scale, int64_t rows_a,
                              const void* b_codes, const void* b_scales, const float* b_tensor_scale, int64_t rows_b, int64_t k,
                              const void* bias, int bias_dtype, int activation, void* out, int out_dtype, vrb_stream stream) {
    VRB_REQUIRE(format == VRB_NVFP4 || format == VRB_MXFP4, VRB_ERR_INVALID, "fp4_linear: unknown 4-bit format %d", format);
    VRB_REQUIRE(a_codes && a_scales && b_codes && b_scales && out, VRB_ERR_INVALID, "fp4_linear: null tensor");
    VRB_REQUIRE(is_float_dtype(out_dtype) && (!bias || is_float_dtype(bias_dtype)), VRB_ERR_UNSUPPORTED, "fp4_linear: out and bias must be F32 or BF16");
    VRB_REQUIRE(rows_a > 0 && rows_b > 0 && k > 0, VRB_ERR_INVALID, "fp4_linear: rows and k must be positive");
    VRB_REQUIRE(rows_a <= INT32_MAX - 256 && rows_b <= INT32_MAX - 256 && k <= INT32_MAX - 512, VRB_ERR_INVALID, "fp4_linear: rows and k must be below 2^31 - 512");
    VRB_REQUIRE(format == VRB_NVFP4 || (!a_tensor_scale && !b_tensor_scale), VRB_ERR_INVALID, "fp4_linear: MXFP4 has no tensor scale");
    VRB_REQUIRE(activation >= VRB_NO_ACTIVATION && activation <= VRB_RELU, VRB_ERR_INVALID, "fp4_linear: unknown activation %d", activation);
    VRB_REQUIRE(aligned16(a_codes) && aligned16(a_scales) && aligned16(b_codes) && aligned16(b_scales), VRB_ERR_INVALID,
                "fp4_linear: codes and scales must be 16-byte aligned");
    LinearArgs p{};
    p.a_scales = static_cast<const uint8_t*>(a_scales); p.b_scales = static_cast<const uint8_t*>(b_scales);
    p.a_scale = a_tensor_scale; p.b_scale = b_tensor_scale;
    p.bias = bias; p.bias_dt = bias_dtype; p.out = out; p.out_dt = out_dtype; p.activation = activation;
    p.m = rows_a; p.n = rows_b; p.k = k; p.block_tiles = fp4_block_tiles(format, k);
    p.vector_out = aligned16(out) && rows_b % (16 / static_cast<int64_t>(dtype_bytes(out_dtype))) == 0;
    CUtensorMap a, b;
    VRB_REQUIRE(encode_codes(&a, a_codes, rows_a, fp4_row_bytes(k), kTile) && encode_codes(&b, b_codes, rows_b, fp4_row_bytes(k), kTile),
                VRB_ERR_UNSUPPORTED, "fp4_linear: the driver offers no tensor maps for these operands");
    return format == VRB_NVFP4 ? launch_linear<VRB_NVFP4>(a, b, p, as_stream(stream)) : launch_linear<VRB_MXFP4>(a, b, p, as_stream(stream));
}
