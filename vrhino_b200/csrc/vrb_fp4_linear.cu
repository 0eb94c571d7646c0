// The linear over packed 4-bit operands: out[m, n] = act(ga gb sum_k a[m, k] b[n, k] + bias[n]).
//
// The tensor core multiplies e2m1 elements 64 to an instruction and applies the block scales itself; they have to lie in
// tensor memory, a 32-bit word of four scales per row and column, which is the order of the packed scale tiles (one
// 32 x 128-bit copy per 128 rows x 4 blocks).
//
// Pair kernel: persistent pairs of CTAs (two SMs of a TPC) on 256 x 256 output tiles.  Each CTA holds 128 rows of a and
// 128 of b; the products read both halves, so a byte brought to an SM takes part in twice the products of a
// 128 x 128 tile, which L2 bandwidth asks for.  Eighteen warps:
//   warp 0      copies 256 elements of k at a time into a ring of buffers: codes by tensor map (128-byte swizzle,
//               zeros outside the operand), scale tiles by a map of 8-byte words
//   warp 1      of the pair's first CTA copies the scale tiles on into tensor memory and issues the products; a
//               buffer's scale columns are its own, so the buffer's barrier also guards them
//   warps 2-17  take the accumulator out of tensor memory in one go (64 registers a thread: 256 accumulator columns and
//               the scales leave no room for a second one), release it, and apply scale, bias and activation and
//               store boxes of 32 rows through shared memory while the next tile's products run
//
// Split kernel, for few rows of a (single tokens) and for results of few tiles: CTAs on 128 rows of b x 16 to 128 rows of a, b's
// rows on the accumulator's lanes so that even one row of a fills the tensor core's 128, and a cluster of up to eight CTAs
// along k, which reads the weight with as many SMs as there are.  The CTAs of a cluster put their accumulators into shared
// memory, and each adds a share of the columns over the cluster in rank order, so results do not depend on timing.
//
// Every wait is bounded: one that runs out sets a flag that the host can read and ends the CTA.
#include <cuda.h>

#include "vrb_fp4.cuh"
#include "vrb_tma.cuh"

namespace vrb {
namespace {

constexpr int kStageBytes = 128;           // bytes of codes per row and stage: 256 elements
constexpr int kStageElements = 256;
constexpr int kRows = 128;                 // operand rows of a CTA
constexpr int kCodeBytes = kRows * kStageBytes;
constexpr int kScaleBytes = 2048;          // scales of 128 rows and a stage: NVFP4 4 tiles of 512 bytes; MXFP4 uses half
constexpr int kBand = 8;                   // row tiles that share a sweep over the columns (L2 reuse)
constexpr unsigned long long kWaitNs = 2000000000ull;

__device__ int g_fp4_wait_gave_up = 0;

struct LinearArgs {
    const float* a_scale;      // tensor scales or nullptr
    const float* b_scale;
    const void* bias;
    void* out;
    int64_t m, n;
    int64_t k;
    int bias_dt, out_dt, activation;
    int boxed;                 // rows of out lie on 16-byte boundaries: stored as boxes
    int quads;                 // and on boundaries of four elements
};

__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// Waits for the phase with the given parity; false: gave up (or another warp of the CTA did).
__device__ __forceinline__ bool wait_barrier(uint64_t* barrier, unsigned parity, volatile int* abort) {
    const unsigned address = shared_address(barrier);
    unsigned long long start = 0;
    for (unsigned tries = 0;; ++tries) {
        unsigned done;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(done) : "r"(address), "r"(parity) : "memory");
        if (done) return true;
        if ((tries & 63u) == 63u) {
            if (*abort) return false;
            const unsigned long long t = now_ns();
            if (start == 0) start = t;
            else if (t - start > kWaitNs) {
                *abort = 1;
                g_fp4_wait_gave_up = 1;
                return false;
            }
        }
    }
}
// The same for a whole warp, with one outcome for all lanes: lanes may meet the limit or another warp's abort apart from each
// other, and what follows a wait (elect.sync, __syncwarp, aligned tensor-memory reads) needs all of them.  The vote costs the
// pair kernel 1 to 2 % (32760 x 1536 x 8960 with GELU 301 -> 306 us among passes); a single thread for each loop cost 2 to 4.
__device__ __forceinline__ bool wait_warp(uint64_t* barrier, unsigned parity, volatile int* abort) {
    return __all_sync(0xffffffffu, wait_barrier(barrier, parity, abort));
}
// After a wait that gave up: lets copies and products in flight end before their memory goes
__device__ __noinline__ void let_end() {
    const unsigned long long start = now_ns();
    for (int i = 0; i < 100000 && now_ns() - start < 20000000ull; ++i) __nanosleep(1000);
}
__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned map_to_rank(unsigned address, unsigned rank) {
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(address), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// Arrives on a barrier of either CTA.  CTA scope is enough: what it orders is tensor memory, by the tcgen05 fences around
// it (a release at cluster scope waits for every earlier store of the warp, 1000 to 1800 cycles a tile).
__device__ __forceinline__ void arrive_cluster(unsigned barrier_address) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(barrier_address) : "memory");
}
__device__ __forceinline__ bool elect_one() {
    unsigned r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
// into this CTA's shared memory; the barrier may lie in the other CTA of the pair
__device__ __forceinline__ void load_box(unsigned dst, const CUtensorMap* map, int x, int y, unsigned barrier_address) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(barrier_address)
                 : "memory");
}

__device__ __forceinline__ void load_own_box(unsigned dst, const CUtensorMap* map, int x, int y, unsigned barrier_address) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(barrier_address)
                 : "memory");
}

// Shared-memory operand descriptors (start address, offsets in units of 16 bytes; bit 46: descriptor version).
// Codes: rows of 128 bytes under the 128-byte swizzle, 8 rows = 1024 bytes apart.  Scale tile: 32 rows of 16 bytes, 8 rows
// = 128 bytes apart, no swizzle.
constexpr uint64_t kCodeDescriptor = (uint64_t{1} << 16) | (uint64_t{64} << 32) | (uint64_t{1} << 46) | (uint64_t{2} << 61);
constexpr uint64_t kScaleDescriptor = (uint64_t{8} << 16) | (uint64_t{8} << 32) | (uint64_t{1} << 46);
// bits 4-5 / 29-30: which byte pair of the scale word (MXFP4), 7-9 and 10-12: e2m1, 17-22: N / 8, 23: e8m0 scales,
// 24-28: M / 16
template <int FORMAT>
__host__ __device__ constexpr uint32_t instruction_descriptor(int m, int n) {
    return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (FORMAT == VRB_MXFP4 ? 1u << 23 : 0u) | (static_cast<uint32_t>(m >> 4) << 24);
}
template <int CTAS>
__device__ __forceinline__ void copy_scales(uint32_t column, uint64_t descriptor) {
    if constexpr (CTAS == 2) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(column), "l"(descriptor) : "memory");
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(column), "l"(descriptor) : "memory");
}
template <int FORMAT, int CTAS>
__device__ __forceinline__ void multiply(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, uint32_t sa, uint32_t sb, uint32_t add) {
#define VRB_MMA(GROUP, KIND)                                                                                                          \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\ttcgen05.mma.cta_group::" GROUP ".kind::" KIND                        \
                 " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(instruction), "r"(sa), "r"(sb), "r"(add) : "memory")
    if constexpr (FORMAT == VRB_NVFP4 && CTAS == 2) VRB_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X");
    else if constexpr (FORMAT == VRB_NVFP4) VRB_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X");
    else if constexpr (CTAS == 2) VRB_MMA("2", "mxf4.block_scale.scale_vec::2X");
    else VRB_MMA("1", "mxf4.block_scale.scale_vec::2X");
#undef VRB_MMA
}
__device__ __forceinline__ void commit_one(uint64_t* barrier) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(shared_address(barrier)) : "memory");
}
__device__ __forceinline__ void commit_pair(uint64_t* barrier) {   // arrives on the barrier at this offset in both CTAs
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(shared_address(barrier)),
                 "h"(static_cast<uint16_t>(3))
                 : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// 32 columns of this warp's 32 lanes into v[0 .. 32); completes with wait_reads()
__device__ __forceinline__ void read_columns(uint32_t address, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
        "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(address));
}
__device__ __forceinline__ void read_columns16(uint32_t address, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(address));
}
__device__ __forceinline__ void wait_reads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// The tile of a linear index: bands of kBand row tiles, row tiles innermost, so that the CTAs at work share operand rows
__device__ __forceinline__ void tile_of(unsigned index, unsigned row_tiles, unsigned column_tiles, unsigned& row_tile, unsigned& column_tile) {
    const unsigned band = index / (kBand * column_tiles), first = band * kBand;
    const unsigned height = min(row_tiles - first, static_cast<unsigned>(kBand)), within = index - band * kBand * column_tiles;
    column_tile = within / height;
    row_tile = first + within - column_tile * height;
}

// ACT: 0 none, 1 SiLU and 2 GELU-tanh for bf16 results, 3 any other kind, 4 and 5 as 1 and 2 for F32 results.  v[0 .. N) =
// act(alpha * v + bias); without an activation the product is rounded to F32 before the bias is added, so that the result has the
// bits of vrb_linear_output on the stored accumulation.  bias: F32 in shared memory or nullptr.
template <int ACT, int N>
__device__ __forceinline__ void finish_columns(float* v, const float* bias, float alpha, int kind) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        float4 b = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (bias) b = *reinterpret_cast<const float4*>(bias + i);
        unsigned long long lo, hi;
        if constexpr (ACT == 0 || ACT == 3) {
            lo = add_f32x2(pack_f32x2(__fmul_rn(v[i], alpha), __fmul_rn(v[i + 1], alpha)), pack_f32x2(b.x, b.y));
            hi = add_f32x2(pack_f32x2(__fmul_rn(v[i + 2], alpha), __fmul_rn(v[i + 3], alpha)), pack_f32x2(b.z, b.w));
        } else {
            lo = fma_f32x2(pack_f32x2(v[i], v[i + 1]), pack_f32x2(alpha, alpha), pack_f32x2(b.x, b.y));
            hi = fma_f32x2(pack_f32x2(v[i + 2], v[i + 3]), pack_f32x2(alpha, alpha), pack_f32x2(b.z, b.w));
        }
        if constexpr (ACT == 1 || ACT == 2) {
            gate_pair<ACT, true>(lo, v[i], v[i + 1]);
            gate_pair<ACT, true>(hi, v[i + 2], v[i + 3]);
        } else {
            unpack_f32x2(lo, v[i], v[i + 1]);
            unpack_f32x2(hi, v[i + 2], v[i + 3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (ACT == 3) v[i + e] = activation_value(kind, v[i + e]);
                if constexpr (ACT > 3) v[i + e] = gate_value<ACT - 3>(v[i + e]);
            }
        }
    }
}
// The product of the tensor scales as two factors: accumulations take `before` (1 as a rule) ahead of `alpha`.  Where the product
// leaves F32's normal range, as that of two ordinary scales can, the larger scale comes first: what it makes overflow the smaller
// one, above 1 then, does not bring back, and only the last product falls below the normal range.
struct Scale {
    float before, alpha;
};
__device__ __forceinline__ Scale tensor_scale(const float* a, const float* b) {
    const float ga = a ? *a : 1.0f, gb = b ? *b : 1.0f, product = __fmul_rn(ga, gb);
    if ((product < 1.17549435e-38f || product > 3.402823466e38f) && ga != 0.0f && gb != 0.0f) return {fmaxf(ga, gb), fminf(ga, gb)};
    return {1.0f, product};
}
// 64 bytes of this lane's row into the warp's box of 32 rows (64-byte swizzle: 16-byte pieces by bits 1-2 of the row)
__device__ __forceinline__ void stage_row(unsigned box, int lane, const uint32_t (&w)[16]) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(box + lane * 64 + ((c ^ (lane >> 1 & 3)) << 4)), "r"(w[4 * c]), "r"(w[4 * c + 1]),
                     "r"(w[4 * c + 2]), "r"(w[4 * c + 3])
                     : "memory");
}
__device__ __forceinline__ void store_box(const CUtensorMap* map, int x, int y, unsigned box) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(box)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// ------------------------------------------------------------------------------------- pair kernel --
constexpr int kPairThreads = 576;
constexpr int kPairTile = 256;
constexpr int kPairStages = 5;
constexpr int kPairBufferBytes = 2 * kCodeBytes + 3 * kScaleBytes;   // a codes, b codes, a scales, b scales of all 256 columns
constexpr int kPairColumns = 512;          // tensor memory: 256 accumulator columns, then 48 scale columns a buffer
constexpr int kPairScaleColumns = 48;
constexpr int kWriters = 16;               // warps that write results: 32 rows x 64 columns of a tile each
constexpr int kWriterColumns = 64;
constexpr int kBoxBytes = 32 * 64;         // a stored box: 32 rows of 64 bytes
static_assert(kPairTile + kPairStages * kPairScaleColumns <= kPairColumns, "scales do not fit tensor memory");

struct PairControl {
    uint64_t full[kPairStages], empty[kPairStages], done, drained;
    uint32_t tensor_base;
    volatile int abort;
};
struct __align__(1024) PairShared {        // fills an SM's shared memory, so it may not need room for alignment
    uint8_t buffers[kPairStages][kPairBufferBytes];
    uint8_t boxes[kWriters][kBoxBytes];
    float bias[kWriters][kWriterColumns];
    PairControl control;
};

template <int FORMAT, int ACT, int OUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
fp4_linear_pair_kernel(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map,
                       const __grid_constant__ CUtensorMap a_scale_map, const __grid_constant__ CUtensorMap b_scale_map,
                       const __grid_constant__ CUtensorMap out_map, const LinearArgs p) {
    extern __shared__ __align__(1024) uint8_t dynamic_shared[];
    PairShared& shared = *reinterpret_cast<PairShared*>(dynamic_shared);
    PairControl& control = shared.control;
    const unsigned buffers = shared_address(dynamic_shared);
    if ((buffers & 1023u) != 0) {   // the same for every thread of the launch: no static shared memory precedes it
        g_fp4_wait_gave_up = 1;
        return;
    }
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;   // known to be the same for a warp
    const unsigned rank = cluster_rank();
    constexpr int kPerTile = FORMAT == VRB_NVFP4 ? 64 : 128;        // elements of k of a scale tile
    constexpr int kTiles = kStageElements / kPerTile;               // scale tiles of 128 rows a stage
    constexpr unsigned kStageTotal = 2 * kCodeBytes + 3 * kTiles * 512;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairStages; ++s) { mbarrier_init(&control.full[s], 1); mbarrier_init(&control.empty[s], 1); }
        mbarrier_init(&control.done, 1);
        mbarrier_init(&control.drained, 2 * kWriters);
        control.abort = 0;
        mbarrier_init_fence();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_address(&control.tensor_base)), "r"(kPairColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    cluster_sync();
    fence_after();
    const uint32_t base = control.tensor_base;
    pdl_wait();

    const unsigned row_tiles = static_cast<unsigned>((p.m + kPairTile - 1) / kPairTile), column_tiles = static_cast<unsigned>((p.n + kPairTile - 1) / kPairTile);
    const unsigned tiles = row_tiles * column_tiles;
    const int stages = static_cast<int>((p.k + kStageElements - 1) / kStageElements);
    const unsigned pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (warp == 0) {
        int slot = 0;
        unsigned phase = 1;
        bool ok = true;
        for (unsigned t = pair; ok && t < tiles; t += pairs) {
            unsigned row_tile, column_tile;
            tile_of(t, row_tiles, column_tiles, row_tile, column_tile);
            for (int stage = 0; stage < stages; ++stage) {
                if (!wait_warp(&control.empty[slot], phase, &control.abort)) { ok = false; break; }
                if (elect_one()) {
                    const unsigned buffer = buffers + slot * kPairBufferBytes;
                    const unsigned full = map_to_rank(shared_address(&control.full[slot]), 0);
                    if (rank == 0) mbarrier_expect_bytes(&control.full[slot], 2 * kStageTotal);
                    load_box(buffer, &a_map, stage * kStageBytes, static_cast<int>(row_tile * kPairTile + rank * kRows), full);
                    load_box(buffer + kCodeBytes, &b_map, stage * kStageBytes, static_cast<int>(column_tile * kPairTile + rank * kRows), full);
                    load_box(buffer + 2 * kCodeBytes, &a_scale_map, stage * kTiles * 64, static_cast<int>(row_tile * 2 + rank), full);
                    load_box(buffer + 2 * kCodeBytes + kScaleBytes, &b_scale_map, stage * kTiles * 64, static_cast<int>(column_tile * 2), full);
                }
                __syncwarp();
                if (++slot == kPairStages) { slot = 0; phase ^= 1u; }
            }
        }
        // the last products' arrivals on the barriers of empty buffers: none may be under way when the CTA ends
        for (int left = kPairStages; ok && left > 0; --left) {
            ok = wait_warp(&control.empty[slot], phase, &control.abort);
            if (++slot == kPairStages) { slot = 0; phase ^= 1u; }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            constexpr uint32_t instruction = instruction_descriptor<FORMAT>(kPairTile, kPairTile);
            int slot = 0;
            unsigned phase = 0, drained_phase = 1;
            bool ok = true;
            for (unsigned t = pair; ok && t < tiles; t += pairs) {
                if (!wait_warp(&control.drained, drained_phase, &control.abort)) break;
                drained_phase ^= 1u;
                fence_after();
                for (int stage = 0; stage < stages; ++stage) {
                    if (!wait_warp(&control.full[slot], phase, &control.abort)) { ok = false; break; }
                    fence_after();
                    if (elect_one()) {
                        const unsigned buffer = buffers + slot * kPairBufferBytes;
                        const uint32_t sa = base + kPairTile + slot * kPairScaleColumns, sb = sa + 16;
                        const uint64_t codes = kCodeDescriptor | ((buffer & 0x3ffffu) >> 4);
                        const uint64_t scales = kScaleDescriptor | (((buffer + 2 * kCodeBytes) & 0x3ffffu) >> 4);
                        const int64_t left = p.k - static_cast<int64_t>(stage) * kStageElements;
                        const int steps = left < kStageElements ? static_cast<int>((left + 63) / 64) : 4;
                        // scale tiles past the operand are zeros: copied all the same
#pragma unroll
                        for (int i = 0; i < kTiles; ++i) {
                            copy_scales<2>(sa + i * 4, scales + i * 32);
                            copy_scales<2>(sb + i * 8, scales + (kScaleBytes >> 4) + i * 32);
                            copy_scales<2>(sb + i * 8 + 4, scales + (kScaleBytes >> 4) + kTiles * 32 + i * 32);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (i < steps) {
                                constexpr int per = kPerTile / 64;
                                const uint32_t half = FORMAT == VRB_MXFP4 ? static_cast<uint32_t>(i & 1) * 2u : 0u;
                                multiply<FORMAT, 2>(base, codes + i * 2, codes + (kCodeBytes >> 4) + i * 2, instruction | (half << 4) | (half << 29),
                                                    sa + i / per * 4, sb + i / per * 8, (stage | i) != 0 ? 1u : 0u);
                            }
                        commit_pair(&control.empty[slot]);
                        if (stage == stages - 1) commit_pair(&control.done);
                    }
                    __syncwarp();
                    if (++slot == kPairStages) { slot = 0; phase ^= 1u; }
                }
            }
        }
    } else {
        const int quarter = warp & 3;                  // the 32 tensor-memory lanes this warp may read
        const int writer = warp - 2, group = writer >> 2;   // its 64 of the columns
        const Scale scale = tensor_scale(p.a_scale, p.b_scale);
        const unsigned box = shared_address(shared.boxes[writer]);
        float* scratch = reinterpret_cast<float*>(shared.boxes[writer]);
        float* bias = shared.bias[writer];
        const unsigned drained = map_to_rank(shared_address(&control.drained), 0);
        unsigned phase = 0;
        for (unsigned t = pair; t < tiles; t += pairs) {
            unsigned row_tile, column_tile;
            tile_of(t, row_tiles, column_tiles, row_tile, column_tile);
            const int64_t column0 = static_cast<int64_t>(column_tile) * kPairTile + group * kWriterColumns;
            if (p.bias) {   // before the wait: the loads are over when the accumulator is
                __syncwarp();
#pragma unroll
                for (int c = 0; c < kWriterColumns; c += 32) bias[c + lane] = column0 + c + lane < p.n ? load1(p.bias, p.bias_dt, column0 + c + lane) : 0.0f;
            }
            if (!wait_warp(&control.done, phase, &control.abort)) break;
            phase ^= 1u;
            fence_after();
            float v[kWriterColumns];
            const uint32_t address = base + group * kWriterColumns + (static_cast<uint32_t>(quarter * 32) << 16);
            read_columns(address, v);
            read_columns(address + 32, v + 32);
            wait_reads();
            fence_before();
            __syncwarp();
            if (lane == 0) arrive_cluster(drained);
            if (scale.before != 1.0f)
#pragma unroll
                for (int c = 0; c < kWriterColumns; ++c) v[c] *= scale.before;
            const int64_t row0 = static_cast<int64_t>(row_tile) * kPairTile + rank * kRows + quarter * 32;
            if (p.boxed) {
                constexpr int N = OUT == VRB_BF16 ? 32 : 16;   // columns of a box
#pragma unroll
                for (int c = 0; c < kWriterColumns; c += N) {
                    finish_columns<ACT, N>(v + c, p.bias ? bias + c : nullptr, scale.alpha, p.activation);
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) w[i] = OUT == VRB_BF16 ? pack_bf16x2(v[c + 2 * i % N], v[c + (2 * i + 1) % N]) : __float_as_uint(v[c + i % N]);
                    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // the last store has read the box
                    __syncwarp();
                    stage_row(box, lane, w);
                    async_proxy_fence();
                    __syncwarp();
                    if (lane == 0 && row0 < p.m && column0 + c < p.n) store_box(&out_map, static_cast<int>(column0 + c), static_cast<int>(row0), box);
                }
            } else {
                // rows off the 16-byte boundaries that a box needs: through scratch, 16 columns at a time, a lane to a column and
                // every other row
                const int height = static_cast<int>(p.m - row0 < 32 ? p.m - row0 : 32);
#pragma unroll
                for (int c = 0; c < kWriterColumns; c += 16) {
                    finish_columns<ACT, 16>(v + c, p.bias ? bias + c : nullptr, scale.alpha, p.activation);
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 16; ++i) scratch[lane * 16 + (i ^ (lane >> 1 & 15))] = v[c + i];
                    __syncwarp();
                    const int64_t column = column0 + c + (lane & 15);
                    if (column < p.n)
                        for (int r = lane >> 4; r < height; r += 2) store1(p.out, OUT, (row0 + r) * p.n + column, scratch[r * 16 + ((lane & 15) ^ (r >> 1 & 15))]);
                }
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (control.abort) let_end();
    cluster_sync();        // the other CTA's products and arrivals reach into this one
    fence_after();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(kPairColumns));
}

// ------------------------------------------------------------------------------------ split kernel --
constexpr int kSplitThreads = 192;
constexpr int kSplitRing = 6;
constexpr int kMostSplits = kMostCluster;
constexpr size_t kSharedPerSm = 228 * 1024, kSharedPerCta = 1024;   // 1 KB of each CTA's is the system's
constexpr int kTensorColumns = 512;        // of an SM
constexpr int kSplitMostColumns = 256;     // of them for a CTA of the split kernel
constexpr size_t kSplitMostShared = kSplitRing * (kCodeBytes + 2 * kScaleBytes + 64 * kStageBytes) + 1024;   // six buffers of 64 columns; four of 128 take less

struct SplitArgs {
    LinearArgs linear;
    int columns;               // rows of a of a tile: 16, 32, 64 or 128
    int tensor_columns;        // tensor memory: the accumulator's columns (32 at least), then 32 scale columns a buffer; a power of two
    int ring;                  // buffers
    int splits;                // CTAs along k: the cluster
    int stages;                // of all of k
    unsigned a_tiles;
};
struct SplitControl {
    uint64_t full[kSplitRing], empty[kSplitRing], done;
    uint32_t tensor_base;
    volatile int abort;
};

__device__ __forceinline__ float4 load_cluster(unsigned address) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(address));
    return v;
}
template <int FORMAT, int ACT>
__global__ void __launch_bounds__(kSplitThreads, 1)
fp4_linear_split_kernel(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map,
                        const __grid_constant__ CUtensorMap a_scale_map, const __grid_constant__ CUtensorMap b_scale_map, const SplitArgs q) {
    extern __shared__ uint8_t dynamic_shared[];
    __shared__ SplitControl control;
    const LinearArgs& p = q.linear;
    const unsigned buffers = (shared_address(dynamic_shared) + 1023u) & ~1023u;
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;   // known to be the same for a warp
    constexpr int kPerTile = FORMAT == VRB_NVFP4 ? 64 : 128;
    constexpr int kTiles = kStageElements / kPerTile;
    const unsigned a_bytes = q.columns * kStageBytes, buffer_bytes = kCodeBytes + 2 * kScaleBytes + ((a_bytes + 1023u) & ~1023u);
    if (threadIdx.x == 0) {
        for (int s = 0; s < kSplitRing; ++s) { mbarrier_init(&control.full[s], 1); mbarrier_init(&control.empty[s], 1); }
        mbarrier_init(&control.done, 1);
        control.abort = 0;
        mbarrier_init_fence();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_address(&control.tensor_base)), "r"(q.tensor_columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t base = control.tensor_base;
    pdl_wait();

    // blockIdx.x = (column tile of b * tiles of a + tile of a) * splits + rank
    const int rank = static_cast<int>(blockIdx.x % q.splits);
    const unsigned tile = blockIdx.x / q.splits;
    const int64_t b0 = static_cast<int64_t>(tile / q.a_tiles) * kRows, a0 = static_cast<int64_t>(tile % q.a_tiles) * q.columns;
    const int first = static_cast<int>(static_cast<unsigned>(q.stages) * rank / q.splits), last = static_cast<int>(static_cast<unsigned>(q.stages) * (rank + 1) / q.splits);

    if (warp == 0) {
        int slot = 0;
        unsigned phase = 1;
        bool ok = true;
        for (int stage = first; stage < last; ++stage) {
            if (!wait_warp(&control.empty[slot], phase, &control.abort)) { ok = false; break; }
            if (elect_one()) {
                const unsigned buffer = buffers + slot * buffer_bytes, full = shared_address(&control.full[slot]);
                mbarrier_expect_bytes(&control.full[slot], kCodeBytes + a_bytes + 2 * kTiles * 512);
                load_own_box(buffer, &b_map, stage * kStageBytes, static_cast<int>(b0), full);
                load_own_box(buffer + kCodeBytes, &b_scale_map, stage * kTiles * 64, static_cast<int>(b0 / 128), full);
                load_own_box(buffer + kCodeBytes + kScaleBytes, &a_scale_map, stage * kTiles * 64, static_cast<int>(a0 / 128), full);
                load_own_box(buffer + kCodeBytes + 2 * kScaleBytes, &a_map, stage * kStageBytes, static_cast<int>(a0), full);
            }
            __syncwarp();
            if (++slot == q.ring) { slot = 0; phase ^= 1u; }
        }
        for (int left = q.ring; ok && left > 0; --left) {   // as in the pair kernel
            ok = wait_warp(&control.empty[slot], phase, &control.abort);
            if (++slot == q.ring) { slot = 0; phase ^= 1u; }
        }
    } else if (warp == 1) {
        const uint32_t instruction = instruction_descriptor<FORMAT>(kRows, q.columns);
        const uint32_t scales_base = base + max(q.columns, 32);
        const uint32_t a_column = static_cast<uint32_t>(a0 % 128) / 32;   // where the tile's scales begin within the 128-row scale tile
        int slot = 0;
        unsigned phase = 0;
        // one thread for the whole loop: electing one a stage takes as long as the products of a narrow tile
        if (elect_one()) for (int stage = first; stage < last; ++stage) {
            if (!wait_barrier(&control.full[slot], phase, &control.abort)) break;
            fence_after();
            const unsigned buffer = buffers + slot * buffer_bytes;
            const uint32_t sb = scales_base + slot * 32, sa = sb + 16;
            const uint64_t b_codes = kCodeDescriptor | ((buffer & 0x3ffffu) >> 4), a_codes = b_codes + ((kCodeBytes + 2 * kScaleBytes) >> 4);
            const uint64_t scales = kScaleDescriptor | (((buffer + kCodeBytes) & 0x3ffffu) >> 4);
            const int64_t left = p.k - static_cast<int64_t>(stage) * kStageElements;
            const int steps = left < kStageElements ? static_cast<int>((left + 63) / 64) : 4;
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
                copy_scales<1>(sb + i * 4, scales + i * 32);
                copy_scales<1>(sa + i * 4, scales + (kScaleBytes >> 4) + i * 32);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < steps) {
                    constexpr int per = kPerTile / 64;
                    const uint32_t half = FORMAT == VRB_MXFP4 ? static_cast<uint32_t>(i & 1) * 2u : 0u;
                    multiply<FORMAT, 1>(base, b_codes + i * 2, a_codes + i * 2, instruction | (half << 4) | (half << 29), sb + i / per * 4,
                                        sa + i / per * 4 + a_column, stage > first || i > 0 ? 1u : 0u);
                }
            commit_one(&control.empty[slot]);
            if (stage == last - 1) commit_one(&control.done);
            if (++slot == q.ring) { slot = 0; phase ^= 1u; }
        }
    }
    const int height = static_cast<int>(p.m - a0 < q.columns ? p.m - a0 : q.columns);
    const int64_t n0 = b0 + lane * 4;                  // the four rows of b that this thread finishes
    const Scale scale = tensor_scale(p.a_scale, p.b_scale);
    __align__(16) float bias[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = p.bias && n0 + e < p.n ? load1(p.bias, p.bias_dt, n0 + e) : 0.0f;
    if (warp >= 2 && wait_warp(&control.done, 0, &control.abort)) {
        // all copies into the ring and all products out of it are over: its memory takes the accumulator, 128 floats a column
        fence_after();
        const unsigned mine = buffers + ((warp & 3) * 32 + lane) * 4;       // the tensor-memory lane is the row of b
        for (int c = 0; c < height; c += 16) {
            float v[16];
            read_columns16(base + (static_cast<uint32_t>((warp & 3) * 32) << 16) + c, v);
            wait_reads();
#pragma unroll
            for (int i = 0; i < 16; ++i) asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine + (c + i) * 512), "f"(v[i]) : "memory");
        }
    }
    // Tensor memory goes back before the cluster meets: a CTA that held it while it waited for the others could wait for good, where
    // one of those waits for the tensor memory of another kernel's cluster, which waits for this CTA's.
    __syncwarp();
    fence_before();
    __syncthreads();
    if (control.abort) let_end();
    fence_after();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(q.tensor_columns));
    if (q.splits > 1) cluster_sync();
    // this CTA's share of the columns, four columns x four rows of b to a thread: a warp writes 128 consecutive elements of four
    // rows of the result, and the loads of four columns from four CTAs are in flight together
    const int share = (height + q.splits * 4 - 1) / (q.splits * 4) * 4, begin = rank * share, end = min(height, begin + share);
    if (n0 < p.n && !control.abort) {
#pragma unroll 1
        for (int c = begin + warp * 4; c < end; c += kSplitThreads / 32 * 4) {
            float y[4][4] = {};
            const unsigned offset = (c * 128 + lane * 4) * 4;   // columns up to a multiple of 16 hold memory, if no values
#pragma unroll 1
            for (int r = 0; r < q.splits; r += 4) {
                float4 part[4][4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (r + k < q.splits) {
                        const unsigned from = map_to_rank(buffers, q.splits > 1 ? r + k : cluster_rank()) + offset;
#pragma unroll
                        for (int i = 0; i < 4; ++i) part[k][i] = load_cluster(from + i * 512);
                    }
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (r + k < q.splits)
#pragma unroll
                        for (int i = 0; i < 4; ++i) { y[i][0] += part[k][i].x; y[i][1] += part[k][i].y; y[i][2] += part[k][i].z; y[i][3] += part[k][i].w; }
            }
            int64_t at = (a0 + c) * p.n + n0;
#pragma unroll
            for (int i = 0; i < 4; ++i, at += p.n) {
                if (scale.before != 1.0f)
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[i][e] *= scale.before;
                finish_columns<ACT, 4>(y[i], bias, scale.alpha, p.activation);
                if (c + i >= end) break;
                if (p.quads && p.out_dt == VRB_BF16) {
                    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = make_uint2(pack_bf16x2(y[i][0], y[i][1]), pack_bf16x2(y[i][2], y[i][3]));
                } else if (p.quads) {
                    *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = make_float4(y[i][0], y[i][1], y[i][2], y[i][3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (n0 + e < p.n) store1(p.out, p.out_dt, at + e, y[i][e]);
                }
            }
        }
    }
    __syncwarp();
    if (q.splits > 1) cluster_sync();   // no CTA's memory goes while another reads it
}

// ----------------------------------------------------------------------------------------- host side --
using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                            const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

bool encode_2d(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t inner, int64_t outer, int64_t row_bytes, int box_inner, int box_outer,
               CUtensorMapSwizzle swizzle) {
    const Encode encode = reinterpret_cast<Encode>(tensor_map_encoder());
    if (!encode) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_bytes)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_inner), static_cast<cuuint32_t>(box_outer)};
    const cuuint32_t steps[2] = {1, 1};
    return encode(map, type, 2, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Codes as rows of bytes: box_rows rows of 128 bytes, 128-byte swizzle, zeros outside
bool encode_codes(CUtensorMap* map, const void* codes, int64_t rows, int64_t k, int box_rows) {
    return encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, fp4_row_bytes(k), rows, fp4_row_bytes(k), kStageBytes, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}
// Scale tiles as 8-byte words, a row of tiles for every 128 operand rows; a box holds a stage's tiles of box_rows rows
bool encode_scales(CUtensorMap* map, int format, const void* scales, int64_t rows, int64_t k, int box_rows) {
    const int64_t tiles = fp4_block_tiles(format, k), per_stage = format == VRB_NVFP4 ? 4 : 2;
    return encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT64, scales, tiles * 64, (rows + 127) / 128, tiles * 512, static_cast<int>(per_stage * 64), box_rows,
                     CU_TENSOR_MAP_SWIZZLE_NONE);
}

struct LinearMaps {
    CUtensorMap a, b, a_scales, b_scales, out;
};

template <int FORMAT, int ACT, int OUT>
int launch_pair(const LinearMaps& maps, const LinearArgs& p, cudaStream_t s) {
    static_assert(sizeof(PairShared) <= 227 * 1024, "ring does not fit shared memory");
    static std::atomic<uint64_t> allowed{0};
    if (int rc = allow_shared(fp4_linear_pair_kernel<FORMAT, ACT, OUT>, sizeof(PairShared), allowed, "fp4_linear")) return rc;
    const int64_t tiles = ((p.m + kPairTile - 1) / kPairTile) * ((p.n + kPairTile - 1) / kPairTile), pairs = sm_count() / 2;
    launch_overlapped(fp4_linear_pair_kernel<FORMAT, ACT, OUT>, dim3(static_cast<unsigned>(2 * (tiles < pairs ? tiles : pairs))), dim3(kPairThreads),
                      sizeof(PairShared), s, maps.a, maps.b, maps.a_scales, maps.b_scales, maps.out, p);
    return after_launch("fp4_linear");
}
// Which kernel, and the split kernel's tile and cluster: the least of the times that a model gives, in nanoseconds, fitted to
// both kernels on B200 (back to back in a graph; the choice is within 3 % of the best on 24 shapes from 1 x 512 x 512
// to 4000 x 6000 and to k past 30000), with operands that L2 held: a weight that comes from HBM takes longer a stage (18 KB a CTA in
// 265 ns are 10 TB/s over the SMs), and the choice of clusters for it is not measured.  Pair kernel: 4300 + 500 a tile + 290 a stage.  Split kernel: 2300 + 19 a column
// of the tile + 265 a stage, and 800 + 130 a CTA to meet in a cluster; one CTA to an SM, what does not fit at once takes turns.
struct LinearPlan {
    int columns;   // 0: pair kernel
    int splits;
};
LinearPlan plan_linear(int64_t m, int64_t n, int stages) {
    auto ceil_div = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    LinearPlan best{0, 1};
    const int64_t pair_tiles = ceil_div(m, kPairTile) * ceil_div(n, kPairTile), pairs = sm_count() / 2 > 0 ? sm_count() / 2 : 1;
    int64_t least = 4300 + ceil_div(pair_tiles, pairs) * (static_cast<int64_t>(stages) * 290 + 500);
    const int* room = cluster_room(reinterpret_cast<const void*>(fp4_linear_split_kernel<VRB_NVFP4, 0>), kSplitThreads, kSplitMostShared);
    for (int columns = 16; columns <= 128; columns *= 2) {
        if (columns <= 32 && m > columns) continue;   // tiles narrower than 64 would begin inside a scale word's lanes
        const int64_t tiles = ceil_div(m, columns) * ceil_div(n, kRows);
        for (int splits = 1; splits <= kMostSplits && splits <= stages; ++splits) {
            const int64_t time = ceil_div(tiles * splits, room[splits]) * (2300 + columns * 19 + ceil_div(stages, splits) * 265 + (splits > 1 ? 800 + 130 * splits : 0));
            if (time < least) { least = time; best = {columns, splits}; }
        }
        if (m <= columns) break;
    }
    return best;
}

template <int FORMAT, int ACT>
int launch_split(const LinearMaps& maps, const LinearArgs& p, const LinearPlan& plan, cudaStream_t s) {
    SplitArgs q{};
    q.linear = p;
    q.columns = plan.columns;
    q.splits = plan.splits;
    q.stages = static_cast<int>((p.k + kStageElements - 1) / kStageElements);
    q.a_tiles = static_cast<unsigned>((p.m + q.columns - 1) / q.columns);
    const int own = (q.stages + q.splits - 1) / q.splits;
    const int accumulator = q.columns < 32 ? 32 : q.columns, most = (kSplitMostColumns - accumulator) / 32;   // three buffers do as well as six, given time
    q.ring = own < kSplitRing ? own : kSplitRing;
    if (q.ring > most) q.ring = most;
    const size_t buffer = kCodeBytes + 2 * kScaleBytes + ((static_cast<size_t>(q.columns) * kStageBytes + 1023) & ~size_t{1023});
    size_t bytes = q.ring * buffer;
    if (bytes < static_cast<size_t>(q.columns) * 512) bytes = static_cast<size_t>(q.columns) * 512;
    bytes += 1024;
    // A CTA takes at least the share of an SM's shared memory that it takes of the tensor memory (as the pair kernel does, with
    // all of both).  So whatever CTAs of these kernels share an SM, from one launch or several streams, no tensor memory
    // allocation ever waits for another CTA of these kernels.
    q.tensor_columns = 32;
    while (q.tensor_columns < accumulator + 32 * q.ring) q.tensor_columns *= 2;
    const size_t share = kSharedPerSm * q.tensor_columns / kTensorColumns;
    if (bytes + kSharedPerCta < share) bytes = share - kSharedPerCta;
    static_assert(kSplitMostShared + sizeof(SplitControl) <= 227 * 1024, "ring does not fit shared memory");
    static_assert(kSplitMostShared + kSharedPerCta >= kSharedPerSm * kSplitMostColumns / kTensorColumns &&
                      kSplitMostShared >= (kSplitMostColumns - 128) / 32 * (2 * kCodeBytes + 2 * kScaleBytes) + 1024,
                  "the most shared memory covers the most tensor memory and the widest tile");
    static std::atomic<uint64_t> allowed{0};
    if (int rc = allow_shared(fp4_linear_split_kernel<FORMAT, ACT>, kSplitMostShared, allowed, "fp4_linear")) return rc;
    const int64_t tiles = ((p.m + q.columns - 1) / q.columns) * ((p.n + kRows - 1) / kRows);
    launch_clusters(fp4_linear_split_kernel<FORMAT, ACT>, dim3(static_cast<unsigned>(tiles * q.splits)), dim3(kSplitThreads), bytes, q.splits, s, maps.a, maps.b, maps.a_scales,
                    maps.b_scales, q);
    return after_launch("fp4_linear");
}

template <int FORMAT>
int launch_split(const LinearMaps& maps, const LinearArgs& p, const LinearPlan& plan, cudaStream_t s) {
    if (p.activation == VRB_NO_ACTIVATION) return launch_split<FORMAT, 0>(maps, p, plan, s);
    const bool f32 = p.out_dt == VRB_F32;
    if (p.activation == VRB_SILU) return f32 ? launch_split<FORMAT, 4>(maps, p, plan, s) : launch_split<FORMAT, 1>(maps, p, plan, s);
    if (p.activation == VRB_GELU_TANH) return f32 ? launch_split<FORMAT, 5>(maps, p, plan, s) : launch_split<FORMAT, 2>(maps, p, plan, s);
    return launch_split<FORMAT, 3>(maps, p, plan, s);
}

template <int FORMAT, int OUT>
int launch_linear(const LinearMaps& maps, const LinearArgs& p, cudaStream_t s) {
    if (p.activation == VRB_NO_ACTIVATION) return launch_pair<FORMAT, 0, OUT>(maps, p, s);
    if (p.activation == VRB_SILU) return launch_pair<FORMAT, OUT == VRB_F32 ? 4 : 1, OUT>(maps, p, s);
    if (p.activation == VRB_GELU_TANH) return launch_pair<FORMAT, OUT == VRB_F32 ? 5 : 2, OUT>(maps, p, s);
    return launch_pair<FORMAT, 3, OUT>(maps, p, s);
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
    VRB_REQUIRE(rows_a <= (int64_t{1} << 40) / rows_b, VRB_ERR_INVALID, "fp4_linear: the result may have at most 2^40 elements");
    VRB_REQUIRE(format == VRB_NVFP4 || (!a_tensor_scale && !b_tensor_scale), VRB_ERR_INVALID, "fp4_linear: MXFP4 has no tensor scale");
    VRB_REQUIRE(activation >= VRB_NO_ACTIVATION && activation <= VRB_RELU, VRB_ERR_INVALID, "fp4_linear: unknown activation %d", activation);
    VRB_REQUIRE(aligned16(a_codes) && aligned16(a_scales) && aligned16(b_codes) && aligned16(b_scales), VRB_ERR_INVALID,
                "fp4_linear: codes and scales must be 16-byte aligned");
    VRB_REQUIRE(aligned_to(out, dtype_bytes(out_dtype)) && (!bias || aligned_to(bias, dtype_bytes(bias_dtype))) && aligned_to(a_tensor_scale, 4) &&
                    aligned_to(b_tensor_scale, 4),
                VRB_ERR_INVALID, "fp4_linear: tensors must be aligned to their elements");
    LinearArgs p{};
    p.a_scale = a_tensor_scale; p.b_scale = b_tensor_scale;
    p.bias = bias; p.bias_dt = bias_dtype; p.out = out; p.out_dt = out_dtype; p.activation = activation;
    p.m = rows_a; p.n = rows_b; p.k = k;
    const int64_t element = static_cast<int64_t>(dtype_bytes(out_dtype));
    p.boxed = aligned16(out) && rows_b * element % 16 == 0;
    p.quads = reinterpret_cast<uintptr_t>(out) % (4 * element) == 0 && rows_b % 4 == 0;
    const LinearPlan plan = plan_linear(rows_a, rows_b, static_cast<int>((k + kStageElements - 1) / kStageElements));
    const bool pair = plan.columns == 0;
    LinearMaps maps{};
    VRB_REQUIRE(encode_codes(&maps.a, a_codes, rows_a, k, pair ? kRows : plan.columns) && encode_codes(&maps.b, b_codes, rows_b, k, kRows) &&
                    encode_scales(&maps.a_scales, format, a_scales, rows_a, k, 1) && encode_scales(&maps.b_scales, format, b_scales, rows_b, k, pair ? 2 : 1) &&
                    (!pair || !p.boxed || encode_2d(&maps.out, out_dtype == VRB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, out, rows_b,
                                                    rows_a, rows_b * element, static_cast<int>(64 / element), 32, CU_TENSOR_MAP_SWIZZLE_64B)),
                VRB_ERR_UNSUPPORTED, "fp4_linear: the driver offers no tensor maps for these operands");
    cudaStream_t s = as_stream(stream);
    if (!pair) return format == VRB_NVFP4 ? launch_split<VRB_NVFP4>(maps, p, plan, s) : launch_split<VRB_MXFP4>(maps, p, plan, s);
    if (format == VRB_NVFP4) return out_dtype == VRB_BF16 ? launch_linear<VRB_NVFP4, VRB_BF16>(maps, p, s) : launch_linear<VRB_NVFP4, VRB_F32>(maps, p, s);
    return out_dtype == VRB_BF16 ? launch_linear<VRB_MXFP4, VRB_BF16>(maps, p, s) : launch_linear<VRB_MXFP4, VRB_F32>(maps, p, s);
}
