// GroupNorm of channels-last feature maps [batch, spatial, channels], with an optional activation.
//
//   mean_g = sum x / n,  var_g = sum (x - mean_g)^2 / n  over the n = spatial * channels / groups elements of a group
//   out    = act((x - mean_g) * rsqrt(var_g + eps) * weight[c] + bias[c])          F32, rounded once to x's dtype
//
// The bound is HBM: x is read for the statistics and again for the result, which is written once (the reference would
// add two permutes).  A thread owns V consecutive channels (16 bytes where the layout allows) of every rpp-th row,
// so the affine terms and the group look-up are per thread, not per element, and consecutive threads read consecutive
// bytes of a row.
//   1. gcl_partial   per thread F32 sums of (x - K) and (x - K)^2 per channel over runs of kRun rows, K the run's
//                    first value (an offset common to the channel cancels exactly), rebuilt in double:
//                    S = s1 + n K, Q = s2 + K (2 s1 + n K); the threads of a group are added in a fixed order
//   2. gcl_finalize  adds the CTAs' partials of a (batch entry, group) in a fixed order; mean, rsqrt(var + eps)
//   3. gcl_apply     sweeps the rows backwards, so that it starts with what the statistics pass left in L2
#include "vrb_common.cuh"

namespace vrb {
namespace {

constexpr int kThreads = 256;
constexpr int kRun = 32;           // rows of a thread between two rebuilds in double
constexpr int kSplitsPerSm = 2;    // CTAs of the statistics pass per SM

struct GclGeom {
    int64_t batch, spatial;
    int channels, groups, per;     // per = channels / groups
    int vectors;                   // channels / V
    int slab;                      // vectors a CTA covers at a time (<= kThreads)
    int rpp;                       // rows a CTA covers at a time
    int splits;                    // CTAs per batch entry (statistics)
};

template <typename T, int V>
struct Vec;
template <int V>
struct Vec<uint16_t, V> {
    uint16_t raw[V];
    __device__ __forceinline__ float get(int e) const { return bf16_bits_to_float(raw[e]); }
};
template <int V>
struct Vec<float, V> {
    float raw[V];
    __device__ __forceinline__ float get(int e) const { return raw[e]; }
};
template <int BYTES> struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<2> { using type = uint16_t; };

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p) {
    using W = typename Word<sizeof(T) * V>::type;
    const W w = __ldcs(reinterpret_cast<const W*>(p));
    Vec<T, V> r;
    *reinterpret_cast<W*>(r.raw) = w;
    return r;
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec_keep(const T* p) {   // default policy: the line should stay in L2
    using W = typename Word<sizeof(T) * V>::type;
    const W w = *reinterpret_cast<const W*>(p);
    Vec<T, V> r;
    *reinterpret_cast<W*>(r.raw) = w;
    return r;
}
template <int V>
__device__ __forceinline__ void store_vec(uint16_t* p, const float (&v)[V]) {
    using W = typename Word<2 * V>::type;
    union { W w; uint16_t h[V]; uint32_t d[V / 2 > 0 ? V / 2 : 1]; } r;
    if constexpr (V == 1) r.h[0] = static_cast<uint16_t>(float_to_bf16_bits(v[0]));
    else
#pragma unroll
        for (int e = 0; e < V; e += 2) r.d[e / 2] = pack_bf16x2(v[e], v[e + 1]);
    __stcs(reinterpret_cast<W*>(p), r.w);
}
template <int V>
__device__ __forceinline__ void store_vec(float* p, const float (&v)[V]) {
    using W = typename Word<4 * V>::type;
    union { W w; float f[V]; } r;
#pragma unroll
    for (int e = 0; e < V; ++e) r.f[e] = v[e];
    __stcs(reinterpret_cast<W*>(p), r.w);
}

// The activation on an F32 value that is rounded once afterwards.  SiLU and GELU-tanh go through one exponential and
// one reciprocal (x sigmoid(x); x sigmoid(2u), u the tanh form's argument): relative error below 2^-20 where the result
// is not negligible, far under the bf16 step and the F32 statistics' own error.  ACT 3: any other kind.
template <int ACT>
__device__ __forceinline__ float activate(float y, int kind) {
    if constexpr (ACT == 0) return y;
    if constexpr (ACT == 1) return __fdividef(y, 1.0f + __expf(-y));
    if constexpr (ACT == 2) {
        const float u = 0.7978845608028654f * (y + 0.044715f * y * y * y);
        return __fdividef(y, 1.0f + __expf(-2.0f * u));
    }
    return activation_value(kind, y);
}

// partial[((b * splits + split) * groups + g) * 2 + {0, 1}] = {sum x, sum x^2} over the CTA's rows
template <typename T, int V>
__global__ void __launch_bounds__(kThreads, V >= 4 ? 2 : 4) gcl_partial_kernel(const T* x, double* __restrict__ partial, GclGeom g) {
    __shared__ double sums[2][kThreads * V];
    pdl_wait();
    const int b = blockIdx.x / g.splits, split = blockIdx.x - b * g.splits;
    const int lane_vector = threadIdx.x % g.slab, lane_row = threadIdx.x / g.slab;
    double* out = partial + static_cast<int64_t>(blockIdx.x) * g.groups * 2;
    for (int slab0 = 0; slab0 < g.vectors; slab0 += g.slab) {
        const int slab = min(g.slab, g.vectors - slab0);
        double S[V], Q[V];
#pragma unroll
        for (int e = 0; e < V; ++e) S[e] = Q[e] = 0.0;
        if (lane_row < g.rpp && lane_vector < slab) {
            const int64_t step = static_cast<int64_t>(g.splits) * g.rpp;
            int64_t row = static_cast<int64_t>(split) * g.rpp + lane_row;
            const T* p = x + (static_cast<int64_t>(b) * g.spatial + row) * g.channels + (slab0 + lane_vector) * V;
            const int64_t p_step = step * g.channels;
            while (row < g.spatial) {
                float K[V], s1[V], s2[V];
                int n = 0;
#pragma unroll
                for (int e = 0; e < V; ++e) s1[e] = s2[e] = 0.0f;
                for (; n < kRun && row < g.spatial; ) {
                    constexpr int U = 4;
                    Vec<T, V> v[U];
                    int have = 0;
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (row + u * step < g.spatial) { v[u] = load_vec_keep<T, V>(p + u * p_step); have = u + 1; }
                    if (n == 0)
#pragma unroll
                        for (int e = 0; e < V; ++e) K[e] = v[0].get(e);
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (u < have)
#pragma unroll
                            for (int e = 0; e < V; ++e) {
                                const float d = v[u].get(e) - K[e];
                                s1[e] += d;
                                s2[e] = fmaf(d, d, s2[e]);
                            }
                    n += have;
                    row += U * step;
                    p += U * p_step;
                }
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const double k = K[e], nk = n * k;
                    S[e] += s1[e] + nk;
                    Q[e] += s2[e] + k * (2.0 * s1[e] + nk);
                }
            }
        }
        if (slab0) __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) {
            sums[0][threadIdx.x * V + e] = S[e];
            sums[1][threadIdx.x * V + e] = Q[e];
        }
        __syncthreads();
        // one warp per group: the slab's channels of the group, over the CTA's rows, strided over the lanes
        const int c_begin = slab0 * V, c_end = c_begin + slab * V;
        const int lane = threadIdx.x & 31;
        for (int group = c_begin / g.per + (threadIdx.x >> 5); group * g.per < c_end; group += kThreads / 32) {
            const int from = max(group * g.per, c_begin) - c_begin, width = min((group + 1) * g.per, c_end) - c_begin - from;
            double s = 0.0, q = 0.0;
            for (int i = lane; i < width * g.rpp; i += 32) {
                const int r = i / width, at = r * g.slab * V + from + (i - r * width);
                s += sums[0][at];
                q += sums[1][at];
            }
            for (int offset = 16; offset > 0; offset >>= 1) {
                s += __shfl_xor_sync(0xffffffffu, s, offset);
                q += __shfl_xor_sync(0xffffffffu, q, offset);
            }
            if (lane == 0) {
                if (group * g.per < c_begin) { s += out[group * 2]; q += out[group * 2 + 1]; }   // begun in an earlier slab
                out[group * 2] = s;
                out[group * 2 + 1] = q;
            }
        }
        __syncthreads();
    }
}

// stats[(b * groups + g) * 2 + {0, 1}] = {mean, rsqrt(var + eps)}; one warp per (batch entry, group)
__global__ void __launch_bounds__(128) gcl_finalize_kernel(const double* __restrict__ partial, float* __restrict__ stats, GclGeom g, float eps) {
    pdl_wait();
    const int64_t unit = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (unit >= g.batch * g.groups) return;
    const int64_t b = unit / g.groups;
    const int group = static_cast<int>(unit - b * g.groups);
    double s = 0.0, q = 0.0;
    for (int i = lane; i < g.splits; i += 32) {
        const double* p = partial + ((b * g.splits + i) * g.groups + group) * 2;
        s += p[0];
        q += p[1];
    }
    for (int offset = 16; offset > 0; offset >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, offset);
        q += __shfl_xor_sync(0xffffffffu, q, offset);
    }
    if (lane == 0) {
        const double n = static_cast<double>(g.spatial) * g.per, mean = s / n;
        double var = q / n - mean * mean;
        if (var < 0.0) var = 0.0;
        stats[unit * 2] = static_cast<float>(mean);
        stats[unit * 2 + 1] = static_cast<float>(1.0 / sqrt(var + static_cast<double>(eps)));
    }
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads, 4) gcl_apply_kernel(const T* x, const void* weight, int w_dt, const void* bias, int b_dt,
                                                               T* out, const float* __restrict__ stats, GclGeom g, int ctas, int kind) {
    pdl_wait();
    const int slabs = (g.vectors + g.slab - 1) / g.slab;
    const int unit = blockIdx.x / ctas, cta = ctas - 1 - (blockIdx.x - unit * ctas);
    const int b = unit / slabs, slab0 = (unit - b * slabs) * g.slab;
    const int lane_vector = threadIdx.x % g.slab, lane_row = threadIdx.x / g.slab;
    if (lane_row >= g.rpp || slab0 + lane_vector >= g.vectors) return;
    const int c0 = (slab0 + lane_vector) * V;
    float mean[V], scale[V], shift[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int64_t at = (static_cast<int64_t>(b) * g.groups + (c0 + e) / g.per) * 2;
        mean[e] = stats[at];
        scale[e] = stats[at + 1] * (weight ? load1(weight, w_dt, c0 + e) : 1.0f);
        shift[e] = bias ? load1(bias, b_dt, c0 + e) : 0.0f;
    }
    constexpr int U = 4;
    const int64_t step = static_cast<int64_t>(ctas) * g.rpp, p_step = step * g.channels;
    // rows of this thread are cta * rpp + lane_row + i * step, visited from the last one down
    int64_t row = static_cast<int64_t>(cta) * g.rpp + lane_row;
    if (row >= g.spatial) return;
    row += (g.spatial - 1 - row) / step * step;
    int64_t at = (static_cast<int64_t>(b) * g.spatial + row) * g.channels + c0;
    for (; row >= 0; row -= U * step, at -= U * p_step) {
        Vec<T, V> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (row - u * step >= 0) v[u] = load_vec<T, V>(x + at - u * p_step);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (row - u * step >= 0) {
                float y[V];
#pragma unroll
                for (int e = 0; e < V; ++e) y[e] = activate<ACT>(fmaf(v[u].get(e) - mean[e], scale[e], shift[e]), kind);
                store_vec<V>(out + at - u * p_step, y);
            }
    }
}

int vector_width(int dtype, int64_t channels, const void* x, const void* out) {
    const int element = static_cast<int>(dtype_bytes(dtype));
    for (int v = 16 / element; v > 1; v /= 2)
        if (channels % v == 0 && ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) % (v * element)) == 0) return v;
    return 1;
}

int make_geom(GclGeom& g, int64_t batch, int64_t spatial, int64_t channels, int groups) {
    VRB_REQUIRE(batch > 0 && spatial > 0 && channels > 0 && groups > 0 && channels % groups == 0, VRB_ERR_INVALID,
                "group_norm_channels_last: group norm shape/groups mismatch");
    VRB_REQUIRE(channels <= (int64_t{1} << 24) && batch <= (int64_t{1} << 20), VRB_ERR_INVALID,
                "group_norm_channels_last: group norm launch extent exceeds CUDA grid capacity");
    g.batch = batch; g.spatial = spatial;
    g.channels = static_cast<int>(channels); g.groups = groups; g.per = static_cast<int>(channels / groups);
    return VRB_OK;
}
// CTAs of the statistics pass per batch entry: kSplitsPerSm per SM over the whole batch, none without a row.  Depends on
// V only through rpp, so the workspace is sized with the most a layout can ask for.
int splits_for(const GclGeom& g, int rpp) {
    int64_t want = (static_cast<int64_t>(sm_count()) * kSplitsPerSm + g.batch - 1) / g.batch;
    const int64_t most = (g.spatial + rpp - 1) / rpp;
    if (want > most) want = most;
    return static_cast<int>(want < 1 ? 1 : want);
}
void set_width(GclGeom& g, int v) {
    g.vectors = g.channels / v;
    g.slab = g.vectors < kThreads ? g.vectors : kThreads;
    g.rpp = kThreads / g.slab;
    if (g.rpp > g.spatial) g.rpp = static_cast<int>(g.spatial);
    g.splits = splits_for(g, g.rpp);
}

size_t up256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }
size_t partial_bytes(const GclGeom& g) { return up256(static_cast<size_t>(g.batch) * splits_for(g, 1) * g.groups * 2 * sizeof(double)); }
size_t workspace_size(const GclGeom& g) { return partial_bytes(g) + up256(static_cast<size_t>(g.batch) * g.groups * 2 * sizeof(float)); }

template <typename T, int V>
int run_two_pass(const T* x, const void* weight, int w_dt, const void* bias, int b_dt, T* out, GclGeom g, float eps, int activation,
                 char* workspace, cudaStream_t s) {
    set_width(g, V);
    double* partial = reinterpret_cast<double*>(workspace);
    float* stats = reinterpret_cast<float*>(workspace + partial_bytes(g));
    launch_overlapped(gcl_partial_kernel<T, V>, dim3(static_cast<unsigned>(g.batch * g.splits)), dim3(kThreads), 0, s, x, partial, g);
    if (int rc = after_launch("group_norm_channels_last statistics")) return rc;
    launch_overlapped(gcl_finalize_kernel, dim3(static_cast<unsigned>((g.batch * g.groups * 32 + 127) / 128)), dim3(128), 0, s, partial, stats, g, eps);
    if (int rc = after_launch("group_norm_channels_last finalize")) return rc;
    const int64_t slabs = (g.vectors + g.slab - 1) / g.slab, units = g.batch * slabs;
    int64_t ctas = (static_cast<int64_t>(sm_count()) * 8 + units - 1) / units;
    const int64_t most = (g.spatial + g.rpp - 1) / g.rpp;
    if (ctas > most) ctas = most;
    const dim3 grid(static_cast<unsigned>(units * ctas));
#define VRB_GCL_APPLY(ACT) launch_overlapped(gcl_apply_kernel<T, V, ACT>, grid, dim3(kThreads), 0, s, x, weight, w_dt, bias, b_dt, out, stats, g, static_cast<int>(ctas), activation)
    if (activation == VRB_NO_ACTIVATION) VRB_GCL_APPLY(0);
    else if (activation == VRB_SILU) VRB_GCL_APPLY(1);
    else if (activation == VRB_GELU_TANH) VRB_GCL_APPLY(2);
    else VRB_GCL_APPLY(3);
#undef VRB_GCL_APPLY
    return after_launch("group_norm_channels_last apply");
}

}  // namespace
}  // namespace vrb

using namespace vrb;

extern "C" size_t vrb_group_norm_channels_last_workspace_bytes(int dtype, int64_t batch, int64_t spatial, int64_t channels, int groups) {
    GclGeom g;
    if (!is_float_dtype(dtype) || make_geom(g, batch, spatial, channels, groups)) return 0;
    return workspace_size(g);
}

extern "C" int vrb_group_norm_channels_last(const void* x, int dtype, const void* weight, int weight_dtype,
                                            const void* bias, int bias_dtype, void* out,
                                            int64_t batch, int64_t spatial, int64_t channels, int groups, float eps,
                                            int activation, void* workspace, size_t workspace_bytes, vrb_stream stream) {
    VRB_REQUIRE(x && out, VRB_ERR_INVALID, "group_norm_channels_last: null tensor");
    VRB_REQUIRE(is_float_dtype(dtype), VRB_ERR_UNSUPPORTED, "group_norm_channels_last: dtype must be F32 or BF16");
    VRB_REQUIRE((!weight || is_float_dtype(weight_dtype)) && (!bias || is_float_dtype(bias_dtype)), VRB_ERR_UNSUPPORTED,
                "group_norm_channels_last: weight and bias must be F32 or BF16");
    VRB_REQUIRE(activation >= VRB_NO_ACTIVATION && activation <= VRB_RELU, VRB_ERR_INVALID,
                "group_norm_channels_last: unknown activation %d", activation);
    GclGeom g;
    if (int rc = make_geom(g, batch, spatial, channels, groups)) return rc;
    const size_t need = workspace_size(g);
    VRB_REQUIRE(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, VRB_ERR_WORKSPACE,
                "group_norm_channels_last: workspace needs %zu bytes, 256-byte aligned", need);
    char* ws = static_cast<char*>(workspace);
    cudaStream_t s = as_stream(stream);
#define VRB_GCL_RUN(T, V) run_two_pass<T, V>(static_cast<const T*>(x), weight, weight_dtype, bias, bias_dtype, static_cast<T*>(out), g, eps, activation, ws, s)
    const int v = vector_width(dtype, channels, x, out);
    if (dtype == VRB_BF16) {
        if (v == 8) return VRB_GCL_RUN(uint16_t, 8);
        if (v == 4) return VRB_GCL_RUN(uint16_t, 4);
        if (v == 2) return VRB_GCL_RUN(uint16_t, 2);
        return VRB_GCL_RUN(uint16_t, 1);
    }
    if (v == 4) return VRB_GCL_RUN(float, 4);
    if (v == 2) return VRB_GCL_RUN(float, 2);
    return VRB_GCL_RUN(float, 1);
#undef VRB_GCL_RUN
}
