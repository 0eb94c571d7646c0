// GroupNorm of channels-last feature maps [batch, spatial, channels], with an optional activation.
//
//   mean_g = sum x / n,  var_g = sum (x - mean_g)^2 / n  over the n = spatial * channels / groups elements of a group
//   out    = act((x - mean_g) * rsqrt(var_g + eps) * weight[c] + bias[c])          F32, rounded once to x's dtype
//
// The bound is HBM: x is read for the statistics and again for the result, which is written once (the reference would
// add two permutes).  A thread owns V consecutive channels (16 bytes where the layout allows) of every rpp-th row,
// so the affine terms and the group look-up are per thread, not per element, and consecutive threads read consecutive
// bytes of a row.  Statistics everywhere: per thread and channel F32 sums of (x - K) and (x - K)^2 over at most kRun rows, K
// the first value of the run (an offset common to the channel cancels exactly), rebuilt in double: S = s1 + n K,
// Q = s2 + K (2 s1 + n K); threads, CTAs and clusters are added in a fixed order.
//   Feature maps that fit the registers of one cluster per slab of channels: gcl_cluster reads x once, keeps it, adds the sums
//   over distributed shared memory and writes the result: one launch.
//   Feature maps that fit the shared memory of clusters at work at once: gcl_resident does the same from there.
//   Others: 1. gcl_partial   a CTA's sums per (batch entry, group)
//           2. gcl_finalize  only for many groups: adds the CTAs' sums once, where adding them in every CTA of 3. would cost more
//           3. gcl_apply     sweeps the rows backwards, so that it starts with what the statistics pass left in L2
#include "vrb_common.cuh"

namespace vrb {
namespace {

constexpr int kThreads = 512;      // of the statistics pass
constexpr int kApplyThreads = 1024;// of the normalise pass: one CTA to an SM, so that the sums are added once on each
constexpr int kClusterThreads = 256;
constexpr int kResidentThreads = 512;
constexpr int kRun = 32;           // rows of a thread between two rebuilds in double
constexpr int kClusterGroups = 128;// groups of a cluster's slab, at most
constexpr int kInlineGroups = 64;  // groups up to which gcl_apply adds the CTAs' sums itself

// Rows whose byte count is no multiple of a vector's are folded: `fold` of them make a row of whole vectors, and what is left of
// the last such row (`tail` elements) is handled element by element.
struct GclGeom {
    int64_t batch, spatial;        // spatial: folded rows
    int64_t entry;                 // elements of a batch entry
    int channels, groups, per;     // channels: elements of a folded row; per: channels of a group
    int fold, row, tail;           // row: elements of an unfolded row
    int vectors;                   // channels / V
    int slab;                      // vectors a CTA covers at a time (<= kThreads)
    int rpp;                       // rows a CTA covers at a time
    int splits;                    // CTAs of the statistics pass per batch entry
    int cluster;                   // CTAs of a cluster of gcl_cluster
    double share;                  // 1 / elements of a group
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
// the double at `local` in the shared memory of the cluster's CTA `rank`
__device__ __forceinline__ double load_cluster(const double* local, unsigned rank) {
    double v;
    asm volatile("{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f64 %0, [a];\n\t}"
                 : "=d"(v) : "r"(static_cast<unsigned>(__cvta_generic_to_shared(local))), "r"(rank) : "memory");
    return v;
}

// V elements as the 32-bit words they are loaded as (an array of halves would be moved half by half)
template <typename T, int V>
struct Vec {
    static constexpr int kBytes = static_cast<int>(sizeof(T)) * V, kWords = (kBytes + 3) / 4;
    uint32_t word[kWords];
    __device__ __forceinline__ float get(int e) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(word[e]);
        else return __uint_as_float(e & 1 ? word[e / 2] & 0xffff0000u : word[e / 2] << 16);
    }
};
template <int BYTES> struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<2> { using type = uint16_t; };

template <bool STREAM, typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p) {   // STREAM: not worth keeping in L2
    using W = typename Word<Vec<T, V>::kBytes>::type;
    const W w = STREAM ? __ldcs(reinterpret_cast<const W*>(p)) : *reinterpret_cast<const W*>(p);
    Vec<T, V> r;
    if constexpr (sizeof(W) == 16) { r.word[0] = w.x; r.word[1] = w.y; r.word[2] = w.z; r.word[3] = w.w; }
    else if constexpr (sizeof(W) == 8) { r.word[0] = w.x; r.word[1] = w.y; }
    else r.word[0] = w;
    return r;
}
template <int V>
__device__ __forceinline__ void store_vec(uint16_t* p, const float (&v)[V]) {
    if constexpr (V == 8)
        __stcs(reinterpret_cast<uint4*>(p), make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])));
    else if constexpr (V == 4) __stcs(reinterpret_cast<uint2*>(p), make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])));
    else if constexpr (V == 2) __stcs(reinterpret_cast<uint32_t*>(p), pack_bf16x2(v[0], v[1]));
    else __stcs(p, static_cast<uint16_t>(float_to_bf16_bits(v[0])));
}
template <int V>
__device__ __forceinline__ void store_vec(float* p, const float (&v)[V]) {
    if constexpr (V == 4) __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
    else if constexpr (V == 2) __stcs(reinterpret_cast<float2*>(p), make_float2(v[0], v[1]));
    else __stcs(p, v[0]);
}

// act((v - mean) scale + shift) of a thread's V channels: F32 values that are rounded once afterwards.  SiLU and GELU-tanh in
// bf16 by pairs (gate_pair: three special functions for two values; with four the normalise pass of 25 MB waits for that unit), in
// F32, twice the bytes a value, one by one to F32's accuracy.  ACT 3: any other kind.
template <int ACT, typename T, int V>
__device__ __forceinline__ void normalise(const Vec<T, V>& v, const float (&mean)[V], const float (&scale)[V], const float (&shift)[V], int kind, float (&y)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) y[e] = fmaf(v.get(e) - mean[e], scale[e], shift[e]);
    if constexpr ((ACT == 1 || ACT == 2) && sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = gate_value<ACT>(y[e]);
    } else if constexpr (ACT == 1 || ACT == 2) {
#pragma unroll
        for (int e = 0; e + 1 < V; e += 2) gate_pair<ACT, false>(pack_f32x2(y[e], y[e + 1]), y[e], y[e + 1]);
        if constexpr (V == 1) {
            float unused;
            gate_pair<ACT, false>(pack_f32x2(y[0], 0.0f), y[0], unused);
        }
    } else if constexpr (ACT == 3) {
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = activation_value(kind, y[e]);
    }
}

// Sums of a thread's V channels over a run, and what has been rebuilt from earlier runs.  E consecutive channels lie in one group
// and share the double sums.
template <typename T, int V, int E>
struct Sums {
    static constexpr int D = V / E;
    double S[D], Q[D];
    float K[V], s1[V], s2[V];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int e = 0; e < D; ++e) S[e] = Q[e] = 0.0;
    }
    __device__ __forceinline__ void begin(const Vec<T, V>& v) {
#pragma unroll
        for (int e = 0; e < V; ++e) { K[e] = v.get(e); s1[e] = s2[e] = 0.0f; }
    }
    __device__ __forceinline__ void add(const Vec<T, V>& v) {
        if constexpr (V > 1) {
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                const unsigned long long d = sub_f32x2(pack_f32x2(v.get(e), v.get(e + 1)), pack_f32x2(K[e], K[e + 1]));
                unpack_f32x2(add_f32x2(pack_f32x2(s1[e], s1[e + 1]), d), s1[e], s1[e + 1]);
                unpack_f32x2(fma_f32x2(d, d, pack_f32x2(s2[e], s2[e + 1])), s2[e], s2[e + 1]);
            }
        } else {
            const float d = v.get(0) - K[0];
            s1[0] += d;
            s2[0] = fmaf(d, d, s2[0]);
        }
    }
    __device__ __forceinline__ void single(int e, float v) {
        const double d = v;
        S[e / E] += d;
        Q[e / E] += d * d;
    }
    __device__ __forceinline__ void rebuild(int n) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const double k = K[e], nk = n * k;
            S[e / E] += s1[e] + nk;
            Q[e / E] += s2[e] + k * (2.0 * s1[e] + nk);
        }
    }
};

// Adds the CTA's sums of one slab per group: a warp to a group, lanes strided over (row, D-channel entry), a fixed tree.  Every
// group's {S, Q} goes to `take(group - first group of the slab, S, Q)` on lane 0.
template <int THREADS, int D, int V, typename Take>
__device__ __forceinline__ void add_groups(double (&sums)[2][THREADS * D], const GclGeom& g, int slab0, int slab, Take take) {
    constexpr int E = V / D;   // channels of an entry
    const int lane = threadIdx.x & 31, c_begin = slab0 * V, c_end = c_begin + slab * V, first = c_begin / g.per;
    // a folded row (one slab) holds a group's channels `times` times, the only group's one after the other
    const int times = g.groups == 1 ? 1 : g.fold, span = g.groups == 1 ? g.channels : g.per;
    for (int group = first + (threadIdx.x >> 5); group < g.groups && group * span < c_end; group += THREADS / 32) {
        const int from = (max(group * span, c_begin) - c_begin) / E, width = (min((group + 1) * span, c_end) - c_begin) / E - from;
        double s = 0.0, q = 0.0;
#pragma unroll 1
        for (int i = lane; i < g.rpp * times * width; i += 32) {
            const int rt = i / width, r = times > 1 ? rt / times : rt;
            const int k = r * g.slab * D + (rt - r * times) * g.row / E + from + (i - rt * width);
            s += sums[0][k];
            q += sums[1][k];
        }
#pragma unroll 1
        for (int offset = 16; offset > 0; offset >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, offset);
            q += __shfl_xor_sync(0xffffffffu, q, offset);
        }
        if (lane == 0) take(group - first, s, q);
    }
}
// {mean, rsqrt(var + eps)}; share = 1 / n.  Products in double, where the squared mean cancels; no double division or square
// root, which took a third of the normalise pass on 25 MB.
__device__ __forceinline__ float2 moments_to_stats(double s, double q, double share, float eps) {
    const double mean = s * share;
    float var = static_cast<float>(q * share - mean * mean);
    if (var < 0.0f) var = 0.0f;                        // a NaN stays
    return make_float2(static_cast<float>(mean), rsqrtf(var + eps));
}

// partial[((b * splits + split) * groups + g) * 2 + {0, 1}] = {sum x, sum x^2} over the CTA's rows.  One CTA to an SM.
template <typename T, int V, int E>
__global__ void __launch_bounds__(kThreads, 1) gcl_partial_kernel(const T* x, double* __restrict__ partial, GclGeom g) {
    using Acc = Sums<T, V, E>;
    __shared__ double sums[2][kThreads * Acc::D];
    pdl_wait();
    const int b = blockIdx.x / g.splits, split = blockIdx.x - b * g.splits;
    const int lane_vector = threadIdx.x % g.slab, lane_row = threadIdx.x / g.slab;
    double* out = partial + static_cast<int64_t>(blockIdx.x) * g.groups * 2;
    for (int slab0 = 0; slab0 < g.vectors; slab0 += g.slab) {
        const int slab = min(g.slab, g.vectors - slab0);
        Acc acc;
        acc.clear();
        if (lane_row < g.rpp && lane_vector < slab) {
            constexpr int U = E == V && sizeof(T) * V == 16 ? 8 : 4;
            const int64_t step = static_cast<int64_t>(g.splits) * g.rpp, p_step = step * g.channels;
            const int64_t row = static_cast<int64_t>(split) * g.rpp + lane_row;
            const T* p = x + b * g.entry + row * g.channels + (slab0 + lane_vector) * V;
            int64_t left = row < g.spatial ? (g.spatial - 1 - row) / step + 1 : 0;   // rows of this thread from p on
            // U rows at a time, the next U on their way while these are added
            Vec<T, V> now[U], next[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (u < left) now[u] = load_vec<false, T, V>(p + u * p_step);
            int run = 0;
            for (; left > 0; left -= U) {
                p += U * p_step;
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (U + u < left) next[u] = load_vec<false, T, V>(p + u * p_step);
                if (run == 0) acc.begin(now[0]);
                if (left >= U) {
#pragma unroll
                    for (int u = 0; u < U; ++u) acc.add(now[u]);
                } else {
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (u < left) acc.add(now[u]);
                }
                run += left < U ? static_cast<int>(left) : U;
                if (run >= kRun || left <= U) {
                    acc.rebuild(run);
                    run = 0;
                }
#pragma unroll
                for (int u = 0; u < U; ++u) now[u] = next[u];
            }
            if (g.tail > 0 && row <= g.spatial && (g.spatial - row) % step == 0) {
                const T* rest = x + b * g.entry + g.spatial * g.channels;
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (lane_vector * V + e < g.tail) acc.single(e, load1(rest, sizeof(T) == 2 ? VRB_BF16 : VRB_F32, lane_vector * V + e));
            }
        }
        if (slab0) __syncthreads();
#pragma unroll
        for (int e = 0; e < Acc::D; ++e) {
            sums[0][threadIdx.x * Acc::D + e] = acc.S[e];
            sums[1][threadIdx.x * Acc::D + e] = acc.Q[e];
        }
        __syncthreads();
        const int first = slab0 * V / g.per;
        add_groups<kThreads, Acc::D, V>(sums, g, slab0, slab, [&](int group, double s, double q) {
            double* o = out + (first + group) * 2;
            if ((first + group) * g.per < slab0 * V) { s += o[0]; q += o[1]; }   // begun in an earlier slab
            o[0] = s;
            o[1] = q;
        });
        __syncthreads();
    }
}

// {mean, rsqrt(var + eps)} of groups [first, first + count) of a batch entry from the CTAs' sums, count <= THREADS: neighbouring
// threads read neighbouring groups, THREADS / count of them share a group's clusters; all threads of the CTA together.
template <int THREADS, typename Take>
__device__ __forceinline__ void collect_groups(const double* partial, int64_t b, int first, int count, const GclGeom& g, float eps, Take take) {
    __shared__ double2 parts[THREADS];
    const int shares = THREADS / count, group = threadIdx.x % count, share = threadIdx.x / count;
    double2 sum = make_double2(0.0, 0.0);
    if (share < shares) {
        const double2* p = reinterpret_cast<const double2*>(partial) + b * g.splits * g.groups + first + group;
        constexpr int U = 8;   // loads in flight: one after the other, each waits for L2
        for (int i = share; i < g.splits; i += U * shares) {
            double2 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = i + u * shares < g.splits ? p[static_cast<int64_t>(i + u * shares) * g.groups] : make_double2(0.0, 0.0);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                sum.x += v[u].x;
                sum.y += v[u].y;
            }
        }
    }
    parts[threadIdx.x] = sum;
    __syncthreads();
    for (int group = threadIdx.x >> 5; group < count; group += THREADS / 32) {
        sum = make_double2(0.0, 0.0);
        for (int i = threadIdx.x & 31; i < shares; i += 32) {
            const double2 v = parts[i * count + group];
            sum.x += v.x;
            sum.y += v.y;
        }
#pragma unroll 1
        for (int offset = 16; offset > 0; offset >>= 1) {
            sum.x += __shfl_xor_sync(0xffffffffu, sum.x, offset);
            sum.y += __shfl_xor_sync(0xffffffffu, sum.y, offset);
        }
        if ((threadIdx.x & 31) == 0) take(group, moments_to_stats(sum.x, sum.y, g.share, eps));
    }
    __syncthreads();
}
// stats[b * groups + g] = {mean, rsqrt(var + eps)}; a CTA to 32 groups
constexpr int kFinalizeGroups = 32;
__global__ void __launch_bounds__(kThreads) gcl_finalize_kernel(const double* __restrict__ partial, float2* __restrict__ stats, GclGeom g, float eps) {
    pdl_wait();
    const int chunks = (g.groups + kFinalizeGroups - 1) / kFinalizeGroups;
    const int64_t b = blockIdx.x / chunks;
    const int first = (blockIdx.x - static_cast<int>(b) * chunks) * kFinalizeGroups;
    collect_groups<kThreads>(partial, b, first, min(kFinalizeGroups, g.groups - first), g, eps,
                             [&](int group, float2 v) { stats[b * g.groups + first + group] = v; });
}

// A thread's affine terms: y = (x - mean) * scale + shift per channel; weight and bias are loaded before the statistics are
// there.  stat(group) gives {mean, inverse}.
template <int V>
__device__ __forceinline__ void load_channels(const void* p, int dt, int c0, int channels, float fill, float (&v)[V]) {
    if (p == nullptr) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = fill;
        return;
    }
    int c = c0;
    // one or two wide loads where they lie whole and aligned: V loads of 2 bytes cost a CTA of 1024 threads 3 us
    if (V >= 4 && c0 + V <= channels && (reinterpret_cast<uintptr_t>(p) + (dt == VRB_F32 ? 4 : 2) * static_cast<uintptr_t>(c0)) % (dt == VRB_F32 ? 16 : 2 * V) == 0) {
        if (dt == VRB_F32) {
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const Vec<float, 4> w = load_vec<false, float, 4>(static_cast<const float*>(p) + c0 + e);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[(e + i) % V] = w.get(i);
            }
        } else {
            const Vec<uint16_t, V> w = load_vec<false, uint16_t, V>(static_cast<const uint16_t*>(p) + c0);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = w.get(e);
        }
    } else if (dt == VRB_F32) {
#pragma unroll
        for (int e = 0; e < V; ++e) { v[e] = static_cast<const float*>(p)[c]; if (++c == channels) c = 0; }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) { v[e] = bf16_bits_to_float(static_cast<const uint16_t*>(p)[c]); if (++c == channels) c = 0; }
    }
}
// c0: the first channel, modulo the unfolded row
template <int V, typename Stat>
__device__ __forceinline__ void apply_stats(const GclGeom& g, int c0, Stat stat, float (&mean)[V], float (&scale)[V]) {
    int group = c0 / g.per, within = c0 - group * g.per;
    float2 v = stat(group);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        mean[e] = v.x;
        scale[e] *= v.y;
        if (++within == g.per && e + 1 < V) {
            within = 0;
            if (++group == g.groups) group = 0;
            v = stat(group);
        }
    }
}

// stats: finished, or nullptr: every CTA adds the CTAs' sums of its batch entry (groups <= kInlineGroups)
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kApplyThreads, 1) gcl_apply_kernel(const T* x, const void* weight, int w_dt, const void* bias, int b_dt, T* out,
                                                               const double* __restrict__ partial, const float2* __restrict__ stats, GclGeom g, float eps,
                                                               int ctas, int kind) {
    __shared__ float2 own[kInlineGroups];
    pdl_wait();
    const int slabs = (g.vectors + g.slab - 1) / g.slab;
    const int unit = blockIdx.x / ctas, cta = ctas - 1 - (blockIdx.x - unit * ctas);
    const int b = unit / slabs, slab0 = (unit - b * slabs) * g.slab;
    const int lane_vector = threadIdx.x % g.slab, lane_row = threadIdx.x / g.slab;
    const bool live = lane_row < g.rpp && slab0 + lane_vector < g.vectors;
    const int c0 = (slab0 + lane_vector) * V, channel = g.fold > 1 ? c0 % g.row : c0;
    constexpr int U = 4;
    const int64_t step = static_cast<int64_t>(ctas) * g.rpp, p_step = step * g.channels;
    float mean[V], scale[V], shift[V];
    if (live) {
        load_channels<V>(weight, w_dt, channel, g.row, 1.0f, scale);
        load_channels<V>(bias, b_dt, channel, g.row, 0.0f, shift);
    }
    if (stats == nullptr) collect_groups<kApplyThreads>(partial, b, 0, g.groups, g, eps, [&](int group, float2 v) { own[group] = v; });
    if (!live) return;
    apply_stats<V>(g, channel, [&](int group) { return stats ? stats[static_cast<int64_t>(b) * g.groups + group] : own[group]; }, mean, scale);
    // rows of this thread are cta * rpp + lane_row + i * step, visited from the last one down
    const int64_t row0 = static_cast<int64_t>(cta) * g.rpp + lane_row;
    int64_t row = row0 < g.spatial ? row0 + (g.spatial - 1 - row0) / step * step : -1;
    int64_t at = b * g.entry + row * g.channels + c0;
    for (; row >= 0; row -= U * step, at -= U * p_step) {
        Vec<T, V> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (row - u * step >= 0) v[u] = load_vec<true, T, V>(x + at - u * p_step);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (row - u * step >= 0) {
                float y[V];
                normalise<ACT>(v[u], mean, scale, shift, kind, y);
                store_vec<V>(out + at - u * p_step, y);
            }
    }
    if (g.tail > 0 && row0 <= g.spatial && (g.spatial - row0) % step == 0) {
        constexpr int dt = sizeof(T) == 2 ? VRB_BF16 : VRB_F32;
        const int64_t rest = b * g.entry + g.spatial * g.channels + c0;
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (c0 + e < g.tail) {
                const Vec<T, 1> v = load_vec<true, T, 1>(x + rest + e);
                const float m[1] = {mean[e]}, f[1] = {scale[e]}, o[1] = {shift[e]};
                float y[1];
                normalise<ACT>(v, m, f, o, kind, y);
                store1(out, dt, rest + e, y[0]);
            }
    }
}

// The statistics of a slab's groups from the sums of all CTAs of a cluster (eight at most), in `own`: eight lanes to a group, a
// CTA's sums to each, a fixed tree.  All threads of the cluster; the CTA's own sums stay until cluster_wait().
template <int THREADS>
__device__ __forceinline__ void join_cluster(const double (*mine)[2], float2* own, int groups, const GclGeom& g, float eps) {
    __syncwarp();
    if (g.cluster > 1) { cluster_arrive(); cluster_wait(); } else __syncthreads();
    for (int at = threadIdx.x; at < (groups * 8 + 31) / 32 * 32; at += THREADS) {
        const int group = at >> 3, r = at & 7;
        double s = 0.0, q = 0.0;
        if (group < groups && r < g.cluster) {
            s = g.cluster > 1 ? load_cluster(&mine[group][0], r) : mine[group][0];
            q = g.cluster > 1 ? load_cluster(&mine[group][1], r) : mine[group][1];
        }
#pragma unroll
        for (int offset = 4; offset > 0; offset >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, offset);
            q += __shfl_xor_sync(0xffffffffu, q, offset);
        }
        if (group < groups && r == 0) own[group] = moments_to_stats(s, q, g.share, eps);
    }
    __syncthreads();
    if (g.cluster > 1) cluster_arrive();   // has read the others' sums
}

// One cluster per (batch entry, slab of whole groups): up to kMostRows rows of a thread stay in registers between the statistics
// and the result.  Row i of a thread is (i * cluster + rank) * rpp + lane_row.
constexpr int kMostRows = 4;
template <typename T, int V, int E, int ACT>
__global__ void __launch_bounds__(kClusterThreads) gcl_cluster_kernel(const T* x, const void* weight, int w_dt, const void* bias, int b_dt, T* out, GclGeom g,
                                                              float eps, int kind) {
    using Acc = Sums<T, V, E>;
    __shared__ double sums[2][kClusterThreads * Acc::D];
    __shared__ double mine[kClusterGroups][2];
    __shared__ float2 own[kClusterGroups];
    const int unit = blockIdx.x / g.cluster, rank = blockIdx.x - unit * g.cluster;
    const int slabs = (g.vectors + g.slab - 1) / g.slab, b = unit / slabs, slab0 = (unit - b * slabs) * g.slab;
    const int slab = min(g.slab, g.vectors - slab0);
    const int lane_vector = threadIdx.x % g.slab, lane_row = threadIdx.x / g.slab;
    const bool live = lane_row < g.rpp && lane_vector < slab;
    const int row0 = rank * g.rpp + lane_row, step = g.cluster * g.rpp, spatial = static_cast<int>(g.spatial);
    const int64_t at0 = (static_cast<int64_t>(b) * g.spatial + row0) * g.channels + (slab0 + lane_vector) * V;
    const int64_t p_step = static_cast<int64_t>(step) * g.channels;
    pdl_wait();
    constexpr int R = kMostRows;
    Vec<T, V> v[R];
    Acc acc;
    acc.clear();
    const int c0 = (slab0 + lane_vector) * V;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (live && row0 + i * step < spatial) v[i] = load_vec<true, T, V>(x + at0 + i * p_step);
    float scale[V], shift[V];
    if (live) {
        load_channels<V>(weight, w_dt, c0, g.row, 1.0f, scale);
        load_channels<V>(bias, b_dt, c0, g.row, 0.0f, shift);
    }
    if (live && row0 < spatial) {
        acc.begin(v[0]);
        int n = 0;
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (row0 + i * step < spatial) { acc.add(v[i]); ++n; }
        acc.rebuild(n);
    }
#pragma unroll
    for (int e = 0; e < Acc::D; ++e) {
        sums[0][threadIdx.x * Acc::D + e] = acc.S[e];
        sums[1][threadIdx.x * Acc::D + e] = acc.Q[e];
    }
    __syncthreads();
    add_groups<kClusterThreads, Acc::D, V>(sums, g, slab0, slab, [&](int group, double s, double q) { mine[group][0] = s; mine[group][1] = q; });
    join_cluster<kClusterThreads>(mine, own, slab * V / g.per, g, eps);
    if (live) {
        const int first = slab0 * V / g.per;
        float mean[V];
        apply_stats<V>(g, c0, [&](int group) { return own[group - first]; }, mean, scale);
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (row0 + i * step < spatial) {
                float y[V];
                normalise<ACT>(v[i], mean, scale, shift, kind, y);
                store_vec<V>(out + at0 + i * p_step, y);
            }
    }
    __syncwarp();
    if (g.cluster > 1) cluster_wait();   // no CTA's memory goes while another reads it
}

// The same with the rows in shared memory: up to most_resident_rows() 16-byte vectors a thread (which alone reads what it copied, so
// no barrier stands between), kResidentAhead batches of kResidentBatch on their way at a time.  A batch's rows are added while
// later ones arrive.
constexpr int kResidentBatch = 4, kResidentAhead = 4;
constexpr int most_resident_rows(int entries) { return 27 - entries; }   // with the double sums of `entries` (1, 2 or 4) a thread: 219 KB
static_assert(most_resident_rows(1) <= kRun, "one run of F32 sums");
template <typename T, int E, int ACT>
__global__ void __launch_bounds__(kResidentThreads) gcl_resident_kernel(const T* x, const void* weight, int w_dt, const void* bias, int b_dt, T* out, GclGeom g,
                                                                float eps, int kind) {
    constexpr int V = 16 / sizeof(T), B = kResidentBatch;
    using Acc = Sums<T, V, E>;
    extern __shared__ __align__(16) uint4 resident_rows[];   // [row of the thread][thread]
    __shared__ double sums[2][kResidentThreads * Acc::D];
    __shared__ double mine[kClusterGroups][2];
    __shared__ float2 own[kClusterGroups];
    const int unit = blockIdx.x / g.cluster, rank = blockIdx.x - unit * g.cluster;
    const int slabs = g.vectors / g.slab, b = unit / slabs, slab0 = (unit - b * slabs) * g.slab;
    const int lane_vector = threadIdx.x % g.slab, lane_row = threadIdx.x / g.slab;
    const int row0 = rank * g.rpp + lane_row, step = g.cluster * g.rpp, spatial = static_cast<int>(g.spatial);
    const int rows = lane_row < g.rpp && row0 < spatial ? (spatial - 1 - row0) / step + 1 : 0;
    const int64_t at0 = (static_cast<int64_t>(b) * g.spatial + row0) * g.channels + (slab0 + lane_vector) * V;
    const int64_t p_step = static_cast<int64_t>(step) * g.channels;
    const int c0 = (slab0 + lane_vector) * V;
    const unsigned place = static_cast<unsigned>(__cvta_generic_to_shared(resident_rows + threadIdx.x));
    pdl_wait();
    auto copy = [&](int i0) {
#pragma unroll
        for (int u = 0; u < B; ++u)
            if (i0 + u < rows)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(place + (i0 + u) * kResidentThreads * 16), "l"(x + at0 + (i0 + u) * p_step) : "memory");
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto row = [&](int i) {
        const uint4 w = resident_rows[i * kResidentThreads + threadIdx.x];
        Vec<T, V> v;
        v.word[0] = w.x; v.word[1] = w.y; v.word[2] = w.z; v.word[3] = w.w;
        return v;
    };
#pragma unroll
    for (int i = 0; i < kResidentAhead; ++i) copy(i * B);
    float scale[V], shift[V];
    load_channels<V>(weight, w_dt, c0, g.row, 1.0f, scale);
    load_channels<V>(bias, b_dt, c0, g.row, 0.0f, shift);
    Acc acc;
    acc.clear();
#pragma unroll 1
    for (int i = 0; i < rows; i += B) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kResidentAhead - 1) : "memory");
        if (i == 0) acc.begin(row(0));
#pragma unroll
        for (int u = 0; u < B; ++u)
            if (i + u < rows) acc.add(row(i + u));
        copy(i + kResidentAhead * B);
    }
    if (rows > 0) acc.rebuild(rows);
#pragma unroll
    for (int e = 0; e < Acc::D; ++e) {
        sums[0][threadIdx.x * Acc::D + e] = acc.S[e];
        sums[1][threadIdx.x * Acc::D + e] = acc.Q[e];
    }
    __syncthreads();
    add_groups<kResidentThreads, Acc::D, V>(sums, g, slab0, g.slab, [&](int group, double s, double q) { mine[group][0] = s; mine[group][1] = q; });
    join_cluster<kResidentThreads>(mine, own, g.slab * V / g.per, g, eps);
    if (rows > 0) {
        const int first = slab0 * V / g.per;
        float mean[V];
        apply_stats<V>(g, c0, [&](int group) { return own[group - first]; }, mean, scale);
#pragma unroll 1
        for (int i = 0; i < rows; i += B) {
#pragma unroll
            for (int u = 0; u < B; ++u)
                if (i + u < rows) {
                    float y[V];
                    normalise<ACT>(row(i + u), mean, scale, shift, kind, y);
                    store_vec<V>(out + at0 + (i + u) * p_step, y);
                }
        }
    }
    __syncwarp();
    if (g.cluster > 1) cluster_wait();
}

int gcd(int a, int b) { return b == 0 ? a : gcd(b, a % b); }
// Elements of a vector: the most, up to 16 bytes, for which every batch entry begins on a vector's boundary; rows that are no
// multiple of it are folded where the folded row is not too long for a CTA.  Eight bf16 channels only where they lie in one
// group or two by two: eight pairs of double sums a thread are more than the registers take.
int vector_width(int dtype, int64_t batch, int64_t spatial, int64_t channels, int groups, bool fold, const void* x, const void* out) {
    const int element = static_cast<int>(dtype_bytes(dtype));
    for (int v = 16 / element; v > 1; v /= 2) {
        const int64_t folded = channels / gcd(static_cast<int>(channels), v);
        if (channels % v != 0 && (!fold || folded > kThreads || spatial < v || (batch > 1 && spatial * channels % v != 0))) continue;
        if (v == 8 && groups > 1 && (channels % 2 != 0 || channels / groups % 2 != 0)) continue;
        if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) % (v * element) == 0) return v;
    }
    return 1;
}
// Consecutive channels of a vector that always lie in one group and share their double sums: all, two or one.  (Two rather than
// one: 300000 rows of 160 channels in groups of 10, bf16 with SiLU, 58.7 us against 69.6, 3 x 1035 of 320 5.9 against 17.3.)
int entry_channels(const GclGeom& g, int v) {
    if (g.groups == 1 || (g.row % v == 0 && g.per % v == 0)) return v;
    return v > 2 && g.row % 2 == 0 && g.per % 2 == 0 ? 2 : 1;
}

int make_geom(GclGeom& g, int64_t batch, int64_t spatial, int64_t channels, int groups) {
    VRB_REQUIRE(batch > 0 && spatial > 0 && channels > 0 && groups > 0 && channels % groups == 0, VRB_ERR_INVALID,
                "group_norm_channels_last: group norm shape/groups mismatch");
    VRB_REQUIRE(channels <= (int64_t{1} << 24) && batch <= (int64_t{1} << 20) && spatial <= (int64_t{1} << 40) / channels / batch, VRB_ERR_INVALID,
                "group_norm_channels_last: group norm launch extent exceeds CUDA grid capacity");
    g.batch = batch; g.spatial = spatial; g.entry = spatial * channels;
    g.channels = g.row = static_cast<int>(channels); g.fold = 1; g.tail = 0; g.groups = groups; g.per = static_cast<int>(channels / groups);
    g.share = 1.0 / (static_cast<double>(spatial) * g.per);
    return VRB_OK;
}
int64_t all_rows(const GclGeom& g) { return g.spatial + (g.tail > 0 ? 1 : 0); }
void set_width(GclGeom& g, int v) {
    if (g.row % v != 0) {
        g.fold = v / gcd(g.row, v);
        g.channels = g.row * g.fold;
        g.spatial = g.entry / g.channels;
        g.tail = static_cast<int>(g.entry - g.spatial * g.channels);
    }
    g.vectors = g.channels / v;
    g.slab = g.vectors < kThreads ? g.vectors : kThreads;
    g.rpp = kThreads / g.slab;
    if (g.rpp > all_rows(g)) g.rpp = static_cast<int>(all_rows(g));
}
// CTAs of the statistics pass per batch entry: one per SM over the whole batch, no more than passes over the rows.  Rounded up, here
// and in the normalise pass: batches that divide the SMs unevenly start a few CTAs more than there are SMs, which run after the rest
// (1433600 rows of 256 channels, bf16 with SiLU: 362 us in 1, 2 or 4 entries, 540 to 586 in 3, 5, 8, 16 or 28).
void set_splits(GclGeom& g) {
    const int64_t want = (sm_count() + g.batch - 1) / g.batch, most = (all_rows(g) + g.rpp - 1) / g.rpp;
    g.splits = static_cast<int>(want < most ? want : most);
}
// The slab and cluster of gcl_cluster, or false: the slab is the least run of whole groups and whole vectors of 64 bytes or
// more (a row's piece of a slab should fill memory sectors), its rows have to fit kMostRows rows of a thread in up to eight
// CTAs, and all clusters should be at work at once.  Measured against the passes (bf16 with SiLU, back to back): 64 rows of 512
// channels 3.5 us against 10.1, 256 rows 4.1 against 10.6, 2048 rows 5.5 against 11.1; with 16 rows a thread the code of a
// once-run kernel costs more than a second read of x (4096 rows 15.9 against 12.6).
bool set_cluster(GclGeom& g, int v, int element) {
    int groups = 1;
    while (groups < g.groups && (groups * g.per % v != 0 || groups * g.per * element < 64 || g.groups % groups != 0)) ++groups;
    const int64_t slab = static_cast<int64_t>(groups) * g.per;
    if (slab % v != 0 || slab / v > kClusterThreads || groups > kClusterGroups) return false;
    g.vectors = g.channels / v;
    g.slab = static_cast<int>(slab / v);
    g.rpp = kClusterThreads / g.slab;
    if (g.rpp > g.spatial) g.rpp = static_cast<int>(g.spatial);
    const int64_t passes = (g.spatial + g.rpp - 1) / g.rpp;
    g.cluster = static_cast<int>(passes < 8 ? passes : 8);
    return passes <= static_cast<int64_t>(g.cluster) * kMostRows && g.batch * (g.vectors / g.slab) * g.cluster <= 4 * static_cast<int64_t>(sm_count());
}

// The slab and cluster of gcl_resident, or false: slabs of whole groups and of 16-byte vectors (whose channels lie in one group or
// two by two), at least 64 bytes or else 32 of every row, whose rows fit the shared memory of up to eight CTAs; all clusters at work
// at once, a CTA to an SM, on half of the SMs or else a quarter (`room`: CTAs that fit for clusters of 1 to 8; a second wave costs
// as much as the first).  Measured against the passes (bf16 with SiLU, back to back): 2400 rows of 512 channels 6.9 us against 11.5,
// 8000 rows 10.6 against 13.1, 16000 rows 15.2 against 15.8; 4 x 4096 rows 12.9 against 15.5; 8 x 4096 rows of 320 channels 17.6
// against 30.1.  Pieces of 32 bytes come at half the rate: 20000 rows of 512 channels, 20 of a thread, 16.5 against 17.9, 24960 rows
// 20.4 against 20.1, so those end at 20 rows.  On a quarter of the SMs: 3000 rows of 192 channels, 3 of a thread, 7.8 against 11.1,
// 16384 of 128, 8 of a thread, 10.6 against 12.0, 9216 of 320, 12 of a thread, 12.7 against 12.3.
bool set_resident(GclGeom& g, int v, int element, const int* room) {
    const int entries = v / entry_channels(g, v);
    if (v * element != 16 || entries > 4 || (entries > 2 && element == 4) || g.spatial > INT32_MAX) return false;
    for (int choice = 0; choice < 4; ++choice) {   // half of the SMs before a quarter, wide pieces before narrow ones
        const int least = choice % 2 ? 32 : 64, share = choice < 2 ? 2 : 4;
        int groups = 1;
        while (groups < g.groups && (groups * g.per % v != 0 || groups * g.per * element < least || g.groups % groups != 0)) ++groups;
        const int64_t slab = static_cast<int64_t>(groups) * g.per;
        if (slab % v != 0 || slab / v > kResidentThreads || groups > kClusterGroups) continue;
        g.vectors = g.channels / v;
        g.slab = static_cast<int>(slab / v);
        g.rpp = kResidentThreads / g.slab;
        const int64_t passes = (g.spatial + g.rpp - 1) / g.rpp, most = share > 2 ? 8 : least < 64 ? 20 : most_resident_rows(entries);
        for (g.cluster = 8; g.cluster > 0; --g.cluster) {
            const int64_t ctas = g.batch * (g.vectors / g.slab) * g.cluster;
            if (g.cluster <= passes && passes <= most * g.cluster && ctas <= room[g.cluster] && ctas * share >= sm_count()) return true;
        }
    }
    return false;
}
size_t resident_bytes(const GclGeom& g) {
    const int64_t step = static_cast<int64_t>(g.cluster) * g.rpp;
    return static_cast<size_t>((g.spatial + step - 1) / step) * kResidentThreads * 16;
}
constexpr size_t resident_most(int entries) { return static_cast<size_t>(most_resident_rows(entries)) * kResidentThreads * 16; }

size_t up256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }
// the most any vector width asks for
size_t partial_bytes(const GclGeom& g) {
    const int64_t ctas = sm_count() + g.batch;
    return up256(static_cast<size_t>(ctas) * g.groups * 2 * sizeof(double));
}
size_t workspace_size(const GclGeom& g) {
    return partial_bytes(g) + (g.groups > kInlineGroups ? up256(static_cast<size_t>(g.batch) * g.groups * sizeof(float2)) : 0);
}

struct GclCall {
    const void *x, *weight, *bias;
    void* out;
    int w_dt, b_dt, activation;
    float eps;
};

template <typename T, int V, int E, int ACT>
int run_cluster(const GclCall& c, const GclGeom& g, cudaStream_t s) {
    const int64_t units = g.batch * ((g.vectors + g.slab - 1) / g.slab);
    launch_clusters(gcl_cluster_kernel<T, V, E, ACT>, dim3(static_cast<unsigned>(units * g.cluster)), dim3(kClusterThreads), 0, g.cluster, s, static_cast<const T*>(c.x), c.weight, c.w_dt, c.bias,
                    c.b_dt, static_cast<T*>(c.out), g, c.eps, c.activation);
    return after_launch("group_norm_channels_last");
}
template <typename T, int V, int E>
int run_cluster(const GclCall& c, const GclGeom& g, cudaStream_t s) {
    if (c.activation == VRB_NO_ACTIVATION) return run_cluster<T, V, E, 0>(c, g, s);
    if (c.activation == VRB_SILU) return run_cluster<T, V, E, 1>(c, g, s);
    if (c.activation == VRB_GELU_TANH) return run_cluster<T, V, E, 2>(c, g, s);
    return run_cluster<T, V, E, 3>(c, g, s);
}

template <typename T, int E, int ACT>
int run_resident(const GclCall& c, const GclGeom& g, cudaStream_t s) {
    static std::atomic<uint64_t> allowed{0};
    if (int rc = allow_shared(gcl_resident_kernel<T, E, ACT>, resident_most(static_cast<int>(16 / sizeof(T)) / E), allowed, "group_norm_channels_last")) return rc;
    launch_clusters(gcl_resident_kernel<T, E, ACT>, dim3(static_cast<unsigned>(g.batch * (g.vectors / g.slab) * g.cluster)), dim3(kResidentThreads), resident_bytes(g), g.cluster, s,
                    static_cast<const T*>(c.x), c.weight, c.w_dt, c.bias, c.b_dt, static_cast<T*>(c.out), g, c.eps, c.activation);
    return after_launch("group_norm_channels_last");
}
template <typename T, int E>
int run_resident(const GclCall& c, const GclGeom& g, cudaStream_t s) {
    if (c.activation == VRB_NO_ACTIVATION) return run_resident<T, E, 0>(c, g, s);
    if (c.activation == VRB_SILU) return run_resident<T, E, 1>(c, g, s);
    if (c.activation == VRB_GELU_TANH) return run_resident<T, E, 2>(c, g, s);
    return run_resident<T, E, 3>(c, g, s);
}
template <typename T>
int run_resident(const GclCall& c, const GclGeom& g, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    return entry_channels(g, V) == V ? run_resident<T, V>(c, g, s) : run_resident<T, 2>(c, g, s);
}

template <typename T, int V>
int run_passes(const GclCall& c, GclGeom g, char* workspace, cudaStream_t s) {
    set_width(g, V);
    set_splits(g);
    double* partial = reinterpret_cast<double*>(workspace);
    float2* stats = g.groups > kInlineGroups ? reinterpret_cast<float2*>(workspace + partial_bytes(g)) : nullptr;
    const dim3 ctas_stats(static_cast<unsigned>(g.batch * g.splits));
    const T* x = static_cast<const T*>(c.x);
    const int entry = entry_channels(g, V);
    if (entry == V) launch_overlapped(gcl_partial_kernel<T, V, V>, ctas_stats, dim3(kThreads), 0, s, x, partial, g);
    if constexpr (V > 2)
        if (entry == 2) launch_overlapped(gcl_partial_kernel<T, V, 2>, ctas_stats, dim3(kThreads), 0, s, x, partial, g);
    if constexpr (V > 1 && V < 8)
        if (entry == 1) launch_overlapped(gcl_partial_kernel<T, V, 1>, ctas_stats, dim3(kThreads), 0, s, x, partial, g);
    if (int rc = after_launch("group_norm_channels_last statistics")) return rc;
    if (stats) {
        launch_overlapped(gcl_finalize_kernel, dim3(static_cast<unsigned>(g.batch * ((g.groups + kFinalizeGroups - 1) / kFinalizeGroups))), dim3(kThreads), 0, s, partial,
                          stats, g, c.eps);
        if (int rc = after_launch("group_norm_channels_last finalize")) return rc;
    }
    g.rpp = kApplyThreads / g.slab;
    if (g.rpp > all_rows(g)) g.rpp = static_cast<int>(all_rows(g));
    const int64_t slabs = (g.vectors + g.slab - 1) / g.slab, units = g.batch * slabs;
    int64_t ctas = (static_cast<int64_t>(sm_count()) + units - 1) / units;
    const int64_t most = (all_rows(g) + g.rpp - 1) / g.rpp;
    if (ctas > most) ctas = most;
    const dim3 grid(static_cast<unsigned>(units * ctas));
#define VRB_GCL_APPLY(ACT) launch_overlapped(gcl_apply_kernel<T, V, ACT>, grid, dim3(kApplyThreads), 0, s, static_cast<const T*>(c.x), c.weight, c.w_dt, c.bias, c.b_dt, \
                                             static_cast<T*>(c.out), partial, stats, g, c.eps, static_cast<int>(ctas), c.activation)
    if (c.activation == VRB_NO_ACTIVATION) VRB_GCL_APPLY(0);
    else if (c.activation == VRB_SILU) VRB_GCL_APPLY(1);
    else if (c.activation == VRB_GELU_TANH) VRB_GCL_APPLY(2);
    else VRB_GCL_APPLY(3);
#undef VRB_GCL_APPLY
    return after_launch("group_norm_channels_last apply");
}

template <typename T, int V>
int run_width(const GclCall& c, GclGeom g, bool cluster, char* workspace, cudaStream_t s) {
    if (!cluster) return run_passes<T, V>(c, g, workspace, s);
    set_cluster(g, V, sizeof(T));
    const int entry = entry_channels(g, V);
    if constexpr (V > 2)
        if (entry == 2) return run_cluster<T, V, 2>(c, g, s);
    if constexpr (V > 1 && V < 8)
        if (entry == 1) return run_cluster<T, V, 1>(c, g, s);
    return run_cluster<T, V, V>(c, g, s);
}

}  // namespace
}  // namespace vrb

using namespace vrb;

extern "C" size_t vrb_group_norm_channels_last_workspace_bytes(int dtype, int64_t batch, int64_t spatial, int64_t channels, int groups) {
    GclGeom g;
    if (!is_float_dtype(dtype) || make_geom(g, batch, spatial, channels, groups)) return 0;
    // none where the cluster kernel takes the shape at every alignment a tensor can have
    const int element = static_cast<int>(dtype_bytes(dtype));
    bool cluster = true;
    for (int v = 16 / element; v >= 1 && cluster; v /= 2) {
        GclGeom h = g;
        if (channels % v == 0 && (v < 8 || groups == 1 || h.per % 2 == 0)) cluster = set_cluster(h, v, element);
    }
    return cluster ? 0 : workspace_size(g);
}

extern "C" int vrb_group_norm_channels_last(const void* x, int dtype, const void* weight, int weight_dtype,
                                            const void* bias, int bias_dtype, void* out,
                                            int64_t batch, int64_t spatial, int64_t channels, int groups, float eps,
                                            int activation, void* workspace, size_t workspace_bytes, vrb_stream stream) {
    VRB_REQUIRE(x && out, VRB_ERR_INVALID, "group_norm_channels_last: null tensor");
    VRB_REQUIRE(is_float_dtype(dtype), VRB_ERR_UNSUPPORTED, "group_norm_channels_last: dtype must be F32 or BF16");
    VRB_REQUIRE((!weight || is_float_dtype(weight_dtype)) && (!bias || is_float_dtype(bias_dtype)), VRB_ERR_UNSUPPORTED,
                "group_norm_channels_last: weight and bias must be F32 or BF16");
    VRB_REQUIRE(aligned_to(x, dtype_bytes(dtype)) && aligned_to(out, dtype_bytes(dtype)) && (!weight || aligned_to(weight, dtype_bytes(weight_dtype))) &&
                    (!bias || aligned_to(bias, dtype_bytes(bias_dtype))),
                VRB_ERR_INVALID, "group_norm_channels_last: tensors must be aligned to their elements");
    VRB_REQUIRE(activation >= VRB_NO_ACTIVATION && activation <= VRB_RELU, VRB_ERR_INVALID,
                "group_norm_channels_last: unknown activation %d", activation);
    GclGeom g;
    if (int rc = make_geom(g, batch, spatial, channels, groups)) return rc;
    int v = vector_width(dtype, batch, spatial, channels, groups, false, x, out);
    GclGeom h = g;
    const bool cluster = set_cluster(h, v, static_cast<int>(dtype_bytes(dtype)));
    GclGeom r = g;
    const bool resident = !cluster && set_resident(r, v, static_cast<int>(dtype_bytes(dtype)),
                                                   cluster_room(reinterpret_cast<const void*>(gcl_resident_kernel<uint16_t, 8, 0>), kResidentThreads, resident_most(1)));
    if (!cluster && !resident) v = vector_width(dtype, batch, spatial, channels, groups, true, x, out);
    const size_t need = cluster || resident ? 0 : workspace_size(g);
    VRB_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0), VRB_ERR_WORKSPACE,
                "group_norm_channels_last: workspace needs %zu bytes, 256-byte aligned", need);
    char* ws = static_cast<char*>(workspace);
    cudaStream_t s = as_stream(stream);
    const GclCall c{x, weight, bias, out, weight_dtype, bias_dtype, activation, eps};
    if (resident) return dtype == VRB_BF16 ? run_resident<uint16_t>(c, r, s) : run_resident<float>(c, r, s);
    if (dtype == VRB_BF16) {
        if (v == 8) return run_width<uint16_t, 8>(c, g, cluster, ws, s);
        if (v == 4) return run_width<uint16_t, 4>(c, g, cluster, ws, s);
        if (v == 2) return run_width<uint16_t, 2>(c, g, cluster, ws, s);
        return run_width<uint16_t, 1>(c, g, cluster, ws, s);
    }
    if (v == 4) return run_width<float, 4>(c, g, cluster, ws, s);
    if (v == 2) return run_width<float, 2>(c, g, cluster, ws, s);
    return run_width<float, 1>(c, g, cluster, ws, s);
}
