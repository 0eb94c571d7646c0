// The launch helpers of vrb_common.cuh against a runtime that refuses the programmatic attribute: every launch has to be tried
// again without it, clusters kept.  The runtime's calls are stood in for here; nothing reaches a GPU.
#include <vector>

#include "vrb_common.cuh"

namespace vrb {
std::atomic<int> g_launch_overlap{1};
std::atomic<uint64_t> g_launches{0};
std::atomic<uint64_t> g_device_allocations{0};
void set_error(const char*, ...) {}
int sm_count() { return 148; }
}  // namespace vrb

struct Launch {
    unsigned grid, block, cluster;
    size_t shared;
    bool programmatic;
};
static std::vector<Launch> launches;
static bool refuse = false;
static cudaError_t last = cudaSuccess;

extern "C" cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* config, const void*, void** args) {
    Launch l{config->gridDim.x, config->blockDim.x, 0, config->dynamicSmemBytes, false};
    for (unsigned i = 0; i < config->numAttrs; ++i) {
        if (config->attrs[i].id == cudaLaunchAttributeClusterDimension) l.cluster = config->attrs[i].val.clusterDim.x;
        if (config->attrs[i].id == cudaLaunchAttributeProgrammaticStreamSerialization) l.programmatic = true;
    }
    if (*static_cast<int*>(args[0]) != 7) return last = cudaErrorInvalidValue;
    launches.push_back(l);
    return last = refuse && l.programmatic ? cudaErrorNotSupported : cudaSuccess;
}
extern "C" cudaError_t cudaGetLastError() {
    const cudaError_t e = last;
    last = cudaSuccess;
    return e;
}
extern "C" const char* cudaGetErrorString(cudaError_t) { return "refused"; }

static void kernel(int, const float*) {}
static int failures = 0;
#define CHECK(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); ++failures; } } while (0)

int main() {
    using namespace vrb;
    const float* data = nullptr;
    for (int cluster : {1, 2, 8}) {
        for (bool refused : {false, true}) {
            refuse = refused;
            launches.clear();
            g_launch_overlap = 1;
            launch_clusters(kernel, dim3(16), dim3(256), 4096, cluster, nullptr, 7, data);
            CHECK(after_launch("clusters") == VRB_OK);
            CHECK(launches.size() == (refused ? 2u : 1u));
            CHECK(launches.front().programmatic && launches.back().programmatic == !refused);
            CHECK(g_launch_overlap.load() == (refused ? 0 : 1));
            for (const Launch& l : launches) CHECK(l.grid == 16 && l.block == 256 && l.shared == 4096 && l.cluster == static_cast<unsigned>(cluster));
            launch_clusters(kernel, dim3(8), dim3(64), 0, cluster, nullptr, 7, data);   // the attribute stays away from then on
            CHECK(after_launch("clusters") == VRB_OK);
            CHECK(launches.back().programmatic == !refused && launches.back().grid == 8 && launches.size() == (refused ? 3u : 2u));
            launches.clear();
            g_launch_overlap = 1;
            launch_overlapped(kernel, dim3(5), dim3(32), 16, nullptr, 7, data);
            CHECK(after_launch("plain") == VRB_OK);
            CHECK(launches.back().programmatic == !refused && launches.back().cluster == 0 && launches.back().grid == 5);
        }
    }
    std::printf(failures ? "failed\n" : "all launches went through\n");
    return failures != 0;
}
