// How many clusters of a kernel the device runs at a time.
#pragma once
#include <cuda_runtime.h>

#include <map>
#include <mutex>
#include <utility>

namespace b200 {

// Asked once per kernel and device (which SMs share a group differs from device to device).  0 where the runtime cannot
// say: the caller does without clusters this time, and the next call asks again.
inline int clusters_at_once(const void* kern, const cudaLaunchConfig_t& cfg) {
    static std::mutex mu;
    static std::map<std::pair<const void*, int>, int> known;
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) == cudaSuccess) {
        std::lock_guard<std::mutex> l(mu);
        const auto it = known.find({kern, dev});
        if (it != known.end()) return it->second;
        if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) == cudaSuccess) return known[{kern, dev}] = n;
    }
    cudaGetLastError();   // (or the next launch reports it)
    return 0;
}

}  // namespace b200
