// How many clusters run at a time: kept per kernel and device, failures not at all; with a CUDA runtime of this file's own.
#include "../../indexsdk_b200/csrc/cluster_limit.h"

#include <cstdio>

static int current_device = 0, asked = 0, cleared = 0;
static bool fail = false;
extern "C" {
cudaError_t cudaGetDevice(int* d) { *d = current_device; return cudaSuccess; }
cudaError_t cudaGetLastError() { ++cleared; return cudaSuccess; }
cudaError_t cudaOccupancyMaxActiveClusters(int* n, const void* kern, const cudaLaunchConfig_t*) {
    ++asked;
    if (fail) return cudaErrorInvalidClusterSize;
    *n = 70 + current_device + (kern ? 2 : 0);
    return cudaSuccess;
}
}
static int failed = 0;
static void check(bool ok, const char* what) {
    if (ok) return;
    std::printf("FAILED: %s\n", what);
    ++failed;
}

int main() {
    cudaLaunchConfig_t cfg{};
    const char kernel[2] = {};
    auto ask = [&](int k) { return b200::clusters_at_once(kernel + k, cfg); };
    fail = true;
    check(ask(0) == 0 && asked == 1 && cleared == 1, "a failure is 0, and no error stays behind");
    fail = false;
    check(ask(0) == 72 && asked == 2, "the next call asks again");
    check(ask(0) == 72 && asked == 2, "and the one after it knows");
    current_device = 1;
    check(ask(0) == 73 && asked == 3, "another device has a number of its own");
    check(ask(1) == 73 && asked == 4, "so has another kernel");
    current_device = 0;
    check(ask(0) == 72 && asked == 4, "both are kept");
    std::printf("%d failed\n", failed);
    return failed != 0;
}
