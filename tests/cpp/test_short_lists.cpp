// MX4 searches whose thresholds are too low, as if the kernel that made them had rounded its sums otherwise than the
// one that collects candidates: the results are those of the search without that.  Linked with the library's objects and
// --wrap, which puts __wrap_... below between the index and its threshold kernel.
#include <b200idx.h>
#include <cuda_runtime.h>

#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

#include "../../indexsdk_b200/csrc/select.cuh"

static int planted = 0;   // steps of fp32
#define THRESHOLDS(prefix) prefix##_ZN4b20020launch_kth_thresholdEPKjiiiiPKfjPjRKNS_7TauFoldEP11CUstream_st
extern "C" cudaError_t THRESHOLDS(__real_)(const uint32_t*, int, int, int, int, const float*, uint32_t, uint32_t*, const b200::TauFold&, cudaStream_t);
extern "C" cudaError_t THRESHOLDS(__wrap_)(const uint32_t* mins, int stride, int n, int nq, int k, const float* eps, uint32_t all, uint32_t* tau, const b200::TauFold& fold, cudaStream_t st) {
    cudaError_t e = THRESHOLDS(__real_)(mins, stride, n, nq, k, eps, all, tau, fold, st);
    if (e != cudaSuccess || !planted) return e;
    std::vector<uint32_t> t(nq);
    e = cudaMemcpyAsync(t.data(), tau, nq * 4, cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    for (uint32_t& v : t) v -= v < all ? planted : 0;
    if (e == cudaSuccess) e = cudaMemcpyAsync(tau, t.data(), nq * 4, cudaMemcpyHostToDevice, st);
    return e == cudaSuccess ? cudaStreamSynchronize(st) : e;
}

static int failed = 0;
static void must(bool ok, const char* what, int metric, int nq, int k) {
    if (ok) return;
    std::printf("FAILED: %s (metric %d, %d queries, k %d)\n", what, metric, nq, k);
    ++failed;
}

int main() {
    constexpr int d = 64, n = 30000;
    std::mt19937 g(1);
    std::normal_distribution<float> f;
    std::vector<float> x(static_cast<size_t>(n) * d), q(static_cast<size_t>(130) * d);
    for (float& v : x) v = f(g);
    for (float& v : q) v = f(g);
    for (int metric : {0, 1}) {
        b200idx_t* ix = nullptr;
        must(b200idx_create_flat(d, metric, B200IDX_MX4, 0, &ix) == 0 && b200idx_add(ix, n, x.data(), nullptr) == 0, "add", metric, 0, 0);
        for (int nq : {1, 17, 128, 130})
            for (int k : {1, 4, 600}) {
                std::vector<float> D[2];
                std::vector<int64_t> I[2];
                b200idx_stats_t st;
                for (int side : {0, 1}) {
                    D[side].resize(static_cast<size_t>(nq) * k);
                    I[side].resize(static_cast<size_t>(nq) * k);
                    // A threshold is the upper edge of a bin that the k-th smallest minimum lies in, 2^-16 of the 2^32 ordered
                    // keys wide at most: 2^17 steps lower it is below that minimum.  (k = 1: nothing is left.)  Half a binade
                    // lower: hundreds of keys are lost.
                    planted = side ? (k == 600 ? 1 << 22 : 1 << 17) : 0;
                    b200idx_stats(ix, &st, 1);
                    must(b200idx_search(ix, nq, q.data(), k, D[side].data(), I[side].data()) == 0, b200idx_last_error(ix), metric, nq, k);
                    planted = 0;
                    b200idx_stats(ix, &st, 0);
                    must(side || st.fallback_queries == 0, "nothing is searched for again without need", metric, nq, k);
                    if (side && k != 4) must(st.fallback_queries == static_cast<uint64_t>(nq), "short lists are searched for again", metric, nq, k);
                }
                must(!std::memcmp(D[0].data(), D[1].data(), D[0].size() * 4) && !std::memcmp(I[0].data(), I[1].data(), I[0].size() * 8), "the same results", metric, nq, k);
            }
        // fewer rows than k: a short list is the whole answer
        std::vector<float> D(700);
        std::vector<int64_t> I(700);
        b200idx_reset(ix);
        b200idx_add(ix, 3, x.data(), nullptr);
        must(b200idx_search(ix, 1, q.data(), 700, D.data(), I.data()) == 0 && I[2] >= 0 && I[3] == -1, "three rows", metric, 1, 700);
        b200idx_destroy(ix);
    }
    std::printf("%d failed\n", failed);
    return failed != 0;
}
