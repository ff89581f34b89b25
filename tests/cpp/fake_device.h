// A device for tests of host code without a GPU: a CUDA runtime on host memory, whose pointers say of themselves what a
// test has told them to, and launches that do nothing unless a test gives them something to do.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <map>
#include <string>

#include "../../indexsdk_b200/csrc/flat_index.h"
#include "../../indexsdk_b200/csrc/mx4_gemm.cuh"
#include "../../indexsdk_b200/csrc/row_ops.cuh"
#include "../../indexsdk_b200/csrc/select.cuh"

static int current_device = 0;
static std::map<const void*, cudaPointerAttributes> known;   // addresses that are not device memory of device 0
static void place(const void* p, cudaMemoryType type, int device) {
    cudaPointerAttributes at{};
    at.type = type;
    at.device = device;
    known[p] = at;
}

extern "C" {
cudaError_t cudaMalloc(void** p, size_t n) { *p = std::calloc(1, n); return cudaSuccess; }
cudaError_t cudaMallocHost(void** p, size_t n) { *p = std::calloc(1, n); return cudaSuccess; }
cudaError_t cudaFree(void* p) { std::free(p); return cudaSuccess; }
cudaError_t cudaFreeHost(void* p) { std::free(p); return cudaSuccess; }
cudaError_t cudaMemcpy(void* d, const void* s, size_t n, cudaMemcpyKind) { std::memcpy(d, s, n); return cudaSuccess; }
cudaError_t cudaMemcpyAsync(void* d, const void* s, size_t n, cudaMemcpyKind, cudaStream_t) { std::memcpy(d, s, n); return cudaSuccess; }
cudaError_t cudaMemcpy2DAsync(void*, size_t, const void*, size_t, size_t, size_t, cudaMemcpyKind, cudaStream_t) { return cudaErrorNotSupported; }
cudaError_t cudaMemset(void* d, int v, size_t n) { std::memset(d, v, n); return cudaSuccess; }
cudaError_t cudaMemsetAsync(void* d, int v, size_t n, cudaStream_t) { std::memset(d, v, n); return cudaSuccess; }
cudaError_t cudaStreamCreateWithFlags(cudaStream_t* s, unsigned) { *s = reinterpret_cast<cudaStream_t>(1); return cudaSuccess; }
cudaError_t cudaStreamDestroy(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaEventCreate(cudaEvent_t*) { return cudaSuccess; }
cudaError_t cudaEventDestroy(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t, cudaStream_t) { return cudaSuccess; }
cudaError_t cudaEventElapsedTime(float*, cudaEvent_t, cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaGetDevice(int* d) { *d = current_device; return cudaSuccess; }
cudaError_t cudaSetDevice(int d) { current_device = d; return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int) { *v = 148; return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "an error"; }
cudaError_t cudaPointerGetAttributes(cudaPointerAttributes* at, const void* p) {
    const auto it = known.find(p);
    *at = cudaPointerAttributes{};
    at->type = cudaMemoryTypeDevice;
    if (it != known.end()) *at = it->second;
    return cudaSuccess;
}
}

namespace b200 {
static std::function<void(const GemmLaunch&, const GemmArgs&)> on_dist_gemm;
static std::function<void(uint64_t* cand, const uint32_t* counts, uint32_t cap, uint8_t* over, const EmitArgs&)> on_select;
static std::function<void(const Mx4ProductArgs&)> on_product;

int encode_mx4_map(CUtensorMap*, const uint8_t*, int64_t, int, int) { return 0; }
int encode_operand_map(CUtensorMap*, int, const void*, int64_t, int, int) { return 0; }
cudaError_t launch_mx4_dist(const GemmLaunch& L, const GemmArgs& a, const uint8_t*, const uint8_t*, const CUtensorMap*, const CUtensorMap*, cudaStream_t) {
    if (on_dist_gemm) on_dist_gemm(L, a);
    return cudaSuccess;
}
cudaError_t launch_dist_gemm(const GemmLaunch& L, const GemmArgs& a, const CUtensorMap*, const CUtensorMap*, cudaStream_t) {
    if (on_dist_gemm) on_dist_gemm(L, a);
    return cudaSuccess;
}
void launch_mx4_product(int, const Mx4ProductArgs& a, int, cudaStream_t) {
    if (on_product) on_product(a);
}
cudaError_t launch_fill_u32(uint32_t* p, int64_t n, uint32_t v, cudaStream_t) {
    for (int64_t i = 0; i < n; ++i) p[i] = v;
    return cudaSuccess;
}
cudaError_t launch_iota_i64(int64_t* p, int64_t n, int64_t start, cudaStream_t) {
    for (int64_t i = 0; i < n; ++i) p[i] = start + i;
    return cudaSuccess;
}
cudaError_t launch_gather_rows(const void*, const int32_t*, int, int, void*, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_rms_norm_i8(int, const RmsNormArgs&, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_i8_dequantize(int64_t, int, const int8_t*, int64_t, const float*, const float*, int, void*, int64_t, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_mx4_quantize(int, int64_t, int, const void*, int64_t, int64_t, uint8_t*, uint8_t*, float*, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_mx4_dequantize(int64_t, int64_t, int, const uint8_t*, const uint8_t*, int, void*, int64_t, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_mx4_move_scales(int, int64_t, int64_t, uint8_t*, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_mx4_pack_rows(int64_t, int, int64_t, uint8_t*, uint8_t*, uint8_t*, bool, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_mx4_norms(int64_t, int, int64_t, const uint8_t*, const uint8_t*, float*, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_f32_to_f16(const float*, int64_t, void*, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_base_prep_f32(const float*, int64_t, int, int, void*, int64_t, float*, float*, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_base_prep_f16(const void*, int64_t, int, float*, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_base_prep_i8(const int8_t*, int64_t, int, int32_t*, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_prep_queries_f32(const float*, int, int, int, float, void*, float*, float*, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_prep_queries_f16(const void*, int, int, float*, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_prep_queries_i8(const int8_t*, int, int, int32_t*, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_kth_threshold(const uint32_t*, int, int, int, int, const float*, uint32_t, uint32_t*, const TauFold&, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_tighten_tau(const uint64_t*, const uint32_t*, uint32_t, int, int, const float*, uint32_t*, const TauFold&, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_prune_candidates(uint64_t*, uint32_t*, uint32_t, int, int, const float*, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_refine_f32(uint64_t*, const uint32_t*, uint32_t, uint32_t, int, int, int, const float*, const float*, cudaStream_t, int, const MemberView*) { return cudaSuccess; }
cudaError_t launch_finish_f32(const uint64_t*, const uint32_t*, uint32_t, int, const float*, const float*, const float*, uint8_t*, uint32_t*, const EmitArgs&, bool, cudaStream_t) { return cudaSuccess; }
cudaError_t launch_select_emit(const uint64_t* cand, const uint32_t* counts, uint32_t, uint32_t cap, uint8_t* over, uint32_t*, const EmitArgs& e, cudaStream_t) {
    if (on_select) on_select(const_cast<uint64_t*>(cand), counts, cap, over, e);
    if (e.err && e.err_host && *e.err) *e.err_host = *e.err;   // (as the kernel does)
    return cudaSuccess;
}
}  // namespace b200

static int failed = 0;
static void check(bool ok, const std::string& what) {
    if (ok) return;
    std::printf("FAILED: %s\n", what.c_str());
    ++failed;
}
// The message of the exception that f ends with, "" where it ends with none.
static std::string thrown(const std::function<void()>& f) {
    try {
        f();
    } catch (const std::exception& e) {
        return e.what();
    }
    return "";
}
