// Products of microscaled 4-bit rows (format and layout: include/b200idx.h) on the block-scaled tensor pipe:
// all scores as a matrix, or distances with the selection in the epilogue (the MX4 counterpart of dist_gemm.cuh).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "dist_gemm.cuh"

namespace b200 {

struct Mx4ProductArgs {
    int64_t m, n;
    int d;
    const uint8_t* a_codes;
    const uint8_t* a_scales;
    const uint8_t* b_codes;
    const uint8_t* b_scales;
    void* out;        // [m][ldo] in dtype
    int64_t ldo;
    int* err = nullptr;   // gets kDevErrPipelineTimeout where a wait runs out (plain stores, so it may lie in pinned memory)
};
// throws where a launch fails; num_sms: of the current device
void launch_mx4_product(int dtype, const Mx4ProductArgs& a, int num_sms, cudaStream_t stream);

// A pass of the exact search, as launch_dist_gemm's: a.A / a.B are the codes, a.d the elements of a row.
cudaError_t launch_mx4_dist(const GemmLaunch& L, const GemmArgs& a, const uint8_t* a_scales, const uint8_t* b_scales,
                            const CUtensorMap* mapA, const CUtensorMap* mapB, cudaStream_t stream);

// The same for up to 128 queries and thresholds (kModeAppend, not direct, consecutive tiles), with the base rows on the
// accumulator's lanes; cudaErrorNotSupported where the queries do not fit.
cudaError_t launch_mx4_few_search(const GemmArgs& a, const uint8_t* a_scales, const uint8_t* b_scales, int num_sms, cudaStream_t stream);

// Tensor map of codes: boxes of box_rows rows x 128 bytes (256 elements), SWIZZLE_128B.  0 on success.
int encode_mx4_map(CUtensorMap* out, const uint8_t* codes, int64_t rows, int d, int box_rows);

}  // namespace b200
