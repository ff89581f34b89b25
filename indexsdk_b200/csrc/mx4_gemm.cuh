// Products of microscaled 4-bit rows (format and layout: include/b200idx.h).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

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
};
// throws std::runtime_error where a launch fails
void launch_mx4_product(int dtype, const Mx4ProductArgs& a, cudaStream_t stream);

}  // namespace b200
