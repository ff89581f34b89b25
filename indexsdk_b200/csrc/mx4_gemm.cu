#include "mx4_gemm.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "row_ops.cuh"

namespace b200 {
namespace {

__device__ __forceinline__ float scale_value(uint32_t byte) {
    return byte == 0u ? __int_as_float(0x00400000) : __int_as_float(byte == 255u ? 0x7fc00000 : byte << 23);
}
// twice the value of a code
__device__ __forceinline__ int code2(uint32_t c) {
    const int m = static_cast<int>(0xC8643210u >> (4 * (c & 7u)) & 15u);
    return c & 8u ? -m : m;
}

// A thread per output: the 32 products of a block are whole quarters, so their sum is exact.
template <typename T>
__global__ void __launch_bounds__(256) mx4_product_kernel(const Mx4ProductArgs a) {
    const int nb = mx4_blocks(a.d), ng = mx4_groups(a.d);
    const int64_t pitch = mx4_pitch(a.d), total = a.m * a.n;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t r = i / a.n, c = i - r * a.n;
        const uint4* pa = reinterpret_cast<const uint4*>(a.a_codes + r * pitch);
        const uint4* pb = reinterpret_cast<const uint4*>(a.b_codes + c * pitch);
        float acc = 0.f;
        for (int b = 0; b < nb; ++b) {
            const uint4 va = pa[b], vb = pb[b];
            const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
            int dot = 0;
            for (int w = 0; w < 4; ++w)
                for (int e = 0; e < 8; ++e) dot += code2(wa[w] >> (4 * e) & 15u) * code2(wb[w] >> (4 * e) & 15u);
            const float sa = scale_value(a.a_scales[mx4_scale_word(r, b >> 2, ng) + (b & 3)]);
            const float sb = scale_value(a.b_scales[mx4_scale_word(c, b >> 2, ng) + (b & 3)]);
            acc += 0.25f * static_cast<float>(dot) * sa * sb;
        }
        T* o = static_cast<T*>(a.out) + r * a.ldo + c;
        if constexpr (std::is_same<T, float>::value) *o = acc;
        else if constexpr (std::is_same<T, __half>::value) *o = __float2half_rn(acc);
        else *o = __float2bfloat16_rn(acc);
    }
}

}  // namespace

void launch_mx4_product(int dtype, const Mx4ProductArgs& a, cudaStream_t st) {
    const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((a.m * a.n + 255) / 256, 148 * 64));
    if (dtype == kF32) mx4_product_kernel<float><<<blocks, 256, 0, st>>>(a);
    else if (dtype == kF16) mx4_product_kernel<__half><<<blocks, 256, 0, st>>>(a);
    else mx4_product_kernel<__nv_bfloat16><<<blocks, 256, 0, st>>>(a);
    B200_CUDA_CHECK(cudaGetLastError());
}

}  // namespace b200
