// Operators on rows in few bits: RMS norm with int8 output, int8 reconstruction, and rounding to and from
// microscaled 4-bit blocks (formats and layouts: include/b200idx.h).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace b200 {

constexpr int kMx4Block = 32;         // elements that share a scale
constexpr int kMaxRowElems = 16384;

inline __host__ __device__ int mx4_blocks(int d) { return (d + kMx4Block - 1) / kMx4Block; }
inline __host__ __device__ int mx4_groups(int d) { return (mx4_blocks(d) + 3) / 4; }
inline __host__ __device__ int64_t mx4_pitch(int d) { return int64_t(16) * mx4_blocks(d); }
inline __host__ __device__ int64_t mx4_scale_bytes(int64_t n, int d) { return (n + 127) / 128 * mx4_groups(d) * 512; }
// Byte offset of the four scales of group g (blocks 4 g .. 4 g + 3) of row r.
inline __host__ __device__ int64_t mx4_scale_word(int64_t r, int g, int ng) {
    return ((r >> 7) * ng + g) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4;
}

struct RmsNormArgs {
    int64_t n;
    int d;
    const void* x;
    int64_t ldx;
    const void* residual;   // or nullptr
    int64_t ldr;
    void* sum;              // or nullptr; with residual only
    int64_t lds;
    const void* weight;
    float eps;
    const float* static_scale;   // exactly one of static_scale and scales
    int8_t* q;
    int64_t ldq;
    float* scales;
};
cudaError_t launch_rms_norm_i8(int dtype, const RmsNormArgs& a, cudaStream_t stream);
cudaError_t launch_i8_dequantize(int64_t n, int d, const int8_t* q, int64_t ldq, const float* scales,
                                 const float* static_scale, int dtype, void* out, int64_t ldo, cudaStream_t stream);

// codes / scales: the whole buffers; the n rows of x become rows row0, row0 + 1, ...  norms: nullptr or (kF32 only) an fp32
// array indexed like the rows, which gets the squared norms of the ROUNDED rows.
cudaError_t launch_mx4_quantize(int dtype, int64_t n, int d, const void* x, int64_t ldx, int64_t row0, uint8_t* codes,
                                uint8_t* scales, float* norms, cudaStream_t stream);
cudaError_t launch_mx4_dequantize(int64_t row0, int64_t n, int d, const uint8_t* codes, const uint8_t* scales, int dtype,
                                  void* out, int64_t ldo, cudaStream_t stream);

// Scales of row `from` -> row `to`.
cudaError_t launch_mx4_move_scales(int d, int64_t from, int64_t to, uint8_t* scales, cudaStream_t stream);
// n rows from row0 on <-> a plain array that holds each row's codes and then its nb scale bytes (out: true, into it).
cudaError_t launch_mx4_pack_rows(int64_t n, int d, int64_t row0, uint8_t* codes, uint8_t* scales, uint8_t* plain, bool out,
                                 cudaStream_t stream);
// Squared norms of rows row0 .. row0 + n - 1 into the same places of norms.
cudaError_t launch_mx4_norms(int64_t n, int d, int64_t row0, const uint8_t* codes, const uint8_t* scales, float* norms,
                             cudaStream_t stream);

}  // namespace b200
