#include "row_ops.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace b200 {
namespace {

// ---- eight consecutive elements of a row <-> fp32 ----
template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T>
union Pack8 {
    uint4 v[sizeof(T) / 2];
    T e[8];
    __device__ Pack8() {}
};
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {   // 16-byte aligned
    Pack8<T> k;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) k.v[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f<T>(k.e[i]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
    Pack8<T> k;
#pragma unroll
    for (int i = 0; i < 8; ++i) k.e[i] = from_f<T>(f[i]);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = k.v[i];
}

// ---------------------------------------------------------------------------------------
// RMS norm -> int8.  A row belongs to NT threads (a warp or a block), which keep it in registers: one pass
// over memory, one reduction (sum of squares and the largest |s w| together -- the norm's factor is the same
// for the whole row, so it is not needed to find the largest element, and q = round(s w * 127 / max|s w|)
// does not contain it at all).  Thread t owns the chunks of 8 elements t, t + NT, ... (VEC) or the elements
// t, t + NT, ... (rows that are not 16-byte aligned; loads stay coalesced).
// ---------------------------------------------------------------------------------------
template <int NT>
__device__ __forceinline__ void reduce_row(float& sum, float& top, float (&sh)[2][NT / 32 + 1]) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    }
    if (NT > 32) {
        const int w = threadIdx.x >> 5;
        __syncthreads();   // (the values of the reduction before have been read)
        if ((threadIdx.x & 31) == 0) { sh[0][w] = sum; sh[1][w] = top; }
        __syncthreads();
        sum = sh[0][0];
        top = sh[1][0];
#pragma unroll
        for (int i = 1; i < NT / 32; ++i) {
            sum += sh[0][i];
            top = fmaxf(top, sh[1][i]);
        }
    }
}

template <typename T, bool VEC, int NT, int J>
__global__ void __launch_bounds__(NT == 32 ? 128 : NT) rms_norm_i8_kernel(const RmsNormArgs a) {
    __shared__ float sh[2][NT / 32 + 1];
    constexpr int kRows = NT == 32 ? 4 : 1;   // rows a block works on at a time
    const int t = NT == 32 ? threadIdx.x & 31 : threadIdx.x;
    const T* weight = static_cast<const T*>(a.weight);
    // element e of chunk j of this thread
    auto at = [&](int j, int e) { return VEC ? (t + NT * j) * 8 + e : t + NT * (8 * j + e); };
    auto whole = [&](int j) { return VEC && at(j, 8) <= a.d; };
    auto fetch = [&](const T* p, int j, float (&f)[8]) {
        if (whole(j)) {
            load8<T>(p + at(j, 0), f);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = at(j, e) < a.d ? to_f<T>(p[at(j, e)]) : 0.f;
        }
    };
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + (NT == 32 ? threadIdx.x >> 5 : 0); row < a.n;
         row += static_cast<int64_t>(gridDim.x) * kRows) {
        const T* x = static_cast<const T*>(a.x) + row * a.ldx;
        float v[J][8];
#pragma unroll
        for (int j = 0; j < J; ++j) fetch(x, j, v[j]);
        T* sum_row = static_cast<T*>(a.sum) + row * a.lds;
        if (a.residual) {
            const T* r = static_cast<const T*>(a.residual) + row * a.ldr;
            float f[J][8];
#pragma unroll
            for (int j = 0; j < J; ++j) fetch(r, j, f[j]);
#pragma unroll
            for (int j = 0; j < J; ++j) {
                // The sum is rounded to the rows' type BEFORE it is normalised: what is normalised is what the
                // model carries on, so the result is that of the two steps done one after the other.
#pragma unroll
                for (int e = 0; e < 8; ++e) v[j][e] = to_f<T>(from_f<T>(v[j][e] + f[j][e]));
                if (!a.sum) continue;
                if (whole(j)) {
                    store8<T>(sum_row + at(j, 0), v[j]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (at(j, e) < a.d) sum_row[at(j, e)] = from_f<T>(v[j][e]);
                }
            }
        }
        float ssq = 0.f, top = 0.f, pre = 1.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            float w[8];
            fetch(weight, j, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                ssq = fmaf(v[j][e], v[j][e], ssq);
                v[j][e] *= w[e];
                top = fmaxf(top, fabsf(v[j][e]));
            }
        }
        reduce_row<NT>(ssq, top, sh);
        if (!(ssq <= 3.4e38f) || !(top <= 3.4e38f)) {
            // The squares left the range of fp32 (or the row holds no numbers): once more with values scaled by
            // 2^-100.  The sum may have taken x's or the residual's place; this thread wrote what it reads.
            pre = 7.8886090522101181e-31f;
            ssq = top = 0.f;
            const T* again = a.sum ? sum_row : x;
            const T* r = a.residual && !a.sum ? static_cast<const T*>(a.residual) + row * a.ldr : nullptr;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                float w[8];
                fetch(again, j, v[j]);
                if (r) {
                    fetch(r, j, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[j][e] = to_f<T>(from_f<T>(v[j][e] + w[e]));
                }
                fetch(weight, j, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float s = v[j][e] * pre;
                    ssq = fmaf(s, s, ssq);
                    v[j][e] = s * w[e];
                    top = fmaxf(top, fabsf(v[j][e]));
                }
            }
            reduce_row<NT>(ssq, top, sh);
        }
        const float rinv = 1.f / sqrtf(ssq / static_cast<float>(a.d) + a.eps * pre * pre);   // y = v * rinv
        const bool numbers = ssq <= 3.4e38f;   // false for NaN and infinities
        float c, up = 1.f;   // q = round(v * up * c)
        if (a.static_scale) {
            const float s = __ldg(a.static_scale);
            c = numbers && s > 0.f && s <= 3.4e38f ? rinv / s : 0.f;
        } else {
            up = top < 1e-20f ? 18446744073709551616.f : 1.f;   // keeps 127 / top in range; a power of two
            c = numbers && top > 0.f ? 127.f / (top * up) : 0.f;
            if (t == 0) a.scales[row] = numbers ? top * rinv / 127.f : __int_as_float(0x7fc00000);
        }
        int8_t* q = a.q + row * a.ldq;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            int b[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float u = v[j][e] * up * c;
                b[e] = c == 0.f ? 0 : __float2int_rn(fminf(fmaxf(u, -127.f), 127.f));
            }
            if (whole(j)) {
                uint2 o;
                o.x = (b[0] & 255) | (b[1] & 255) << 8 | (b[2] & 255) << 16 | b[3] << 24;
                o.y = (b[4] & 255) | (b[5] & 255) << 8 | (b[6] & 255) << 16 | b[7] << 24;
                *reinterpret_cast<uint2*>(q + at(j, 0)) = o;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (at(j, e) < a.d) q[at(j, e)] = static_cast<int8_t>(b[e]);
            }
        }
    }
}

// ---- int8 rows -> values; a thread per 8 elements ----
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) i8_dequantize_kernel(int64_t n, int d, const int8_t* q, int64_t ldq,
                                                            const float* scales, const float* static_scale, T* out,
                                                            int64_t ldo) {
    const int per = (d + 7) / 8;   // VEC: chunks of a row;  else threads of a row, each with every per-th element
    const int64_t total = n * per;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t row = i / per;
        const int c = static_cast<int>(i - row * per);
        const float s = __ldg(scales ? scales + row : static_scale);
        const int8_t* p = q + row * ldq;
        T* o = out + row * ldo;
        if (VEC && c * 8 + 8 <= d) {
            const uint2 u = *reinterpret_cast<const uint2*>(p + c * 8);
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                f[e] = static_cast<float>(static_cast<int8_t>((e < 4 ? u.x : u.y) >> (8 * (e & 3)))) * s;
            store8<T>(o + c * 8, f);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int k = VEC ? c * 8 + e : c + e * per;
                if (k < d) o[k] = from_f<T>(static_cast<float>(p[k]) * s);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------
// MX4
// ---------------------------------------------------------------------------------------
// Two fp32 values -> two E2M1 codes (lo in bits 0-3): nearest, ties to even, magnitudes above 6 become 6.
__device__ __forceinline__ uint32_t e2m1_pair(float lo, float hi) {
    uint32_t r;
    asm("{\n"
        ".reg .b8 t;\n"
        "cvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n"
        "cvt.u32.u8 %0, t;\n"
        "}\n"
        : "=r"(r)
        : "f"(lo), "f"(hi));
    return r;
}
// Two codes (bits 0-3, 4-7 of the low byte) -> their values.
__device__ __forceinline__ float2 e2m1_values(uint32_t byte) {
    uint32_t h;
    asm("{\n"
        ".reg .b8 t;\n"
        "cvt.u8.u32 t, %1;\n"
        "cvt.rn.f16x2.e2m1x2 %0, t;\n"
        "}\n"
        : "=r"(h)
        : "r"(byte));
    return __half22float2(*reinterpret_cast<__half2*>(&h));
}
__device__ __forceinline__ float e8m0_value(uint32_t byte) {   // 2^(byte - 127), NaN for 255
    return byte == 0u ? __int_as_float(0x00400000) : __int_as_float(byte == 255u ? 0x7fc00000 : byte << 23);
}

// Rounding to MX4.  Half a warp (16 threads of 8 elements, four threads a block of 32) works on one group of
// 128 elements, so that the four scale bytes of a group leave as one word and the codes of a group as 64
// contiguous bytes.  A warp takes whole rows (two groups at a time), which lets it add up the squared norm of
// the rounded row on the way where an index asks for it; `split` warps share a row where there are few rows
// (each warp then starts at a group of its own; not with norms).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) mx4_quantize_kernel(int64_t n, int d, const T* x, int64_t ldx, int64_t row0,
                                                           uint8_t* codes, uint8_t* scales, float* norms, int split) {
    __shared__ float stage[VEC ? 1 : 8][2][132];
    const int lane = threadIdx.x & 31, half = lane >> 4, t = lane & 15, warp = threadIdx.x >> 5;
    const int nb = mx4_blocks(d), ng = mx4_groups(d);
    const int64_t pitch = mx4_pitch(d);
    const int64_t warps = static_cast<int64_t>(gridDim.x) * 8;
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * 8 + warp; u < n * split; u += warps) {
        const int64_t row = u / split;
        const int part = static_cast<int>(u - row * split);
        const T* xr = x + row * ldx;
        uint8_t* crow = codes + (row0 + row) * pitch;
        float nrm = 0.f;
        for (int g0 = 2 * part; g0 < ng; g0 += 2 * split) {
            const int g = g0 + half, k = g * 128 + t * 8;   // this thread's first element
            float f[8];
            if (VEC) {
                if (k + 8 <= d) {
                    load8<T>(xr + k, f);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] = k + e < d ? to_f<T>(xr[k + e]) : 0.f;
                }
            } else {
                // coalesced loads, turned to eight consecutive elements a thread in shared memory
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int m = g * 128 + e * 16 + t;
                    stage[warp][half][e * 16 + t] = m < d ? to_f<T>(xr[m]) : 0.f;
                }
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = stage[warp][half][t * 8 + e];
                __syncwarp();
            }
            float top = 0.f;
            bool fine = true;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                top = fmaxf(top, fabsf(f[e]));
                fine = fine && fabsf(f[e]) <= 3.402823466e+38f;   // (NaN compares false)
            }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
                fine = __shfl_xor_sync(0xFFFFFFFFu, static_cast<int>(fine), o) != 0 && fine;
            }
            // floor(log2(top)) is the exponent field; a subnormal or zero top ends at the smallest scale anyway
            const int field = static_cast<int>(__float_as_uint(top) >> 23) - 2;
            const int byte = fine ? max(field, 0) : 255;
            const float inv = fine ? __int_as_float((254 - byte) << 23) : 0.f;   // 2^(127 - byte)
            uint32_t c = 0;
            if (fine) {
#pragma unroll
                for (int e = 0; e < 4; ++e) c |= e2m1_pair(f[2 * e] * inv, f[2 * e + 1] * inv) << (8 * e);
            }
            if (norms) {
                float part_sum = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 v = e2m1_values(c >> (8 * e));
                    part_sum = fmaf(v.x, v.x, fmaf(v.y, v.y, part_sum));   // exact: at most 288, in quarters
                }
                if (g * 4 + (t >> 2) < nb) {
                    const float s = e8m0_value(byte);
                    nrm = fmaf(part_sum * s, s, nrm);
                }
            }
            if (g * 4 + (t >> 2) < nb) *reinterpret_cast<uint32_t*>(crow + static_cast<int64_t>(g) * 64 + t * 4) = c;
            uint32_t word = static_cast<uint32_t>(g * 4 + (t >> 2) < nb ? byte : 127) << (8 * (t >> 2));
            word |= __shfl_xor_sync(0xFFFFFFFFu, word, 4);
            word |= __shfl_xor_sync(0xFFFFFFFFu, word, 8);
            if (t == 0 && g < ng) *reinterpret_cast<uint32_t*>(scales + mx4_scale_word(row0 + row, g, ng)) = word;
        }
        if (norms) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) nrm += __shfl_xor_sync(0xFFFFFFFFu, nrm, o);
            if (lane == 0) norms[row0 + row] = nrm;
        }
    }
}

// MX4 -> values; a thread per 8 elements (one word of codes).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) mx4_dequantize_kernel(int64_t row0, int64_t n, int d, const uint8_t* codes,
                                                             const uint8_t* scales, T* out, int64_t ldo) {
    const int per = (d + 7) / 8, ng = mx4_groups(d);
    const int64_t pitch = mx4_pitch(d), total = n * per;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t row = i / per;
        const int c = static_cast<int>(i - row * per);
        const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + (row0 + row) * pitch + c * 4);
        const int b = c >> 2;
        const float s = e8m0_value(__ldg(scales + mx4_scale_word(row0 + row, b >> 2, ng) + (b & 3)));
        T* o = out + row * ldo + c * 8;
        float f[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 v = e2m1_values(w >> (8 * e) & 255u);
            f[2 * e] = v.x * s;
            f[2 * e + 1] = v.y * s;
        }
        if (VEC && c * 8 + 8 <= d) {
            store8<T>(o, f);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c * 8 + e < d) o[e] = from_f<T>(f[e]);
        }
    }
}

__global__ void mx4_move_scales_kernel(int ng, int64_t from, int64_t to, uint8_t* scales) {
    for (int g = threadIdx.x; g < ng; g += blockDim.x)
        *reinterpret_cast<uint32_t*>(scales + mx4_scale_word(to, g, ng)) = *reinterpret_cast<const uint32_t*>(scales + mx4_scale_word(from, g, ng));
}

// A warp per row.
__global__ void __launch_bounds__(256) mx4_pack_rows_kernel(int64_t n, int d, int64_t row0, uint8_t* codes, uint8_t* scales,
                                                            uint8_t* plain, int out) {
    const int nb = mx4_blocks(d), ng = mx4_groups(d), lane = threadIdx.x & 31;
    const int64_t pitch = mx4_pitch(d);
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); r < n; r += static_cast<int64_t>(gridDim.x) * 8) {
        uint8_t* c = codes + (row0 + r) * pitch;
        uint8_t* p = plain + r * (pitch + nb);
        for (int i = lane; i < pitch; i += 32) {
            if (out) p[i] = c[i];
            else c[i] = p[i];
        }
        for (int b = lane; b < 4 * ng; b += 32) {
            uint8_t* s = scales + mx4_scale_word(row0 + r, b >> 2, ng) + (b & 3);
            if (!out) *s = b < nb ? p[pitch + b] : 127;
            else if (b < nb) p[pitch + b] = *s;
        }
    }
}

__global__ void __launch_bounds__(256) mx4_norms_kernel(int64_t n, int d, int64_t row0, const uint8_t* codes,
                                                        const uint8_t* scales, float* norms) {
    const int nb = mx4_blocks(d), ng = mx4_groups(d), lane = threadIdx.x & 31;
    const int64_t pitch = mx4_pitch(d);
    for (int64_t r = row0 + static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); r < row0 + n; r += static_cast<int64_t>(gridDim.x) * 8) {
        const uint32_t* c = reinterpret_cast<const uint32_t*>(codes + r * pitch);
        float nrm = 0.f;
        for (int i = lane; i < nb * 4; i += 32) {
            const uint32_t w = c[i];
            float part = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 v = e2m1_values(w >> (8 * e) & 255u);
                part = fmaf(v.x, v.x, fmaf(v.y, v.y, part));
            }
            const float s = e8m0_value(scales[mx4_scale_word(r, i >> 4, ng) + ((i >> 2) & 3)]);
            nrm = fmaf(part * s, s, nrm);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) nrm += __shfl_xor_sync(0xFFFFFFFFu, nrm, o);
        if (lane == 0) norms[r] = nrm;
    }
}

inline unsigned warp_blocks(int64_t n) { return static_cast<unsigned>(std::min<int64_t>((n + 7) / 8, 148 * 64)); }

template <typename T>
bool rows_aligned(const void* p, int64_t ld) {   // 16-byte loads of eight elements
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * static_cast<int64_t>(sizeof(T)) % 16 == 0;
}

template <typename T, bool VEC>
cudaError_t rms_rows(const RmsNormArgs& a, cudaStream_t st) {
    const int64_t most = 148 * 64;
    auto go = [&](auto nt, auto j) {
        constexpr int NT = decltype(nt)::value, J = decltype(j)::value;
        constexpr int kRows = NT == 32 ? 4 : 1;
        const int64_t blocks = std::min<int64_t>((a.n + kRows - 1) / kRows, most);
        rms_norm_i8_kernel<T, VEC, NT, J><<<static_cast<unsigned>(blocks), NT == 32 ? 128 : NT, 0, st>>>(a);
        return cudaGetLastError();
    };
    using std::integral_constant;
    if (a.d <= 256) return go(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    if (a.d <= 512) return go(integral_constant<int, 32>{}, integral_constant<int, 2>{});
    if (a.d <= 1024) return go(integral_constant<int, 128>{}, integral_constant<int, 1>{});
    if (a.d <= 2048) return go(integral_constant<int, 128>{}, integral_constant<int, 2>{});
    if (a.d <= 4096) return go(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    if (a.d <= 8192) return go(integral_constant<int, 512>{}, integral_constant<int, 2>{});
    return go(integral_constant<int, 512>{}, integral_constant<int, 4>{});
}
template <typename T>
cudaError_t rms_type(const RmsNormArgs& a, cudaStream_t st) {
    const bool vec = rows_aligned<T>(a.x, a.ldx) && rows_aligned<T>(a.weight, 0) &&
                     (!a.residual || rows_aligned<T>(a.residual, a.ldr)) && (!a.sum || rows_aligned<T>(a.sum, a.lds)) &&
                     reinterpret_cast<uintptr_t>(a.q) % 8 == 0 && a.ldq % 8 == 0;
    return vec ? rms_rows<T, true>(a, st) : rms_rows<T, false>(a, st);
}

inline unsigned chunk_blocks(int64_t n, int d) {   // a thread per 8 elements
    const int64_t b = (n * ((d + 7) / 8) + 255) / 256;
    return static_cast<unsigned>(std::min<int64_t>(b, 148 * 256));
}
template <typename T>
cudaError_t i8_values(int64_t n, int d, const int8_t* q, int64_t ldq, const float* scales, const float* one, void* out,
                      int64_t ldo, cudaStream_t st) {
    const bool vec = rows_aligned<T>(out, ldo) && reinterpret_cast<uintptr_t>(q) % 8 == 0 && ldq % 8 == 0;
    if (vec) i8_dequantize_kernel<T, true><<<chunk_blocks(n, d), 256, 0, st>>>(n, d, q, ldq, scales, one, static_cast<T*>(out), ldo);
    else i8_dequantize_kernel<T, false><<<chunk_blocks(n, d), 256, 0, st>>>(n, d, q, ldq, scales, one, static_cast<T*>(out), ldo);
    return cudaGetLastError();
}
template <typename T>
cudaError_t mx4_round(int64_t n, int d, const void* x, int64_t ldx, int64_t row0, uint8_t* codes, uint8_t* scales,
                      float* norms, cudaStream_t st) {
    const int pairs = (mx4_groups(d) + 1) / 2;
    int split = 1;
    if (!norms)   // few long rows: a warp for every two groups
        while (split < pairs && n * split < 148 * 8) ++split;
    const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((n * split + 7) / 8, 148 * 64));
    const T* xt = static_cast<const T*>(x);
    if (rows_aligned<T>(x, ldx)) mx4_quantize_kernel<T, true><<<blocks, 256, 0, st>>>(n, d, xt, ldx, row0, codes, scales, norms, split);
    else mx4_quantize_kernel<T, false><<<blocks, 256, 0, st>>>(n, d, xt, ldx, row0, codes, scales, norms, split);
    return cudaGetLastError();
}
template <typename T>
cudaError_t mx4_values(int64_t row0, int64_t n, int d, const uint8_t* codes, const uint8_t* scales, void* out,
                       int64_t ldo, cudaStream_t st) {
    if (rows_aligned<T>(out, ldo)) mx4_dequantize_kernel<T, true><<<chunk_blocks(n, d), 256, 0, st>>>(row0, n, d, codes, scales, static_cast<T*>(out), ldo);
    else mx4_dequantize_kernel<T, false><<<chunk_blocks(n, d), 256, 0, st>>>(row0, n, d, codes, scales, static_cast<T*>(out), ldo);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_mx4_move_scales(int d, int64_t from, int64_t to, uint8_t* scales, cudaStream_t st) {
    mx4_move_scales_kernel<<<1, 64, 0, st>>>(mx4_groups(d), from, to, scales);
    return cudaGetLastError();
}

cudaError_t launch_mx4_pack_rows(int64_t n, int d, int64_t row0, uint8_t* codes, uint8_t* scales, uint8_t* plain, bool out,
                                 cudaStream_t st) {
    mx4_pack_rows_kernel<<<warp_blocks(n), 256, 0, st>>>(n, d, row0, codes, scales, plain, out ? 1 : 0);
    return cudaGetLastError();
}

cudaError_t launch_mx4_norms(int64_t n, int d, int64_t row0, const uint8_t* codes, const uint8_t* scales, float* norms,
                             cudaStream_t st) {
    mx4_norms_kernel<<<warp_blocks(n), 256, 0, st>>>(n, d, row0, codes, scales, norms);
    return cudaGetLastError();
}

cudaError_t launch_rms_norm_i8(int dtype, const RmsNormArgs& a, cudaStream_t st) {
    switch (dtype) {
        case kF32: return rms_type<float>(a, st);
        case kF16: return rms_type<__half>(a, st);
        case kBF16: return rms_type<__nv_bfloat16>(a, st);
        default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_i8_dequantize(int64_t n, int d, const int8_t* q, int64_t ldq, const float* scales,
                                 const float* static_scale, int dtype, void* out, int64_t ldo, cudaStream_t st) {
    switch (dtype) {
        case kF32: return i8_values<float>(n, d, q, ldq, scales, static_scale, out, ldo, st);
        case kF16: return i8_values<__half>(n, d, q, ldq, scales, static_scale, out, ldo, st);
        case kBF16: return i8_values<__nv_bfloat16>(n, d, q, ldq, scales, static_scale, out, ldo, st);
        default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_mx4_quantize(int dtype, int64_t n, int d, const void* x, int64_t ldx, int64_t row0, uint8_t* codes,
                                uint8_t* scales, float* norms, cudaStream_t st) {
    switch (dtype) {
        case kF32: return mx4_round<float>(n, d, x, ldx, row0, codes, scales, norms, st);
        case kF16: return mx4_round<__half>(n, d, x, ldx, row0, codes, scales, norms, st);
        case kBF16: return mx4_round<__nv_bfloat16>(n, d, x, ldx, row0, codes, scales, norms, st);
        default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_mx4_dequantize(int64_t row0, int64_t n, int d, const uint8_t* codes, const uint8_t* scales, int dtype,
                                  void* out, int64_t ldo, cudaStream_t st) {
    switch (dtype) {
        case kF32: return mx4_values<float>(row0, n, d, codes, scales, out, ldo, st);
        case kF16: return mx4_values<__half>(row0, n, d, codes, scales, out, ldo, st);
        case kBF16: return mx4_values<__nv_bfloat16>(row0, n, d, codes, scales, out, ldo, st);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace b200
