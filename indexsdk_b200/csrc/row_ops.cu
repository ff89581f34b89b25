#include "row_ops.cuh"
#include "ptx_sm100.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

namespace b200 {
namespace {

constexpr int64_t kSms = 148;   // shapes grids, nothing else

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

__device__ __forceinline__ float max_nan(float a, float b) {   // NaN where one of them is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Eight elements as they lie in memory: four or eight words.
template <typename T>
struct Row8 {
    uint32_t w[2 * sizeof(T)];
};
template <typename T>
__device__ __forceinline__ void unpack8(const Row8<T>& k, float (&f)[8]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(k.w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
                const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&k.w[i]));
                f[2 * i] = v.x;
                f[2 * i + 1] = v.y;
            } else {   // bf16 is the upper half of an fp32
                f[2 * i] = __uint_as_float(k.w[i] << 16);
                f[2 * i + 1] = __uint_as_float(k.w[i] & 0xFFFF0000u);
            }
        }
    }
}
template <typename T>
__device__ __forceinline__ void pack8(const float (&f)[8], Row8<T>& k) {   // to nearest, ties to even
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) k.w[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
                const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
                k.w[i] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
                k.w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
    }
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, Row8<T>& k) {   // 16-byte aligned
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
        const uint4 u = reinterpret_cast<const uint4*>(p)[i];
        k.w[4 * i] = u.x; k.w[4 * i + 1] = u.y; k.w[4 * i + 2] = u.z; k.w[4 * i + 3] = u.w;
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const Row8<T>& k) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
        reinterpret_cast<uint4*>(p)[i] = make_uint4(k.w[4 * i], k.w[4 * i + 1], k.w[4 * i + 2], k.w[4 * i + 3]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
    Row8<T> k;
    pack8<T>(f, k);
    store8<T>(p, k);
}

// ---------------------------------------------------------------------------------------
// RMS norm -> int8.  A row belongs to NT threads, up to 32 lanes of a warp (short rows: a reduction over few lanes,
// several rows a warp) or a block; they keep it in registers: one pass over memory, one reduction (sum of squares and
// the largest |s w| together -- the norm's factor is the same for the whole row, so it is not needed to find the
// largest element, and q = round(s w * 127 / max|s w|) does not contain it at all).  Thread t owns the
// chunks of 8 elements t, t + NT, ... (VEC) or the elements t, t + NT, ... (rows that are not 16-byte aligned;
// loads stay coalesced).  The next row's loads are on their way while this one is reduced and written.
//
// A rounding to whole numbers shows every error of its argument where that lies next to a border, and for 16-bit
// rows with weights of 16 bits one element in 20 000 lies exactly ON a border.  So squares are added up in
// 64 bits (with a scale per row over eight elements in fp32 first), fp32 rows keep their largest product unrounded, and an element whose fp32
// quotient is within 2^-14 of a border (that quotient is off by at most 127 * 6 * 2^-24) is compared with it in 64 bits.
// ---------------------------------------------------------------------------------------
template <int NT>
struct RowSums {   // two sets in turn: one is written again only behind the other's barrier
    double ssq[2][NT / 32 + 1], top[2][NT / 32 + 1];
};
// The sum of `sum` and the largest `top` of the row's threads.
template <int NT, typename F>
__device__ __forceinline__ void reduce_row(double& sum, F& top, RowSums<NT>& sh, int& turn) {
#pragma unroll
    for (int o = (NT < 32 ? NT : 32) / 2; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        const F other = __shfl_xor_sync(0xFFFFFFFFu, top, o);
        top = other > top ? other : top;
    }
    if (NT > 32) {
        turn ^= 1;
        if ((threadIdx.x & 31) == 0) {
            sh.ssq[turn][threadIdx.x >> 5] = sum;
            *reinterpret_cast<F*>(&sh.top[turn][threadIdx.x >> 5]) = top;
        }
        __syncthreads();
        sum = sh.ssq[turn][0];
        top = *reinterpret_cast<const F*>(&sh.top[turn][0]);
#pragma unroll
        for (int i = 1; i < NT / 32; ++i) {
            sum += sh.ssq[turn][i];
            const F other = *reinterpret_cast<const F*>(&sh.top[turn][i]);
            top = other > top ? other : top;
        }
    }
}

// What is rare, element by element from memory and in 64 bits.
template <typename T, bool RES>
__device__ __forceinline__ double row_element(const RmsNormArgs& a, int64_t row, int k) {
    if (!RES) return to_f<T>(static_cast<const T*>(a.x)[row * a.ldx + k]);
    if (a.sum) return to_f<T>(static_cast<const T*>(a.sum)[row * a.lds + k]);   // (this thread's own; it may have x's place)
    return to_f<T>(from_f<T>(to_f<T>(static_cast<const T*>(a.x)[row * a.ldx + k]) +
                             to_f<T>(static_cast<const T*>(a.residual)[row * a.ldr + k])));
}
// One element: its product times num / den.
template <typename T, bool RES>
__device__ __noinline__ void round_precisely(const RmsNormArgs& a, int64_t row, int k, double num, double den) {
    const double y = row_element<T, RES>(a, row, k) * to_f<T>(static_cast<const T*>(a.weight)[k]) * num / den;
    a.q[row * a.ldq + k] = static_cast<int8_t>(__double2int_rn(fmin(fmax(y, -127.), 127.)));
}
// A whole row: squares or products outside the range of fp32, or no numbers at all.  Every thread of the row.
template <typename T, bool VEC, bool RES, int NT, int J>
__device__ __noinline__ int hard_row(const RmsNormArgs& a, int64_t row, int t, bool mine, RowSums<NT>& sh, int turn) {
    double ssq = 0., top = 0.;
    for (int i = 0; i < 8 * J; ++i) {
        const int k = VEC ? (t + NT * (i >> 3)) * 8 + (i & 7) : t + NT * i;
        if (!mine || k >= a.d) continue;
        const double s = row_element<T, RES>(a, row, k);
        const double p = fabs(s * to_f<T>(static_cast<const T*>(a.weight)[k]));
        ssq += p < __longlong_as_double(0x7ff0000000000000ll) ? s * s : p;   // (a weight that is no number: nor is the row)
        top = fmax(top, p);
    }
    reduce_row<NT>(ssq, top, sh, turn);
    if (!mine) return turn;
    const double inf = __longlong_as_double(0x7ff0000000000000ll);
    bool live = ssq < inf && top < inf;   // false for NaN and infinities
    const double root = sqrt(ssq / a.d + static_cast<double>(a.eps));
    if (!a.static_scale && t == 0) a.scales[row] = live ? static_cast<float>(top / (127. * root)) : __int_as_float(0x7fc00000);
    double num = 127., den = top;
    if (a.static_scale) {
        const float given = __ldg(a.static_scale);
        live = live && given > 0.f && given <= 3.4e38f;
        num = 1.;
        den = root * given;
    }
    live = live && den > 0.;
    for (int i = 0; i < 8 * J; ++i) {
        const int k = VEC ? (t + NT * (i >> 3)) * 8 + (i & 7) : t + NT * i;
        if (k >= a.d) continue;
        if (live) round_precisely<T, RES>(a, row, k, num, den);
        else a.q[row * a.ldq + k] = 0;
    }
    return turn;
}

template <typename T, bool VEC, bool RES, int NT, int J, int FIT>
__global__ void __launch_bounds__(NT <= 32 ? 128 : NT, FIT) rms_norm_i8_kernel(const __grid_constant__ RmsNormArgs a) {
    __shared__ RowSums<NT> sh;
    int turn = 0;
    constexpr int kRows = NT <= 32 ? 128 / NT : 1;   // rows a block works on at a time
    constexpr bool kLow = sizeof(T) == 4;            // (products of 16-bit numbers are exact in fp32)
    constexpr bool kAhead = sizeof(T) == 2;          // (fp32: the registers of a second row cost more blocks than they hide)
    const int t = NT <= 32 ? threadIdx.x & (NT - 1) : threadIdx.x;
    // element e of chunk j of this thread
    auto at = [&](int j, int e) { return VEC ? (t + NT * j) * 8 + e : t + NT * (8 * j + e); };
    auto whole = [&](int j) { return VEC && at(j, 8) <= a.d; };
    auto fetch = [&](const void* base, int j, Row8<T>& k) {
        const T* p = static_cast<const T*>(base);
        if (whole(j)) {
            load8<T>(p + at(j, 0), k);
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 8; ++e) k.w[e] = at(j, e) < a.d ? reinterpret_cast<const uint32_t*>(p)[at(j, e)] : 0u;
        } else {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const uint32_t lo = at(j, e) < a.d ? h[at(j, e)] : 0u, hi = at(j, e + 1) < a.d ? h[at(j, e + 1)] : 0u;
                k.w[e / 2] = lo | hi << 16;
            }
        }
    };
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
    const int slot = NT <= 32 ? threadIdx.x / NT : 0;
    int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + slot;
    // (the lanes of a warp meet in the reductions: they leave together)
    const int64_t first = NT < 32 ? row - slot % (NT < 32 ? 32 / NT : 1) : row;
    Row8<T> x[J], r[RES ? J : 1];
    auto fetch_row = [&](int64_t i) {
        const T* xp = static_cast<const T*>(a.x) + i * a.ldx;
#pragma unroll
        for (int j = 0; j < J; ++j) fetch(xp, j, x[j]);
        if (RES) {
            const T* rp = static_cast<const T*>(a.residual) + i * a.ldr;
#pragma unroll
            for (int j = 0; j < J; ++j) fetch(rp, j, r[j]);
        }
    };
    if (kAhead && row < a.n) fetch_row(row);
    for (int64_t lead = first; lead < a.n; lead += step, row += step) {
        const bool real = row < a.n;
        if (!kAhead && real) fetch_row(row);
        double ssq = 0.;
        float top = 0.f, top_s = 0.f, top_w = 0.f;
        float v[J][8];   // s w
#pragma unroll
        for (int j = 0; j < J; ++j) {
            float f[8], w[8];
            unpack8<T>(x[j], f);
            if (RES) {
                // The sum is rounded to the rows' type BEFORE it is normalised: what is normalised is what the
                // model carries on, so the result is that of the two steps done one after the other.
                float g[8];
                unpack8<T>(r[j], g);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] += g[e];
                Row8<T> s;
                pack8<T>(f, s);
                unpack8<T>(s, f);
                // (written before the next row is fetched, which may have x's or the residual's place)
                if (a.sum && real) {
                    T* sum_row = static_cast<T*>(a.sum) + row * a.lds;
                    if (whole(j)) {
                        store8<T>(sum_row + at(j, 0), s);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            if (at(j, e) >= a.d) continue;
                            if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(sum_row)[at(j, e)] = s.w[e];
                            else reinterpret_cast<uint16_t*>(sum_row)[at(j, e)] = static_cast<uint16_t>(s.w[e / 2] >> (16 * (e & 1)));
                        }
                    }
                }
            }
            Row8<T> wt;
            fetch(a.weight, j, wt);
            unpack8<T>(wt, w);
            float part = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                part = fmaf(f[e], f[e], part);
                v[j][e] = f[e] * w[e];
                // (as whole numbers, which puts a NaN above all)
                if (kLow && (__float_as_uint(v[j][e]) & 0x7fffffffu) > __float_as_uint(top)) {
                    top = fabsf(v[j][e]);
                    top_s = f[e];
                    top_w = w[e];
                }
            }
            if (a.static_scale) {   // (nothing cancels an error of the sum there)
#pragma unroll
                for (int e = 0; e < 8; ++e) ssq = fma(static_cast<double>(f[e]), static_cast<double>(f[e]), ssq);
            } else {
                ssq += part;
            }
            if (!kLow) {
#pragma unroll
                for (int e = 0; e < 8; e += 2) top = max_nan(top, fabsf(v[j][e]), fabsf(v[j][e + 1]));
            }
        }
        if (top != top) ssq = __longlong_as_double(0x7ff8000000000000ll);   // (a weight; reductions of `top` do not pass a NaN on)
        // Products below fp32's least number come out as zeros: that number stands for them, so that a row that has nothing
        // larger is done in 64 bits.  (Rows of zeros, as in a padded batch, stay here.)
        if (!std::is_same<T, __half>::value && top == 0.f) {
            uint32_t any = 0;
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int i = 0; i < static_cast<int>(2 * sizeof(T)); ++i) any |= RES ? x[j].w[i] | r[RES ? j : 0].w[i] : x[j].w[i];
            if (any & (kLow ? 0x7fffffffu : 0x7fff7fffu)) {
                top = top_s = __int_as_float(1);
                top_w = 1.f;
            }
        }
        if (kAhead && row + step < a.n) fetch_row(row + step);
        const float mine = top;
        double most = 0.;   // the largest product
        if (kLow) {
            most = fabs(static_cast<double>(top_s) * top_w);
            reduce_row<NT>(ssq, most, sh, turn);
            top = static_cast<float>(most);
        } else {
            reduce_row<NT>(ssq, top, sh, turn);
            most = top;
        }
        // (a given scale this small divides products that are no fp32 numbers)
        const bool hard = !(ssq <= 3e38) || !(top <= 1e36f) || (top < 1e-20f && top > 0.f) || (a.static_scale && !(__ldg(a.static_scale) >= 1e-30f));
        if (NT < 32 ? __any_sync(0xFFFFFFFFu, hard) : hard) {
            turn = hard_row<T, VEC, RES, NT, J>(a, row, t, hard && real, sh, turn);
            if (hard) continue;
        }
        // (a warp's rows that were not hard go on)
        const float root = sqrtf(static_cast<float>(ssq) / a.d + a.eps);   // y = v / root
        float c = 0.f;   // q = round(v c); 0: zeros
        if (a.static_scale) {
            const float given = __ldg(a.static_scale);
            if (given <= 3.4e38f) c = 1.f / root / given;
            if (mine * c > 127.f) {   // (few values: a scale is made for its rows)
                const float cut = 127.f / c;
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[j][e] = fminf(fmaxf(v[j][e], -cut), cut);
            }
        } else {
            if (t == 0 && real) {
                // The values that users take back carry the scale's error, so it is rounded to fp32 once: 1 / root by one
                // step of Newton's method in 64 bits.  What is left is the fp32 sum of eight squares in `part`, at most 4 steps of
                // 2^-24 after the root (65 536 x 4096: one scale in 26 is not the nearest fp32 number, but the next).
                const double ms = ssq / a.d + static_cast<double>(a.eps), r0 = rsqrtf(static_cast<float>(ms));
                a.scales[row] = static_cast<float>(most * (r0 * (1.5 - 0.5 * ms * r0 * r0)) * (1. / 127.));
            }
            if (top > 0.f) c = 127.f / top;
        }
        if (!real) continue;
        int8_t* q = a.q + row * a.ldq;
        const uint32_t keep = c != 0.f ? 0xFFFFFFFFu : 0u;   // rows that are zeros
        uint32_t near = 0;   // chunks with an element next to a border
#pragma unroll
        for (int j = 0; j < J; ++j) {
            // v c + 1.5 * 2^23: the last bit of such a sum is one, so it is rounded to a whole number, whose two's
            // complement stands in the low bits (a multiply-add instead of a conversion)
            uint32_t b[8];
            float off = 0.f;   // largest distance to the whole number
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float r0 = fmaf(v[j][e], c, 12582912.f), r1 = fmaf(v[j][e + 1], c, 12582912.f);
                b[e] = __float_as_uint(r0);
                b[e + 1] = __float_as_uint(r1);
                off = ptx::max3(off, fabsf(fmaf(v[j][e], c, 12582912.f - r0)), fabsf(fmaf(v[j][e + 1], c, 12582912.f - r1)));
            }
            if (off > 0.5f - 1.f / 16384.f) near |= 1u << j;
            uint2 o;
            o.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410) & keep;
            o.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410) & keep;
            if (whole(j)) {
                *reinterpret_cast<uint2*>(q + at(j, 0)) = o;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (at(j, e) < a.d) q[at(j, e)] = static_cast<int8_t>((e < 4 ? o.x : o.y) >> (8 * (e & 3)));
            }
        }
        if (near & keep) {
            double num = 127., den = most;
            if (a.static_scale) {
                num = 1.;
                den = sqrt(ssq / a.d + static_cast<double>(a.eps)) * __ldg(a.static_scale);
            }
#pragma unroll
            for (int j = 0; j < J; ++j) {
                if (!(near >> j & 1u)) continue;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float p = fabsf(v[j][e] * c), k = floorf(p);
                    if (fabsf(p - k - 0.5f) > 1.f / 8192.f || at(j, e) >= a.d) continue;
                    // |product| num / den against k + 1/2, without a division
                    const double product = kLow ? row_element<T, RES>(a, row, at(j, e)) * to_f<T>(static_cast<const T*>(a.weight)[at(j, e)])
                                                : static_cast<double>(v[j][e]);
                    const double l = fabs(product) * num, h = (k + 0.5) * den;
                    const int up = l > h || (l == h && (static_cast<int>(k) & 1)) ? 1 : 0;
                    const int whole_number = static_cast<int>(k) + up;
                    q[at(j, e)] = static_cast<int8_t>(v[j][e] < 0.f ? -whole_number : whole_number);
                }
            }
        }
    }
}

// Quotients by a number known to the host, of 32-bit numbers: the estimate is right or one too small.
struct Divisor {
    uint32_t d, m;
    explicit Divisor(uint32_t v) : d(v), m(static_cast<uint32_t>((uint64_t(1) << 32) / v - (v == 1 ? 1 : 0))) {}
    __device__ __forceinline__ uint32_t quotient(uint32_t x) const {
        uint32_t q = __umulhi(x, m);
        if (x - q * d >= d) ++q;
        return q;
    }
};
constexpr int64_t kFlat = int64_t(1) << 31;   // elements (or groups) one launch covers

// ---- int8 rows -> values; a thread per 8 elements ----
// Rows without gaps (FLAT) are one long array of outputs: a thread writes 8 of them on a 16-byte boundary,
// whatever d is, and takes the scale of the next row where a row ends among them.
template <typename T, bool FLAT>
__global__ void __launch_bounds__(256) i8_dequantize_kernel(uint32_t total, Divisor by, const int8_t* q, int64_t ldq,
                                                            const float* scales, const float* static_scale, T* out,
                                                            int64_t ldo) {
    const uint32_t step = gridDim.x * 256 * (FLAT ? 8 : 1);
    uint32_t i = (blockIdx.x * 256 + threadIdx.x) * (FLAT ? 8 : 1);
    if constexpr (!FLAT) {
        for (; i < total; i += step) {
            const uint32_t row = by.quotient(i), k = i - row * by.d;
            const float s = __ldg(scales ? scales + row : static_scale);
            out[row * ldo + k] = from_f<T>(static_cast<float>(q[row * ldq + k]) * s);
        }
    } else {
        for (; i < total; i += 2 * step) {   // two pieces at a time: their loads are on the way together
            uint2 u[2];
            float s[2], s2[2];
            uint32_t first[2];   // elements that belong to the first row
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const uint32_t at = i + p * step;
                if (at + 8 > total) continue;
                const uint32_t row = by.quotient(at);
                first[p] = by.d - (at - row * by.d);
                u[p] = *reinterpret_cast<const uint2*>(q + at);
                s[p] = __ldg(scales ? scales + row : static_scale);
                s2[p] = first[p] < 8 && scales ? __ldg(scales + row + 1) : s[p];   // (d >= 8)
            }
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const uint32_t at = i + p * step;
                if (at + 8 <= total) {
                    float f[8];
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e)
                        f[e] = static_cast<float>(static_cast<int8_t>((e < 4 ? u[p].x : u[p].y) >> (8 * (e & 3)))) * (e < first[p] ? s[p] : s2[p]);
                    store8<T>(out + at, f);
                } else {
                    for (uint32_t e = at; e < total; ++e)
                        out[e] = from_f<T>(static_cast<float>(q[e]) * __ldg(scales ? scales + by.quotient(e) : static_scale));
                }
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

// 32 consecutive bytes of a row that starts off a 16-byte boundary: the aligned words around them, shifted.
// `shift` is the address modulo 16 (the same for a whole row); nothing before `p` rounded down and nothing from
// `end` on is read.
__device__ __forceinline__ bool load32_shifted(const char* p, uint32_t shift, const char* end, uint32_t (&k)[8]) {
    const uint4* base = reinterpret_cast<const uint4*>(p - shift);
    if (reinterpret_cast<const char*>(base + 3) > end) return false;
    uint32_t w[12];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const uint4 u = __ldg(base + i);
        w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
    }
    if (shift & 8) {
#pragma unroll
        for (int i = 0; i < 10; ++i) w[i] = w[i + 2];
    }
    if (shift & 4) {
#pragma unroll
        for (int i = 0; i < 9; ++i) w[i] = w[i + 1];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) k[i] = __funnelshift_r(w[i], w[i + 1], (shift & 3) * 8);
    return true;
}

// Rounding to MX4 works in pieces of 32 bytes of the input, P elements to a thread (8 fp32, 16 of 16 bits): 32 / P
// neighbouring threads make a block of 32, 128 / P a group of 128 elements, whose four scale bytes leave as one
// word and whose codes as 64 contiguous bytes.  With half as many elements a thread, the addresses and the
// reductions of the 16-bit types cost more than the rounding (65 536 x 4096 bf16: 153 us instead of 110).
template <typename T>
constexpr int kPiece = 32 / sizeof(T);

enum Mx4Load { kLoadAligned, kLoadShifted, kLoadSingle };   // rows on 16-byte boundaries; only the first one; not even that
template <typename T, int LOAD>
__device__ __forceinline__ void fetch_piece(const T* xr, int k, int d, const T* end, float (&f)[kPiece<T>]) {
    constexpr int P = kPiece<T>;
    uint32_t w[8];
    bool got = false;
    if (k + P <= d) {
        if (LOAD == kLoadAligned) {
            const uint4* p = reinterpret_cast<const uint4*>(xr + k);
            const uint4 u = __ldg(p), v = __ldg(p + 1);
            w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
            w[4] = v.x; w[5] = v.y; w[6] = v.z; w[7] = v.w;
            got = true;
        } else if (LOAD == kLoadShifted) {
            got = load32_shifted(reinterpret_cast<const char*>(xr + k), static_cast<uint32_t>(reinterpret_cast<uintptr_t>(xr)) & 15u,
                                 reinterpret_cast<const char*>(end), w);
        }
    }
    if (got) {
#pragma unroll
        for (int h = 0; h < P / 8; ++h) {
            Row8<T> r;
            float g[8];
#pragma unroll
            for (int i = 0; i < static_cast<int>(2 * sizeof(T)); ++i) r.w[i] = w[h * 2 * sizeof(T) + i];
            unpack8<T>(r, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[h * 8 + e] = g[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < P; ++e) f[e] = k + e < d ? to_f<T>(xr[k + e]) : 0.f;
    }
}

// The block's scale byte and the thread's codes.
template <int P>
__device__ __forceinline__ void round_piece(const float (&f)[P], uint32_t (&c)[P / 8], uint32_t& byte) {
    float top = fabsf(f[0]);
#pragma unroll
    for (int e = 1; e + 1 < P; e += 2) top = max_nan(top, fabsf(f[e]), fabsf(f[e + 1]));
    top = max_nan(top, fabsf(f[P - 1]));
#pragma unroll
    for (int o = 1; o < 32 / P; o <<= 1) top = max_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    // floor(log2(top)) is the exponent field; a subnormal or zero top ends at the smallest scale anyway.  NaN and
    // infinities have a field of 255.
    const int field = static_cast<int>(__float_as_uint(top) >> 23 & 255u);
    const bool fine = field < 255;
    byte = fine ? static_cast<uint32_t>(max(field - 2, 0)) : 255u;
    const float inv = __uint_as_float((254u - byte) << 23);   // 2^(127 - byte)
#pragma unroll
    for (int h = 0; h < P / 8; ++h) {
        uint32_t b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = e2m1_pair(f[8 * h + 2 * e] * inv, f[8 * h + 2 * e + 1] * inv);
        c[h] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
        if (!fine) c[h] = 0u;
    }
}
// The scales of a group's four blocks as a word, in every thread of the group.
template <int P>
__device__ __forceinline__ uint32_t scale_word(uint32_t byte, uint32_t t) {
    uint32_t word = byte << (8 * (t / (32 / P)));
#pragma unroll
    for (int o = 32 / P; o < 128 / P; o <<= 1) word |= __shfl_xor_sync(0xFFFFFFFFu, word, o);
    return word;
}
template <int P>
__device__ __forceinline__ void store_codes(uint8_t* p, const uint32_t (&c)[P / 8]) {
    if constexpr (P == 8) *reinterpret_cast<uint32_t*>(p) = c[0];
    else *reinterpret_cast<uint2*>(p) = make_uint2(c[0], c[1]);
}

// The groups of all rows in turn.
template <typename T, int LOAD>
__global__ void __launch_bounds__(256) mx4_quantize_kernel(uint32_t groups, Divisor by, int d, const T* x, int64_t ldx,
                                                           const T* end, int64_t row0, uint8_t* codes, uint8_t* scales) {
    constexpr int P = kPiece<T>, TG = 128 / P, PB = 256 / TG;   // threads of a group, groups of a thread block
    const uint32_t t = threadIdx.x % TG;
    const int nb = mx4_blocks(d);
    const int64_t pitch = mx4_pitch(d);
    const uint32_t step = gridDim.x * PB;
    // (a warp stays until the last of its groups is done: they meet in the shuffles)
    for (uint32_t u = blockIdx.x * PB + threadIdx.x / TG; u - threadIdx.x % 32 / TG < groups; u += step) {
        const bool real = u < groups;
        const uint32_t row = by.quotient(real ? u : 0u), g = (real ? u : 0u) - row * by.d;
        const int k = static_cast<int>(g * 128u + t * P);   // this thread's first element
        float f[P];
        fetch_piece<T, LOAD>(x + row * ldx, k, d, end, f);
        uint32_t byte, c[P / 8];
        round_piece<P>(f, c, byte);
        const bool here = k < nb * 32;   // the block exists
        const uint32_t word = scale_word<P>(here ? byte : 127u, t);
        if (!real) continue;
        if (here) store_codes<P>(codes + (row0 + row) * pitch + k / 2, c);
        if (t == 0) *reinterpret_cast<uint32_t*>(scales + mx4_scale_word(row0 + row, g, by.d)) = word;
    }
}

// The same with the squared norms of the rounded rows, for an index: a warp takes whole rows.
template <typename T, int LOAD>
__global__ void __launch_bounds__(256) mx4_quantize_norms_kernel(int64_t n, int d, const T* x, int64_t ldx, const T* end,
                                                                 int64_t row0, uint8_t* codes, uint8_t* scales, float* norms) {
    constexpr int P = kPiece<T>, TG = 128 / P;
    const int lane = threadIdx.x & 31, t = lane % TG;
    const int nb = mx4_blocks(d), ng = mx4_groups(d);
    const int64_t pitch = mx4_pitch(d);
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); row < n; row += static_cast<int64_t>(gridDim.x) * 8) {
        const T* xr = x + row * ldx;
        uint8_t* crow = codes + (row0 + row) * pitch;
        float nrm = 0.f;
        for (int g0 = 0; g0 < ng; g0 += 32 / TG) {
            const int g = g0 + lane / TG, k = g * 128 + t * P;
            float f[P];
            fetch_piece<T, LOAD>(xr, k, d, end, f);
            uint32_t byte, c[P / 8];
            round_piece<P>(f, c, byte);
            const bool here = k < nb * 32;
            if (here) {
                float part = 0.f;
#pragma unroll
                for (int e = 0; e < P / 2; ++e) {
                    const float2 v = e2m1_values(c[e / 4] >> (8 * (e & 3)) & 255u);
                    part = fmaf(v.x, v.x, fmaf(v.y, v.y, part));   // exact: at most 576, in quarters
                }
                const float s = e8m0_value(byte);
                nrm = fmaf(part * s, s, nrm);
                store_codes<P>(crow + k / 2, c);
            }
            const uint32_t word = scale_word<P>(here ? byte : 127u, t);
            if (t == 0 && g < ng) *reinterpret_cast<uint32_t*>(scales + mx4_scale_word(row0 + row, g, ng)) = word;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) nrm += __shfl_xor_sync(0xFFFFFFFFu, nrm, o);
        if (lane == 0) norms[row0 + row] = nrm;
    }
}

// MX4 -> values where a thread's 16 bytes of output lie in one block: d a multiple of O, rows on 16-byte boundaries.
// Neighbouring threads write neighbouring pieces (32 bytes a thread: 65 536 x 4096 to bf16 149 us instead of 135).
template <typename T>
__global__ void __launch_bounds__(256) mx4_dequantize_aligned_kernel(uint32_t pieces, Divisor by, int64_t row0, int ng, int64_t pitch,
                                                                     const uint8_t* codes, const uint8_t* scales, T* out, int64_t ldo) {
    constexpr int O = 16 / sizeof(T);
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < pieces; i += gridDim.x * 256) {
        const uint32_t row = by.quotient(i), c = i - row * by.d, b = c / (32 / O);   // by.d: pieces of a row; b: block
        const uint8_t* p = codes + (row0 + row) * pitch + c * (O / 2);
        const uint32_t w = O == 8 ? __ldg(reinterpret_cast<const uint32_t*>(p)) : __ldg(reinterpret_cast<const uint16_t*>(p));
        const float s = e8m0_value(__ldg(scales + mx4_scale_word(row0 + row, b >> 2, ng) + (b & 3u)));
        float f[8];
#pragma unroll
        for (int e = 0; e < O / 2; ++e) {
            const float2 v = e2m1_values(w >> (8 * e));
            f[2 * e] = v.x * s;
            f[2 * e + 1] = v.y * s;
        }
        T* o = out + row * ldo + c * O;
        if constexpr (O == 8) store8<T>(o, f);
        else *reinterpret_cast<float4*>(o) = make_float4(f[0], f[1], f[2], f[3]);
    }
}

// MX4 -> values.  FLAT as in i8_dequantize_kernel: 8 outputs on a 16-byte boundary need two words of codes, shifted,
// and up to two scales; where a row ends among them, also the next row's first word and scale.
__device__ __forceinline__ float mx4_value(const uint8_t* crow, const uint8_t* scales, int64_t row, uint32_t k, int ng) {
    const uint32_t b = k >> 5, code = crow[k >> 1] >> (4 * (k & 1u)) & 15u;
    return e2m1_values(code).x * e8m0_value(__ldg(scales + mx4_scale_word(row, b >> 2, ng) + (b & 3u)));
}
template <typename T, bool FLAT>
__global__ void __launch_bounds__(256) mx4_dequantize_kernel(uint32_t total, Divisor by, int64_t row0, const uint8_t* codes,
                                                             const uint8_t* scales, T* out, int64_t ldo) {
    const int d = static_cast<int>(by.d), nb = mx4_blocks(d), ng = mx4_groups(d);
    const int64_t pitch = mx4_pitch(d);
    const uint32_t step = gridDim.x * 256 * (FLAT ? 8 : 1);
    uint32_t i = (blockIdx.x * 256 + threadIdx.x) * (FLAT ? 8 : 1);
    if (!FLAT) {
        for (; i < total; i += step) {
            const uint32_t row = by.quotient(i), k = i - row * by.d;
            out[row * ldo + k] = from_f<T>(mx4_value(codes + (row0 + row) * pitch, scales, row0 + row, k, ng));
        }
        return;
    }
    const int64_t granule = static_cast<int64_t>(ng) * 512;
    for (; i < total; i += step) {
        const uint32_t r = by.quotient(i), k = i - r * by.d, rest = by.d - k;   // rest: elements up to the row's end
        const int64_t row = row0 + r;
        if (i + 8 > total) {   // the array's last elements
            for (uint32_t e = i; e < total; ++e) {
                const uint32_t re = by.quotient(e);
                out[e] = from_f<T>(mx4_value(codes + (row0 + re) * pitch, scales, row0 + re, e - re * by.d, ng));
            }
            continue;
        }
        const uint32_t* w = reinterpret_cast<const uint32_t*>(codes + row * pitch) + (k >> 3);
        const uint8_t* srow = scales + (row >> 7) * granule + (row & 31) * 16 + (row >> 5 & 3) * 4;
        const uint32_t last = static_cast<uint32_t>(nb - 1), b = k >> 5, b2 = min((k + 7) >> 5, last);
        const uint32_t w0 = __ldg(w), w1 = (k & 7u) && (k >> 3) < 4 * last + 3 ? __ldg(w + 1) : 0u;
        const float f0 = e8m0_value(__ldg(srow + (b >> 2) * 512 + (b & 3u)));
        const float f1 = e8m0_value(__ldg(srow + (b2 >> 2) * 512 + (b2 & 3u)));
        uint32_t c = __funnelshift_r(w0, w1, 4 * (k & 7u));
        const uint32_t first = 32u - (k & 31u);   // elements of the first block
        float f[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; e += 2) {
            const float2 v = e2m1_values(c >> (4 * e));
            f[e] = v.x * (e < first ? f0 : f1);
            f[e + 1] = v.y * (e + 1 < first ? f0 : f1);
        }
        if (rest < 8) {   // the row ends here (d >= 8): the others come from the next row's first block
            c = __ldg(reinterpret_cast<const uint32_t*>(codes + (row + 1) * pitch)) << (4 * rest);
            const float f2 = e8m0_value(__ldg(scales + mx4_scale_word(row + 1, 0, ng)));
#pragma unroll
            for (uint32_t e = 0; e < 8; e += 2) {
                const float2 v = e2m1_values(c >> (4 * e));
                if (e >= rest) f[e] = v.x * f2;
                if (e + 1 >= rest) f[e + 1] = v.y * f2;
            }
        }
        store8<T>(out + i, f);
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

template <typename T, bool VEC, bool RES, int NT, int J, int FIT = 1>
cudaError_t rms_launch(const RmsNormArgs& a, cudaStream_t st) {
    const int threads = NT <= 32 ? 128 : NT, rows = NT <= 32 ? 128 / NT : 1;
    auto kern = rms_norm_i8_kernel<T, VEC, RES, NT, J, FIT>;
    // as many blocks as fit at a time: a row is on its way while its predecessor is worked on
    int fit = 0;
    cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kern, threads, 0);
    if (e != cudaSuccess) return e;
    const int64_t blocks = std::min<int64_t>((a.n + rows - 1) / rows, kSms * std::max(fit, 1));
    kern<<<static_cast<unsigned>(blocks), threads, 0, st>>>(a);
    return cudaGetLastError();
}
template <typename T, bool VEC, bool RES>
cudaError_t rms_rows(const RmsNormArgs& a, cudaStream_t st) {
    // Threads a row, chunks of 8 elements a thread, blocks an SM (which hold the registers down; forms that then spill were
    // the faster ones all the same).  What carries the memory's rate is bytes on the way: 32 of x and 32 of the residual for
    // each of 700 to 1000 threads of an SM, 64 of x alone.  A line ends where its threads hold no longer row; us of 2^27
    // elements with this line / with the next one (threads x chunks / blocks where that is no neighbour), a scale per row:
    //   16 bits, residual      d 128: 177 / 379; 256: 177 / 364; 512: 166 / 250; 768: 166 / 232; 1024: 158 / 361 (32 x 4 / 5: 181);
    //                          2048: 160 / 373 (64 x 4 / 12: 191); 4096: 164 / 406 (128 x 4 / 6: 187); 8192: 179 / 392
    //   16 bits, x alone       128: 128 (four blocks 130) / 285; 256: 132 / 259 (8 x 4 / 5: 138); 512: 117 / 177; 768: 115 / 148;
    //                          1024: 105 (64 x 2 / 12: 117) / 234; 2048: 105 (128 x 2 / 6: 119) / 236;
    //                          4096: 103 (256 x 2 / 3: 123) / 336; 8192: 170 / 291
    //   rows off the 16-byte boundaries, one element a load, 16 bits:
    //     residual             128: 411 (five blocks 440) / 592; 256: 332 / 534; 512: 281 (32 x 2 / 5: 414) / 519; 1001: 285
    //                          (64 x 2 / 12: 338) / 568; 2048: 304 (128 x 2 / 6: 371) / 625; 4096: 353 (256 x 2 / 3: 404) / 637
    //     x alone              128: 264 (five blocks 297) / 490; 256: 261 / 396; 512: 205 (32 x 2 / 5: 238) / 343; 600: 295
    //                          (32 x 3 / 4: 473, 128 x 1 / 8: 324); 1001: 195 (128 x 1 / 8: 205) / 355; 2048: 201 (256 x 1 / 4:
    //                          218) / 414; 4096: 222 (512 x 1 / 2: 263) / 435
    //   fp32, residual         128: 342 / 652; 256: 302 / 537; 512: 312 / 451; 1024: 288 / 461; 2048: 283 / 485; 4096: 297 / 603;
    //                          8192: 353 / 600
    //   fp32, x alone          128: 226 / 523; 256: 226 / 334; 512: 166 / 328; 1024: 162 / 332; 2048: 168 / 349; 4096: 181 / 474;
    //                          8192: 259 / 383
    // One given scale (64-bit sums of squares) costs 16-bit rows 5 to 30 % more (4096, x alone: 103 -> 134), fp32 rows 2 to 7 with
    // a residual and 8 to 22 without.
    if constexpr (sizeof(T) == 2 && !VEC) {
        if (a.d > 256 && a.d <= 512) return rms_launch<T, VEC, RES, 64, 1, 16>(a, st);
    }
    if constexpr (sizeof(T) == 2 && !VEC && RES) {
        if (a.d > 512 && a.d <= 1024) return rms_launch<T, VEC, RES, 128, 1, 8>(a, st);
        if (a.d > 1024 && a.d <= 2048) return rms_launch<T, VEC, RES, 256, 1, 4>(a, st);
        if (a.d > 2048 && a.d <= 4096) return rms_launch<T, VEC, RES, 512, 1, 2>(a, st);
    }
    if constexpr (sizeof(T) == 2 && VEC && !RES) {
        if (a.d > 768 && a.d <= 1024) return rms_launch<T, VEC, RES, 32, 4, 5>(a, st);
        if (a.d > 1024 && a.d <= 2048) return rms_launch<T, VEC, RES, 64, 4, 12>(a, st);
        if (a.d > 2048 && a.d <= 4096) return rms_launch<T, VEC, RES, 128, 4, 6>(a, st);
    }
    if constexpr (sizeof(T) == 2 && VEC) {
        if (a.d > 256 && a.d <= 512) return rms_launch<T, VEC, RES, 32, 2, 5>(a, st);
        if (a.d > 512 && a.d <= 768) return rms_launch<T, VEC, RES, 32, 3, 4>(a, st);
    }
    if constexpr (sizeof(T) == 2) {
        if (a.d <= 128) return rms_launch<T, VEC, RES, 8, 2, VEC && !RES ? 5 : 4>(a, st);
        if (a.d <= 256) return rms_launch<T, VEC, RES, 16, 2, 4>(a, st);
        // (what a line above takes for these is not built a second time)
        if constexpr (VEC == RES) {
            if (a.d <= 1024) return rms_launch<T, VEC, RES, 64, 2, 12>(a, st);
            if (a.d <= 2048) return rms_launch<T, VEC, RES, 128, 2, 6>(a, st);
            if (a.d <= 4096) return rms_launch<T, VEC, RES, 256, 2, 3>(a, st);
        }
        if (a.d <= 8192) return rms_launch<T, VEC, RES, 512, 2, 2>(a, st);
        return rms_launch<T, VEC, RES, 512, 4>(a, st);
    } else {
        if (a.d <= 128) return rms_launch<T, VEC, RES, 16, 1, 8>(a, st);
        if (a.d <= 256) return rms_launch<T, VEC, RES, 32, 1, 8>(a, st);
        if (a.d <= 512) return rms_launch<T, VEC, RES, 32, 2, 6>(a, st);
        if (a.d <= 1024) return rms_launch<T, VEC, RES, 64, 2, 12>(a, st);
        if (a.d <= 2048) return rms_launch<T, VEC, RES, 128, 2, 6>(a, st);
        if (a.d <= 4096) return rms_launch<T, VEC, RES, 256, 2, 3>(a, st);
        if (a.d <= 8192) return rms_launch<T, VEC, RES, 512, 2, 1>(a, st);
        return rms_launch<T, VEC, RES, 512, 4>(a, st);
    }
}
template <typename T>
cudaError_t rms_type(const RmsNormArgs& a, cudaStream_t st) {
    const bool vec = rows_aligned<T>(a.x, a.ldx) && rows_aligned<T>(a.weight, 0) &&
                     (!a.residual || rows_aligned<T>(a.residual, a.ldr)) && (!a.sum || rows_aligned<T>(a.sum, a.lds)) &&
                     reinterpret_cast<uintptr_t>(a.q) % 8 == 0 && a.ldq % 8 == 0;
    if (a.residual) return vec ? rms_rows<T, true, true>(a, st) : rms_rows<T, false, true>(a, st);
    return vec ? rms_rows<T, true, false>(a, st) : rms_rows<T, false, false>(a, st);
}

// A launch per stretch of rows whose elements 32 bits count; a stretch is a multiple of 8 rows, which keeps
// the 16-byte boundaries of rows without gaps.
template <typename F>
cudaError_t by_stretches(int64_t n, int64_t per_row, F&& go) {
    const int64_t most = kFlat / per_row / 8 * 8;
    for (int64_t r = 0; r < n; r += most) {
        const cudaError_t e = go(r, std::min(most, n - r));
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}
inline unsigned flat_blocks(int64_t threads) { return static_cast<unsigned>(std::min<int64_t>((threads + 255) / 256, kSms * 64)); }

template <typename T>
cudaError_t i8_values(int64_t n, int d, const int8_t* q, int64_t ldq, const float* scales, const float* one, void* out,
                      int64_t ldo, cudaStream_t st) {
    const bool flat = ldo == d && ldq == d && d >= 8 && rows_aligned<T>(out, 0) && reinterpret_cast<uintptr_t>(q) % 8 == 0;
    return by_stretches(n, d, [&](int64_t r, int64_t m) {
        const int8_t* qr = q + r * ldq;
        const float* sr = scales ? scales + r : nullptr;
        T* o = static_cast<T*>(out) + r * ldo;
        const uint32_t total = static_cast<uint32_t>(m * d);
        if (flat) i8_dequantize_kernel<T, true><<<flat_blocks((total + 7) / 8), 256, 0, st>>>(total, Divisor(d), qr, ldq, sr, one, o, ldo);
        else i8_dequantize_kernel<T, false><<<flat_blocks(total), 256, 0, st>>>(total, Divisor(d), qr, ldq, sr, one, o, ldo);
        return cudaGetLastError();
    });
}
template <typename T, int LOAD>
cudaError_t mx4_round_rows(int64_t n, int d, const T* x, int64_t ldx, int64_t row0, uint8_t* codes, uint8_t* scales,
                           float* norms, cudaStream_t st) {
    const T* end = x + (n - 1) * ldx + d;
    if (norms) {   // (rows and queries of an index, which are fp32)
        if constexpr (std::is_same<T, float>::value) {
            mx4_quantize_norms_kernel<T, LOAD><<<warp_blocks(n), 256, 0, st>>>(n, d, x, ldx, end, row0, codes, scales, norms);
            return cudaGetLastError();
        }
        return cudaErrorInvalidValue;
    }
    const int ng = mx4_groups(d);
    return by_stretches(n, ng, [&](int64_t r, int64_t m) {
        const uint32_t groups = static_cast<uint32_t>(m * ng);
        mx4_quantize_kernel<T, LOAD><<<flat_blocks(int64_t(groups) * (128 / kPiece<T>)), 256, 0, st>>>(groups, Divisor(ng), d, x + r * ldx, ldx, end, row0 + r, codes, scales);
        return cudaGetLastError();
    });
}
template <typename T>
cudaError_t mx4_round(int64_t n, int d, const void* x, int64_t ldx, int64_t row0, uint8_t* codes, uint8_t* scales,
                      float* norms, cudaStream_t st) {
    const T* xt = static_cast<const T*>(x);
    if (rows_aligned<T>(x, ldx)) return mx4_round_rows<T, kLoadAligned>(n, d, xt, ldx, row0, codes, scales, norms, st);
    if (rows_aligned<T>(x, 0)) return mx4_round_rows<T, kLoadShifted>(n, d, xt, ldx, row0, codes, scales, norms, st);
    return mx4_round_rows<T, kLoadSingle>(n, d, xt, ldx, row0, codes, scales, norms, st);
}
template <typename T>
cudaError_t mx4_values(int64_t row0, int64_t n, int d, const uint8_t* codes, const uint8_t* scales, void* out,
                       int64_t ldo, cudaStream_t st) {
    constexpr int O = 16 / sizeof(T);
    if (d % O == 0 && rows_aligned<T>(out, ldo))
        return by_stretches(n, d, [&](int64_t r, int64_t m) {
            const uint32_t pieces = static_cast<uint32_t>(m * (d / O));
            mx4_dequantize_aligned_kernel<T><<<flat_blocks(pieces), 256, 0, st>>>(pieces, Divisor(d / O), row0 + r, mx4_groups(d), mx4_pitch(d), codes, scales, static_cast<T*>(out) + r * ldo, ldo);
            return cudaGetLastError();
        });
    const bool flat = ldo == d && d >= 8 && rows_aligned<T>(out, 0);
    return by_stretches(n, d, [&](int64_t r, int64_t m) {
        T* o = static_cast<T*>(out) + r * ldo;
        const uint32_t total = static_cast<uint32_t>(m * d);
        if (flat) mx4_dequantize_kernel<T, true><<<flat_blocks((total + 7) / 8), 256, 0, st>>>(total, Divisor(d), row0 + r, codes, scales, o, ldo);
        else mx4_dequantize_kernel<T, false><<<flat_blocks(total), 256, 0, st>>>(total, Divisor(d), row0 + r, codes, scales, o, ldo);
        return cudaGetLastError();
    });
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
