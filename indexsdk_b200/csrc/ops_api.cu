// extern "C" surface of the operators on rows in few bits (include/b200idx.h): argument checks, the device
// the pointers live on, launches.  The calls without an index allocate nothing and wait for nothing, so they can be captured
// into graphs; those on an index (states in and against one, all scores) use its scratch memory and its stream, and return
// when they are done.
#include "../../include/b200idx.h"

#include <initializer_list>
#include <stdexcept>
#include <string>

#include "c_api_internal.h"
#include "device_mem.h"
#include "mx4_gemm.cuh"
#include "row_ops.cuh"

using namespace b200;

namespace {

constexpr int64_t kMaxRows = 1000000000;   // n < 1e9, as everywhere in this library

void check_rows(int64_t n, const char* what) {
    if (n <= 0 || n >= kMaxRows) throw std::invalid_argument(std::string(what) + " must be > 0 and < 1e9");
}
void check_dim(int d) {
    if (d <= 0 || d > kMaxRowElems) throw std::invalid_argument("Unsupported dims: d must be in (0, 16384]");
}
size_t elem_bytes(int dtype) {
    if (dtype == B200IDX_F32) return 4;
    if (dtype == B200IDX_F16 || dtype == B200IDX_BF16) return 2;
    throw std::invalid_argument("Unsupported dtype");
}
int64_t stride(int64_t ld, int d, const char* what) {
    if (ld == 0) return d;
    if (ld < d) throw std::invalid_argument(std::string(what) + " must be 0 or >= d");
    return ld;
}

void check_eps(float eps) {
    if (!(eps >= 1e-12f && eps <= 1.f)) throw std::invalid_argument("eps must be in [1e-12, 1]");
}

struct Operand {
    const char* name;
    const void* p;
    size_t align;
};
constexpr int kAnyDevice = -1;   // of managed memory, which every device reaches
// Presence and alignment first (no device needed), then the device that holds all of them, or kAnyDevice.
int device_of(std::initializer_list<Operand> ops) {
    for (const Operand& o : ops) {
        if (!o.p) throw std::invalid_argument(std::string("Invalid ") + o.name + ": nullptr.");
        if (reinterpret_cast<uintptr_t>(o.p) % o.align != 0)
            throw std::invalid_argument(std::string(o.name) + " must be aligned to " + std::to_string(o.align) + " bytes");
    }
    int device = kAnyDevice;
    for (const Operand& o : ops) {
        cudaPointerAttributes at;
        const cudaError_t e = cudaPointerGetAttributes(&at, o.p);
        if (e == cudaErrorNoDevice || e == cudaErrorInsufficientDriver) {
            cudaGetLastError();
            throw std::runtime_error("no CUDA device is available; this library has no CPU path");
        }
        if (e != cudaSuccess || (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)) {
            cudaGetLastError();
            throw std::invalid_argument(std::string(o.name) + " must be a device pointer");
        }
        if (at.type == cudaMemoryTypeManaged) continue;
        if (device != kAnyDevice && at.device != device) throw std::invalid_argument("the pointers lie on different devices");
        device = at.device;
    }
    return device;
}
// Where a call without an index runs: the operands' device, the current one where none is named.
int device_for(std::initializer_list<Operand> ops) {
    int device = device_of(ops);
    if (device == kAnyDevice) B200_CUDA_CHECK(cudaGetDevice(&device));
    return device;
}
// A call on an index runs on the index's device.
void check_on(const FlatIndex* ix, std::initializer_list<Operand> ops, const char* what) {
    const int device = device_of(ops);
    if (device != kAnyDevice && device != ix->device()) throw std::invalid_argument(std::string(what) + " must lie on the index's device");
}

FlatIndex* states_index(b200idx_t* h) {
    FlatIndex* ix = b200_capi::flat_of(h);
    if (!ix || ix->dtype() != kI8) throw std::invalid_argument("states are accepted by Int8Flat indexes only");
    return ix;
}
RmsNormArgs states_args(const FlatIndex* ix, int64_t n, int dtype, const void* x, const void* residual,
                        const void* weight, float eps, const float* static_scale) {
    check_rows(n, "n");
    const size_t eb = elem_bytes(dtype);
    check_eps(eps);
    if (!static_scale && ix->metric() != kMetricCos)
        throw std::invalid_argument("inner products and L2 distances need a static_scale: rows with scales of their own do not compare");
    const Operand xo{"x", x, eb};
    check_on(ix, {xo, {"weight", weight, eb}, residual ? Operand{"residual", residual, eb} : xo,
                  static_scale ? Operand{"static_scale", static_scale, 4} : xo}, "the states");
    RmsNormArgs a{};
    a.x = x;
    a.ldx = a.ldr = ix->d();
    a.residual = residual;
    a.weight = weight;
    a.eps = eps;
    a.static_scale = static_scale;
    return a;
}

int sm_count(int device) {
    int sms = 0;
    B200_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    return sms;
}

}  // namespace

extern "C" {

int b200idx_rms_norm_i8_device(int64_t n, int d, int dtype, const void* x, int64_t ldx, const void* residual,
                               int64_t ldr, void* sum, int64_t lds, const void* weight, float eps,
                               const float* static_scale, int8_t* q, int64_t ldq, float* scales, void* stream) {
    return b200_capi::guarded_call([&] {
        check_rows(n, "n");
        check_dim(d);
        const size_t eb = elem_bytes(dtype);
        check_eps(eps);
        if (sum && !residual) throw std::invalid_argument("a sum needs a residual");
        if (!static_scale == !scales) throw std::invalid_argument("give exactly one of static_scale and scales");
        RmsNormArgs a{n, d, x, stride(ldx, d, "ldx"), residual, stride(ldr, d, "ldr"), sum, stride(lds, d, "lds"),
                      weight, eps, static_scale, q, stride(ldq, d, "ldq"), scales};
        if (sum && ((sum == x && a.lds != a.ldx) || (sum == residual && a.lds != a.ldr)))
            throw std::invalid_argument("sum in place of x or residual needs the same stride");
        const float* sc = static_scale ? static_scale : scales;
        const Operand no{"q", q, 1};   // (repeats a required one where the optional ones are absent)
        DeviceGuard g(device_for({{"x", x, eb}, {"weight", weight, eb}, no, {"scales", sc, 4},
                                 residual ? Operand{"residual", residual, eb} : no, sum ? Operand{"sum", sum, eb} : no}));
        B200_CUDA_CHECK(launch_rms_norm_i8(dtype, a, static_cast<cudaStream_t>(stream)));
    });
}

int b200idx_add_states_device(b200idx_t* h, int64_t n, int dtype, const void* x, const void* residual, const void* weight,
                              float eps, const float* static_scale, const int64_t* ids_host) {
    if (!h) return B200IDX_ERR_INVALID_PARAM;
    return b200_capi::guarded(h, [&] {
        FlatIndex* ix = states_index(h);
        const RmsNormArgs a = states_args(ix, n, dtype, x, residual, weight, eps, static_scale);
        ix->add_states(n, dtype, a, ids_host);
    });
}

int b200idx_search_states_device(b200idx_t* h, int64_t n, int dtype, const void* x, const void* residual,
                                 const void* weight, float eps, const float* static_scale, int k, float* distances,
                                 int64_t* labels) {
    if (!h) return B200IDX_ERR_INVALID_PARAM;
    return b200_capi::guarded(h, [&] {
        FlatIndex* ix = states_index(h);
        const RmsNormArgs a = states_args(ix, n, dtype, x, residual, weight, eps, static_scale);
        if (k <= 0 || k > 4096) throw std::invalid_argument("k must be > 0 and <= 4096");
        check_on(ix, {{"distances", distances, 4}, {"labels", labels, 8}}, "distances and labels");
        ix->search_states(n, dtype, a, k, distances, labels);
    });
}

int b200idx_i8_dequantize_device(int64_t n, int d, const int8_t* q, int64_t ldq, const float* scales,
                                 const float* static_scale, int dtype, void* out, int64_t ldo, void* stream) {
    return b200_capi::guarded_call([&] {
        check_rows(n, "n");
        check_dim(d);
        const size_t eb = elem_bytes(dtype);
        if (!static_scale == !scales) throw std::invalid_argument("give exactly one of static_scale and scales");
        const int64_t lq = stride(ldq, d, "ldq"), lo = stride(ldo, d, "ldo");
        DeviceGuard g(device_for({{"q", q, 1}, {"scales", scales ? scales : static_scale, 4}, {"out", out, eb}}));
        B200_CUDA_CHECK(launch_i8_dequantize(n, d, q, lq, scales, static_scale, dtype, out, lo, static_cast<cudaStream_t>(stream)));
    });
}

int b200idx_scores_device(b200idx_t* h, int64_t n, const float* x, int dtype, void* out, int64_t ldo) {
    if (!h) return B200IDX_ERR_INVALID_PARAM;
    return b200_capi::guarded(h, [&] {
        FlatIndex* ix = b200_capi::flat_of(h);
        if (!ix || ix->dtype() != kMX4) throw std::invalid_argument("scores apply to MX4 indexes");
        check_rows(n, "n");
        const size_t eb = elem_bytes(dtype);
        if (ldo != 0 && ldo < ix->ntotal()) throw std::invalid_argument("ldo must be 0 or >= ntotal");
        check_on(ix, {{"x", x, 4}, {"out", out, eb}}, "x and out");
        ix->scores_device(n, x, dtype, out, ldo ? ldo : ix->ntotal());
    });
}

int64_t b200idx_mx4_row_bytes(int d) { return d <= 0 || d > kMaxRowElems ? -1 : mx4_pitch(d); }
int64_t b200idx_mx4_scale_bytes(int64_t n, int d) {
    return n <= 0 || n >= kMaxRows || d <= 0 || d > kMaxRowElems ? -1 : mx4_scale_bytes(n, d);
}

int b200idx_mx4_quantize_device(int64_t n, int d, int dtype, const void* x, int64_t ldx, uint8_t* codes, uint8_t* scales,
                                void* stream) {
    return b200_capi::guarded_call([&] {
        check_rows(n, "n");
        check_dim(d);
        const size_t eb = elem_bytes(dtype);
        const int64_t lx = stride(ldx, d, "ldx");
        DeviceGuard g(device_for({{"x", x, eb}, {"codes", codes, 16}, {"scales", scales, 16}}));
        B200_CUDA_CHECK(launch_mx4_quantize(dtype, n, d, x, lx, 0, codes, scales, nullptr, static_cast<cudaStream_t>(stream)));
    });
}

int b200idx_mx4_dequantize_device(int64_t n, int d, const uint8_t* codes, const uint8_t* scales, int dtype, void* out,
                                  int64_t ldo, void* stream) {
    return b200_capi::guarded_call([&] {
        check_rows(n, "n");
        check_dim(d);
        const size_t eb = elem_bytes(dtype);
        const int64_t lo = stride(ldo, d, "ldo");
        DeviceGuard g(device_for({{"codes", codes, 16}, {"scales", scales, 16}, {"out", out, eb}}));
        B200_CUDA_CHECK(launch_mx4_dequantize(0, n, d, codes, scales, dtype, out, lo, static_cast<cudaStream_t>(stream)));
    });
}

int b200idx_mx4_product_device(int64_t m, int64_t n, int d, const uint8_t* a_codes, const uint8_t* a_scales,
                               const uint8_t* b_codes, const uint8_t* b_scales, int dtype, void* out, int64_t ldo,
                               void* stream) {
    return b200_capi::guarded_call([&] {
        check_rows(m, "m");
        check_rows(n, "n");
        check_dim(d);
        const size_t eb = elem_bytes(dtype);
        if (ldo != 0 && ldo < n) throw std::invalid_argument("ldo must be 0 or >= n");
        const int device = device_for({{"a_codes", a_codes, 16}, {"a_scales", a_scales, 16}, {"b_codes", b_codes, 16},
                                       {"b_scales", b_scales, 16}, {"out", out, eb}});
        DeviceGuard g(device);
        launch_mx4_product(dtype, Mx4ProductArgs{m, n, d, a_codes, a_scales, b_codes, b_scales, out, ldo ? ldo : n},
                           sm_count(device), static_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"
