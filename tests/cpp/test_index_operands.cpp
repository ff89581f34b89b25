// Which device a call's operands have to lie on (entry points of the operators on rows in few bits), on a device of the
// test's own.
#include "fake_device.h"

#include "../../indexsdk_b200/csrc/c_api_internal.h"

static std::string last;
static b200::FlatIndex* index_of_handle = nullptr;
namespace b200_capi {
int guarded_call(const std::function<void()>& f) {
    last = thrown(f);
    return last.empty() ? B200IDX_OK : B200IDX_ERR_INVALID_PARAM;
}
int guarded(const b200idx_t*, const std::function<void()>& f) { return guarded_call(f); }
b200::FlatIndex* flat_of(b200idx_t*) { return index_of_handle; }
}  // namespace b200_capi

static void refused(int rc, const char* text, const char* what) {
    check(rc != B200IDX_OK && last.find(text) != std::string::npos, std::string(what) + ": " + last);
}
static void taken(int rc, const char* what) { check(rc == B200IDX_OK, std::string(what) + ": " + last); }

int main() {
    alignas(16) static char here[8][64], there[8][64], managed[8][64], host[64];
    for (auto& p : there) place(p, cudaMemoryTypeDevice, 1);
    for (auto& p : managed) place(p, cudaMemoryTypeManaged, 0);
    place(host, cudaMemoryTypeHost, 0);
    b200idx_t* h = reinterpret_cast<b200idx_t*>(here);
    auto f = [](void* p) { return static_cast<float*>(p); };
    auto l = [](void* p) { return static_cast<int64_t*>(p); };

    for (int device : {0, 1}) {
        char(*own)[64] = device ? there : here;
        char(*other)[64] = device ? here : there;
        b200::FlatIndex i8(64, b200::kMetricIP, b200::kI8, device);
        index_of_handle = &i8;
        auto search = [&](char* x, char* w, char* s, char* D, char* I) {
            return b200idx_search_states_device(h, 1, B200IDX_F32, x, nullptr, w, 1e-6f, f(s), 1, f(D), l(I));
        };
        taken(search(own[0], own[1], own[2], own[3], own[4]), "all on the index's device");
        refused(search(own[0], own[1], own[2], other[3], other[4]), "index's device", "both results elsewhere");
        refused(search(own[0], own[1], own[2], own[3], other[4]), "different devices", "labels elsewhere");
        refused(search(other[0], other[1], other[2], own[3], own[4]), "index's device", "states elsewhere");
        refused(search(own[0], other[1], own[2], own[3], own[4]), "different devices", "weight elsewhere");
        refused(search(own[0], own[1], own[2], host, own[4]), "device pointer", "results on the host");
        // managed memory is reached from every device, whichever is the current one
        for (int current : {0, 1}) {
            current_device = current;
            taken(search(managed[0], managed[1], managed[2], managed[3], managed[4]), "managed memory");
            taken(search(managed[0], own[1], managed[2], managed[3], own[4]), "managed and the index's memory");
            refused(search(managed[0], managed[1], managed[2], managed[3], other[4]), "index's device", "managed and other memory");
            taken(b200idx_add_states_device(h, 1, B200IDX_F32, managed[0], managed[5], managed[1], 1e-6f, f(managed[2]), nullptr), "add, managed memory");
            refused(b200idx_add_states_device(h, 1, B200IDX_F32, managed[0], other[5], managed[1], 1e-6f, f(managed[2]), nullptr), "index's device", "add, residual elsewhere");
            check(current_device == current, "the current device stays");
        }
        b200::FlatIndex mx(64, b200::kMetricIP, b200::kMX4, device);
        mx.add(2, own[0], false, nullptr, true);
        index_of_handle = &mx;
        taken(b200idx_scores_device(h, 1, f(own[0]), B200IDX_F32, own[1], 0), "scores");
        taken(b200idx_scores_device(h, 1, f(managed[0]), B200IDX_F32, managed[1], 0), "scores, managed memory");
        refused(b200idx_scores_device(h, 1, f(managed[0]), B200IDX_F32, other[1], 0), "index's device", "scores elsewhere");
    }
    // calls without an index run where their operands are
    for (int current : {0, 1}) {
        current_device = current;
        int seen = -1;
        b200::on_product = [&](const b200::Mx4ProductArgs&) { seen = current_device; };
        auto product = [&](char(*a)[64], char* out) {
            auto u = [&](int i) { return reinterpret_cast<uint8_t*>(a[i]); };
            return b200idx_mx4_product_device(1, 1, 32, u(0), u(1), u(2), u(3), B200IDX_F32, out, 0, nullptr);
        };
        taken(product(there, there[4]), "product");
        check(seen == 1, "product on its operands' device");
        taken(product(managed, there[4]), "product, managed operands");
        check(seen == 1, "product on its output's device");
        taken(product(managed, managed[4]), "product, managed memory");
        check(seen == current, "product on the current device");
        refused(product(here, there[4]), "different devices", "product of two devices");
        check(current_device == current, "the current device stays");
    }
    std::printf("%d failed\n", failed);
    return failed != 0;
}
