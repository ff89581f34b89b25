// A wait that runs out in a kernel of an exact index: the call that launched it says so, and the next one does not.  The
// kernels are the test's own (fake_device.h); they set the error word that the real ones set.
#include "fake_device.h"

using namespace b200;

static bool names_the_wait(const std::string& s) { return s.find("bounded wait") != std::string::npos; }

static void searches_again(int dtype) {
    constexpr int kN = 70000, kD = 64, kQ = 3, kK = 5;
    FlatIndex ix(kD, kMetricL2, dtype, 0);
    std::vector<float> x(static_cast<size_t>(kN) * kD), q(kQ * kD), D(kQ * kK);
    std::vector<int64_t> I(kQ * kK);
    ix.add(kN, x.data(), false, nullptr, false);
    auto search = [&] { return thrown([&] { ix.search_device(kQ, q.data(), false, kK, D.data(), I.data(), kK); }); };
    bool overflow = false, first_pass = false, second_pass = false;
    int again = 0;
    on_dist_gemm = [&](const GemmLaunch& L, const GemmArgs& a) {
        if (L.mode != kModeAppend) return;
        if (a.direct) ++again;
        if (a.direct ? second_pass : first_pass) *a.err = kDevErrPipelineTimeout;
    };
    on_select = [&](uint64_t*, const uint32_t*, uint32_t, uint8_t* over, const EmitArgs& e) {
        if (overflow && over && !e.qmap) over[1] = 1;
    };
    check(search().empty() && again == 0, "a search");
    overflow = true;
    check(search().empty() && again == 1, "a query searched for again");
    second_pass = true;
    check(names_the_wait(search()), "the wait of a query searched for again runs out: this call says so");
    second_pass = overflow = false;
    check(search().empty(), "and the next does not");
    first_pass = true;
    check(names_the_wait(search()), "the wait of the first pass runs out");
    first_pass = false;
    check(search().empty(), "and the next search is fine");
    on_dist_gemm = nullptr;
    on_select = nullptr;
}

static void scores() {
    constexpr int kN = 300, kD = 64;
    FlatIndex ix(kD, kMetricIP, kMX4, 0);
    std::vector<float> x(kN * kD), out(kN);
    ix.add(kN, x.data(), false, nullptr, false);
    bool late = false;
    on_product = [&](const Mx4ProductArgs& a) {
        if (late && a.err) *a.err = kDevErrPipelineTimeout;
    };
    auto call = [&] { return thrown([&] { ix.scores_device(1, x.data(), kF32, out.data(), kN); }); };
    check(call().empty(), "scores");
    late = true;
    check(names_the_wait(call()), "the wait of a product of scores runs out: the call says so");
    late = false;
    check(call().empty(), "and the next does not");
    on_product = nullptr;
}

// The selection gets the thresholds where another kernel may have made them, and none where every row is a candidate.
static void thresholds(int dtype, bool want) {
    constexpr int kN = 70000, kD = 64;
    FlatIndex ix(kD, kMetricL2, dtype, 0);
    std::vector<float> x(static_cast<size_t>(kN) * kD), D(4);
    std::vector<int64_t> I(4);
    ix.add(kN, x.data(), false, nullptr, false);
    int calls = 0;
    on_select = [&](uint64_t*, const uint32_t* counts, uint32_t, uint8_t* over, const EmitArgs& e) {
        ++calls;
        check((e.tau != nullptr) == (want && counts != nullptr), "thresholds for the selection");
        if (e.tau && over) over[0] = 1;   // (came short)
    };
    ix.search_device(1, x.data(), false, 4, D.data(), I.data(), 4);
    check(calls == (want ? 2 : 1) && ix.stats().fallback_queries == (want ? 1u : 0u), "a short list is searched for again");
    on_select = nullptr;
}

int main() {
    searches_again(kMX4);
    searches_again(kF16);
    scores();
    thresholds(kMX4, true);
    thresholds(kF16, false);
    std::printf("%d failed\n", failed);
    return failed != 0;
}
