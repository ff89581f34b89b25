// Distances of microscaled 4-bit rows with tcgen05.mma kind::mxf4 (E2M1 codes, a scale per 32 elements) and the
// selection in the epilogue.
//
// A CTA computes 128 x 256 tiles (queries x base rows) of fp32 accumulators in TMEM:
//   warp 0      : producer.  Per K chunk of 128 bytes (256 elements) a tensor copy of 256 base rows (SWIZZLE_128B) and
//                 their scales, which lie in memory in the order the tensor core wants, 512 bytes for 128 rows x 4
//                 blocks, so nothing is rearranged.  Up to d = 1024 the query tile stays in shared memory and its
//                 scales in TMEM for a whole query block; longer rows travel through the ring.
//   warp 1      : a stage's scales into TMEM (tcgen05.cp, a slot of columns per stage), up to four 128 x 256 x 64
//                 products.
//   warps 2-17  : epilogue.  Thread = (row, 64 of the tile's 256 columns), both 32-column chunks in
//                 registers at once, so that the accumulator goes back before the slow part begins.
// TMEM has 512 columns: two accumulators of 256 and the scales do not fit side by side.  The two accumulators
// therefore SHARE 104 columns (0-255 and 152-407; scales 408-511): tile t + 1 may start once tile t's shared columns
// are in registers, which half of the epilogue warps report.
#include "mx4_gemm.cuh"

#include <algorithm>
#include <cstring>
#include <type_traits>

#include "ptx_sm100.cuh"
#include "row_epilogue.cuh"
#include "row_ops.cuh"
#include "smem_limit.h"

namespace b200 {
namespace {

constexpr int kABytes = kTileQ * kChunkBytes, kBBytes = kTileB * kChunkBytes;   // 16 KB, 32 KB
constexpr int kSfaBytes = 1024, kSfbBytes = 2048;                               // two groups of 128 elements
constexpr int kResidentChunks = 4;   // of the query tile
constexpr int kMaxStages = 6;
constexpr int kSmemMost = 216 * 1024;   // beside the epilogue's norms
constexpr int kEpiWarps = 16;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr uint32_t kAcc1 = 152, kScaleCols = 408, kAllScaleCols = 104;   // TMEM columns
// A stage: base rows and their scales, or with them the queries and theirs.
constexpr int stage_bytes(bool resident) { return kBBytes + kSfbBytes + (resident ? 0 : kABytes + kSfaBytes); }
constexpr uint32_t scale_slot(bool resident) { return resident ? 16 : 24; }
constexpr int ring_stages(bool resident, int chunks) {
    const int kept = resident ? chunks : 0;
    const int by_smem = (kSmemMost - 1024 - kept * (kABytes + kSfaBytes)) / stage_bytes(resident);
    const int by_tmem = (static_cast<int>(kAllScaleCols) - 8 * kept) / static_cast<int>(scale_slot(resident));
    const int n = by_smem < by_tmem ? by_smem : by_tmem;
    return n < kMaxStages ? n : kMaxStages;
}
static_assert(ring_stages(true, 1) == 5 && ring_stages(true, kResidentChunks) == 4 && ring_stages(false, 8) == 4, "ring");

struct Mx4Args {
    GemmArgs g;
    const uint8_t* a_scales;
    const uint8_t* b_scales;
    int nb, ng;      // blocks of a row, groups of four
    int stages;
};

// Bit 31 - c: column c's key is below tau_up, the value above the threshold (L2; RowEpilogue::ip_mask otherwise).
__device__ __forceinline__ uint32_t l2_pass_mask(const uint32_t (&r)[32], const float* norms, float tau_up) {
    uint32_t m[2] = {0u, 0u};
#pragma unroll
    for (int g = 0; g < 8; ++g) {
        const float4 n = reinterpret_cast<const float4*>(norms)[g];
        uint32_t& h = m[g >> 2];
        h = __funnelshift_l(__float_as_uint(fmaf(-2.f, __uint_as_float(r[4 * g]), n.x) - tau_up), h, 1);
        h = __funnelshift_l(__float_as_uint(fmaf(-2.f, __uint_as_float(r[4 * g + 1]), n.y) - tau_up), h, 1);
        h = __funnelshift_l(__float_as_uint(fmaf(-2.f, __uint_as_float(r[4 * g + 2]), n.z) - tau_up), h, 1);
        h = __funnelshift_l(__float_as_uint(fmaf(-2.f, __uint_as_float(r[4 * g + 3]), n.w) - tau_up), h, 1);
    }
    return m[0] << 16 | (m[1] & 0xFFFFu);
}

template <int MODE, int BURST, bool L2, bool RESIDENT>
__global__ void __launch_bounds__(kThreads, 1)
mx4_gemm_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB, const __grid_constant__ Mx4Args m) {
    const GemmArgs& a = m.g;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bar_full[kMaxStages], bar_empty[kMaxStages], bar_acc_full[2], bar_shared_free[2];
    __shared__ uint64_t bar_a_full, bar_a_free;   // RESIDENT: the query tile landed; it was read for the last time
    __shared__ __align__(16) float tile_norms[L2 ? kEpiWarps : 1][2][64];   // of a warp's columns, two tiles in turn
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int nkc = (m.ng + 1) / 2;   // chunks of 256 elements
    constexpr int kStage = stage_bytes(RESIDENT);
    uint8_t* a_scales = smem + nkc * kABytes;                                   // RESIDENT: [nkc] codes, [nkc] scales, ring
    uint8_t* ring = RESIDENT ? a_scales + nkc * kSfaBytes : smem;
    if (threadIdx.x == 0) {
        for (int s = 0; s < m.stages; ++s) {
            ptx::mbar_init(&bar_full[s], 1);
            ptx::mbar_init(&bar_empty[s], 1);
        }
        ptx::mbar_init(&bar_acc_full[0], 1);
        ptx::mbar_init(&bar_acc_full[1], 1);
        ptx::mbar_init(&bar_shared_free[0], kEpiWarps / 2);
        ptx::mbar_init(&bar_shared_free[1], kEpiWarps / 2);
        ptx::mbar_init(&bar_a_full, 1);
        ptx::mbar_init(&bar_a_free, 1);
        abort_flag = 0;
        ptx::mbar_fence_init();
        ptx::prefetch_tensormap(&mapA);
        ptx::prefetch_tensormap(&mapB);
    }
    if (warp == 1) {
        ptx::tmem_alloc(&tmem_base_slot, 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem_base = tmem_base_slot;
    const int n_qb = (a.nq + kTileQ - 1) / kTileQ;
    const ItemRange range(a, n_qb);
    const uint32_t col_a = tmem_base + kScaleCols, col_b = col_a + (RESIDENT ? 8 * nkc : 0);

    if (warp == 0) {
        const bool leader = ptx::elect_one();
        uint32_t s = 0, ph = 0, loads = 0;
        int cur_qb = -1;
        bool ok = true;
        ItemCursor cur(range);
        const int64_t b_granules = (a.N + 127) / 128;
        for (int64_t i = 0; i < range.count && ok; ++i, cur.next()) {
            const uint8_t* sa = m.a_scales + static_cast<int64_t>(cur.qb) * m.ng * 512;
            if (RESIDENT && cur.qb != cur_qb) {
                if (loads && !ptx::mbar_wait_warp(&bar_a_free, (loads - 1u) & 1u, &abort_flag)) { ok = false; break; }
                if (leader) {
                    ptx::mbar_expect_tx(&bar_a_full, nkc * kABytes + m.ng * 512u);
                    for (int kc = 0; kc < nkc; ++kc) ptx::tma_load_2d(smem + kc * kABytes, &mapA, &bar_a_full, kc * kChunkBytes, cur.qb * kTileQ);
                    ptx::bulk_load_1d(a_scales, sa, m.ng * 512u, &bar_a_full);
                }
                __syncwarp();
                ++loads;
                cur_qb = cur.qb;
            }
            const int64_t tile = tile_of(a, cur.sel);
            const bool second = 2 * tile + 1 < b_granules;   // the tile's upper 128 rows exist
            const uint8_t* sb = m.b_scales + 2 * tile * m.ng * 512;
            for (int kc = 0; kc < nkc; ++kc) {
                if (!ptx::mbar_wait_warp(&bar_empty[s], ph ^ 1u, &abort_flag)) { ok = false; break; }
                if (leader) {
                    uint8_t* st = ring + s * kStage;
                    uint8_t* sf = st + kBBytes;
                    uint64_t* full = &bar_full[s];
                    const uint32_t bytes = min(2, m.ng - 2 * kc) * 512u;
                    ptx::mbar_expect_tx(full, kBBytes + bytes * (second ? 2u : 1u) + (RESIDENT ? 0u : kABytes + bytes));
                    ptx::tma_load_2d(st, &mapB, full, kc * kChunkBytes, static_cast<int>(tile * kTileB));
                    ptx::bulk_load_1d(sf, sb + kc * 1024, bytes, full);
                    if (second) ptx::bulk_load_1d(sf + 1024, sb + m.ng * 512 + kc * 1024, bytes, full);
                    if (!RESIDENT) {
                        ptx::tma_load_2d(st + kBBytes + kSfbBytes, &mapA, full, kc * kChunkBytes, cur.qb * kTileQ);
                        ptx::bulk_load_1d(st + kBBytes + kSfbBytes + kABytes, sa + kc * 1024, bytes, full);
                    }
                }
                __syncwarp();
                if (++s == static_cast<uint32_t>(m.stages)) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 1) {
        constexpr uint32_t kIdesc0 = ptx::umma_idesc_mxf4(kTileQ, kTileB, 0), kIdesc2 = ptx::umma_idesc_mxf4(kTileQ, kTileB, 2);
        const uint64_t desc_hi = ptx::umma_desc_k_sw128(0);
        const uint64_t sf_hi = ptx::umma_desc_k_plain(0, 128u, 128u);
        const uint32_t a_lo = (ptx::smem_u32(smem) & 0x3FFFFu) >> 4, ring_lo = (ptx::smem_u32(ring) & 0x3FFFFu) >> 4;
        const uint32_t a_sf_lo = (ptx::smem_u32(a_scales) & 0x3FFFFu) >> 4;
        const bool leader = ptx::elect_one();
        uint32_t s = 0, ph = 0, t = 0, seen = 0;
        int cur_qb = -1;
        bool ok = true;
        ItemCursor cur(range);
        for (int64_t i = 0; i < range.count && ok; ++i, ++t, cur.next()) {
            if (RESIDENT && cur.qb != cur_qb) {
                if (!ptx::mbar_wait_warp(&bar_a_full, seen & 1u, &abort_flag)) { ok = false; break; }
                ptx::tc_fence_after();
                if (leader)
                    for (int g = 0; g < m.ng; ++g) ptx::tmem_cp_scales(col_a + 4 * g, sf_hi | static_cast<uint64_t>(a_sf_lo + 32 * g));
                __syncwarp();
                ++seen;
                cur_qb = cur.qb;
            }
            // the columns this accumulator shares with tile t - 1's (and with them all of tile t - 2's).
            if (t && !ptx::mbar_wait_warp(&bar_shared_free[(t - 1u) & 1u], ((t - 1u) >> 1) & 1u, &abort_flag)) { ok = false; break; }
            const uint32_t tacc = tmem_base + (t & 1u ? kAcc1 : 0u);
            for (int kc = 0; kc < nkc; ++kc) {
                if (!ptx::mbar_wait_warp(&bar_full[s], ph, &abort_flag)) { ok = false; break; }
                ptx::tc_fence_after();
                const uint32_t st = ring_lo + s * (kStage >> 4), sf_lo = st + (kBBytes >> 4);
                const uint32_t slot = col_b + s * scale_slot(RESIDENT);   // 8 columns of b's scales per group, then 4 of a's
                const uint32_t at = RESIDENT ? a_lo + kc * (kABytes >> 4) : st + ((kBBytes + kSfbBytes) >> 4);
                const uint32_t sa = RESIDENT ? col_a + 8 * kc : slot + 16;
                const int steps = min(4, (m.nb - 8 * kc + 1) / 2);   // 64 elements each
                if (leader) {
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        if (2 * g >= steps) continue;
                        ptx::tmem_cp_scales(slot + 8 * g, sf_hi | static_cast<uint64_t>(sf_lo + g * 32));
                        ptx::tmem_cp_scales(slot + 8 * g + 4, sf_hi | static_cast<uint64_t>(sf_lo + 64 + g * 32));
                        if (!RESIDENT) ptx::tmem_cp_scales(sa + 4 * g, sf_hi | static_cast<uint64_t>(at + (kABytes >> 4) + g * 32));
                    }
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        if (ks < steps)
                            ptx::umma_mxf4(tacc, desc_hi | static_cast<uint64_t>(at + ks * 2), desc_hi | static_cast<uint64_t>(st + ks * 2),
                                           (ks & 1) ? kIdesc2 : kIdesc0, sa + (ks >> 1) * 4, slot + (ks >> 1) * 8, (kc | ks) ? 1u : 0u);
                    ptx::umma_commit(&bar_empty[s]);
                    if (kc + 1 == nkc) ptx::umma_commit(&bar_acc_full[t & 1u]);
                }
                __syncwarp();
                if (++s == static_cast<uint32_t>(m.stages)) { s = 0; ph ^= 1u; }
            }
            if (!ok) break;
            if (RESIDENT && (i + 1 == range.count || cur.last_of_qb())) {   // nothing of this query block is left
                if (leader) ptx::umma_commit(&bar_a_free);
                __syncwarp();
            }
        }
    } else {
        const int quarter = warp & 3, part = (warp - 2) >> 2;   // TMEM lanes, columns of this warp
        RowEpilogue<float, MODE, BURST, false, 2, false, !L2> epi(a);
        // L2, threshold mode: which columns of `r` (positions from c0 on) pass this row's threshold, and their keys
        auto mask_l2 = [&](const uint32_t (&r)[32], const float* norms, int64_t c0, int valid) {
            uint32_t mask = l2_pass_mask(r, norms, epi.tau_up) | epi.admit_all;
            if (valid < 32) mask &= ~(0xFFFFFFFFu >> valid);
            if (!epi.row_ok) return 0u;
            return a.qmask ? mask & __brev(epi.mask_word(c0)) : mask;
        };
        auto extract_l2 = [&](const uint32_t (&r)[32], uint32_t mask, const float* norms, uint32_t c0) {
            while (mask) {
                const uint32_t c = __clz(mask);
                mask &= ~(0x80000000u >> c);
                const float key = fmaf(-2.f, __uint_as_float(epi.pick(r, c)), norms[c]);
                if (!(key <= epi.tau)) continue;   // NaN
                epi.append(pack_cand(float_to_ord(key), c0 + c));
            }
        };
        // A tile's norms are on their way while the tile before it is worked on (read where they are used, they held up
        // every tile for a trip to memory: 16 queries against 1 M x 256, 5 000 cycles a tile).
        float next_norm[2] = {0.f, 0.f};
        auto fetch_norms = [&](const ItemCursor& c) {
            const float* p = static_cast<const float*>(a.bnorm) + static_cast<int64_t>(tile_of(a, c.sel)) * kTileB + part * 64 + lane;
            next_norm[0] = __ldg(p);
            next_norm[1] = __ldg(p + 32);
        };
        if (L2 && range.count > 0) fetch_norms(ItemCursor(range));
        uint32_t t = 0;
        ItemCursor cur(range);
        for (int64_t i = 0; i < range.count; ++i, ++t, cur.next()) {
            const int sel = cur.sel, q = cur.qb * kTileQ + quarter * 32 + lane;
            const int64_t tile = tile_of(a, sel);
            const int64_t col0 = tile * kTileB + part * 64;
            const uint32_t ab = t & 1u;
            const int64_t rem = a.N - col0;
            const int va = rem >= 32 ? 32 : (rem > 0 ? static_cast<int>(rem) : 0);
            const int vb = rem >= 64 ? 32 : (rem > 32 ? static_cast<int>(rem) - 32 : 0);
            uint32_t ra[32], rb[32];
            float* norms = tile_norms[L2 ? warp - 2 : 0][ab];
            if (L2) {   // (the buffer's last tile was the one before the last)
                norms[lane] = next_norm[0];
                norms[lane + 32] = next_norm[1];
                if (i + 1 < range.count) {
                    ItemCursor ahead = cur;
                    ahead.next();
                    fetch_norms(ahead);
                }
                __syncwarp();
            }
            const bool rows = cur.qb * kTileQ + quarter * 32 < a.nq;   // of this warp
            if (rows) epi.begin_tile(q, q < a.nq);
            if (!ptx::mbar_wait_warp(&bar_acc_full[ab], (t >> 1) & 1u, &abort_flag)) break;
            if (!rows) {
                __syncwarp();
                if (lane == 0 && (ab ? part < 2 : part >= 2)) ptx::mbar_arrive(&bar_shared_free[ab]);
                continue;
            }
            ptx::tc_fence_after();
            const uint32_t tacc = tmem_base + (ab ? kAcc1 : 0u) + part * 64 + (static_cast<uint32_t>(quarter * 32) << 16);
            ptx::tmem_ld_32x32(tacc, ra);
            ptx::tmem_ld_32x32(tacc + 32, rb);
            ptx::tmem_ld_wait(ra);
            ptx::tmem_ld_wait(rb);
            ptx::tc_fence_before();
            __syncwarp();
            // shared columns: 152 .. 255 of accumulator 0, 0 .. 103 of accumulator 1
            if (lane == 0 && (ab ? part < 2 : part >= 2)) ptx::mbar_arrive(&bar_shared_free[ab]);
            if (MODE == kModeAppend && !a.direct) {
                if (L2) {
                    const uint32_t ma = mask_l2(ra, norms, col0, va), mb = mask_l2(rb, norms + 32, col0 + 32, vb);
                    extract_l2(ra, ma, norms, static_cast<uint32_t>(col0));
                    extract_l2(rb, mb, norms + 32, static_cast<uint32_t>(col0) + 32);
                } else {
                    epi.ip_extract(ra, epi.ip_mask(ra, col0, va), col0);
                    epi.ip_extract(rb, epi.ip_mask(rb, col0 + 32, vb), col0 + 32);
                }
                epi.end_tile(0);
            } else {
                const uint32_t* nb = reinterpret_cast<const uint32_t*>(norms);
                const int slot = sel * (kTileB / BURST) + part * (64 / BURST);
                epi.chunk(ra, nb, col0, va, slot, 0, 0);
                epi.chunk(rb, nb + 32, col0 + 32, vb, slot + 32 / BURST, 1, 0);
                epi.end_tile(slot);
            }
        }
        epi.finish();
    }

    // After an abort, copies in flight get time to land before the CTA's shared memory is released.
    __syncwarp();
    if (abort_flag) {
        const long long t0 = clock64();
        while (clock64() - t0 < 4000000LL) { }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem_base, 512);
    }
    if (threadIdx.x == 0 && abort_flag) atomicOr(a.err, kDevErrPipelineTimeout);
}

template <int MODE, int BURST, bool L2>
cudaError_t launch_one(Mx4Args m, const CUtensorMap* mapA, const CUtensorMap* mapB, int num_sms, cudaStream_t stream) {
    GemmArgs& a = m.g;
    const int n_qb = (a.nq + kTileQ - 1) / kTileQ;
    const int64_t total = static_cast<int64_t>(n_qb) * a.n_tiles_sel;
    if (total <= 0) return cudaSuccess;
    if (a.tile_step < 1) a.tile_step = 1;
    const int chunks = (m.ng + 1) / 2;
    const bool resident = chunks <= kResidentChunks;
    m.stages = ring_stages(resident, chunks);
    const int smem = 1024 + (resident ? chunks * (kABytes + kSfaBytes) : 0) + m.stages * stage_bytes(resident);
    auto kern = resident ? mx4_gemm_kernel<MODE, BURST, L2, true> : mx4_gemm_kernel<MODE, BURST, L2, false>;
    cudaError_t e = allow_max_smem(kern);
    if (e != cudaSuccess) return e;
    const int grid = static_cast<int>(std::min<int64_t>(total, num_sms));
    // CTAs of different query blocks on the same stretch of the base at the same time, where the split stays even
    a.aligned_ranges = 0;
    if (n_qb <= grid && a.n_tiles_sel >= grid / n_qb) {
        const int nl_min = grid / n_qb;
        const double worst = static_cast<double>((a.n_tiles_sel + nl_min - 1) / nl_min);
        if (worst <= 1.06 * (static_cast<double>(total) / grid) + 1.0) a.aligned_ranges = 1;
    }
    const bool shared = n_qb == 1 && a.row_cands < 3LL * 4 * grid;   // (the rule of launch_dist_gemm)
    a.eager = total >= 16LL * grid && !shared ? 1 : 0;
    kern<<<grid, kThreads, smem, stream>>>(*mapA, *mapB, m);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_mx4_dist(const GemmLaunch& L, const GemmArgs& a, const uint8_t* a_scales, const uint8_t* b_scales,
                            const CUtensorMap* mapA, const CUtensorMap* mapB, cudaStream_t stream) {
    Mx4Args m{};
    m.g = a;
    m.a_scales = a_scales;
    m.b_scales = b_scales;
    m.nb = mx4_blocks(a.d);
    m.ng = mx4_groups(a.d);
    const bool l2 = a.metric == kMetricL2;
    if (L.mode == kModeAppend && !a.direct && a.tile_first >= 0 && a.tile_step <= 1) {
        const cudaError_t e = launch_mx4_few_search(a, a_scales, b_scales, L.num_sms, stream);
        if (e != cudaErrorNotSupported) return e;
    }
    if (L.mode == kModeAppend)
        return l2 ? launch_one<kModeAppend, 32, true>(m, mapA, mapB, L.num_sms, stream)
                  : launch_one<kModeAppend, 32, false>(m, mapA, mapB, L.num_sms, stream);
    if (L.burst == 8)
        return l2 ? launch_one<kModeBurstMin, 8, true>(m, mapA, mapB, L.num_sms, stream)
                  : launch_one<kModeBurstMin, 8, false>(m, mapA, mapB, L.num_sms, stream);
    return l2 ? launch_one<kModeBurstMin, 32, true>(m, mapA, mapB, L.num_sms, stream)
              : launch_one<kModeBurstMin, 32, false>(m, mapA, mapB, L.num_sms, stream);
}

}  // namespace b200
