// tcgen05 / TMEM / TMA distance GEMM with fused selection epilogues, plus a plain CUDA-core
// variant that shares the epilogue code and serves as an on-device cross-check.
//
// Pipeline of the tcgen05 variant (one persistent CTA per SM, 320 or 576 threads):
//   warp 0 (one lane)  : TMA producer.  Per K chunk of 128 bytes: query box 128 x 128 B and base
//                        box 256 x 128 B into a 4-stage ring of 48 KB stages (SWIZZLE_128B).
//   warp 1 (one lane)  : issues tcgen05.mma 128 x 256 x (32 bytes of K) from shared-memory
//                        descriptors into one of two 256-column TMEM accumulators; commits free
//                        the stage (per chunk) and publish the accumulator (per tile).
//   warps 2-9 / 2-17   : epilogue, two or four warps per scheduler (see epi_warps).  Thread = (query
//                        row = TMEM lane, a half or a quarter of the tile's columns); reads 32
//                        columns at a time with tcgen05.ld (double-buffered) and applies the
//                        selection predicate (after the norm-add where the operands are not folded).
// Work items are (query block, base tile) pairs, query block fastest, so the CTAs running at
// the same time read the same base tiles and HBM sees each base tile about once per pass.
#include "dist_gemm.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "cos16.cuh"

#include <cstring>
#include <type_traits>

#include "common.cuh"
#include "ptx_sm100.cuh"
#include "row_epilogue.cuh"

namespace b200 {
namespace {

constexpr int kMaxStages = 8;
// int8 with the fp16 cosine epilogue: a kernel instantiation of its own (chosen by launch_dist_gemm from
// GemmArgs::metric), so that the inner-product / L2 kernels carry none of its code
constexpr int kKindI8Cos = 3;
// int8 inner product: reads no norms, so its epilogue is light enough for sixteen warps of two
// chunks (96 registers) instead of eight of four -- the eight, two per scheduler, cannot hide their
// own instruction latency
constexpr int kKindI8IP = 4;
constexpr int kKindF16IP = 5;   // the same for fp16 operands
constexpr int kKindI8L2 = 6;    // sixteen-warp L2 kinds, see l2_global
constexpr int kKindF16L2 = 7;
__host__ __device__ constexpr bool is_i8(int kind) {
    return kind == kKindI8 || kind == kKindI8Cos || kind == kKindI8IP || kind == kKindI8L2;
}
__host__ __device__ constexpr bool ip_only(int kind) { return kind == kKindI8IP || kind == kKindF16IP; }
// L2 with sixteen epilogue warps as well: the norms are not staged in shared memory (which costs a
// barrier per item and 32 registers per chunk) but read from global memory where they are used --
// the 32 lanes of a warp want the same 32 norms, so a load is one broadcast that hits L1 after the
// first warp of the CTA has asked for it.
__host__ __device__ constexpr bool l2_global(int kind) { return kind == kKindI8L2 || kind == kKindF16L2; }
constexpr int kStageABytes = kTileQ * kChunkBytes;               // 16 KB
constexpr int kStageBBytes = kTileB * kChunkBytes;               // 32 KB
constexpr int kStageBytes = kStageABytes + kStageBBytes;         // 48 KB
constexpr int kGemmSmemBudget = 224 * 1024;                      // dynamic shared memory incl. 1 KB alignment slack
constexpr int kResidentMaxChunks = 4;                            // query tile kept in shared memory up to 64 KB
// Epilogue warps: two per scheduler, each thread draining half of a row's columns, where the
// epilogue is bound by shared-memory norm loads (fp16, int8); four per scheduler and a quarter
// of the columns each for the folded bf16 kind, whose short ALU-only epilogue is latency-bound
// and scales with the number of warps.
__host__ __device__ constexpr int epi_warps(int kind) {
    return (kind == kKindBF16 || ip_only(kind) || l2_global(kind) || kind == kKindI8Cos) ? 16 : 8;
}
// + the producer warp, the MMA warp and, behind the epilogue warps, a second MMA warp and a second
// producer warp (even and odd items have their own issuing threads and their own stage sub-ring)
__host__ __device__ constexpr int gemm_threads(int kind) { return 64 + 32 * epi_warps(kind) + 64; }
__host__ __device__ constexpr int mma2_warp(int kind) { return 2 + epi_warps(kind); }
__host__ __device__ constexpr int prod2_warp(int kind) { return 3 + epi_warps(kind); }
constexpr uint32_t kTmemCols = 512;
// Per-role cycle counters (GemmArgs::prof) exist in development builds only (-DB200IDX_DEV_PROF):
// the epilogue is bound by instruction issue, and even predicated-off clock reads cost slots.
#ifdef B200IDX_DEV_PROF
constexpr bool kDevProf = true;
#else
constexpr bool kDevProf = false;
#endif

// Shared-memory side of the epilogue: the tile's base norms, double-buffered with the TMEM
// accumulators (kinds whose operands are not folded).
struct EpiShared {
    uint32_t norm[2][kTileB];
};

// ---------------------------------------------------------------------------------------
// tcgen05 variant
// ---------------------------------------------------------------------------------------
// Shared memory is the scarce resource of this kernel: a 128 x 256 x 16 UMMA reads 12 KB of
// operands, and with K of a few hundred every operand byte that TMA writes is read about once, so
// TMA writes and UMMA reads together are bounded by the 128 B/clk of the shared-memory pipe.  When
// the query tile is small enough (a.a_resident) it is therefore loaded once per query block and
// only base chunks (32 KB) travel through the stage ring.
template <int KIND, int MODE, int BURST>
__global__ void __launch_bounds__(gemm_threads(KIND), 1)
dist_gemm_tc_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB,
                    const GemmArgs a) {
    using AccT = typename std::conditional<is_i8(KIND), int32_t, float>::type;
    constexpr int kElemBytes = is_i8(KIND) ? 1 : 2;
    constexpr int kChunkElems = kChunkBytes / kElemBytes;
    constexpr bool FOLD = KIND == kKindBF16;
    constexpr uint32_t kIdesc = is_i8(KIND) ? ptx::umma_idesc(2, 1, kTileQ, kTileB)
                                                : ptx::umma_idesc(1, KIND == kKindBF16 ? 1 : 0, kTileQ, kTileB);

    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bar_full[kMaxStages];
    __shared__ uint64_t bar_empty[kMaxStages];
    __shared__ uint64_t bar_acc_full[2];
    __shared__ uint64_t bar_acc_empty[2];
    __shared__ uint64_t bar_a_full;      // resident query tile landed
    __shared__ uint64_t bar_a_free;      // every UMMA that read the resident query tile has completed
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag;
    __shared__ __align__(16) EpiShared epi_sh;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    // Packed operands (bf16 kind only): the query tile and a base tile are one contiguous image each;
    // an item is ONE stage of its parity's sub-ring (nst = 1) and ONE hand-off per role.
    const bool packed = KIND == kKindBF16 && a.packed != 0;
    const uint32_t a_img_bytes = static_cast<uint32_t>(kTileQ) * a.d * 2u;
    const int nkc = packed ? 1 : (a.d + kChunkElems - 1) / kChunkElems;
    const bool resident = a.a_resident != 0;
    const int nst = a.n_stages / 2;          // stages per sub-ring (even / odd items)
    const uint32_t stage_bytes = packed ? static_cast<uint32_t>(kTileB) * a.d * 2u : (resident ? kStageBBytes : kStageBytes);
    uint8_t* ring = smem + (packed ? ((a_img_bytes + 1023u) & ~1023u) : (resident ? nkc * kStageABytes : 0));

    if (threadIdx.x == 0) {
        for (int r = 0; r < 2; ++r)
            for (int s = 0; s < nst; ++s) {
                ptx::mbar_init(&bar_full[r * (kMaxStages / 2) + s], 1);
                ptx::mbar_init(&bar_empty[r * (kMaxStages / 2) + s], 1);
            }
        for (int b = 0; b < 2; ++b) {
            ptx::mbar_init(&bar_acc_full[b], 1);
            ptx::mbar_init(&bar_acc_empty[b], epi_warps(KIND));
        }
        ptx::mbar_init(&bar_a_full, 1);
        ptx::mbar_init(&bar_a_free, 2);   // both MMA-issuing threads
        abort_flag = 0;
        ptx::mbar_fence_init();
        if (!packed) {
            ptx::prefetch_tensormap(&mapA);
            ptx::prefetch_tensormap(&mapB);
        }
    }
    if (warp == 1) {
        ptx::tmem_alloc(&tmem_base_slot, kTmemCols);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem_base = tmem_base_slot;

    const int n_qb = (a.nq + kTileQ - 1) / kTileQ;
    const ItemRange range(a, n_qb);

    if (warp == 0 || warp == prod2_warp(KIND)) {
        if (lane == 0) {
            const uint32_t pidx = warp == 0 ? 0u : 1u;   // this producer serves the items of this parity
            // Two sub-rings of nst / 2 stages: even items travel through the first, odd items through
            // the second, so that each ring's barriers have exactly one consuming thread (a consumer a
            // whole revolution ahead of the other would otherwise read a parity that has not happened).
            // The resident query tile is loaded by producer 0.
            int rs = 0;
            uint32_t rph = 0;
            int cur_qb = -1;
            uint32_t a_loads = 0, t = 0;
            bool ok = true;
            long long pw = 0;
            const bool prof_on = kDevProf && a.prof && pidx == 0;
            const long long k0 = prof_on ? clock64() : 0;
            const uint32_t r = pidx;
            ItemCursor cur(range);
            for (int64_t i = 0; i < range.count && ok; ++i, ++t, cur.next()) {
                const int qb = cur.qb;
                if (resident && pidx == 0 && qb != cur_qb) {
                    // the previous query block's UMMAs must be done with the tile before it is overwritten
                    if (a_loads && !ptx::mbar_wait_bounded(&bar_a_free, (a_loads - 1u) & 1u, &abort_flag)) { ok = false; break; }
                    if (packed) {
                        ptx::mbar_expect_tx(&bar_a_full, a_img_bytes);
                        ptx::bulk_load_1d(smem, static_cast<const uint8_t*>(a.A) + static_cast<size_t>(qb) * a_img_bytes,
                                          a_img_bytes, &bar_a_full);
                    } else {
                        ptx::mbar_expect_tx(&bar_a_full, static_cast<uint32_t>(nkc) * kStageABytes);
                        for (int kc = 0; kc < nkc; ++kc)
                            ptx::tma_load_2d(smem + kc * kStageABytes, &mapA, &bar_a_full, kc * kChunkElems, qb * kTileQ);
                    }
                    ++a_loads;
                    cur_qb = qb;
                }
                if ((t & 1u) != pidx) continue;
                const int tile = tile_of(a, cur.sel);
                for (int kc = 0; kc < nkc; ++kc) {
                    const int s = rs;
                    uint64_t* full = &bar_full[r * (kMaxStages / 2) + s];
                    const long long w0 = prof_on ? clock64() : 0;
                    if (!ptx::mbar_wait_bounded(&bar_empty[r * (kMaxStages / 2) + s], rph ^ 1u, &abort_flag)) { ok = false; break; }
                    if (prof_on) pw += clock64() - w0;
                    ptx::mbar_expect_tx(full, stage_bytes);
                    uint8_t* st = ring + static_cast<size_t>(r * nst + s) * stage_bytes;
                    if (packed) {
                        const void* src = a.seg_tile ? a.seg_tile[tile]
                                                     : static_cast<const uint8_t*>(a.B) + static_cast<size_t>(tile) * stage_bytes;
                        ptx::bulk_load_1d(st, src, stage_bytes, full);
                        if (++rs == nst) { rs = 0; rph ^= 1u; }
                        continue;
                    }
                    if (!resident) {
                        ptx::tma_load_2d(st, &mapA, full, kc * kChunkElems, qb * kTileQ);
                        st += kStageABytes;
                    }
                    ptx::tma_load_2d(st, &mapB, full, kc * kChunkElems, tile * kTileB);
                    if (++rs == nst) { rs = 0; rph ^= 1u; }
                }
                if (kDevProf && a.trace && blockIdx.x == 0 && t < 64) a.trace[0 * 64 + t] = clock64();
            }
            if (prof_on) {
                atomicAdd(a.prof + 0, static_cast<unsigned long long>(pw));
                atomicAdd(a.prof + 7, static_cast<unsigned long long>(clock64() - k0));
            }
        }
    } else if (warp == 1 || warp == mma2_warp(KIND)) {
        // Two threads issue the UMMAs, one for the even items (accumulator 0) and one for the odd
        // items (accumulator 1), on different schedulers: a single issuing thread, sharing its
        // scheduler with busy epilogue warps, could not keep the tensor pipe fed.  Both walk the
        // whole item list so that their view of the query-block runs agrees; each consumes its own
        // sub-ring of stages.
        if (lane == 0) {
            const uint32_t parity = warp == 1 ? 0u : 1u;
            const bool prof_on = kDevProf && a.prof && parity == 0;
            int s = 0;
            uint32_t ph = 0, t = 0;
            int cur_qb = -1;
            uint32_t a_seen = 0;
            bool ok = true;
            long long mw0 = 0, mw1 = 0;
            // Descriptors differ only in their 14-bit address field: build the constant part once
            // and add byte offsets / 16 (the single issuing thread is on the critical path).
            const uint64_t desc_hi = ptx::umma_desc_k_sw128(0);
            // packed operands: core matrices adjacent along K are 128 bytes apart, 8-row groups a.d / 8 of them
            const uint64_t desc_hi_p = ptx::umma_desc_k_plain(0, 128u, static_cast<uint32_t>(a.d) * 16u);
            const uint32_t a_res_lo = (ptx::smem_u32(smem) & 0x3FFFFu) >> 4;
            const uint32_t ring_lo = (ptx::smem_u32(ring) & 0x3FFFFu) >> 4;
            const uint32_t stage_lo = stage_bytes >> 4;
            const int tail_bytes = a.d * kElemBytes - (nkc - 1) * kChunkBytes;   // bytes of K in the last chunk
            const int tail_nks = tail_bytes >= kChunkBytes ? kChunkBytes / 32 : (tail_bytes + 31) / 32;
            ItemCursor cur(range);
            for (int64_t i = 0; i < range.count && ok; ++i, ++t, cur.next()) {
                const int qb = cur.qb;
                if (resident && qb != cur_qb) {
                    if (!ptx::mbar_wait_bounded(&bar_a_full, a_seen & 1u, &abort_flag)) { ok = false; break; }
                    ++a_seen;
                    cur_qb = qb;
                }
                const bool run_ends = resident && (i + 1 == range.count || cur.last_of_qb());
                if ((t & 1u) != parity) {
                    // the other thread's item (it travels through the other sub-ring)
                    if (run_ends) ptx::umma_commit(&bar_a_free);   // nothing of this run left on this thread
                    continue;
                }
                const uint32_t ab = parity;
                const uint32_t aph = (t >> 1) & 1u;
                long long w0 = prof_on ? clock64() : 0;
                if (!ptx::mbar_wait_bounded(&bar_acc_empty[ab], aph ^ 1u, &abort_flag)) { ok = false; break; }
                if (prof_on) mw0 += clock64() - w0;
                if (kDevProf && a.trace && blockIdx.x == 0 && t < 64) a.trace[1 * 64 + t] = clock64();
                ptx::tc_fence_after();
                const uint32_t tacc = tmem_base + ab * kTileB;
                for (int kc = 0; kc < nkc; ++kc) {
                    w0 = prof_on ? clock64() : 0;
                    if (!ptx::mbar_wait_bounded(&bar_full[parity * (kMaxStages / 2) + s], ph, &abort_flag)) { ok = false; break; }
                    if (prof_on) mw1 += clock64() - w0;
                    if (kDevProf && a.trace && blockIdx.x == 0 && t < 64 && kc + 1 == nkc) a.trace[2 * 64 + t] = clock64();
                    ptx::tc_fence_after();
                    const uint32_t st_lo = ring_lo + (parity * static_cast<uint32_t>(nst) + static_cast<uint32_t>(s)) * stage_lo;
                    if (packed) {
                        // K / 16 steps of one 128 x 256 x 16 UMMA; a step advances both images by two core matrices
                        const int nks_p = a.d >> 4;
                        for (int ks = 0; ks < nks_p; ++ks) {
                            const uint64_t da = desc_hi_p | static_cast<uint64_t>(a_res_lo + ks * 16);
                            const uint64_t db = desc_hi_p | static_cast<uint64_t>(st_lo + ks * 16);
                            ptx::umma_f16(tacc, da, db, kIdesc, ks > 0 ? 1u : 0u);
                        }
                        ptx::umma_commit(&bar_empty[parity * (kMaxStages / 2) + s]);
                        if (++s == nst) { s = 0; ph ^= 1u; }
                        continue;
                    }
                    const uint32_t sa_lo = resident ? a_res_lo + static_cast<uint32_t>(kc) * (kStageABytes >> 4) : st_lo;
                    const uint32_t sb_lo = resident ? st_lo : st_lo + (kStageABytes >> 4);
                    // the last chunk may hold fewer than four 32-byte K steps (the rest is zero fill)
                    const int nks = kc + 1 == nkc ? tail_nks : kChunkBytes / 32;
#pragma unroll
                    for (int ks = 0; ks < kChunkBytes / 32; ++ks) {
                        if (ks >= nks) break;
                        const uint64_t da = desc_hi | static_cast<uint64_t>(sa_lo + ks * 2);
                        const uint64_t db = desc_hi | static_cast<uint64_t>(sb_lo + ks * 2);
                        const uint32_t accum = (kc > 0 || ks > 0) ? 1u : 0u;
                        if (kDevProf && (a.dbg & 4)) continue;
                        if (is_i8(KIND)) ptx::umma_i8(tacc, da, db, kIdesc, accum);
                        else ptx::umma_f16(tacc, da, db, kIdesc, accum);
                    }
                    ptx::umma_commit(&bar_empty[parity * (kMaxStages / 2) + s]);
                    if (++s == nst) { s = 0; ph ^= 1u; }
                }
                if (!ok) break;
                ptx::umma_commit(&bar_acc_full[ab]);
                if (kDevProf && a.trace && blockIdx.x == 0 && t < 64) a.trace[3 * 64 + t] = clock64();
                // last item of this CTA for the query block: the resident tile may be replaced once
                // everything both threads issued so far has completed
                if (run_ends) ptx::umma_commit(&bar_a_free);
            }
            if (prof_on) {
                atomicAdd(a.prof + 1, static_cast<unsigned long long>(mw0));
                atomicAdd(a.prof + 2, static_cast<unsigned long long>(mw1));
            }
        }
    } else {
        const int quarter = warp & 3;          // TMEM lane quarter this warp may read
        const int half = (warp - 2) >> 2;      // which kCols columns of the tile this warp drains
        const int row_in_tile = quarter * 32 + lane;
        const int et = threadIdx.x - 64;       // epilogue thread index
        constexpr int kCols = kTileB / (epi_warps(KIND) / 4);   // columns per epilogue thread
        RowEpilogue<AccT, MODE, BURST, FOLD, kCols / 32, KIND == kKindI8Cos, ip_only(KIND)> epi(a);
        // FOLD, plain inner products: no norms; sixteen-warp L2: norms read where they are used
        const bool l2 = a.metric == kMetricL2 && !FOLD && !ip_only(KIND) && !l2_global(KIND);
        constexpr bool cosm = KIND == kKindI8Cos;
        const uint32_t* gnorm = static_cast<const uint32_t*>(a.bnorm);
        uint32_t t = 0;
        bool ok = true;
        long long ew = 0, ec = 0, ef = 0, elw = 0, ebar = 0, ecc = 0;
        const bool profiler = kDevProf && a.prof && warp == 2 && lane == 0;
        ItemCursor cur(range);
        for (int64_t i = 0; i < range.count && ok; ++i, ++t, cur.next()) {
            const int qb = cur.qb;
            const int sel = cur.sel;
            const int tile = tile_of(a, sel);
            const uint32_t ab = t & 1u;
            const uint32_t aph = (t >> 1) & 1u;
            const int q_in = qb * kTileQ + row_in_tile;
            const int64_t tile_col0 = static_cast<int64_t>(tile) * kTileB;
            // segmented base: the tile's index decides the candidate row and the valid extent
            int q = q_in;
            int64_t cbase = 0, n_end = a.N;
            if (a.seg_index) {
                q += (__ldg(a.seg_index + tile) - a.seg_first) * a.nq;
                cbase = __ldg(a.seg_col0 + tile);
                n_end = __ldg(a.seg_end + tile);
            }
            const long long e0 = profiler ? clock64() : 0;
            // The tile's norms travel global -> registers while the MMA is still running.
            uint32_t n0 = 0;
            if ((l2 || cosm) && et < kTileB) {
                n0 = __ldg(gnorm + tile_col0 + et);
                if (cosm) n0 = cos16_rnorm_bits(static_cast<int32_t>(n0));
            }
            epi.begin_tile(q, q_in < a.nq);
            if (!ptx::mbar_wait_bounded(&bar_acc_full[ab], aph, &abort_flag)) {
                // leave without stranding a sibling warp at the named barrier below
                if (!FOLD && (l2 || cosm)) asm volatile("bar.arrive 1, %0;" ::"n"(32 * epi_warps(KIND)) : "memory");
                ok = false;
                break;
            }
            const long long e1 = profiler ? clock64() : 0;
            if (kDevProf && a.trace && blockIdx.x == 0 && t < 64 && lane == 0 && (warp == 2 || warp == 2 + epi_warps(KIND) - 1))
                a.trace[(warp == 2 ? 4 : 6) * 64 + t] = clock64();
            ptx::tc_fence_after();
            const long long b0 = profiler ? clock64() : 0;
            if (!FOLD && (l2 || cosm)) {   // inner product: no norms, and no reason to keep the warps in step
                if (et < kTileB) epi_sh.norm[ab][et] = n0;
                asm volatile("bar.sync 1, %0;" ::"n"(32 * epi_warps(KIND)) : "memory");   // the epilogue warps
            }
            if (profiler) ebar += clock64() - b0;
            const uint32_t tacc =
                tmem_base + ab * kTileB + half * kCols + (static_cast<uint32_t>(quarter * 32) << 16);
            const int64_t half_col0 = tile_col0 + half * kCols;
            // sixteen-warp L2: the generic chunk code (sample pass, direct mode) reads the norms from global memory too
            const uint32_t* hnorm = l2_global(KIND) ? gnorm + tile_col0 + half * kCols : &epi_sh.norm[ab][half * kCols];
            // first burst slot: counted from the pass's first tile, or from the first tile of the segment
            const int slot_tile = a.seg_index ? tile - static_cast<int>(cbase / kTileB) : sel;
            const int hslot = slot_tile * (kTileB / BURST) + half * (kCols / BURST);
            uint32_t ra[32], rb[32];
            if (KIND == kKindI8Cos && MODE == kModeAppend && kCols == 64 && !a.direct) {
                // cosine: the accumulators of both chunks become ordered fp16 scores in place (the
                // reciprocal norms staged above are read here, before the buffer goes back), and from
                // there on they are inner products
                ptx::tmem_ld_32x32(tacc, ra);
                ptx::tmem_ld_32x32(tacc + 32, rb);
                ptx::tmem_ld_wait(ra);
                ptx::tmem_ld_wait(rb);
                epi.cos_scores(ra, hnorm);
                epi.cos_scores(rb, hnorm + 32);
                const int64_t rem_a = n_end - half_col0, rem_b = rem_a - 32;
                const uint32_t ma = epi.ip_mask(ra, half_col0, rem_a >= 32 ? 32 : (rem_a > 0 ? static_cast<int>(rem_a) : 0));
                const uint32_t mb = epi.ip_mask(rb, half_col0 + 32, rem_b >= 32 ? 32 : (rem_b > 0 ? static_cast<int>(rem_b) : 0));
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&bar_acc_empty[ab]);
                epi.ip_extract(ra, ma, half_col0);
                epi.ip_extract(rb, mb, half_col0 + 32);
                epi.end_tile(hslot);
                continue;
            }
            if (ip_only(KIND) && MODE == kModeAppend && kCols == 64 && !a.direct) {
                // as below: both chunks, both masks, the accumulator back, then the candidates
                ptx::tmem_ld_32x32(tacc, ra);
                ptx::tmem_ld_32x32(tacc + 32, rb);
                ptx::tmem_ld_wait(ra);
                ptx::tmem_ld_wait(rb);
                const int64_t rem_a = n_end - half_col0, rem_b = rem_a - 32;
                const uint32_t ma = epi.ip_mask(ra, half_col0, rem_a >= 32 ? 32 : (rem_a > 0 ? static_cast<int>(rem_a) : 0));
                const uint32_t mb = epi.ip_mask(rb, half_col0 + 32, rem_b >= 32 ? 32 : (rem_b > 0 ? static_cast<int>(rem_b) : 0));
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&bar_acc_empty[ab]);
                epi.ip_extract(ra, ma, half_col0);
                epi.ip_extract(rb, mb, half_col0 + 32);
                epi.end_tile(hslot);
                continue;
            }
            if (l2_global(KIND) && MODE == kModeAppend && kCols == 64 && !a.direct) {
                ptx::tmem_ld_32x32(tacc, ra);
                ptx::tmem_ld_32x32(tacc + 32, rb);
                ptx::tmem_ld_wait(ra);
                ptx::tmem_ld_wait(rb);
                const uint32_t* gna = gnorm + half_col0;
                const int64_t rem_a = n_end - half_col0, rem_b = rem_a - 32;
                const uint32_t ma = epi.l2_mask(ra, gna, half_col0, rem_a >= 32 ? 32 : (rem_a > 0 ? static_cast<int>(rem_a) : 0));
                const uint32_t mb = epi.l2_mask(rb, gna + 32, half_col0 + 32, rem_b >= 32 ? 32 : (rem_b > 0 ? static_cast<int>(rem_b) : 0));
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&bar_acc_empty[ab]);
                epi.l2_extract(ra, ma, half_col0, gna);
                epi.l2_extract(rb, mb, half_col0 + 32, gna + 32);
                epi.end_tile(hslot);
                continue;
            }
            if (FOLD && MODE == kModeAppend && kCols == 64 && !a.direct && !(kDevProf && a.dbg)) {
                // Both chunks into registers, the pass masks, and the accumulator goes back to the MMA
                // side at once: taking the candidates out (the slow, uneven part -- a warp with three
                // hits would otherwise hold the buffer for all sixteen) happens afterwards, from the
                // registers, while the tensor core already refills the buffer.
                ptx::tmem_ld_32x32(tacc, ra);
                ptx::tmem_ld_32x32(tacc + 32, rb);
                ptx::tmem_ld_wait(ra);
                ptx::tmem_ld_wait(rb);
                const int64_t rem_a = n_end - half_col0, rem_b = rem_a - 32;
                const int va = rem_a >= 32 ? 32 : (rem_a > 0 ? static_cast<int>(rem_a) : 0);
                const int vb = rem_b >= 32 ? 32 : (rem_b > 0 ? static_cast<int>(rem_b) : 0);
                if (a.seg_bias) {
                    const uint32_t ma = epi.seg_fold_mask(ra, va), mb = epi.seg_fold_mask(rb, vb);
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(&bar_acc_empty[ab]);
                    epi.seg_fold_extract(ra, ma, half_col0);
                    epi.seg_fold_extract(rb, mb, half_col0 + 32);
                    epi.end_tile(hslot);
                    continue;
                }
                const uint32_t ma = epi.fold_mask(ra, half_col0, va);
                const uint32_t mb = epi.fold_mask(rb, half_col0 + 32, vb);
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&bar_acc_empty[ab]);
                epi.fold_extract(ra, ma, half_col0);
                epi.fold_extract(rb, mb, half_col0 + 32);
                epi.end_tile(hslot);
                continue;
            }
            const bool dbg_no_ld = kDevProf && (a.dbg & 2), dbg_no_chunk = kDevProf && (a.dbg & 3);
            if (!dbg_no_ld) ptx::tmem_ld_32x32(tacc, ra);
            // two chunks per step, the TMEM load of the next chunk in flight behind the current one
            auto step = [&](int c) {
                if (dbg_no_ld) return;
                const long long w0 = profiler ? clock64() : 0;
                ptx::tmem_ld_wait(ra);
                if (profiler) elw += clock64() - w0;
                ptx::tmem_ld_32x32(tacc + (c + 1) * 32, rb);
                {
                    const long long c0 = profiler ? clock64() : 0;
                    const int64_t col0 = half_col0 + c * 32;
                    const int64_t rem = n_end - col0;
                    if (!dbg_no_chunk) epi.chunk(ra, hnorm + c * 32, col0, rem >= 32 ? 32 : (rem > 0 ? static_cast<int>(rem) : 0),
                              hslot + c * (32 / BURST), c, cbase);
                    if (profiler) ecc += clock64() - c0;
                }
                const long long w1 = profiler ? clock64() : 0;
                ptx::tmem_ld_wait(rb);
                if (profiler) elw += clock64() - w1;
                if (c + 2 < kCols / 32) ptx::tmem_ld_32x32(tacc + (c + 2) * 32, ra);
                {
                    const int64_t col0 = half_col0 + (c + 1) * 32;
                    const int64_t rem = n_end - col0;
                    if (!dbg_no_chunk) epi.chunk(rb, hnorm + (c + 1) * 32, col0, rem >= 32 ? 32 : (rem > 0 ? static_cast<int>(rem) : 0),
                              hslot + (c + 1) * (32 / BURST), c + 1, cbase);
                }
            };
            if (FOLD) {   // small body: unrolled, so the chunk index is a constant
#pragma unroll
                for (int c = 0; c < kCols / 32; c += 2) step(c);
            } else {
#pragma unroll 1
                for (int c = 0; c < kCols / 32; c += 2) step(c);
            }
            // accumulator drained: hand the TMEM buffer back before the global stores
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&bar_acc_empty[ab]);
            if (kDevProf && a.trace && blockIdx.x == 0 && t < 64 && lane == 0 && (warp == 2 || warp == 2 + epi_warps(KIND) - 1))
                a.trace[(warp == 2 ? 5 : 7) * 64 + t] = clock64();
            const long long e2 = profiler ? clock64() : 0;
            epi.end_tile(hslot);
            if (profiler) {
                const long long e3 = clock64();
                ew += e1 - e0;
                ec += e2 - e1;
                ef += e3 - e2;
            }
        }
        epi.finish();
        if (profiler) {
            atomicAdd(a.prof + 3, static_cast<unsigned long long>(ew));
            atomicAdd(a.prof + 4, static_cast<unsigned long long>(ec));
            atomicAdd(a.prof + 5, static_cast<unsigned long long>(ef));
            atomicAdd(a.prof + 6, static_cast<unsigned long long>(t));
            atomicAdd(a.prof + 8, static_cast<unsigned long long>(elw));
            atomicAdd(a.prof + 9, static_cast<unsigned long long>(ebar));
            atomicAdd(a.prof + 10, static_cast<unsigned long long>(ecc));
        }
    }

    // Teardown.  After an abort, give copies in flight time to land before the CTA's shared
    // memory is released.
    __syncwarp();
    if (abort_flag) {
        const long long t0 = clock64();
        while (clock64() - t0 < 4000000LL) { }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem_base, kTmemCols);
    }
    if (threadIdx.x == 0 && abort_flag) atomicOr(a.err, kDevErrPipelineTimeout);
}

// ---------------------------------------------------------------------------------------
// CUDA-core variant: same work decomposition and epilogue, accumulators computed with
// scalar FMAs.  Used to cross-check the tcgen05 variant on device.
// ---------------------------------------------------------------------------------------
template <int KIND>
__device__ __forceinline__ typename std::conditional<is_i8(KIND), int32_t, float>::type
load_elem(const void* p, int64_t idx) {
    if (is_i8(KIND)) return static_cast<int32_t>(static_cast<const int8_t*>(p)[idx]);
    else if (KIND == kKindBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[idx]);
    else return __half2float(static_cast<const __half*>(p)[idx]);
}

template <int KIND, int MODE, int BURST>
__global__ void __launch_bounds__(kTileQ)
dist_gemm_simt_kernel(const GemmArgs a) {
    using AccT = typename std::conditional<is_i8(KIND), int32_t, float>::type;
    __shared__ __align__(16) EpiShared epi_sh;
    const int n_qb = (a.nq + kTileQ - 1) / kTileQ;
    const ItemRange range(a, n_qb);
    const bool l2 = a.metric == kMetricL2;
    constexpr bool cosm = KIND == kKindI8Cos;
    const uint32_t* gnorm = static_cast<const uint32_t*>(a.bnorm);
    RowEpilogue<AccT, MODE, BURST, KIND == kKindBF16, kTileB / 32, KIND == kKindI8Cos, ip_only(KIND)> epi(a);
    ItemCursor cur(range);
    for (int64_t i = 0; i < range.count; ++i, cur.next()) {
        const int qb = cur.qb;
        const int sel = cur.sel;
        const int tile = tile_of(a, sel);
        const int q_in = qb * kTileQ + threadIdx.x;
        const bool row_ok = q_in < a.nq;
        const int qc = row_ok ? q_in : a.nq - 1;
        const int64_t tile_col0 = static_cast<int64_t>(tile) * kTileB;
        int q = q_in;
        int64_t cbase = 0, n_end = a.N;
        if (a.seg_index) {
            q += (a.seg_index[tile] - a.seg_first) * a.nq;
            cbase = a.seg_col0[tile];
            n_end = a.seg_end[tile];
        }
        const int slot_tile = a.seg_index ? tile - static_cast<int>(cbase / kTileB) : sel;
        __syncthreads();
        for (int h = 0; h < kTileB; h += kTileQ) {
            uint32_t nv = (l2 || cosm) ? __ldg(gnorm + tile_col0 + h + threadIdx.x) : 0u;
            if (cosm) nv = cos16_rnorm_bits(static_cast<int32_t>(nv));
            epi_sh.norm[0][h + threadIdx.x] = nv;
        }
        __syncthreads();
        epi.begin_tile(q, row_ok);
        for (int c = 0; c < kTileB / 32; ++c) {
            const int64_t col0 = tile_col0 + c * 32;
            int64_t rem = n_end - col0;
            const int nvalid = rem >= 32 ? 32 : (rem > 0 ? static_cast<int>(rem) : 0);
            uint32_t r[32];
            for (int j = 0; j < 32; ++j) {
                const int64_t col = (col0 + j < a.N) ? col0 + j : a.N - 1;
                AccT acc = AccT(0);
                const bool packed = packed_operands(KIND, a.d);
                for (int k = 0; k < a.d; ++k)
                    acc += load_elem<KIND>(a.A, operand_elem(packed, qc, k, a.d, kTileQ)) *
                           load_elem<KIND>(a.B, operand_elem(packed, col, k, a.d, kTileB));
                if (is_i8(KIND)) r[j] = static_cast<uint32_t>(acc);
                else r[j] = __float_as_uint(acc);
            }
            const int bslot = slot_tile * (kTileB / BURST) + c * (32 / BURST);
            epi.chunk(r, &epi_sh.norm[0][c * 32], col0, nvalid, bslot, c, cbase);
        }
        epi.end_tile(slot_tile * (kTileB / BURST));
    }
    epi.finish();
}

template <int KIND, int MODE, int BURST>
cudaError_t launch_one(const GemmLaunch& L, GemmArgs a, const CUtensorMap* mapA, const CUtensorMap* mapB,
                       cudaStream_t stream) {
    const int n_qb = (a.nq + kTileQ - 1) / kTileQ;
    const int64_t total = static_cast<int64_t>(n_qb) * a.n_tiles_sel;
    if (total <= 0) return cudaSuccess;
    if (a.tile_step < 1) a.tile_step = 1;
    if (L.simt) {
        const int grid = static_cast<int>(total < 4LL * L.num_sms ? total : 4LL * L.num_sms);
        dist_gemm_simt_kernel<KIND, MODE, BURST><<<grid, kTileQ, 0, stream>>>(a);
        return cudaGetLastError();
    }
    // shared-memory plan: resident query tile (if it is small) + as many ring stages as fit
    const int elem = is_i8(KIND) ? 1 : 2;
    const int nkc = (a.d * elem + kChunkBytes - 1) / kChunkBytes;
    a.packed = packed_operands(KIND, a.d) ? 1 : 0;
    a.a_resident = (a.packed || nkc <= kResidentMaxChunks) ? 1 : 0;
    const int a_bytes = a.packed ? ((kTileQ * a.d * 2 + 1023) & ~1023) : (a.a_resident ? nkc * kStageABytes : 0);
    const int stage_bytes = a.packed ? kTileB * a.d * 2 : (a.a_resident ? kStageBBytes : kStageBytes);
    int nst = a.packed ? 2 : (kGemmSmemBudget - 1024 - a_bytes) / stage_bytes;   // packed: one whole tile per parity
    if (nst > kMaxStages) nst = kMaxStages;
    nst &= ~1;                       // two sub-rings of equal depth
    if (nst < 2) return cudaErrorInvalidConfiguration;
    a.n_stages = nst;
    const int smem = a_bytes + nst * stage_bytes + 1024;
    if (smem > kGemmSmemBudget) return cudaErrorInvalidConfiguration;
    auto kern = dist_gemm_tc_kernel<KIND, MODE, BURST>;
    // per-device attribute; cheap enough to set on every launch
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kGemmSmemBudget);
    if (e != cudaSuccess) return e;
    const int grid = static_cast<int>(total < L.num_sms ? total : L.num_sms);
    // aligned ranges when every query block gets at least one CTA and the split stays balanced
    a.aligned_ranges = 0;
    if (n_qb <= grid && a.n_tiles_sel >= grid / n_qb) {
        const int nl_min = grid / n_qb;
        const double worst = static_cast<double>((a.n_tiles_sel + nl_min - 1) / nl_min);
        const double ideal = static_cast<double>(total) / grid;
        if (worst <= 1.06 * ideal + 1.0) a.aligned_ranges = 1;
    }
    // In a short run most threads never see a candidate, and the blocks they reserved would be what the
    // selection reads: 9 472 slots for the 150 candidates of one query against 100 003 rows.  The same holds for
    // one query block, whose rows every CTA has a share in.  us of a search on demand / ahead, fp32, d 128:
    //   one query block, k = 10:  4 items a CTA 87 / 103, 16 items 115 / 129, 64 items 203 / 220; k = 100: 106 / 114, 142 / 144, 228 / 236
    //   two, 32 items a CTA: k = 10 133 / 138, k = 100 170 / 160;  eight, 32 items: k = 10 151 / 148, k = 100 200 / 191
    //   eight, 211 items (1 M rows): k = 10 389 / 366, k = 100 510 / 493;  79, 34 items (16 384 rows), k = 64: 324 / 312
    //   below 16 items the two differ by less than 4 us from two query blocks on
    // With many candidates a thread it turns round there, too (three and more: 41 queries, 831 508 x 128 int8,
    // k = 113, 129 / 126).  The rows of a segmented base belong to a few CTAs each, however few the query blocks.
    const bool shared = n_qb == 1 && !a.seg_index && a.row_cands < 3LL * 4 * grid;   // (four threads a row and CTA)
    a.eager = total >= 16LL * grid && !shared ? 1 : 0;
    kern<<<grid, gemm_threads(KIND), smem, stream>>>(*mapA, *mapB, a);
    return cudaGetLastError();
}

template <int KIND>
cudaError_t launch_kind(const GemmLaunch& L, const GemmArgs& a, const CUtensorMap* mapA, const CUtensorMap* mapB,
                        cudaStream_t stream) {
    if (L.mode == kModeAppend) return launch_one<KIND, kModeAppend, 32>(L, a, mapA, mapB, stream);
    if (L.burst == 8) return launch_one<KIND, kModeBurstMin, 8>(L, a, mapA, mapB, stream);
    return launch_one<KIND, kModeBurstMin, 32>(L, a, mapA, mapB, stream);
}

}  // namespace

cudaError_t launch_dist_gemm(const GemmLaunch& L, const GemmArgs& a, const CUtensorMap* mapA, const CUtensorMap* mapB,
                             cudaStream_t stream) {
    switch (L.kind) {
        case kKindF16:
            return a.metric == kMetricIP ? launch_kind<kKindF16IP>(L, a, mapA, mapB, stream)
                                         : launch_kind<kKindF16L2>(L, a, mapA, mapB, stream);
        case kKindBF16: return launch_kind<kKindBF16>(L, a, mapA, mapB, stream);
        case kKindI8:
            return a.metric == kMetricCos  ? launch_kind<kKindI8Cos>(L, a, mapA, mapB, stream)
                   : a.metric == kMetricIP ? launch_kind<kKindI8IP>(L, a, mapA, mapB, stream)
                                           : launch_kind<kKindI8L2>(L, a, mapA, mapB, stream);
        default: return cudaErrorInvalidValue;
    }
}

int encode_operand_map(CUtensorMap* out, int kind, const void* base, int64_t rows, int d, int box_rows) {
    if (packed_operands(kind, d)) {   // read with contiguous copies: no tensor map
        std::memset(out, 0, sizeof(*out));
        return 0;
    }
    const int elem = kind == kKindI8 ? 1 : 2;
    const CUtensorMapDataType dt = kind == kKindI8    ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : kind == kKindBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return encode_rows_map(out, dt, elem, base, rows, d, box_rows);
}

namespace {

// dims, box: ndim extents in elements, innermost first; rows without gaps
int encode_map(CUtensorMap* out, CUtensorMapDataType type, int elem, const void* base, int ndim, const cuuint64_t* dims,
               const cuuint32_t* box, CUtensorMapSwizzle swizzle) {
    typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static EncodeFn encode = nullptr;
    if (!encode) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &qres) !=
                cudaSuccess || qres != cudaDriverEntryPointSuccess || !fn)
            return -1;
        encode = reinterpret_cast<EncodeFn>(fn);
    }
    cuuint64_t stride[2] = {dims[0] * elem, ndim > 2 ? dims[0] * dims[1] * elem : 0};
    cuuint32_t estride[3] = {1, 1, 1};
    CUresult r = encode(out, type, static_cast<cuuint32_t>(ndim), const_cast<void*>(base), dims, stride, box, estride,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : static_cast<int>(r);
}

}  // namespace

int encode_rows_map(CUtensorMap* out, CUtensorMapDataType type, int elem, const void* base, int64_t rows, int cols,
                    int box_rows) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(kChunkBytes / elem), static_cast<cuuint32_t>(box_rows)};
    return encode_map(out, type, elem, base, 2, dims, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

int encode_scale_map(CUtensorMap* out, const void* base, int64_t granules, int groups, int box_granules) {
    const cuuint64_t dims[3] = {128, static_cast<cuuint64_t>(groups), static_cast<cuuint64_t>(granules)};
    const cuuint32_t box[3] = {128, 2, static_cast<cuuint32_t>(box_granules)};
    return encode_map(out, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, base, 3, dims, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

}  // namespace b200
