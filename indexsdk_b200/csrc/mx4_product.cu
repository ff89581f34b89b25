// All scores of two sets of microscaled 4-bit rows, with tcgen05.mma kind::mxf4.
//
// out[i][j] is stored with j along a row, so the rows of b are the M side of the product (the 128 lanes of an
// accumulator) and the rows of a its N side (TN columns): a store instruction of a warp then covers 32 neighbouring
// outputs, whatever the output's stride is, and nothing passes through shared memory.  TN follows from m, so that few
// rows of a cost little shared memory and leave the stage ring to the rows of b, which is what is read most.
//   warp 0            : producer.  Per K chunk of 128 bytes (256 elements) 128 rows of b, TN rows of a and their
//                       scales, which lie in memory in the order the tensor core wants.
//   warp 1            : scales to TMEM (tcgen05.cp, a slot of columns per stage), up to four products of K = 64.
//   other warps       : epilogue.  Thread = (row of b, up to 64 rows of a).
// Two accumulators in turn.  Of 512 TMEM columns two of 256 would leave none for the scales: at TN = 256 they share
// 96 columns (0-255 and 160-415), and tile t + 1 starts once tile t's shared columns are in registers.
// Few tiles with a long K are split along K over a cluster, whose CTAs add their parts through shared memory in a
// fixed order.
#include "mx4_gemm.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <stdexcept>
#include <type_traits>

#include "cluster_limit.h"
#include "ptx_sm100.cuh"
#include "row_ops.cuh"
#include "smem_limit.h"

namespace b200 {
namespace {

constexpr int kLanes = 128;                     // rows of b in a tile
constexpr int kChunk = 128;                     // bytes of codes of a row in a stage
constexpr int kMaxStages = 10;
constexpr int kSmemMost = 224 * 1024;
constexpr int kMaxSplit = 8;

template <int TN>
struct Tile {
    static constexpr int kBBytes = kLanes * kChunk, kABytes = TN * kChunk;
    static constexpr int kGranulesA = TN > 128 ? 2 : 1;         // 128 rows of scales each
    static constexpr int kScaleBytes = 1024 * (1 + kGranulesA); // two groups of 128 elements
    static constexpr int kStage = kBBytes + kABytes + kScaleBytes;
    static constexpr int kFit = (kSmemMost - 1024) / kStage;
    static constexpr int kStages = kFit < kMaxStages ? kFit : kMaxStages;
    static constexpr int kSmem = kStages * kStage + 1024;
    static constexpr int kEpiWarps = TN > 64 ? TN / 16 : 4;
    static constexpr int kThreads = 64 + 32 * kEpiWarps;
    static constexpr int kCols = TN > 64 ? 64 : TN;              // columns of an epilogue thread
    static constexpr uint32_t kAcc1 = TN == 256 ? 160 : TN;      // second accumulator
    static constexpr uint32_t kSlotGroup = 4 + 4 * kGranulesA;   // TMEM columns of a group's scales
    static constexpr uint32_t kSlot = 2 * kSlotGroup;
    static constexpr uint32_t kScaleCol = TN == 256 ? 416 : 2 * TN;
    static_assert(kScaleCol + kStages * kSlot <= 512, "TMEM columns");
};

struct ProductArgs {
    const uint8_t* a_scales;
    const uint8_t* b_scales;
    int nb, ng;              // blocks of a row, groups of four
    int64_t m, n;
    void* out;
    int64_t ldo;
    int a_tiles, b_tiles;    // tiles of TN rows of a, of 128 rows of b
    int split;               // CTAs of a cluster that share a tile's K (1: none)
    int* err;                // where a wait that ran out is reported, or nullptr
    int b_first;             // mx4_few_kernel: first tile of b
    GemmArgs g;              // mx4_few_kernel as a pass of a search: thresholds and candidate lists
};

// What mx4_few_kernel does with its accumulators: scores to memory, or a search's keys at or below the row's threshold
// to its candidate list (inner product, L2).
enum FewEnd : int { kEndStore, kEndSearchIP, kEndSearchL2 };

__device__ __forceinline__ void next_tile(const ProductArgs& p, int& bt, int& at) {
    if (++at == p.a_tiles) {
        at = 0;
        ++bt;
    }
}

template <typename T>
__device__ __forceinline__ void store_one(T* o, float v) {
    if constexpr (std::is_same<T, float>::value) *o = v;
    else if constexpr (std::is_same<T, __half>::value) *o = __float2half_rn(v);
    else *o = __float2bfloat16_rn(v);
}

// COLS accumulator columns (rows of a) of this lane's output column j -> out; `cols` of them exist.
template <int COLS, typename T>
__device__ __forceinline__ void store_columns(const uint32_t (&r)[COLS], const ProductArgs& p, int64_t i0, int64_t j, int cols) {
    T* o = static_cast<T*>(p.out) + i0 * p.ldo + j;
    if (j >= p.n) return;
    if (cols >= COLS) {
#pragma unroll
        for (int c = 0; c < COLS; ++c, o += p.ldo) store_one(o, __uint_as_float(r[c]));
    } else {
#pragma unroll
        for (int c = 0; c < COLS; ++c, o += p.ldo)
            if (c < cols) store_one(o, __uint_as_float(r[c]));
    }
}

__device__ __forceinline__ void report_abort(const ProductArgs& p) {
    if (p.err && (threadIdx.x & 31) == 0) *reinterpret_cast<volatile int*>(p.err) = kDevErrPipelineTimeout;
}
// The end of a CTA: TMEM goes back; a split tile (bt, at), whose parts lie in shared memory as [TN][128], is added up.
template <int THREADS, int TN, typename T>
__device__ __forceinline__ void finish(const ProductArgs& p, bool owns_tmem, uint32_t tmem_base, volatile int& abort_flag, uint8_t* smem,
                                       int bt, int at, int part) {
    // After an abort, copies in flight get time to land before the shared memory is used again or released.
    __syncwarp();
    if (abort_flag) {
        report_abort(p);
        const long long t0 = clock64();
        while (clock64() - t0 < 4000000LL) { }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (owns_tmem) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem_base, 512);
    }
    if (p.split > 1) {
        if (abort_flag)   // (a copy that landed late may have overwritten the part)
            for (int e = threadIdx.x; e < TN * kLanes; e += THREADS) reinterpret_cast<uint32_t*>(smem)[e] = 0x7fffffffu;
        ptx::cluster_sync();
        // this CTA's share of the tile's columns: the parts in order of K
        const int c0 = TN * part / p.split, c1 = TN * (part + 1) / p.split;
        uint32_t peer[kMaxSplit];
#pragma unroll
        for (int r = 0; r < kMaxSplit; ++r) peer[r] = r < p.split ? ptx::cluster_addr(ptx::smem_u32(smem), r) : 0u;
        for (int e = c0 * kLanes + threadIdx.x; e < c1 * kLanes; e += THREADS) {
            float v = 0.f;
#pragma unroll
            for (int r = 0; r < kMaxSplit; ++r)
                if (r < p.split) v += ptx::cluster_load(peer[r] + e * 4);
            const int64_t i = static_cast<int64_t>(at) * TN + e / kLanes, j = static_cast<int64_t>(bt) * kLanes + e % kLanes;
            if (i < p.m && j < p.n) store_one(static_cast<T*>(p.out) + i * p.ldo + j, v);
        }
        ptx::cluster_sync();   // (the parts stay until everybody has read them)
    }
}

template <int TN, typename T>
__global__ void __launch_bounds__(Tile<TN>::kThreads, 1)
mx4_product_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_a,
                   const __grid_constant__ ProductArgs p) {
    using K = Tile<TN>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bar_full[K::kStages], bar_empty[K::kStages], bar_acc_full[2], bar_acc_free[2];
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int chunks = (p.ng + 1) / 2;
    // this CTA's tiles (in order of b, so that a tile's rows of b are read again from close by) and chunks of K
    const int64_t total = static_cast<int64_t>(p.a_tiles) * p.b_tiles;
    const int workers = gridDim.x / p.split, worker = blockIdx.x / p.split;
    const int64_t lo = total * worker / workers, hi = total * (worker + 1) / workers;
    const int part = p.split > 1 ? static_cast<int>(ptx::cluster_rank()) : 0;
    const int kc0 = chunks * part / p.split, kc1 = chunks * (part + 1) / p.split;
    if (threadIdx.x == 0) {
        for (int s = 0; s < K::kStages; ++s) {
            ptx::mbar_init(&bar_full[s], 1);
            ptx::mbar_init(&bar_empty[s], 1);
        }
        ptx::mbar_init(&bar_acc_full[0], 1);
        ptx::mbar_init(&bar_acc_full[1], 1);
        // TN = 256: one for both accumulators, told by the warps that hold columns which both have
        ptx::mbar_init(&bar_acc_free[0], TN == 256 ? K::kEpiWarps / 2 : K::kEpiWarps);
        ptx::mbar_init(&bar_acc_free[1], K::kEpiWarps);
        abort_flag = 0;
        ptx::mbar_fence_init();
        ptx::prefetch_tensormap(&map_a);
        ptx::prefetch_tensormap(&map_b);
    }
    if (warp == 1) {
        ptx::tmem_alloc(&tmem_base_slot, 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem_base = tmem_base_slot;

    if (warp == 0) {
        const bool leader = ptx::elect_one();
        uint32_t s = 0, ph = 0;
        bool ok = true;
        const int64_t a_granules = (p.m + 127) / 128;
        int bt = static_cast<int>(lo / p.a_tiles), at = static_cast<int>(lo % p.a_tiles);
        for (int64_t i = lo; i < hi && ok; ++i, next_tile(p, bt, at)) {
            const bool second = K::kGranulesA > 1 && 2 * at + 1 < a_granules;   // the upper 128 rows of a exist
            const uint8_t* sb = p.b_scales + static_cast<int64_t>(bt) * p.ng * 512;
            const uint8_t* sa = p.a_scales + static_cast<int64_t>(K::kGranulesA * at) * p.ng * 512;
            for (int kc = kc0; kc < kc1; ++kc) {
                if (!ptx::mbar_wait_warp(&bar_empty[s], ph ^ 1u, &abort_flag)) { ok = false; break; }
                if (leader) {
                    uint8_t* st = smem + s * K::kStage;
                    uint8_t* sf = st + K::kBBytes + K::kABytes;
                    const uint32_t bytes = min(2, p.ng - 2 * kc) * 512u;
                    ptx::mbar_expect_tx(&bar_full[s], K::kBBytes + K::kABytes + bytes * (second ? 3u : 2u));
                    ptx::tma_load_2d(st, &map_b, &bar_full[s], kc * kChunk, bt * kLanes);
                    ptx::tma_load_2d(st + K::kBBytes, &map_a, &bar_full[s], kc * kChunk, at * TN);
                    ptx::bulk_load_1d(sf, sb + kc * 1024, bytes, &bar_full[s]);
                    ptx::bulk_load_1d(sf + 1024, sa + kc * 1024, bytes, &bar_full[s]);
                    if (second) ptx::bulk_load_1d(sf + 2048, sa + p.ng * 512 + kc * 1024, bytes, &bar_full[s]);
                }
                __syncwarp();
                if (++s == K::kStages) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 1) {
        constexpr uint32_t kIdesc0 = ptx::umma_idesc_mxf4(kLanes, TN, 0), kIdesc2 = ptx::umma_idesc_mxf4(kLanes, TN, 2);
        const uint64_t desc_hi = ptx::umma_desc_k_sw128(0);
        const uint64_t sf_hi = ptx::umma_desc_k_plain(0, 128u, 128u);
        const uint32_t ring_lo = (ptx::smem_u32(smem) & 0x3FFFFu) >> 4;
        const bool leader = ptx::elect_one();
        uint32_t s = 0, ph = 0, t = 0;
        bool ok = true;
        for (int64_t i = lo; i < hi && ok; ++i, ++t) {
            // TN = 256: tile t - 1's shared columns (and with them all of tile t - 2); else tile t - 2
            if (TN == 256 ? t >= 1 && !ptx::mbar_wait_warp(&bar_acc_free[0], (t - 1) & 1u, &abort_flag)
                          : t >= 2 && !ptx::mbar_wait_warp(&bar_acc_free[t & 1u], ((t >> 1) - 1) & 1u, &abort_flag)) { ok = false; break; }
            const uint32_t tacc = tmem_base + (t & 1u ? K::kAcc1 : 0u);
            for (int kc = kc0; kc < kc1; ++kc) {
                if (!ptx::mbar_wait_warp(&bar_full[s], ph, &abort_flag)) { ok = false; break; }
                ptx::tc_fence_after();
                const uint32_t st = ring_lo + s * (K::kStage >> 4);
                const uint32_t sf_lo = st + ((K::kBBytes + K::kABytes) >> 4);
                const uint32_t slot = tmem_base + K::kScaleCol + s * K::kSlot;
                const int steps = min(4, (p.nb - 8 * kc + 1) / 2);   // 64 elements each
                if (leader) {
#pragma unroll
                    for (int g = 0; g < 2; ++g)
                        if (2 * g < steps)
#pragma unroll
                            for (int h = 0; h < 1 + K::kGranulesA; ++h)
                                ptx::tmem_cp_scales(slot + g * K::kSlotGroup + 4 * h, sf_hi | static_cast<uint64_t>(sf_lo + 64 * h + 32 * g));
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) {
                        const uint32_t col = slot + (ks >> 1) * K::kSlotGroup;
                        if (ks < steps)
                            ptx::umma_mxf4(tacc, desc_hi | static_cast<uint64_t>(st + ks * 2),
                                           desc_hi | static_cast<uint64_t>(st + (K::kBBytes >> 4) + ks * 2),
                                           (ks & 1) ? kIdesc2 : kIdesc0, col, col + 4, (kc > kc0 || ks) ? 1u : 0u);
                    }
                    ptx::umma_commit(&bar_empty[s]);
                    if (kc + 1 == kc1) ptx::umma_commit(&bar_acc_full[t & 1u]);
                }
                __syncwarp();
                if (++s == K::kStages) { s = 0; ph ^= 1u; }
            }
        }
    } else {
        const int quarter = warp & 3, group = (warp - 2) >> 2;   // TMEM lanes, columns of this warp
        uint32_t t = 0;
        bool ok = true;
        float* parts = reinterpret_cast<float*>(smem);           // split: [TN][128]
        int bt = static_cast<int>(lo / p.a_tiles), at = static_cast<int>(lo % p.a_tiles);
        for (int64_t i = lo; i < hi; ++i, ++t, next_tile(p, bt, at)) {
            const int64_t j = static_cast<int64_t>(bt) * kLanes + quarter * 32 + lane;
            const int64_t i0 = static_cast<int64_t>(at) * TN + group * K::kCols;
            const uint32_t ab = t & 1u;
            uint32_t r[K::kCols];
            if (ok) ok = ptx::mbar_wait_warp(&bar_acc_full[ab], (t >> 1) & 1u, &abort_flag);
            if (ok) {
                ptx::tc_fence_after();
                const uint32_t tacc = tmem_base + (ab ? K::kAcc1 : 0u) + group * K::kCols + (static_cast<uint32_t>(quarter * 32) << 16);
                if constexpr (K::kCols >= 32) {
#pragma unroll
                    for (int c = 0; c < K::kCols; c += 32) ptx::tmem_ld_32x32(tacc + c, *reinterpret_cast<uint32_t(*)[32]>(r + c));
#pragma unroll
                    for (int c = 0; c < K::kCols; c += 32) ptx::tmem_ld_wait(*reinterpret_cast<uint32_t(*)[32]>(r + c));
                } else {
                    ptx::tmem_ld_32x16(tacc, r);
                    ptx::tmem_ld_wait(*reinterpret_cast<uint32_t(*)[16]>(r));
                }
                ptx::tc_fence_before();
                __syncwarp();
                // TN = 256: shared are 160 .. 255 of accumulator 0, 0 .. 95 of accumulator 1
                if (lane == 0 && (TN != 256 || (ab ? group < 2 : group >= 2))) ptx::mbar_arrive(&bar_acc_free[TN == 256 ? 0 : ab]);
            } else {
                // whether somebody reads an error word or not: results that could not be computed are no numbers
#pragma unroll
                for (int c = 0; c < K::kCols; ++c) r[c] = 0x7fffffffu;
            }
            if (p.split > 1) {   // (one tile)  every load of the ring has been consumed: it holds the part now
#pragma unroll
                for (int c = 0; c < K::kCols; ++c) parts[(group * K::kCols + c) * kLanes + quarter * 32 + lane] = __uint_as_float(r[c]);
                continue;
            }
            store_columns<K::kCols, T>(r, p, i0, j, static_cast<int>(min(p.m - i0, static_cast<int64_t>(K::kCols))));
        }
    }

    finish<K::kThreads, TN, T>(p, warp == 1, tmem_base, abort_flag, smem, static_cast<int>(lo / p.a_tiles), static_cast<int>(lo % p.a_tiles), part);
}

// ---------------------------------------------------------------------------------------
// Few rows of a (up to 128): they and their scales stay in shared memory and in TMEM, and only rows of b travel through
// the ring.  (All CTAs reading the same few rows of a again for every tile queue up at the few L2 lines that hold
// them.)  A tile is little work for anybody, so what counts is how many of the hand-offs between the roles overlap:
// two producers and two MMA warps take even and odd tiles, each with half of the ring, and four groups of epilogue
// warps have four accumulators (two of 128 columns, in halves).
// ---------------------------------------------------------------------------------------
constexpr int kFewStage = kLanes * kChunk + 1024;
constexpr int kFewMaxStages = 12;
constexpr int kFewGroups = 4;
constexpr int kFewThreads = 128 + 128 * kFewGroups;
template <int TN>
struct Few {
    static constexpr int kAcc = TN == 128 ? 2 : 4;              // accumulators
    static constexpr int kCols = TN == 128 ? 64 : TN;           // columns of an epilogue thread
    static constexpr int kMaxChunks = TN >= 64 ? 16 : 32;       // of a: 8 TMEM columns of scales each
    static_assert(kAcc * TN + 8 * kMaxChunks + 8 * kFewMaxStages <= 512, "TMEM columns");
    static constexpr int resident_bytes(int chunks) { return chunks * (TN * kChunk + 1024); }
};

// A CTA's candidates wait in shared memory, kNearAll / TN for each query, and go to the queries' lists at the end
// (or, when there are more, at once).
constexpr int kNearAll = 2048;
template <int TN>
struct NearList {
    enum : int { kSlots = kNearAll / TN };
    uint32_t taken[TN];      // slots reserved, may pass kSlots
    uint32_t base[TN];
    float tau[TN];
};
// A warp's 32 rows of b against COLS queries, accumulators at tacc, values in r: candidates into `list`.
// Rows are lanes here, so a row's norm is one register and a hit's slots are taken for all lanes that have the same
// query in one atomic, 32 queries' at a time.  In shared memory, since most tiles of a warp have a candidate and
// would wait for the global counters (64 queries, 1 M x 128, inner product: the passes 58 us with global ones).
template <bool L2, int TN, int COLS>
__device__ __forceinline__ void take_candidates(const uint32_t (&r)[COLS], const GemmArgs& a, NearList<TN>& near, uint64_t* list, int first,
                                                uint32_t tacc, int64_t j, float norm) {
    constexpr uint32_t kSlots = NearList<TN>::kSlots;
    const float* tau = near.tau + first;
    uint32_t pass[2] = {0u, 0u};
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
        const float v = __uint_as_float(r[c]);
        if ((L2 ? fmaf(-2.f, v, norm) : -v) <= tau[c]) pass[c >> 5] |= 1u << (c & 31);   // (NaN is not)
    }
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int h = 0; h < (COLS + 31) / 32; ++h) {
        uint32_t mine = j < a.N ? pass[h] : 0u;
        uint32_t who = 0u;   // lanes with a candidate of query 32 h + lane
        for (uint32_t any = __reduce_or_sync(0xFFFFFFFFu, mine); any; any &= any - 1) {
            const int c = __ffs(any) - 1;
            if (a.qmask && (mine >> c & 1u) &&
                !(__ldg(a.qmask + static_cast<int64_t>(first + 32 * h + c) * a.qmask_stride + (j >> 5)) >> (j & 31) & 1u))
                mine &= ~(1u << c);
            const uint32_t w = __ballot_sync(0xFFFFFFFFu, mine >> c & 1u);
            if (lane == c) who = w;
        }
        uint32_t slots = 0;   // of the list in shared memory; from kSlots on: of the query's own
        if (who) {
            const uint32_t more = __popc(who);
            slots = atomicAdd(&near.taken[first + 32 * h + lane], more);
            if (slots + more > kSlots) slots = kSlots + atomicAdd(a.counts + first + 32 * h + lane, more);
        }
        for (uint32_t any = __ballot_sync(0xFFFFFFFFu, who != 0u); any; any &= any - 1) {
            const int c = __ffs(any) - 1;
            const float v = __uint_as_float(ptx::tmem_ld_32x1(tacc + 32 * h + c));
            const uint32_t slot = __shfl_sync(0xFFFFFFFFu, slots, c) + __popc(__shfl_sync(0xFFFFFFFFu, who, c) & ((1u << lane) - 1u));
            const float key = L2 ? fmaf(-2.f, v, norm) : -v;
            if (mine >> c & 1u) {
                const uint64_t cand = pack_cand(float_to_ord(key), static_cast<uint32_t>(j));
                const int q = first + 32 * h + c;
                if (slot < kSlots) list[q * kSlots + slot] = cand;
                else if (slot - kSlots < a.cap) a.cand[static_cast<int64_t>(q) * a.cap + slot - kSlots] = cand;
            }
        }
    }
}

template <int TN, typename T, int END = kEndStore>
__global__ void __launch_bounds__(kFewThreads, 1)
mx4_few_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_a,
               const __grid_constant__ ProductArgs p, const int half_stages) {
    using K = Few<TN>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bar_full[kFewMaxStages], bar_empty[kFewMaxStages], bar_acc_full[K::kAcc], bar_acc_free[K::kAcc], bar_a, bar_a_scales;
    __shared__ uint32_t tmem_base_slot;
    __shared__ __align__(16) NearList<END == kEndStore ? 1 : TN> near;
    __shared__ int abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int chunks = (p.ng + 1) / 2;
    const int workers = gridDim.x / p.split, worker = blockIdx.x / p.split;
    const int lo = p.b_first + static_cast<int>(static_cast<int64_t>(p.b_tiles) * worker / workers);
    const int hi = p.b_first + static_cast<int>(static_cast<int64_t>(p.b_tiles) * (worker + 1) / workers);
    const int part = p.split > 1 ? static_cast<int>(ptx::cluster_rank()) : 0;
    const int kc0 = chunks * part / p.split, kc1 = chunks * (part + 1) / p.split, nkc = kc1 - kc0;
    uint8_t* a_codes = smem;                              // [nkc][TN][128 B]
    uint8_t* a_scales = smem + nkc * TN * kChunk;         // [nkc][1 KB]
    uint8_t* ring = a_scales + nkc * 1024;
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2 * half_stages; ++s) {
            ptx::mbar_init(&bar_full[s], 1);
            ptx::mbar_init(&bar_empty[s], 1);
        }
        for (int b = 0; b < K::kAcc; ++b) {
            ptx::mbar_init(&bar_acc_full[b], 1);
            ptx::mbar_init(&bar_acc_free[b], 4 * kFewGroups / K::kAcc);
        }
        ptx::mbar_init(&bar_a, 1);
        ptx::mbar_init(&bar_a_scales, 1);
        abort_flag = 0;
        ptx::mbar_fence_init();
        ptx::prefetch_tensormap(&map_a);
        ptx::prefetch_tensormap(&map_b);
    }
    uint64_t* list = reinterpret_cast<uint64_t*>(ring + 2 * half_stages * kFewStage);   // search only
    if constexpr (END != kEndStore) {
        if (threadIdx.x < TN) {   // (columns behind the last query let nothing pass)
            near.tau[threadIdx.x] = threadIdx.x < p.m ? ord_to_float(__ldg(p.g.tau + threadIdx.x)) : __int_as_float(0x7fffffff);
            near.taken[threadIdx.x] = 0;
        }
        for (int e = threadIdx.x; e < kNearAll; e += kFewThreads) list[e] = kCandInvalid;   // (a reservation past the end leaves some)
    }
    if (warp == 2) {
        ptx::tmem_alloc(&tmem_base_slot, 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem_base = tmem_base_slot;
    const uint32_t col_a = tmem_base + K::kAcc * TN, col_b = col_a + 8 * nkc;
    const uint32_t pipe = warp & 1u;                      // of producers and MMA warps
    const uint32_t s0 = pipe * half_stages;               // first stage of this pipe's half of the ring

    if (warp < 2) {
        const bool leader = ptx::elect_one();
        const uint32_t a_sf = static_cast<uint32_t>(min(p.ng, 2 * kc1) - 2 * kc0) * 512u;
        if (leader && pipe == 0) {
            ptx::mbar_expect_tx(&bar_a, static_cast<uint32_t>(nkc) * TN * kChunk + a_sf);
            for (int kc = kc0; kc < kc1; ++kc) ptx::tma_load_2d(a_codes + (kc - kc0) * TN * kChunk, &map_a, &bar_a, kc * kChunk, 0);
            ptx::bulk_load_1d(a_scales, p.a_scales + kc0 * 1024, a_sf, &bar_a);
        }
        __syncwarp();
        uint32_t s = 0, ph = 0;
        bool ok = true;
        for (int bt = lo + pipe; bt < hi && ok; bt += 2) {
            const uint8_t* sb = p.b_scales + static_cast<int64_t>(bt) * p.ng * 512;
            for (int kc = kc0; kc < kc1; ++kc) {
                if (!ptx::mbar_wait_warp(&bar_empty[s0 + s], ph ^ 1u, &abort_flag)) { ok = false; break; }
                if (leader) {
                    uint8_t* st = ring + (s0 + s) * kFewStage;
                    uint64_t* full = &bar_full[s0 + s];
                    const uint32_t bytes = min(2, p.ng - 2 * kc) * 512u;
                    ptx::mbar_expect_tx(full, kLanes * kChunk + bytes);
                    ptx::tma_load_2d(st, &map_b, full, kc * kChunk, bt * kLanes);
                    ptx::bulk_load_1d(st + kLanes * kChunk, sb + kc * 1024, bytes, full);
                }
                __syncwarp();
                if (++s == static_cast<uint32_t>(half_stages)) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp < 4) {
        constexpr uint32_t kIdesc0 = ptx::umma_idesc_mxf4(kLanes, TN, 0), kIdesc2 = ptx::umma_idesc_mxf4(kLanes, TN, 2);
        const uint64_t desc_hi = ptx::umma_desc_k_sw128(0);
        const uint64_t sf_hi = ptx::umma_desc_k_plain(0, 128u, 128u);
        const uint32_t a_lo = (ptx::smem_u32(a_codes) & 0x3FFFFu) >> 4, ring_lo = (ptx::smem_u32(ring) & 0x3FFFFu) >> 4;
        const uint32_t a_sf_lo = (ptx::smem_u32(a_scales) & 0x3FFFFu) >> 4;
        const bool leader = ptx::elect_one();
        uint32_t s = 0, ph = 0, u = 0;                    // u: tiles of this pipe so far
        bool ok = ptx::mbar_wait_warp(&bar_a, 0u, &abort_flag);
        if (pipe == 0) {
            if (ok && leader) {
                for (int g = 0; g < min(p.ng, 2 * kc1) - 2 * kc0; ++g) ptx::tmem_cp_scales(col_a + 4 * g, sf_hi | static_cast<uint64_t>(a_sf_lo + 32 * g));
                ptx::umma_commit(&bar_a_scales);
            }
            __syncwarp();
        } else if (ok) {   // (copies are in order with the products of the warp that made them only)
            ok = ptx::mbar_wait_warp(&bar_a_scales, 0u, &abort_flag);
            ptx::tc_fence_after();
        }
        for (int bt = lo + pipe; bt < hi && ok; bt += 2, ++u) {
            const uint32_t ab = K::kAcc == 4 ? pipe + 2 * (u & 1u) : pipe, use = K::kAcc == 4 ? u >> 1 : u;   // use: of this accumulator
            if (use && !ptx::mbar_wait_warp(&bar_acc_free[ab], (use - 1) & 1u, &abort_flag)) { ok = false; break; }
            const uint32_t tacc = tmem_base + ab * TN;
            for (int kc = kc0; kc < kc1; ++kc) {
                if (!ptx::mbar_wait_warp(&bar_full[s0 + s], ph, &abort_flag)) { ok = false; break; }
                ptx::tc_fence_after();
                const uint32_t st = ring_lo + (s0 + s) * (kFewStage >> 4), slot = col_b + (s0 + s) * 8;
                const uint32_t at = a_lo + (kc - kc0) * (TN * kChunk >> 4), sa = col_a + (kc - kc0) * 8;
                const int steps = min(4, (p.nb - 8 * kc + 1) / 2);   // 64 elements each
                if (leader) {
                    ptx::tmem_cp_scales(slot, sf_hi | static_cast<uint64_t>(st + (kLanes * kChunk >> 4)));
                    if (steps > 2) ptx::tmem_cp_scales(slot + 4, sf_hi | static_cast<uint64_t>(st + (kLanes * kChunk >> 4) + 32));
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        if (ks < steps)
                            ptx::umma_mxf4(tacc, desc_hi | static_cast<uint64_t>(st + ks * 2), desc_hi | static_cast<uint64_t>(at + ks * 2),
                                           (ks & 1) ? kIdesc2 : kIdesc0, slot + (ks >> 1) * 4, sa + (ks >> 1) * 4, (kc > kc0 || ks) ? 1u : 0u);
                    ptx::umma_commit(&bar_empty[s0 + s]);
                    if (kc + 1 == kc1) ptx::umma_commit(&bar_acc_full[ab]);
                }
                __syncwarp();
                if (++s == static_cast<uint32_t>(half_stages)) { s = 0; ph ^= 1u; }
            }
        }
    } else {
        // group g: accumulator g % kAcc, columns from (g / kAcc) * kCols on; its tiles are kAcc apart
        const int quarter = warp & 3, group = (warp - 4) >> 2, ab = group % K::kAcc, first = group / K::kAcc * K::kCols;
        bool ok = true;
        float* parts = reinterpret_cast<float*>(smem);           // split: [TN][128]
        uint32_t turn = 0;
        // (a tile's norms are on their way while the tile before it is worked on)
        auto norm_of = [&](int bt) {
            return END == kEndSearchL2 && bt < hi ? __ldg(static_cast<const float*>(p.g.bnorm) + static_cast<int64_t>(bt) * kLanes + quarter * 32 + lane) : 0.f;
        };
        float norm = 0.f, next_norm = norm_of(lo + ab);
        for (int bt = lo + ab; bt < hi; bt += K::kAcc, ++turn) {
            const int64_t j = static_cast<int64_t>(bt) * kLanes + quarter * 32 + lane;
            uint32_t r[K::kCols];
            norm = next_norm;
            next_norm = norm_of(bt + K::kAcc);
            if (ok) ok = ptx::mbar_wait_warp(&bar_acc_full[ab], turn & 1u, &abort_flag);
            if (END != kEndStore && !ok) break;   // (the host sees the error word)
            if (ok) {
                ptx::tc_fence_after();
                const uint32_t tacc = tmem_base + ab * TN + first + (static_cast<uint32_t>(quarter * 32) << 16);
                if constexpr (K::kCols >= 32) {
#pragma unroll
                    for (int c = 0; c < K::kCols; c += 32) ptx::tmem_ld_32x32(tacc + c, *reinterpret_cast<uint32_t(*)[32]>(r + c));
#pragma unroll
                    for (int c = 0; c < K::kCols; c += 32) ptx::tmem_ld_wait(*reinterpret_cast<uint32_t(*)[32]>(r + c));
                } else {
                    ptx::tmem_ld_32x16(tacc, r);
                    ptx::tmem_ld_wait(*reinterpret_cast<uint32_t(*)[16]>(r));
                }
                if constexpr (END != kEndStore)
                    take_candidates<END == kEndSearchL2, TN>(r, p.g, near, list, first, tacc, j, norm);
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&bar_acc_free[ab]);
                if (END != kEndStore) continue;
            } else {
                // (as above: no numbers)
#pragma unroll
                for (int c = 0; c < K::kCols; ++c) r[c] = 0x7fffffffu;
            }
            if (p.split > 1) {   // (one tile: its commit says that every copy and product has read what lies there)
#pragma unroll
                for (int c = 0; c < K::kCols; ++c) parts[(first + c) * kLanes + quarter * 32 + lane] = __uint_as_float(r[c]);
                continue;
            }
            store_columns<K::kCols, T>(r, p, first, j, static_cast<int>(p.m) - first);
        }
    }

    finish<kFewThreads, TN, T>(p, warp == 2, tmem_base, abort_flag, smem, lo, 0, part);
    if constexpr (END != kEndStore) {   // (finish has brought all threads together)
        constexpr int kSlots = NearList<TN>::kSlots;
        if (threadIdx.x < TN && near.taken[threadIdx.x])
            near.base[threadIdx.x] = atomicAdd(p.g.counts + threadIdx.x, min(near.taken[threadIdx.x], static_cast<uint32_t>(kSlots)));
        __syncthreads();
        for (int e = threadIdx.x; e < kNearAll; e += kFewThreads) {
            const uint32_t q = e / kSlots, i = e % kSlots;
            if (i >= near.taken[q]) continue;
            const uint32_t slot = near.base[q] + i;
            if (slot < p.g.cap) p.g.cand[static_cast<int64_t>(q) * p.g.cap + slot] = list[e];
        }
        if (threadIdx.x == 0 && abort_flag) atomicOr(p.g.err, kDevErrPipelineTimeout);
    }
}

template <int TN, typename T>
void launch(const Mx4ProductArgs& q, int num_sms, cudaStream_t st) {
    using K = Tile<TN>;
    CUtensorMap map_a, map_b;
    if (encode_mx4_map(&map_a, q.a_codes, q.m, q.d, TN) != 0 || encode_mx4_map(&map_b, q.b_codes, q.n, q.d, kLanes) != 0)
        throw std::runtime_error("cuTensorMapEncodeTiled failed for the rows of a product");
    ProductArgs p{};
    p.a_scales = q.a_scales;
    p.b_scales = q.b_scales;
    p.nb = mx4_blocks(q.d);
    p.ng = mx4_groups(q.d);
    p.m = q.m;
    p.n = q.n;
    p.out = q.out;
    p.ldo = q.ldo;
    p.err = q.err;
    p.a_tiles = div_up(q.m, TN);
    p.b_tiles = div_up(q.n, kLanes);
    const int64_t total = static_cast<int64_t>(p.a_tiles) * p.b_tiles;
    p.split = 1;
    const int chunks = (p.ng + 1) / 2;
    while (p.split < kMaxSplit && total * p.split * 2 <= num_sms && p.split * 2 <= chunks) p.split *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.split > 1 ? total * p.split : std::min<int64_t>(total, num_sms)));
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = static_cast<unsigned>(p.split);
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = p.split > 1 ? 1 : 0;
    if constexpr (TN <= 128) {
        const int mine = (chunks + p.split - 1) / p.split;   // chunks of K of a CTA
        const int half = std::min(kFewMaxStages, (kSmemMost - 1024 - Few<TN>::resident_bytes(mine)) / kFewStage) / 2;
        if (mine <= Few<TN>::kMaxChunks && half >= 3) {   // (64 x 16 384 x 4096 with four stages: 15.7 us; through the ring 12.2)
            auto kern = mx4_few_kernel<TN, T>;
            B200_CUDA_CHECK(allow_max_smem(kern));
            cfg.blockDim = dim3(kFewThreads);
            cfg.dynamicSmemBytes = 1024 + Few<TN>::resident_bytes(mine) + 2 * half * kFewStage;
            B200_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, map_b, map_a, p, half));
            return;
        }
    }
    auto kern = mx4_product_kernel<TN, T>;
    B200_CUDA_CHECK(allow_max_smem(kern));
    cfg.blockDim = dim3(K::kThreads);
    cfg.dynamicSmemBytes = K::kSmem;
    B200_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, map_b, map_a, p));
}

// ---------------------------------------------------------------------------------------
// Many rows of both: a pair of CTAs makes 256 x 256 tiles, 128 rows of b each, and each loads only half of a's rows --
// 32 KB of codes per 256 elements of K instead of 48, which is what a single CTA's ring waits for.  CTA 0 issues for
// both; its barriers count both CTAs' copies, and its commits arrive in both.  TMEM as above, six stages of 24 columns
// of scales: the accumulators share 144 columns (0-255 and 112-367).
// ---------------------------------------------------------------------------------------
constexpr int kPairStages = 6;
constexpr int kPairHalf = 128 * kChunk;                                   // 16 KB: this CTA's rows of b, or of a
constexpr int kPairStage = 2 * kPairHalf + 3 * 1024;                      // and scales: b's own 128 rows, all 256 of a
constexpr int kPairSmem = kPairStages * kPairStage + 1024;
constexpr int kPairThreads = 128 + 32 * 16;
constexpr uint32_t kPairAcc1 = 112, kPairScaleCol = 368;

template <typename T>
__global__ void __launch_bounds__(kPairThreads, 1) __cluster_dims__(2, 1, 1)
mx4_pair_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_a,
                const __grid_constant__ CUtensorMap map_sb, const __grid_constant__ CUtensorMap map_sa,
                const __grid_constant__ ProductArgs p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bar_full[kPairStages], bar_empty[kPairStages], bar_acc_full[2], bar_acc_free;
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = ptx::cluster_rank();
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int chunks = (p.ng + 1) / 2;
    const int64_t total = static_cast<int64_t>(p.a_tiles) * p.b_tiles;     // b_tiles: of 256 rows
    const int workers = gridDim.x / 2, worker = blockIdx.x / 2;
    const int64_t lo = total * worker / workers, hi = total * (worker + 1) / workers;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairStages; ++s) {
            ptx::mbar_init(&bar_full[s], 1);
            ptx::mbar_init(&bar_empty[s], 1);
        }
        ptx::mbar_init(&bar_acc_full[0], 1);
        ptx::mbar_init(&bar_acc_full[1], 1);
        ptx::mbar_init(&bar_acc_free, 24);   // CTA 0's: twelve warps of each CTA
        abort_flag = 0;
        ptx::mbar_fence_init();
        ptx::prefetch_tensormap(&map_a);
        ptx::prefetch_tensormap(&map_b);
        ptx::prefetch_tensormap(&map_sa);
        ptx::prefetch_tensormap(&map_sb);
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(&tmem_base_slot, 512);
        ptx::tmem_relinquish_pair();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_sync();   // (the other CTA's barriers exist)
    ptx::tc_fence_after();
    const uint32_t tmem_base = tmem_base_slot;

    if (warp == 0 || warp == 2) {   // codes; scales
        const bool leader = ptx::elect_one();
        uint32_t s = 0, ph = 0;
        bool ok = true;
        int bt = static_cast<int>(lo / p.a_tiles), at = static_cast<int>(lo % p.a_tiles);
        for (int64_t i = lo; i < hi && ok; ++i, next_tile(p, bt, at)) {
            for (int kc = 0; kc < chunks; ++kc) {
                if (!ptx::mbar_wait_warp(&bar_empty[s], ph ^ 1u, &abort_flag)) { ok = false; break; }
                if (leader) {
                    uint8_t* st = smem + s * kPairStage;
                    const uint32_t full = ptx::cluster_addr(ptx::smem_u32(&bar_full[s]), 0);
                    if (warp == 0) {
                        if (rank == 0) ptx::mbar_expect_tx(&bar_full[s], 2 * kPairStage);
                        ptx::tma_load_2d_pair(st, &map_b, full, kc * kChunk, bt * 256 + static_cast<int>(rank) * 128);
                        ptx::tma_load_2d_pair(st + kPairHalf, &map_a, full, kc * kChunk, at * 256 + static_cast<int>(rank) * 128);
                    } else {   // two groups of 128 rows; zeros behind a row's last group and behind the last rows
                        ptx::tma_load_3d_pair(st + 2 * kPairHalf, &map_sb, full, 0, 2 * kc, bt * 2 + static_cast<int>(rank));
                        ptx::tma_load_3d_pair(st + 2 * kPairHalf + 1024, &map_sa, full, 0, 2 * kc, at * 2);
                    }
                }
                __syncwarp();
                if (++s == kPairStages) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            constexpr uint32_t kIdesc0 = ptx::umma_idesc_mxf4(256, 256, 0), kIdesc2 = ptx::umma_idesc_mxf4(256, 256, 2);
            const uint64_t desc_hi = ptx::umma_desc_k_sw128(0);
            const uint64_t sf_hi = ptx::umma_desc_k_plain(0, 128u, 128u);
            const uint32_t ring_lo = (ptx::smem_u32(smem) & 0x3FFFFu) >> 4;
            const bool leader = ptx::elect_one();
            uint32_t s = 0, ph = 0, t = 0;
            bool ok = true;
            for (int64_t i = lo; i < hi && ok; ++i, ++t) {
                // both CTAs have tile t - 1's shared columns in registers (and with them all of tile t - 2)
                if (t && !ptx::mbar_wait_warp(&bar_acc_free, (t - 1u) & 1u, &abort_flag)) { ok = false; break; }
                ptx::tc_fence_after();
                const uint32_t tacc = tmem_base + (t & 1u ? kPairAcc1 : 0u);
                for (int kc = 0; kc < chunks; ++kc) {
                    if (!ptx::mbar_wait_warp(&bar_full[s], ph, &abort_flag)) { ok = false; break; }
                    ptx::tc_fence_after();
                    const uint32_t st = ring_lo + s * (kPairStage >> 4), sf_lo = st + (2 * kPairHalf >> 4);
                    const uint32_t slot = tmem_base + kPairScaleCol + s * 24;
                    const int steps = min(4, (p.nb - 8 * kc + 1) / 2);   // 64 elements each
                    if (leader) {
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks) {
                            if (ks >= steps) continue;
                            const uint32_t col = slot + (ks >> 1) * 12;
                            if ((ks & 1) == 0)
#pragma unroll
                                for (int h = 0; h < 3; ++h)
                                    ptx::tmem_cp_scales_pair(col + 4 * h, sf_hi | static_cast<uint64_t>(sf_lo + 64 * h + 16 * ks));
                            ptx::umma_mxf4_pair(tacc, desc_hi | static_cast<uint64_t>(st + ks * 2),
                                                desc_hi | static_cast<uint64_t>(st + (kPairHalf >> 4) + ks * 2),
                                                (ks & 1) ? kIdesc2 : kIdesc0, col, col + 4, (kc | ks) ? 1u : 0u);
                        }
                        ptx::umma_commit_pair(&bar_empty[s]);
                        if (kc + 1 == chunks) ptx::umma_commit_pair(&bar_acc_full[t & 1u]);
                    }
                    __syncwarp();
                    if (++s == kPairStages) { s = 0; ph ^= 1u; }
                }
            }
        }
    } else if (warp >= 4) {
        const int quarter = warp & 3, group = (warp - 4) >> 2;   // TMEM lanes, columns of this warp
        const uint32_t free_at = ptx::cluster_addr(ptx::smem_u32(&bar_acc_free), 0);
        uint32_t t = 0;
        bool ok = true;
        int bt = static_cast<int>(lo / p.a_tiles), at = static_cast<int>(lo % p.a_tiles);
        for (int64_t i = lo; i < hi; ++i, ++t, next_tile(p, bt, at)) {
            const int64_t j = static_cast<int64_t>(bt) * 256 + rank * 128 + quarter * 32 + lane;
            const int64_t i0 = static_cast<int64_t>(at) * 256 + group * 64;
            const uint32_t ab = t & 1u;
            uint32_t r[64];
            if (ok) ok = ptx::mbar_wait_warp(&bar_acc_full[ab], (t >> 1) & 1u, &abort_flag);
            if (ok) {
                ptx::tc_fence_after();
                const uint32_t tacc = tmem_base + (ab ? kPairAcc1 : 0u) + group * 64 + (static_cast<uint32_t>(quarter * 32) << 16);
                ptx::tmem_ld_32x32(tacc, *reinterpret_cast<uint32_t(*)[32]>(r));
                ptx::tmem_ld_32x32(tacc + 32, *reinterpret_cast<uint32_t(*)[32]>(r + 32));
                ptx::tmem_ld_wait(*reinterpret_cast<uint32_t(*)[32]>(r));
                ptx::tmem_ld_wait(*reinterpret_cast<uint32_t(*)[32]>(r + 32));
                ptx::tc_fence_before();
                __syncwarp();
                // shared: 112 .. 255 of accumulator 0, 0 .. 143 of accumulator 1
                if (lane == 0 && (ab ? group < 3 : group >= 1)) ptx::mbar_arrive_cluster(free_at);
            } else {
                // (as above: no numbers)
#pragma unroll
                for (int c = 0; c < 64; ++c) r[c] = 0x7fffffffu;
            }
            store_columns<64, T>(r, p, i0, j, static_cast<int>(min(p.m - i0, static_cast<int64_t>(64))));
        }
    }

    // (after an abort, copies in flight get time to land; neither CTA's memory goes before both are done)
    __syncwarp();
    if (abort_flag) {
        report_abort(p);
        const long long t0 = clock64();
        while (clock64() - t0 < 4000000LL) { }
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_sync();
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc_pair(tmem_base, 512);
    }
}

template <typename T>
bool launch_pair(const Mx4ProductArgs& q, cudaStream_t st) {
    auto kern = mx4_pair_kernel<T>;
    B200_CUDA_CHECK(allow_max_smem(kern));
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kPairThreads);
    cfg.dynamicSmemBytes = kPairSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    // pairs that the device runs at a time (an odd number of SMs in a group leaves one without a partner)
    cfg.gridDim = dim3(2);
    const int pairs = clusters_at_once(reinterpret_cast<const void*>(kern), cfg);
    ProductArgs p{};
    p.a_scales = q.a_scales;
    p.b_scales = q.b_scales;
    p.nb = mx4_blocks(q.d);
    p.ng = mx4_groups(q.d);
    p.m = q.m;
    p.n = q.n;
    p.out = q.out;
    p.ldo = q.ldo;
    p.err = q.err;
    p.split = 1;
    p.a_tiles = div_up(q.m, 256);
    p.b_tiles = div_up(q.n, 256);
    const int64_t total = static_cast<int64_t>(p.a_tiles) * p.b_tiles;
    if (pairs <= 0 || total < pairs) return false;
    CUtensorMap map_a, map_b, map_sa, map_sb;
    if (encode_mx4_map(&map_a, q.a_codes, q.m, q.d, 128) != 0 || encode_mx4_map(&map_b, q.b_codes, q.n, q.d, 128) != 0 ||
        encode_scale_map(&map_sa, q.a_scales, (q.m + 127) / 128, p.ng, 2) != 0 ||
        encode_scale_map(&map_sb, q.b_scales, (q.n + 127) / 128, p.ng, 1) != 0)
        throw std::runtime_error("cuTensorMapEncodeTiled failed for the rows of a product");
    cfg.gridDim = dim3(2 * static_cast<unsigned>(pairs));
    B200_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, map_b, map_a, map_sb, map_sa, p));
    return true;
}

template <typename T>
void product(const Mx4ProductArgs& q, int num_sms, cudaStream_t st) {
    if (q.m <= 16) launch<16, T>(q, num_sms, st);
    else if (q.m <= 32) launch<32, T>(q, num_sms, st);
    else if (q.m <= 64) launch<64, T>(q, num_sms, st);
    else if (q.m <= 128) launch<128, T>(q, num_sms, st);
    else if (!launch_pair<T>(q, st)) launch<256, T>(q, num_sms, st);
}

}  // namespace

void launch_mx4_product(int dtype, const Mx4ProductArgs& q, int num_sms, cudaStream_t st) {
    if (dtype == kF32) product<float>(q, num_sms, st);
    else if (dtype == kF16) product<__half>(q, num_sms, st);
    else product<__nv_bfloat16>(q, num_sms, st);
}

namespace {
template <int TN, int END>
cudaError_t few_search(const ProductArgs& p, const CUtensorMap& map_b, const CUtensorMap& map_a, int num_sms, int half, cudaStream_t st) {
    auto kern = mx4_few_kernel<TN, float, END>;
    cudaError_t e = allow_max_smem(kern);
    if (e != cudaSuccess) return e;
    const int chunks = (p.ng + 1) / 2;
    const int grid = std::min(p.b_tiles, num_sms);
    kern<<<grid, kFewThreads, 1024 + Few<TN>::resident_bytes(chunks) + 2 * half * kFewStage + kNearAll * 8, st>>>(map_b, map_a, p, half);
    return cudaGetLastError();
}
template <int TN>
cudaError_t few_search(const GemmArgs& a, const uint8_t* a_scales, const uint8_t* b_scales, int num_sms, cudaStream_t st) {
    ProductArgs p{};
    p.a_scales = a_scales;
    p.b_scales = b_scales;
    p.nb = mx4_blocks(a.d);
    p.ng = mx4_groups(a.d);
    p.m = a.nq;
    p.n = a.N;
    p.split = 1;
    p.a_tiles = 1;
    p.b_first = a.tile_first * (kTileB / kLanes);
    p.b_tiles = std::min(a.n_tiles_sel * (kTileB / kLanes), div_up(a.N, kLanes) - p.b_first);
    p.g = a;
    if (p.b_tiles <= 0) return cudaSuccess;
    const int chunks = (p.ng + 1) / 2;
    const int half = std::min(kFewMaxStages, (kSmemMost - 1024 - kNearAll * 8 - Few<TN>::resident_bytes(chunks)) / kFewStage) / 2;
    if (chunks > Few<TN>::kMaxChunks || half < 3) return cudaErrorNotSupported;
    CUtensorMap map_a, map_b;
    if (encode_mx4_map(&map_a, static_cast<const uint8_t*>(a.A), a.nq, a.d, TN) != 0 ||
        encode_mx4_map(&map_b, static_cast<const uint8_t*>(a.B), a.N, a.d, kLanes) != 0)
        return cudaErrorInvalidValue;
    return a.metric == kMetricL2 ? few_search<TN, kEndSearchL2>(p, map_b, map_a, num_sms, half, st)
                                 : few_search<TN, kEndSearchIP>(p, map_b, map_a, num_sms, half, st);
}
}  // namespace

// Against 1 M rows, the other kernel's passes and this one's: 1 query x 128 L2 75 and 36 us (its tile has 128 lanes for
// queries, and every lane tests); 64 x 128 inner product 73 and 48; 128 x 128 k = 100 78 and 73; 100 x 768 101 and 100, where
// the rows' bytes take 62.
cudaError_t launch_mx4_few_search(const GemmArgs& a, const uint8_t* a_scales, const uint8_t* b_scales, int num_sms, cudaStream_t st) {
    if (a.nq <= 16) return few_search<16>(a, a_scales, b_scales, num_sms, st);
    if (a.nq <= 32) return few_search<32>(a, a_scales, b_scales, num_sms, st);
    if (a.nq <= 64) return few_search<64>(a, a_scales, b_scales, num_sms, st);
    if (a.nq <= 128) return few_search<128>(a, a_scales, b_scales, num_sms, st);
    return cudaErrorNotSupported;
}

int encode_mx4_map(CUtensorMap* out, const uint8_t* codes, int64_t rows, int d, int box_rows) {
    return encode_rows_map(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, codes, rows, static_cast<int>(mx4_pitch(d)), box_rows);
}

}  // namespace b200
