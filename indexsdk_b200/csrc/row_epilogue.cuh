// What a thread of a distance GEMM does with its part of an accumulator tile (thresholds, burst minima,
// candidate lists), and the walk over the (query block, base tile) items of a CTA.  Shared by the kernels
// of dist_gemm.cu and mx4_gemm.cu.
#pragma once
#include "dist_gemm.cuh"

#include "common.cuh"
#include "cos16.cuh"

namespace b200 {
namespace {

template <typename AccT>
struct KeyOps;
template <>
struct KeyOps<float> {
    using Norm = float;
    static __device__ __forceinline__ float from_bits(uint32_t r) { return __uint_as_float(r); }
    static __device__ __forceinline__ float key(float acc, float bn, bool l2) { return l2 ? fmaf(-2.f, acc, bn) : -acc; }
    static __device__ __forceinline__ uint32_t ord(float k) { return float_to_ord(k); }
    static __device__ __forceinline__ float tau(uint32_t o) { return ord_to_float(o); }
    static __device__ __forceinline__ float worst() { return __int_as_float(0x7f800000); }
    // smallest value strictly above t (t itself when t = +inf): key <= t  <=>  key - above(t) < 0
    static __device__ __forceinline__ float above(float t) {
        return t == __int_as_float(0x7f800000) ? t : ord_to_float(float_to_ord(t) + 1u);
    }
    // sign word of (l2 ? bn - 2 acc : -acc) - tup
    static __device__ __forceinline__ uint32_t sign_l2(float acc, float bn, float tup) {
        return __float_as_uint(fmaf(-2.f, acc, bn) - tup);
    }
    static __device__ __forceinline__ uint32_t sign_ip(float acc, float ntup) { return __float_as_uint(ntup - acc); }
    static __device__ __forceinline__ float neg(float v) { return -v; }
};
template <>
struct KeyOps<int32_t> {
    using Norm = int32_t;
    static __device__ __forceinline__ int32_t from_bits(uint32_t r) { return static_cast<int32_t>(r); }
    static __device__ __forceinline__ int32_t key(int32_t acc, int32_t bn, bool l2) { return l2 ? bn - 2 * acc : -acc; }
    static __device__ __forceinline__ uint32_t ord(int32_t k) { return int_to_ord(k); }
    static __device__ __forceinline__ int32_t tau(uint32_t o) { return ord_to_int(o); }
    static __device__ __forceinline__ int32_t worst() { return 0x7fffffff; }
    static __device__ __forceinline__ int32_t above(int32_t t) { return t == 0x7fffffff ? t : t + 1; }
    static __device__ __forceinline__ uint32_t sign_l2(int32_t acc, int32_t bn, int32_t tup) {
        return static_cast<uint32_t>(bn - 2 * acc - tup);
    }
    static __device__ __forceinline__ uint32_t sign_ip(int32_t acc, int32_t ntup) {
        return static_cast<uint32_t>(ntup - acc);
    }
    static __device__ __forceinline__ int32_t neg(int32_t v) { return -v; }
};

constexpr uint32_t kCandBlock = 8;   // candidate slots a thread reserves with one atomic

// Per-thread (= query row x part of the tile's columns) epilogue state.
//   append mode : a thread reserves kCandBlock consecutive slots of its row's candidate list with
//                 ONE atomicAdd and fills them over as many tiles as it takes -- a CTA walks
//                 consecutive base tiles of the same query block, so the row stays the same.
//                 When the row changes (or the kernel ends) the unused slots of the open block are
//                 written as "invalid"; the consumers skip those.  counts[row] is therefore the
//                 number of RESERVED slots, an upper bound of the candidates.
//   direct mode : every key is written to cand[q][position] (no threshold, no atomics).
//   FOLD        : the operands carry 16 extra K columns (GemmArgs / kFoldCols), so the accumulator
//                 already holds  D = q.y - |y|^2/2 + tau/2  (L2; inner product: q.y + tau).  No
//                 norms are read and "key <= tau" is the sign of D: 32 columns are tested with a
//                 16-instruction AND tree, and the burst minimum of the key is a maximum of D.
// NCH: 32-column chunks a thread handles per tile.
template <typename AccT, int MODE, int BURST, bool FOLD, int NCH, bool COS = false, bool IPONLY = false>
struct RowEpilogue {
    using K = KeyOps<AccT>;
    const GemmArgs& a;
    int q;        // query row, valid when row_ok
    bool row_ok;
    bool l2;
    static constexpr bool cosm = COS;   // int8 cosine: the accumulators are turned into ordered fp16 scores first
    __half2 rq2;              // cosine: the row's query term
    AccT tau, tau_up;
    float tq;                 // FOLD append: the row's threshold, for the approximate key
    float bias;               // FOLD append over a segmented base: what the accumulator lacks to (tau - key) / 2
    uint32_t admit_all;       // all ones when the row's threshold admits every key (no difference to it can be formed)
    int blk_q;                // row of the open candidate block (-1: none)
    uint32_t blk_next, blk_left;
    uint32_t pre_base;        // a second block reserved ahead of need (its atomic is issued at the end of a
    bool pre_ok;              // tile and not read before the open block runs out, so nobody waits for it)
    uint32_t res[NCH * (32 / BURST)];   // burst-min results of this thread's part of the tile

    __device__ __forceinline__ explicit RowEpilogue(const GemmArgs& a_)
        : a(a_), q(-1), row_ok(false), l2(!IPONLY && a_.metric == kMetricL2),
          tau(AccT(0)), tau_up(AccT(0)), tq(0.f), bias(0.f), admit_all(0u),
          blk_q(-1), blk_next(0), blk_left(0), pre_base(0), pre_ok(false) {}

    // 32 filter bits of this row for base positions col0 .. col0 + 31 (col0 is a multiple of 32).
    __device__ __forceinline__ uint32_t mask_word(int64_t col0) const {
        return __ldg(a.qmask + static_cast<int64_t>(q) * a.qmask_stride + (col0 >> 5));
    }

    // Fills what is left of the open block with the "invalid" marker.
    __device__ __forceinline__ void close_block() {
        if (blk_q >= 0) {
            uint64_t* crow = a.cand + static_cast<int64_t>(blk_q) * a.cap;
            for (uint32_t i = 0; i < blk_left; ++i)
                if (blk_next + i < a.cap) crow[blk_next + i] = kCandInvalid;
            if (pre_ok)
                for (uint32_t i = 0; i < kCandBlock; ++i)
                    if (pre_base + i < a.cap) crow[pre_base + i] = kCandInvalid;
        }
        blk_q = -1;
        blk_left = 0;
        pre_ok = false;
    }

    __device__ __forceinline__ void begin_tile(int q_, bool ok) {
        const bool new_row = q_ != q || ok != row_ok;
        if (MODE == kModeAppend && !a.direct && (q_ != blk_q || !ok)) close_block();
        q = q_;
        row_ok = ok;
        if (cosm && ok && new_row) {
            const int qn = a.seg_index ? q % a.nq : q;   // segmented base: candidate row -> query
            rq2 = cos16_query_term(__ldg(a.qnorm_i32 + qn));
        }
        if (MODE == kModeAppend && ok && new_row) {
            // once per run of tiles of the same row: the threshold, and (threshold mode, runs long
            // enough to use it) the first candidate block -- reserved now, while the accumulator is
            // still being computed, so that the first candidate of the run does not wait for the atomic
            const uint32_t to = __ldg(a.tau + q);
            if (a.eager && !a.direct && blk_q != q) {
                blk_next = atomicAdd(a.counts + q, kCandBlock);
                blk_left = kCandBlock;
                blk_q = q;
            }
            if (FOLD && !a.direct) {
                tq = ord_to_float(to);
                if (a.seg_bias) bias = __ldg(a.seg_bias + q);
            } else {
                tau = K::tau(to);
                tau_up = K::above(tau);
                admit_all = tau == tau_up ? 0xFFFFFFFFu : 0u;
            }
        }
    }

    __device__ __forceinline__ void append(uint64_t e) {
        if (blk_left == 0) {
            if (pre_ok) {
                blk_next = pre_base;
                pre_ok = false;
            } else {
                blk_next = atomicAdd(a.counts + q, kCandBlock);   // first block of a run, or a burst of candidates
            }
            blk_left = kCandBlock;
            blk_q = q;
        }
        if (blk_next < a.cap) a.cand[static_cast<int64_t>(q) * a.cap + blk_next] = e;
        ++blk_next;
        --blk_left;
    }

    // Value of r[c] for a run-time c without indexing registers dynamically (select tree).
    static __device__ __forceinline__ uint32_t pick(const uint32_t (&r)[32], uint32_t c) {
        uint32_t v16[16], v8[8], v4[4], v2[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) v16[i] = (c & 16u) ? r[16 + i] : r[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) v8[i] = (c & 8u) ? v16[8 + i] : v16[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) v4[i] = (c & 4u) ? v8[4 + i] : v8[i];
#pragma unroll
        for (int i = 0; i < 2; ++i) v2[i] = (c & 2u) ? v4[2 + i] : v4[i];
        return (c & 1u) ? v2[1] : v2[0];
    }

    // Folded operands: r holds D for 32 columns.
    // ci: index of the chunk inside this thread's part of the tile (a constant after unrolling)
    __device__ __forceinline__ void chunk_fold(const uint32_t (&r)[32], int64_t col0, int nvalid, int ci, int64_t cbase) {
        if (!row_ok && (MODE == kModeBurstMin || a.direct)) return;
        if (MODE == kModeBurstMin) {
            constexpr int NB = 32 / BURST;
            const float ninf = __int_as_float(0xff800000);
            // min / max and selects share the half-rate integer pipe, which is what bounds this
            // epilogue: the test for rows past the end of the base is kept out of the common path.
            uint32_t keep = nvalid >= 32 ? 0xFFFFFFFFu : ((1u << nvalid) - 1u);   // bit c: column c takes part
            if (a.qmask) keep &= mask_word(col0);
            const bool full = keep == 0xFFFFFFFFu;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float v[BURST];
                if (full) {
#pragma unroll
                    for (int j = 0; j < BURST; ++j) v[j] = __uint_as_float(r[b * BURST + j]);
                } else {
#pragma unroll
                    for (int j = 0; j < BURST; ++j) {
                        const int c = b * BURST + j;
                        v[j] = ((keep >> c) & 1u) ? __uint_as_float(r[c]) : ninf;
                    }
                }
#pragma unroll
                for (int w = BURST / 2; w > 0; w >>= 1)
#pragma unroll
                    for (int j = 0; j < w; ++j) v[j] = fmaxf(v[j], v[j + w]);   // NaN never wins
                const float key = l2 ? -2.f * v[0] : -v[0];
                res[ci * NB + b] = float_to_ord(key);
            }
        } else if (a.direct) {
            uint64_t* crow = a.cand + static_cast<int64_t>(q) * a.cap + (col0 - cbase);
            uint32_t keep = nvalid >= 32 ? 0xFFFFFFFFu : ((1u << nvalid) - 1u);
            if (a.qmask) keep &= mask_word(col0);
#pragma unroll
            for (int c = 0; c < 32; ++c) {
                const float dv = __uint_as_float(r[c]);
                const float key = l2 ? -2.f * dv : -dv;
                // NaN keys are left at the buffer's "invalid" fill
                if (((keep >> c) & 1u) && key <= tau) crow[c] = pack_cand(float_to_ord(key), static_cast<uint32_t>(col0 + c));
            }
        } else {
            // (the tcgen05 kernel calls fold_mask / fold_extract itself, with the accumulator handed
            // back in between; this is the path of the CUDA-core variant)
            if (a.seg_bias) {
                seg_fold_extract(r, seg_fold_mask(r, nvalid), col0);
                return;
            }
            const uint32_t m = fold_mask(r, col0, nvalid);
            fold_extract(r, m, col0);
        }
    }

    // Folded operands, append mode, split in two so that the accumulator can be handed back between
    // them.  fold_mask: bit (31 - c) of the result = column c of this lane's row passes (D >= 0, a
    // real base row, not filtered out); warp-collective, 0 for everybody when no lane has a hit.
    __device__ __forceinline__ uint32_t fold_mask(const uint32_t (&r)[32], int64_t col0, int nvalid) {
        uint32_t t[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) t[i] = r[2 * i] & r[2 * i + 1];
#pragma unroll
        for (int w = 8; w > 0; w >>= 1)
#pragma unroll
            for (int i = 0; i < w; ++i) t[i] &= t[i + w];
        const bool hit = row_ok && static_cast<int32_t>(t[0]) >= 0;   // not every D negative
        if (!__any_sync(0xFFFFFFFFu, hit)) return 0u;
        uint32_t m0 = 0, m1 = 0;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
            m0 = __funnelshift_l(r[c], m0, 1);
            m1 = __funnelshift_l(r[16 + c], m1, 1);
        }
        uint32_t mask = ~((m0 << 16) | (m1 & 0xFFFFu));
        mask &= nvalid >= 32 ? 0xFFFFFFFFu : ~(0xFFFFFFFFu >> nvalid);
        if (a.qmask && row_ok) mask &= __brev(mask_word(col0));
        return hit ? mask : 0u;
    }
    // Segmented base: the threshold is the candidate row's own (bias), so it joins the accumulator here.
    // The registers keep D without it: the key is read from them directly, and with a threshold of
    // +infinity every column whose key is a number passes, infinite keys included.
    __device__ __forceinline__ uint32_t seg_fold_mask(const uint32_t (&r)[32], int nvalid) {
        uint32_t m0 = 0, m1 = 0;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
            m0 = __funnelshift_l(__float_as_uint(__uint_as_float(r[c]) + bias), m0, 1);
            m1 = __funnelshift_l(__float_as_uint(__uint_as_float(r[16 + c]) + bias), m1, 1);
        }
        const uint32_t mask = ~((m0 << 16) | (m1 & 0xFFFFu)) & (nvalid >= 32 ? 0xFFFFFFFFu : ~(0xFFFFFFFFu >> nvalid));
        return row_ok ? mask : 0u;
    }
    __device__ __forceinline__ void seg_fold_extract(const uint32_t (&r)[32], uint32_t mask, int64_t col0) {
        while (mask) {
            const uint32_t c = __clz(mask);
            mask &= ~(0x80000000u >> c);
            const float dv = __uint_as_float(pick(r, c));
            const float key = l2 ? -2.f * dv : -dv;
            if (key != key) continue;   // NaN
            append(pack_cand(float_to_ord(key), static_cast<uint32_t>(col0 + c)));
        }
    }
    // fold_extract: appends the columns of `mask` from the registers (select tree; no TMEM access).
    __device__ __forceinline__ void fold_extract(const uint32_t (&r)[32], uint32_t mask, int64_t col0) {
        while (mask) {
            const uint32_t c = __clz(mask);
            mask &= ~(0x80000000u >> c);
            const float dv = __uint_as_float(pick(r, c));
            if (!(dv >= 0.f)) continue;   // NaN
            const float key = l2 ? fmaf(-2.f, dv, tq) : tq - dv;
            append(pack_cand(float_to_ord(key), static_cast<uint32_t>(col0 + c)));
        }
    }

    // The same split for an inner product without folded operands and without norms (int8): bit
    // (31 - c) = column c has key = -acc <= tau.
    __device__ __forceinline__ uint32_t ip_mask(const uint32_t (&r)[32], int64_t col0, int nvalid) {
        const AccT ntup = K::neg(tau_up);
        uint32_t m0 = 0, m1 = 0;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
            m0 = __funnelshift_l(K::sign_ip(K::from_bits(r[c]), ntup), m0, 1);
            m1 = __funnelshift_l(K::sign_ip(K::from_bits(r[16 + c]), ntup), m1, 1);
        }
        uint32_t mask = (m0 << 16) | (m1 & 0xFFFFu);
        uint32_t valid = nvalid >= 32 ? 0xFFFFFFFFu : ((1u << nvalid) - 1u);
        if (a.qmask && row_ok) valid &= mask_word(col0);
        return row_ok ? ((mask | admit_all) & __brev(valid)) : 0u;
    }
    __device__ __forceinline__ void ip_extract(const uint32_t (&r)[32], uint32_t mask, int64_t col0) {
        while (mask) {
            const uint32_t c = __clz(mask);
            mask &= ~(0x80000000u >> c);
            const AccT key = K::neg(K::from_bits(pick(r, c)));
            if (!(key <= tau)) continue;
            append(pack_cand(K::ord(key), static_cast<uint32_t>(col0 + c)));
        }
    }

    // ... and for L2 with the norms taken from global memory (gn: the norms of the chunk's 32 columns)
    __device__ __forceinline__ uint32_t l2_mask(const uint32_t (&r)[32], const uint32_t* gn, int64_t col0, int nvalid) {
        uint32_t m0 = 0, m1 = 0;
        const uint4* g4 = reinterpret_cast<const uint4*>(gn);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const uint4 na = __ldg(g4 + g), nb4 = __ldg(g4 + 4 + g);
            m0 = __funnelshift_l(K::sign_l2(K::from_bits(r[4 * g + 0]), K::from_bits(na.x), tau_up), m0, 1);
            m0 = __funnelshift_l(K::sign_l2(K::from_bits(r[4 * g + 1]), K::from_bits(na.y), tau_up), m0, 1);
            m0 = __funnelshift_l(K::sign_l2(K::from_bits(r[4 * g + 2]), K::from_bits(na.z), tau_up), m0, 1);
            m0 = __funnelshift_l(K::sign_l2(K::from_bits(r[4 * g + 3]), K::from_bits(na.w), tau_up), m0, 1);
            m1 = __funnelshift_l(K::sign_l2(K::from_bits(r[16 + 4 * g + 0]), K::from_bits(nb4.x), tau_up), m1, 1);
            m1 = __funnelshift_l(K::sign_l2(K::from_bits(r[16 + 4 * g + 1]), K::from_bits(nb4.y), tau_up), m1, 1);
            m1 = __funnelshift_l(K::sign_l2(K::from_bits(r[16 + 4 * g + 2]), K::from_bits(nb4.z), tau_up), m1, 1);
            m1 = __funnelshift_l(K::sign_l2(K::from_bits(r[16 + 4 * g + 3]), K::from_bits(nb4.w), tau_up), m1, 1);
        }
        uint32_t mask = (m0 << 16) | (m1 & 0xFFFFu);
        uint32_t valid = nvalid >= 32 ? 0xFFFFFFFFu : ((1u << nvalid) - 1u);
        if (a.qmask && row_ok) valid &= mask_word(col0);
        return row_ok ? ((mask | admit_all) & __brev(valid)) : 0u;
    }
    __device__ __forceinline__ void l2_extract(const uint32_t (&r)[32], uint32_t mask, int64_t col0, const uint32_t* gn) {
        while (mask) {
            const uint32_t c = __clz(mask);
            mask &= ~(0x80000000u >> c);
            const AccT key = K::key(K::from_bits(pick(r, c)), K::from_bits(__ldg(gn + c)), true);
            if (!(key <= tau)) continue;   // NaN
            append(pack_cand(K::ord(key), static_cast<uint32_t>(col0 + c)));
        }
    }

    // r: 32 accumulator columns; nb: the matching 32 norms in shared memory; col0: base position
    // of r[0]; nvalid: real base rows among the 32; bslot: first burst slot (burst-min mode);
    // ci: see chunk_fold.  The hot path is straight-line code: the threshold test of the 32
    // columns is folded into a bit mask, and only a non-zero mask (rare) enters the compact
    // candidate loop.
    // cbase: position of the first base row of the segment the tile belongs to (0 without segments)
    __device__ __forceinline__ void chunk(uint32_t (&r)[32], const uint32_t* nb, int64_t col0, int nvalid,
                                          int bslot, int ci, int64_t cbase) {
        if (FOLD) {
            chunk_fold(r, col0, nvalid, ci, cbase);
            return;
        }
        if (!row_ok) return;
        if (cosm) cos_scores(r, nb);
        chunk_keys(r, nb, col0, nvalid, bslot, ci, cbase);
    }

    // nb holds the base rows' fp16 reciprocal norms; the accumulators become ordered scores in place,
    // and from here on they are treated as inner products
    __device__ __forceinline__ void cos_scores(uint32_t (&r)[32], const uint32_t* nb) const {
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
            int32_t s0, s1;
            cos16_pair(static_cast<int32_t>(r[c]), static_cast<int32_t>(r[c + 1]), nb[c], nb[c + 1], rq2, s0, s1);
            r[c] = static_cast<uint32_t>(s0);
            r[c + 1] = static_cast<uint32_t>(s1);
        }
    }

    __device__ __forceinline__ void chunk_keys(const uint32_t (&r)[32], const uint32_t* nb, int64_t col0, int nvalid,
                                               int bslot, int ci, int64_t cbase) {
        // The norms (L2) are taken eight at a time, next to their use: nb may point into shared or
        // into global memory, and 32 of them held in registers beside the 32 accumulator words are
        // what a 96-register kernel cannot afford.
        const uint4* np4 = reinterpret_cast<const uint4*>(nb);
        auto norms8 = [&](int s8, uint32_t (&n8)[8]) {
            if (l2) {
                const uint4 x = np4[2 * s8], y = np4[2 * s8 + 1];
                n8[0] = x.x; n8[1] = x.y; n8[2] = x.z; n8[3] = x.w;
                n8[4] = y.x; n8[5] = y.y; n8[6] = y.z; n8[7] = y.w;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) n8[j] = 0u;   // +0.0f / 0
            }
        };
        uint32_t valid = nvalid >= 32 ? 0xFFFFFFFFu : ((1u << nvalid) - 1u);
        if (a.qmask) valid &= mask_word(col0);
        if (MODE == kModeBurstMin) {
            uint32_t* dst = a.mins + static_cast<int64_t>(q) * a.mins_stride + bslot;
            const bool full = valid == 0xFFFFFFFFu;
            AccT m[4] = {K::worst(), K::worst(), K::worst(), K::worst()};   // independent chains
#pragma unroll
            for (int s8 = 0; s8 < 4; ++s8) {
                uint32_t n8[8];
                norms8(s8, n8);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int c = s8 * 8 + j;
                    const AccT key = K::key(K::from_bits(r[c]), K::from_bits(n8[j]), l2);
                    if (full || ((valid >> c) & 1u)) m[j & 3] = key < m[j & 3] ? key : m[j & 3];
                }
                if (BURST == 8 || s8 == 3) {   // a burst of 8 ends with every group, a burst of 32 with the last
                    const AccT ma = m[0] < m[1] ? m[0] : m[1], mb = m[2] < m[3] ? m[2] : m[3];
                    dst[BURST == 8 ? s8 : 0] = K::ord(ma < mb ? ma : mb);
#pragma unroll
                    for (int i = 0; i < 4; ++i) m[i] = K::worst();
                }
            }
        } else if (a.direct) {
            uint64_t* crow = a.cand + static_cast<int64_t>(q) * a.cap + (col0 - cbase);
#pragma unroll
            for (int s8 = 0; s8 < 4; ++s8) {
                uint32_t n8[8];
                norms8(s8, n8);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int c = s8 * 8 + j;
                    const AccT key = K::key(K::from_bits(r[c]), K::from_bits(n8[j]), l2);
                    // NaN keys are left at the buffer's "invalid" fill
                    if (((valid >> c) & 1u) && key <= tau) crow[c] = pack_cand(K::ord(key), static_cast<uint32_t>(col0 + c));
                }
            }
        } else {
            // bit (31 - c) of mask = "column c passes": the sign of key - above(tau), shifted in
            // with one funnel shift per column (two independent chains for the scheduler).
            uint32_t m0 = 0, m1 = 0;
            if (l2) {
#pragma unroll
                for (int s8 = 0; s8 < 2; ++s8) {
                    uint32_t na[8], nc[8];
                    norms8(s8, na);
                    norms8(s8 + 2, nc);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        m0 = __funnelshift_l(K::sign_l2(K::from_bits(r[s8 * 8 + j]), K::from_bits(na[j]), tau_up), m0, 1);
                        m1 = __funnelshift_l(K::sign_l2(K::from_bits(r[16 + s8 * 8 + j]), K::from_bits(nc[j]), tau_up), m1, 1);
                    }
                }
            } else {
                const AccT ntup = K::neg(tau_up);
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    m0 = __funnelshift_l(K::sign_ip(K::from_bits(r[c]), ntup), m0, 1);
                    m1 = __funnelshift_l(K::sign_ip(K::from_bits(r[16 + c]), ntup), m1, 1);
                }
            }
            uint32_t mask = (m0 << 16) | (m1 & 0xFFFFu);
            mask = (mask | admit_all) & __brev(valid);   // rows past the end of the base, rows the filter excludes
            while (mask) {
                const uint32_t c = __clz(mask);
                mask &= ~(0x80000000u >> c);
                const AccT key = K::key(K::from_bits(pick(r, c)), K::from_bits(l2 ? nb[c] : 0u), l2);
                if (!(key <= tau)) continue;   // NaN
                append(pack_cand(K::ord(key), static_cast<uint32_t>(col0 + c)));
            }
        }
    }

    // hslot: first burst slot of this thread's part of the tile (burst-min mode)
    __device__ __forceinline__ void end_tile(int hslot) {
        if (MODE == kModeAppend && !a.direct && row_ok && blk_q == q && !pre_ok && blk_left <= kCandBlock / 2) {
            pre_base = atomicAdd(a.counts + q, kCandBlock);
            pre_ok = true;
        }
        if (MODE == kModeBurstMin && FOLD && row_ok) {
            // 16-byte (or 8-byte) stores instead of scattered words
            uint32_t* dst = a.mins + static_cast<int64_t>(q) * a.mins_stride + hslot;
            constexpr int NW = NCH * (32 / BURST);
            if (NW % 4 == 0) {
#pragma unroll
                for (int i = 0; i < NW / 4; ++i)
                    reinterpret_cast<uint4*>(dst)[i] = make_uint4(res[4 * i], res[4 * i + 1], res[4 * i + 2], res[4 * i + 3]);
            } else {
#pragma unroll
                for (int i = 0; i < NW / 2; ++i) reinterpret_cast<uint2*>(dst)[i] = make_uint2(res[2 * i], res[2 * i + 1]);
            }
        }
    }

    __device__ __forceinline__ void finish() {
        if (MODE == kModeAppend && !a.direct) close_block();
    }
};

__device__ __forceinline__ int tile_of(const GemmArgs& a, int sel) {
    if (a.tile_first >= 0) return a.tile_first + sel * a.tile_step;   // a stretch of tiles (whole base: first = 0)
    return static_cast<int>(static_cast<int64_t>(sel) * a.n_tiles_total / a.n_tiles_sel);
}

// Work of one CTA: a contiguous range of the (query block, base tile) items in query-block-major
// order.  Consecutive items of a CTA share the query block, which is what lets the query tile stay
// in shared memory and a thread keep one candidate block open across tiles.  With few query blocks
// and a base larger than L2 the ranges are aligned (see below) so that CTAs of different query
// blocks walk the same base tiles at the same time and a base tile is read from HBM about once;
// otherwise the linearised item list is simply cut into equal pieces.
struct ItemRange {
    int64_t count;       // items of this CTA
    int qb0, sel0;       // first item
    int n_sel;
    __device__ __forceinline__ ItemRange(const GemmArgs& a, int n_qb) {
        n_sel = a.n_tiles_sel;
        const int G = gridDim.x, c = blockIdx.x;
        if (a.aligned_ranges) {
            // one query block per CTA; the CTAs of a query block split the tiles evenly, so CTAs of
            // different query blocks sit on the same stretch of the base at the same time
            const int qb = c % n_qb, j = c / n_qb;
            const int nl = G / n_qb + (qb < G % n_qb ? 1 : 0);
            const int64_t lo = static_cast<int64_t>(n_sel) * j / nl;
            const int64_t hi = static_cast<int64_t>(n_sel) * (j + 1) / nl;
            count = hi - lo;
            qb0 = qb;
            sel0 = static_cast<int>(lo);
        } else {
            const int64_t total = static_cast<int64_t>(n_qb) * n_sel;
            const int64_t lo = total * c / G;
            const int64_t hi = total * (c + 1) / G;
            count = hi - lo;
            qb0 = static_cast<int>(lo / n_sel);
            sel0 = static_cast<int>(lo % n_sel);
        }
    }
};
// Walks a range without divisions (the roles that run one thread deep cannot afford them).
struct ItemCursor {
    int qb, sel;
    int n_sel;
    __device__ __forceinline__ explicit ItemCursor(const ItemRange& r) : qb(r.qb0), sel(r.sel0), n_sel(r.n_sel) {}
    __device__ __forceinline__ void next() {
        if (++sel == n_sel) {
            sel = 0;
            ++qb;
        }
    }
    __device__ __forceinline__ bool last_of_qb() const { return sel + 1 == n_sel; }
};

}  // namespace
}  // namespace b200
