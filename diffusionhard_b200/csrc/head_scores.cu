// head_scores.cu -- the int8 output head fused with the scores of its rows
// (log probabilities of given tokens, entropy, logsumexp, the k best tokens);
// logits never reach HBM.  Two kernels:
//
// 1. head_stats_kernel: the persistent, warp-specialised int8 GEMM of
//    gemm_tc.cuh's structure (TMA ring, one MMA thread, accumulators double
//    buffered in TMEM), whose epilogue turns accumulators into logits
//    x = fp32(acc * fp32(a_scale w_scale) + bias) and these into running
//    softmax statistics (row_scores.cuh), 4 rows a thread.  A CTA walks a
//    contiguous span of tiles in (row tile, column tile) order, so that a
//    thread's statistics stay in registers until the row tile changes.  For
//    the k best tokens it stores only maxima: of each part of 64 logits and
//    of each group of 8 (10 bytes a part and row).
// 2. head_rows_kernel: joins a row's partial statistics, bounds the k-th best
//    logit from below by the k-th largest of maxima of disjoint parts, and
//    computes the logits of the groups that reach the bound (about k) again (the
//    same fp32 expression of the same integer sum, so the same bits), like the
//    given tokens' logits.
//
// What bounds them: the first, the epilogue's issue slots beside the tensor cores
// (32768 x 50258, hidden 768: 880 us, of which 785 remain with an epilogue that
// reads nothing, 2.9 Pop/s; with maxima 965); the second, reads of weight rows from
// L2 (5 alternatives 175 us, 32 of 4096 rows 127 us, about 10 TB/s; none 30 us).
// With few rows both are latency: 32 rows 19.5 us, 25.6 with 8 alternatives.
#include <cuda_fp16.h>

#include "dequant.cuh"
#include "row_scores.cuh"
#include "tc_ptx.cuh"
#include "tmap.h"

#include <algorithm>

namespace dh {

uint32_t make_i8_operand_maps(CUtensorMap* ta, CUtensorMap* tb, const int8_t* a, uint64_t lda,
                              const int8_t* w, uint64_t ldw, uint32_t m, uint32_t n, uint32_t k,
                              uint32_t bn);

namespace {

constexpr uint32_t kBM = 128, kBK = 128;
constexpr uint32_t kMaxStages = 6;
constexpr uint32_t kABytes = kBM * kBK;
constexpr uint32_t kPartCols = 64;                      // a tile's columns are cut into parts of 64: two blocks of 32
constexpr uint32_t kGroup = 8;                          // logits per stored maximum (group_token)
constexpr uint32_t kGroupsPerPart = kPartCols / kGroup;
constexpr uint32_t kBarBytes = 1024;
constexpr uint32_t kStagePerWarp = kPartCols * 8;       // bias and w_scale of the warp's columns
// Shared memory: with k <= kResidentK the row tile's A stays for all its column
// tiles and the ring holds B alone (the copies into shared memory compete with
// the MMA's and the epilogue's reads of it: 32768 x 50258, hidden 768, 871 against
// 915 us); otherwise a stage holds both.  Above 768 the ring beside A shrinks to 3 stages
// (hidden 832: resident 55.1 against 52.2 us at 1001 rows, 87.0 against 82.9 at 2048;
// 896: 54.5 against 52.2, 273 against 271 at 8192, but 337 against 351 with 5
// alternatives), and past 896 to 2.  Rows at an odd multiple of 16 bytes are the
// exception: streaming them costs more (784: resident 308 against 416 us at 8192 rows).
constexpr uint32_t kSmemLimit = 227 * 1024;
constexpr uint32_t kResidentK = 768;
constexpr uint32_t kStreamedStages = 4;
template <uint32_t kBN>
struct HeadTile {
    static constexpr uint32_t kParts = kBN / kPartCols;
    static constexpr uint32_t kEpiWarps = 4 * kParts;   // 4 for each part: the lane quadrants of TMEM
    static constexpr uint32_t kThreads = 64 + 32 * kEpiWarps;
    static constexpr uint32_t kBBytes = kBN * kBK;
    static constexpr uint32_t kFixed = 1024 + kBarBytes + kEpiWarps * kStagePerWarp;
    static constexpr uint32_t resident_stages(uint32_t k_blocks) {
        const uint32_t n = (kSmemLimit - kFixed - k_blocks * kABytes) / kBBytes;
        return n < kMaxStages ? n : kMaxStages;
    }
    static_assert(resident_stages(kResidentK / kBK) >= 3, "room for a ring beside A");
    static_assert(kFixed + kStreamedStages * (kABytes + kBBytes) <= kSmemLimit, "room for the streamed ring");
};
// float(acc) is exact up to 2^24: k products of magnitude 127 * 127 (128 * 128).
// (float64 there instead: 8192 x 50258, hidden 1024, 716 against 298 us)
constexpr uint32_t kExactK = 1024;
constexpr uint64_t kMaxTiles = 1u << 30;

// Logits up to this size take the epilogue's short way.  (Bases up to kSlipBase
// carry a slip, at most 64 there; a logit is then 2e8 below any larger base.)
constexpr float kPlainLogit = 8e8f, kSlipBase = 1e9f;

// How a launch splits the work, shared by the two kernels: CTA c takes `each`
// tiles, and one more if c < more, after those of the CTAs before it.
struct HeadSplit {
    uint32_t rows, cols, n_tiles, parts, grid, max_segs, each, more;  // cols, parts: of a tile
    __host__ __device__ uint32_t all_parts() const { return n_tiles * parts; }
    __host__ __device__ uint32_t first_tile(uint32_t cta) const { return cta * each + (cta < more ? cta : more); }
    // the CTA that holds tile t
    __host__ __device__ uint32_t cta_of(uint32_t t) const {
        const uint32_t longer = more * (each + 1);
        return t < longer ? t / (each + 1) : more + (t - longer) / each;
    }
    // where a row's maximum of a part lies
    __host__ __device__ uint64_t padded_rows() const { return (static_cast<uint64_t>(rows) + kBM - 1) / kBM * kBM; }
    __host__ __device__ uint64_t slot(uint32_t part, uint32_t row) const { return part * padded_rows() + row; }
};

struct HeadScoreParams {
    HeadSplit split;
    uint32_t vocab, mask_id, k, stages;
    const float* a_scale;
    const float* w_scale;
    const float* bias;   // or null
    float4* partials;    // [grid][max_segs][parts][128]: base, s, t of a row's part
    uint2* group_max;    // [n_tiles * parts][rows]: 8 groups' (group_at), or null: none asked for
    uint16_t* part_max;  // [n_tiles * parts][rows]; rows rounded up to row tiles
};

// The logit of one accumulator, by an FMA whose only rounding is the logit's.  kWide:
// k > kExactK, where float(acc) would round and the expression is evaluated in float64
// and rounded again.  (The scaled product always does the latter: where the float64
// value is halfway between two fp32 ones and the exact one is not, as with a bias that
// float64 drops beside a product of few bits, the last bits differ.)
template <bool kWide>
DH_DEVINL float score_logit(int32_t acc, float ab, float w, float b) {
    if (kWide) return ref_logit(acc, ab, w, b);
    return __fmaf_rn(static_cast<float>(acc), __fmul_rn(ab, w), b);
}

DH_DEVINL float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

// Maxima are stored as half floats rounded toward zero (past their range: the
// largest finite one; -inf stays), those of groups as the upper byte of that:
// rounding keeps the order, so that every part and group with a logit of the k best
// still reaches the rounded bound.  Parts within a rounding step of it are looked
// at for nothing, so 8 bits are too few for them (bfloat16: 8 us more of 233 for
// 32768 x 50258 and 5 alternatives), but enough to tell the groups of a part apart.
DH_DEVINL uint32_t half_pair(float lo, float hi) {
    uint32_t y;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
}
DH_DEVINL float half_float(uint32_t h) { return __half2float(__ushort_as_half(static_cast<uint16_t>(h))); }
constexpr uint32_t kNonePair = 0xFC00FC00u;  // -inf twice
DH_DEVINL uint32_t max_pairs(uint32_t a, uint32_t b) {
    const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}
DH_DEVINL uint32_t min_pairs(uint32_t a, uint32_t b) {
    const __half2 m = __hmin2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}
// Which group of a part (group_token) is byte `b` of a row's 8.
DH_DEVINL uint32_t group_at(uint32_t b, uint64_t row) { return b ^ (static_cast<uint32_t>(row) / 8 % 4 * 2); }

// A row's running statistics in this kernel: pairs of sums of e = 2^z and of
// e z, z = (x - base) log2 e + slip.  slip is what rounding base log2 e to fp32
// leaves off, so that z of a usual logit is one FMA, x log2 e - neg_base2, and
// no error of base's size enters (dropping it: the log probabilities of logits
// around 1e6 were off by 0.04, and past 1e9 it overflowed).
struct PairStats {
    float base;  // -inf before the first logit above it
    float2 s, t;
    DH_DEVINL void clear() {
        base = -CUDART_INF_F;
        s = t = make_float2(0.f, 0.f);
    }
    // -base log2 e as fp32; bounded, so that the z of a logit far below stays finite
    DH_DEVINL static float neg_base2(float base) { return fmaxf(-__fmul_rn(base, kLog2E), -1e38f); }
    // (a base past kSlipBase is met by usual logits from so far below that their
    // e is 0 whatever the slip)
    DH_DEVINL static float slip(float base) {
        return fabsf(base) < kSlipBase ? __fmaf_rn(base, kLog2E, neg_base2(base)) : 0.f;
    }
    // z of the base in terms of another base
    DH_DEVINL void shift(float z) {
        const float f = exp2_fast(z);
        s = make_float2(s.x * f, s.y * f);
        t = make_float2(__fmaf_rn(s.x, z, f * t.x), __fmaf_rn(s.y, z, f * t.y));
    }
    // a new maximum (rare once a row has begun)
    DH_DEVINL void raise(float m) {
        shift(base == -CUDART_INF_F ? 0.f : max_nan(__fmaf_rn(base - m, kLog2E, slip(m) - slip(base)), -1e30f));
        base = m;
    }
    DH_DEVINL RowStats sum() {
        shift(-slip(base));
        return RowStats{base, s.x + s.y, (t.x + t.y) * kLn2};
    }
};

// 32 columns of 4 rows (8 logits of each, a group): accumulators to logits, to the
// rows' statistics, and their maxima to g.  kClamp: some logit may be -inf or NaN, or
// past kPlainLogit.
template <bool kWide, bool kTop, bool kClamp>
DH_DEVINL void add_block(PairStats (&st)[4], float (&g)[4], const uint32_t (&v)[2][16], const float (&ab)[4],
                         const float2 (&w)[4], const float2 (&b)[4]) {
    float2 x[4][4];
#pragma unroll
    for (uint32_t r = 0; r < 4; ++r) {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const int32_t v0 = static_cast<int32_t>(v[r / 2][4 * j + r % 2 * 2]);
            const int32_t v1 = static_cast<int32_t>(v[r / 2][4 * j + r % 2 * 2 + 1]);
            if (kWide)
                x[r][j] = make_float2(ref_logit(v0, ab[r], w[j].x, b[j].x), ref_logit(v1, ab[r], w[j].y, b[j].y));
            else
                x[r][j] = __ffma2_rn(make_float2(static_cast<float>(v0), static_cast<float>(v1)),
                                     __fmul2_rn(make_float2(ab[r], ab[r]), w[j]), b[j]);
        }
    }
    bool above = false;
    float m[4];
#pragma unroll
    for (uint32_t r = 0; r < 4; ++r) {
        m[r] = max3(fmaxf(x[r][0].x, x[r][0].y), x[r][1].x, x[r][1].y);
        m[r] = fmaxf(m[r], max3(fmaxf(x[r][2].x, x[r][2].y), x[r][3].x, x[r][3].y));
        if (kTop) g[r] = m[r];
        above = above || m[r] > st[r].base + kBaseSlack;
    }
    // (one branch for the four rows: what follows is one block of independent work)
    if (above) {
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r)
            if (m[r] > st[r].base + kBaseSlack) st[r].raise(m[r]);
    }
    const float2 c2 = make_float2(kLog2E, kLog2E);
    float2 nb[4], slip[4];
#pragma unroll
    for (uint32_t r = 0; r < 4; ++r) {
        const float base = st[r].base;
        const float y = kClamp ? (base == -CUDART_INF_F ? 0.f : -base) : PairStats::neg_base2(base);
        nb[r] = make_float2(y, y);
        if (kClamp) slip[r].x = slip[r].y = PairStats::slip(base);
    }
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) {
            float2 z;
            if (kClamp) {
                z = __ffma2_rn(__fadd2_rn(x[r][j], nb[r]), c2, slip[r]);
                z = make_float2(max_nan(z.x, -1e30f), max_nan(z.y, -1e30f));
            } else {
                z = __ffma2_rn(x[r][j], c2, nb[r]);
            }
            const float2 e = make_float2(exp2_fast(z.x), exp2_fast(z.y));
            st[r].s = __fadd2_rn(st[r].s, e);
            st[r].t = __ffma2_rn(e, z, st[r].t);
        }
    }
}

// kTop: some alternatives are asked for.
template <bool kWide, bool kResident, bool kTop, uint32_t kBN>
__global__ void __launch_bounds__(HeadTile<kBN>::kThreads, 1)
head_stats_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                  const __grid_constant__ HeadScoreParams p) {
    constexpr uint32_t kBBytes = HeadTile<kBN>::kBBytes, kEpiWarps = HeadTile<kBN>::kEpiWarps;
    constexpr uint32_t kParts = HeadTile<kBN>::kParts, kTmemCols = 512;  // two accumulators, a power of two
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~static_cast<uintptr_t>(1023));
    const uint32_t n_tiles = p.split.n_tiles, stages = p.stages;
    const uint32_t k_blocks = (p.k + kBK - 1) / kBK;
    uint8_t* a_smem = smem;
    uint8_t* b_smem = smem + (kResident ? k_blocks : stages) * kABytes;
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(b_smem + stages * kBBytes);
    uint64_t* empty_bar = full_bar + kMaxStages;
    uint64_t* accf_bar = empty_bar + kMaxStages;   // [2]
    uint64_t* acce_bar = accf_bar + 2;             // [2]
    uint64_t* a_full = acce_bar + 2;               // resident A is there
    uint64_t* a_free = a_full + 1;                 // and was multiplied for the last time
    uint64_t* drain_bar = a_free + 1;              // [1]
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain_bar + 1);
    uint8_t* staging = reinterpret_cast<uint8_t*>(full_bar) + kBarBytes;

    const uint32_t warp = warp_id(), lane = lane_id();
    if (warp == 0 && lane == 0) {
        for (uint32_t s = 0; s < kMaxStages; ++s) {
            tc::mbar_init(&full_bar[s], 1);
            tc::mbar_init(&empty_bar[s], 1);
        }
        for (uint32_t b = 0; b < 2; ++b) {
            tc::mbar_init(&accf_bar[b], 1);
            tc::mbar_init(&acce_bar[b], kEpiWarps);
        }
        tc::mbar_init(a_full, 1);
        tc::mbar_init(a_free, 1);
        tc::mbar_init(drain_bar, 1);
        tc::fence_barrier_init();
        tc::prefetch_tmap(&tmap_a);
        tc::prefetch_tmap(&tmap_b);
    }
    if (warp == 1) tc::tmem_alloc(tmem_holder, kTmemCols);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem_base = *tmem_holder;

    const uint32_t tile0 = p.split.first_tile(blockIdx.x), tile1 = p.split.first_tile(blockIdx.x + 1);

    if (warp == 0) {
        // ------------------------------------------------------ TMA producer
        if (tc::elect_one()) {
            uint32_t stage = 0, phase = 0, issued = 0, issued_parity = 0, a_phase = 0, a_loads = 0;
            bool ok = true;
            for (uint32_t tile = tile0; tile < tile1 && ok; ++tile) {
                const uint32_t m0 = (tile / n_tiles) * kBM, n0 = (tile % n_tiles) * kBN;
                if (kResident && (tile == tile0 || n0 == 0)) {
                    if (!tc::mbar_wait(a_free, a_phase ^ 1, tc::kErrTimeoutEmpty)) break;
                    a_phase ^= 1;
                    ++a_loads;
                    tc::mbar_arrive_expect_tx(a_full, k_blocks * kABytes);
                    for (uint32_t kb = 0; kb < k_blocks; ++kb)
                        tc::tma_load_2d(a_smem + kb * kABytes, &tmap_a, a_full, static_cast<int32_t>(kb * kBK),
                                        static_cast<int32_t>(m0));
                }
                for (uint32_t kb = 0; kb < k_blocks; ++kb) {
                    if (!tc::mbar_wait(&empty_bar[stage], phase ^ 1, tc::kErrTimeoutEmpty)) {
                        ok = false;
                        break;
                    }
                    tc::mbar_arrive_expect_tx(&full_bar[stage], kResident ? kBBytes : kABytes + kBBytes);
                    if (!kResident)
                        tc::tma_load_2d(a_smem + stage * kABytes, &tmap_a, &full_bar[stage],
                                        static_cast<int32_t>(kb * kBK), static_cast<int32_t>(m0));
                    tc::tma_load_2d(b_smem + stage * kBBytes, &tmap_b, &full_bar[stage],
                                    static_cast<int32_t>(kb * kBK), static_cast<int32_t>(n0));
                    issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
                    ++issued;
                    if (++stage == stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            // Drain: every copy this CTA issued has landed before it may exit.
            for (uint32_t s = 0; s < stages && s < issued; ++s)
                tc::mbar_wait(&full_bar[s], (issued_parity >> s) & 1u, tc::kErrTimeoutFull);
            if (a_loads) tc::mbar_wait(a_full, (a_loads - 1) & 1u, tc::kErrTimeoutFull);
        }
    } else if (warp == 1) {
        // ------------------------------------------------------- MMA issuer
        if (tc::elect_one()) {
            constexpr uint32_t idesc = tc::idesc_i8_s32<kBM, kBN>();
            uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0, a_phase = 0;
            bool ok = true;
            for (uint32_t tile = tile0; tile < tile1 && ok; ++tile) {
                if (!tc::mbar_wait(&acce_bar[acc], acc_phase ^ 1, tc::kErrTimeoutAccEmpty)) break;
                if (kResident && (tile == tile0 || tile % n_tiles == 0)) {
                    if (!tc::mbar_wait(a_full, a_phase, tc::kErrTimeoutFull)) break;
                    a_phase ^= 1;
                }
                tc::tc_fence_after();
                const uint32_t d_tmem = tmem_base + acc * kBN;
                for (uint32_t kb = 0; kb < k_blocks; ++kb) {
                    if (!tc::mbar_wait(&full_bar[stage], phase, tc::kErrTimeoutFull)) {
                        ok = false;
                        break;
                    }
                    tc::tc_fence_after();
                    const uint64_t a_desc = tc::smem_desc_sw128(a_smem + (kResident ? kb : stage) * kABytes);
                    const uint64_t b_desc = tc::smem_desc_sw128(b_smem + stage * kBBytes);
#pragma unroll
                    for (uint32_t kk = 0; kk < kBK / 32; ++kk)
                        tc::mma_i8(d_tmem, tc::desc_advance(a_desc, kk * 32), tc::desc_advance(b_desc, kk * 32),
                                   idesc, (kb | kk) != 0u);
                    tc::mma_commit(&empty_bar[stage]);
                    if (++stage == stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (!ok) break;
                tc::mma_commit(&accf_bar[acc]);
                if (kResident && (tile + 1) % n_tiles == 0) tc::mma_commit(a_free);
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1;
                }
            }
            // Drain: all MMAs issued by this thread complete before TMEM is freed.
            tc::mma_commit(drain_bar);
            tc::mbar_wait(drain_bar, 0, tc::kErrTimeoutAccFull);
        }
    } else {
        // --------------------------------------------------------- epilogue
        // All warps drain the same tile, so that none idles while its buffer is
        // filled again (two groups of 8 warps, a buffer each: 1100 us for 32768
        // rows).  A thread holds 4 rows (lane / 4 + 0, 8, 16, 24 of its
        // quadrant's) and a quarter of its part's columns (2 of every 8), so that
        // it reads a column's scale and bias once for 4 logits: with a row a
        // thread, these reads from shared memory were what set the pace (1000
        // against 860 us without them).  A group is 8 of the thread's 16 columns, those of
        // one 32.
        const uint32_t ew = warp - 2, quad = warp & 3u, part = ew >> 2;
        float* bs = reinterpret_cast<float*>(staging + ew * kStagePerWarp);
        float* ws = bs + kPartCols;
        const uint32_t mt0 = tile0 / n_tiles, row_in = quad * 32 + lane / 4, quarter = lane % 4;
        PairStats st[4];
        uint32_t seg = 0;
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) st[r].clear();
        auto flush = [&]() {
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                // the 4 threads of a row
                RowStats o = st[r].sum();
                float top = fmaxf(o.base, __shfl_xor_sync(kFullMask, o.base, 1));
                top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 2));
                rebase(o, top);
#pragma unroll
                for (uint32_t i = 1; i < 4; i <<= 1) {
                    o.s += __shfl_xor_sync(kFullMask, o.s, i);
                    o.t += __shfl_xor_sync(kFullMask, o.t, i);
                }
                if (quarter == 0)
                    p.partials[((static_cast<uint64_t>(blockIdx.x) * p.split.max_segs + seg) * kParts + part) * kBM +
                               row_in + 8 * r] = make_float4(top, o.s, o.t, 0.f);
                st[r].clear();
            }
            ++seg;
        };
        uint32_t mt = mt0, nt = tile0 % n_tiles;  // this tile
        // the next tile's scales and biases, fetched while one is added: columns
        // that are excluded (past the vocabulary, the masked token) get a logit
        // of -inf from a scale of 0 and that bias (NaN in rows whose own scale is
        // infinite or NaN: settle_row answers these)
        float w_next[kPartCols / 32], b_next[kPartCols / 32], ab[4];
        auto fetch = [&](uint32_t n) {
#pragma unroll
            for (uint32_t i = 0; i < kPartCols / 32; ++i) {
                const uint32_t c = n * kBN + part * kPartCols + i * 32 + lane;
                w_next[i] = 0.f;
                b_next[i] = -CUDART_INF_F;
                if (c < p.vocab && c != p.mask_id) {
                    w_next[i] = __ldg(p.w_scale + c);
                    b_next[i] = p.bias ? __ldg(p.bias + c) : 0.f;
                }
            }
        };
        float reach = 0.f;  // bounds |acc a_scale| of the warp's rows
        auto fetch_rows = [&](uint32_t m) {
            float top = 0.f;
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                const uint32_t row = m * kBM + row_in + 8 * r;
                ab[r] = row < p.split.rows ? __ldg(p.a_scale + row) : 0.f;
                const float size = fabsf(ab[r]);
                top = fmaxf(top, size < CUDART_INF_F ? size : CUDART_INF_F);  // (NaN: infinite)
            }
            reach = lanes_max(top) * (16384.f * static_cast<float>(p.k));
        };
        fetch(nt);
        fetch_rows(mt);
        uint32_t acc = 0, phase = 0;
        for (uint32_t tile = tile0; tile < tile1; ++tile) {
            __syncwarp();
            bool odd = false;  // a logit may be past kPlainLogit, -inf or NaN
#pragma unroll
            for (uint32_t i = 0; i < kPartCols / 32; ++i) {
                bs[i * 32 + lane] = b_next[i];
                ws[i * 32 + lane] = w_next[i];
                odd = odd || !(fabsf(b_next[i]) < kPlainLogit / 2 && fabsf(w_next[i]) * reach < kPlainLogit / 2);
            }
            odd = __any_sync(kFullMask, odd);
            __syncwarp();
            const bool last = nt + 1 == n_tiles;
            if (tile + 1 < tile1) fetch(last ? 0u : nt + 1);
            if (!tc::mbar_wait(&accf_bar[acc], phase, tc::kErrTimeoutAccFull)) break;
            tc::tc_fence_after();
            const uint32_t taddr = tmem_base + ((quad * 32u) << 16) + acc * kBN + part * kPartCols;
            float g[2][4];
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {  // 32 columns at a time
                uint32_t v[2][16];
                tc::tmem_ld_16x256b_x4(taddr + 32 * h, v[0]);
                tc::tmem_ld_16x256b_x4(taddr + 32 * h + (16u << 16), v[1]);
                float2 w[4], b[4];
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    w[j] = *reinterpret_cast<const float2*>(ws + 32 * h + 8 * j + 2 * quarter);
                    b[j] = *reinterpret_cast<const float2*>(bs + 32 * h + 8 * j + 2 * quarter);
                }
                tc::tmem_ld_wait();
                if (h == 1) {
                    // the accumulators are read: their buffer may be filled again
                    tc::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&acce_bar[acc]);
                }
                if (odd) add_block<kWide, kTop, true>(st, g[h], v, ab, w, b);
                else add_block<kWide, kTop, false>(st, g[h], v, ab, w, b);
            }
            if (kTop) {
                // the 4 threads of a row hold 2 groups each of 4 rows: after two
                // exchanges each has a row's 8 groups
                uint32_t own[4], got[2];
#pragma unroll
                for (uint32_t r = 0; r < 4; ++r) own[r] = half_pair(g[0][r], g[1][r]);
                const bool odd_q = quarter & 1u, upper_q = quarter & 2u;
#pragma unroll
                for (uint32_t e = 0; e < 2; ++e) {
                    got[e] = __shfl_xor_sync(kFullMask, upper_q ? own[e] : own[2 + e], 2);
                    own[e] = upper_q ? own[2 + e] : own[e];
                }
                const uint32_t q0 = odd_q ? own[1] : own[0], q2 = odd_q ? got[1] : got[0];
                const uint32_t q1 = __shfl_xor_sync(kFullMask, odd_q ? own[0] : own[1], 1);
                const uint32_t q3 = __shfl_xor_sync(kFullMask, odd_q ? got[0] : got[1], 1);
                // (rows past the last have room, and hold what nothing reads)
                const uint64_t at = p.split.slot(nt * kParts + part, mt * kBM + row_in + 8 * quarter);
                p.group_max[at] = make_uint2(__byte_perm(q0, q1, 0x7531), __byte_perm(q2, q3, 0x7531));
                const uint32_t m = max_pairs(max_pairs(q0, q1), max_pairs(q2, q3));
                p.part_max[at] = static_cast<uint16_t>(max_pairs(m, m >> 16));
            }
            ++nt;
            if (last) {
                flush();
                nt = 0;
                ++mt;
                if (tile + 1 < tile1) fetch_rows(mt);
            }
            acc ^= 1;
            phase ^= acc == 0;
        }
        const uint32_t segs = tile1 > tile0 ? (tile1 - 1) / n_tiles - mt0 + 1 : 0u;
        while (seg < segs) flush();
    }
    tc::tc_fence_before();
    __syncthreads();
    // The second kernel may be brought in; it waits for this one's end before it
    // reads what this one writes.  (Earlier, its few CTAs would crowd on the SMs
    // that are done first: 88 against 66 us for 1001 rows and 8 alternatives.)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (warp == 1) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem_base, kTmemCols);
    }
}

// ------------------------------------------------------------ second kernel

struct HeadRowParams {
    HeadSplit split;
    uint32_t vocab, mask_id, k;
    const int8_t* hidden;
    uint64_t ld_hidden;
    const int8_t* weights;
    uint64_t ld_weights;
    const float* a_scale;
    const float* w_scale;
    const float* bias;
    const float4* partials;
    const uint2* group_max;
    const uint16_t* part_max;
    ScoreOutputs out;
};

// One lane's share of hidden row . weight row: lane `l` of `n` lanes takes
// every n-th 16 bytes, and the bytes past the last whole 16 one by one.
DH_DEVINL int32_t dot_share(const int8_t* h, const int8_t* w, uint32_t k, uint32_t l, uint32_t n) {
    int32_t acc = 0;
    const uint32_t nv = k / 16;
    for (uint32_t j = l; j < nv; j += n) {
        const int4 a = __ldg(reinterpret_cast<const int4*>(h) + j);
        const int4 b = __ldg(reinterpret_cast<const int4*>(w) + j);
        acc = __dp4a(a.x, b.x, acc);
        acc = __dp4a(a.y, b.y, acc);
        acc = __dp4a(a.z, b.z, acc);
        acc = __dp4a(a.w, b.w, acc);
    }
    for (uint32_t j = nv * 16 + l; j < k; j += n) acc += static_cast<int32_t>(h[j]) * w[j];
    return acc;
}

DH_DEVINL void mma_s8(int32_t (&c)[4], int32_t a0, int32_t a1, int32_t a2, int32_t a3, int32_t b0, int32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The j-th of a group's 8 tokens: of 32 columns of a part (group % 2), in every 8
// the two of the quarter group / 2 % 4.
DH_DEVINL uint32_t group_token(uint32_t group, uint32_t j) {
    return group / kGroupsPerPart * kPartCols + group % 2 * 32 + j / 2 * 8 + group / 2 % 4 * 2 + j % 2;
}

// Integer sums of the 8 tokens of two groups with the hidden row, by a warp: a
// 16 x 8 x 32 MMA whose 16 rows are the tokens and whose 8 columns are all the
// hidden row.  Any order of the k dimension serves as long as both operands
// share it, so a lane loads 16 consecutive bytes of token lane / 4 of both, and
// feeds them to two MMAs.  Every lane receives the sums of these two tokens.
// kUnroll: how many 64 bytes of each row are in flight.
template <uint32_t kUnroll>
DH_DEVINL int2 group_sums(const int8_t* h, const int8_t* w, uint64_t ldw, uint32_t group_a, uint32_t group_b,
                          uint32_t vocab, uint32_t k, uint32_t lane) {
    const uint32_t g = lane / 4, t = lane % 4;
    const int8_t* wa = w + min(group_token(group_a, g), vocab - 1) * ldw;
    const int8_t* wb = w + min(group_token(group_b, g), vocab - 1) * ldw;
    const int4 *pa = reinterpret_cast<const int4*>(wa) + t, *pb = reinterpret_cast<const int4*>(wb) + t;
    const int4* px = reinterpret_cast<const int4*>(h) + t;
    int32_t c[4] = {0, 0, 0, 0};
    const uint32_t vecs = k / 16;
    uint32_t at = 0;
#pragma unroll 1
    for (; at + 4 * kUnroll <= vecs; at += 4 * kUnroll, pa += 4 * kUnroll, pb += 4 * kUnroll, px += 4 * kUnroll) {
        int4 a[kUnroll], b[kUnroll], x[kUnroll];
#pragma unroll
        for (uint32_t u = 0; u < kUnroll; ++u) {
            a[u] = __ldg(pa + 4 * u);
            b[u] = __ldg(pb + 4 * u);
            x[u] = __ldg(px + 4 * u);
        }
#pragma unroll
        for (uint32_t u = 0; u < kUnroll; ++u) {
            mma_s8(c, a[u].x, b[u].x, a[u].y, b[u].y, x[u].x, x[u].y);
            mma_s8(c, a[u].z, b[u].z, a[u].w, b[u].w, x[u].z, x[u].w);
        }
    }
    const int4 none = make_int4(0, 0, 0, 0);
#pragma unroll 1
    for (; at < vecs; at += 4, pa += 4, pb += 4, px += 4) {
        const bool in = at + t < vecs;
        const int4 a = in ? __ldg(pa) : none, b = in ? __ldg(pb) : none, x = in ? __ldg(px) : none;
        mma_s8(c, a.x, b.x, a.y, b.y, x.x, x.y);
        mma_s8(c, a.z, b.z, a.w, b.w, x.z, x.w);
    }
    int2 sums = make_int2(c[0], c[2]);
#pragma unroll 1
    for (uint32_t o = vecs * 16; o < k; ++o) {  // the bytes past the last whole 16
        sums.x += static_cast<int32_t>(wa[o]) * h[o];
        sums.y += static_cast<int32_t>(wb[o]) * h[o];
    }
    return sums;
}

// A row whose scale is infinite or NaN, from end to end.  All of its logits are
// infinite or NaN, so it is empty (each -inf) or has no answer, and mostly the first
// tokens tell.  (The first kernel's statistics of such a row are NaN either way, from
// columns that are no token; setting these to -inf there cost every call 1 to 3%.)
// Out of line, and the row ends with it: hardly a row needs it.  Whole warp.
template <bool kWide>
static __device__ __noinline__ void settle_row(const HeadRowParams& p, uint64_t row) {
    const uint32_t lane = lane_id();
    const int8_t* h = p.hidden + row * p.ld_hidden;
    const float ab = __ldg(p.a_scale + row);
    bool bad = false;
#pragma unroll 1
    for (uint32_t c = lane; c - lane < p.vocab && !bad; c += 32) {
        bool other = false;
        if (c < p.vocab && c != p.mask_id) {
            const int32_t acc = dot_share(h, p.weights + c * p.ld_weights, p.k, 0, 1);
            const float x = score_logit<kWide>(acc, ab, __ldg(p.w_scale + c), p.bias ? __ldg(p.bias + c) : 0.f);
            other = !(x == -CUDART_INF_F);
        }
        bad = __any_sync(kFullMask, other);
    }
    const RowResult r = row_result(-CUDART_INF_F, bad ? CUDART_NAN_F : 0.f, 0.f);
    if (lane == 0) store_row(p.out, row, r);
    store_top(p.out, row, r, 0, lane);
    for (uint32_t i = lane; i < p.out.targets_per_row; i += 32)
        p.out.logprobs[row * p.out.targets_per_row + i] = given_logprob(r, target_of(p.out, row, i), p.vocab, 0.f);
}

constexpr uint32_t kRowWarps = 8;
constexpr uint32_t kMaxStaged = 1025;  // words of shared memory a row: vocabularies up to 131,072
constexpr uint32_t kPicks = 256;  // groups kept for the k best (more, by ties: every group is looked at)
// Rows below which each gets a CTA: 512 rows 43 / 43 us (1 / 8 alternatives)
// against 41 / 51 with a warp each, 1001 rows 66 / 68 against 55 / 66.
constexpr uint32_t kTeamRows = 768;

template <uint32_t kTeam>
struct RowsSmem {
    static constexpr uint32_t kTeams = kRowWarps / kTeam;
    float part_base[kRowWarps], part_s[kRowWarps], part_t[kRowWarps];
    uint64_t keys[kRowWarps][32], lists[kTeam > 1 ? kRowWarps : 1][32];
    uint32_t picks[kTeams][kPicks], pick_count[kTeams];
    uint32_t parts[kRowWarps][160];
    float pairs[kTeam > 1 ? kRowWarps : 1][2][32];
};
static_assert(sizeof(RowsSmem<1>) + kMaxStaged * kRowWarps * sizeof(float) <= 48 * 1024,
              "shared memory of a launch without an opt-in");

// kTeam warps a row: 1 when there are rows enough for every warp of the GPU,
// all of a CTA's when there are few.  kPerSM: CTAs an SM holds, 4, or 2 with the
// registers for more loads in flight (32 rows and 8 alternatives 25.6 against 27.6
// us, 256 rows 31.8 against 33.8; 512 rows, in two turns, 48 against 42).
template <bool kWide, uint32_t kTeam, uint32_t kPerSM>
__global__ void __launch_bounds__(32 * kRowWarps, kPerSM)
head_rows_kernel(const __grid_constant__ HeadRowParams p, const uint32_t staged) {
    extern __shared__ uint32_t staged_max[];  // the part maxima of the CTA's rows, if `staged` holds them: [kTeams][staged]
    constexpr uint32_t kTeams = kRowWarps / kTeam;
    __shared__ RowsSmem<kTeam> sm;

    const uint32_t warp = warp_id(), lane = lane_id();
    const uint32_t team = warp / kTeam, member = warp % kTeam;
    auto team_sync = [] {
        if (kTeam == 1) __syncwarp();
        else __syncthreads();
    };
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * kTeams + team;
    const uint32_t k = p.out.top_k, targets = p.out.targets_per_row;
    const bool have = kTeam > 1 || row < p.split.rows;  // (with teams the grid is the rows)
    const int8_t* h = p.hidden + row * p.ld_hidden;
    const float ab = have ? __ldg(p.a_scale + row) : 0.f;

    auto token_logit = [&](uint32_t c, int32_t acc) {
        if (c == p.mask_id) return -CUDART_INF_F;
        return score_logit<kWide>(acc, ab, __ldg(p.w_scale + c), p.bias ? __ldg(p.bias + c) : 0.f);
    };
    // the logit of given token i, by a whole warp (0 if there is none)
    auto target_logit = [&](uint32_t i, int64_t& t) {
        t = target_of(p.out, row, i);
        if (t < 0 || t >= p.vocab) return 0.f;
        const int32_t acc = __reduce_add_sync(kFullMask, dot_share(h, p.weights + t * p.ld_weights, p.k, lane, 32));
        return token_logit(static_cast<uint32_t>(t), acc);
    };
    // the last members take the first given tokens, the first the k best
    const uint32_t first_target = kTeam - 1 - member;
    int64_t target = -1;
    float target_x = 0.f;
    if (have && first_target < targets) target_x = target_logit(first_target, target);

    // so far the call's inputs alone: now the first kernel has to have ended (what
    // it writes is read by plain loads, not through the read-only path)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t n_part = p.split.all_parts(), n_pair = (n_part + 1) / 2;  // parts in pairs, a word each
    if (staged) {
        // the CTA's 8 rows of a part are 16 bytes
        const uint4* from = reinterpret_cast<const uint4*>(p.part_max) + blockIdx.x;
        const uint64_t pitch = p.split.padded_rows() / 8;
#pragma unroll 2
        for (uint32_t j = threadIdx.x; j < n_pair; j += 32 * kRowWarps) {
            const uint4 none = make_uint4(kNonePair, kNonePair, kNonePair, kNonePair);
            const uint4 u = from[2 * j * pitch], v = 2 * j + 1 < n_part ? from[(2 * j + 1) * pitch] : none;
            const uint32_t lo[4] = {u.x, u.y, u.z, u.w}, hi[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (uint32_t r = 0; r < 8; ++r)
                staged_max[r * staged + j] = __byte_perm(lo[r / 2], hi[r / 2], r % 2 ? 0x7632 : 0x5410);
        }
        __syncthreads();
    }
    if (!have) return;
    if (!(fabsf(ab) < CUDART_INF_F)) {  // the whole team's row
        if (member == 0) settle_row<kWide>(p, row);
        return;
    }

    // the row's partial statistics
    const uint32_t mt = static_cast<uint32_t>(row / kBM), r_in = static_cast<uint32_t>(row % kBM);
    const uint32_t t0 = mt * p.split.n_tiles;
    const uint32_t c_lo = p.split.cta_of(t0), c_hi = p.split.cta_of(t0 + p.split.n_tiles - 1);
    const uint32_t parts = p.split.parts;
    RowStats st{-CUDART_INF_F, 0.f, 0.f};
#pragma unroll 4
    for (uint32_t i = member * 32 + lane; i < (c_hi - c_lo + 1) * parts; i += kTeam * 32) {
        const uint32_t c = c_lo + i / parts;
        const uint32_t seg = mt - p.split.first_tile(c) / p.split.n_tiles;
        const float4 q = p.partials[((static_cast<uint64_t>(c) * p.split.max_segs + seg) * parts + i % parts) * kBM + r_in];
        RowStats o{q.x, q.y, q.z};
        const float m = fmaxf(st.base, o.base);
        rebase(st, m);
        rebase(o, m);
        st.s += o.s;
        st.t += o.t;
    }
    float top = lanes_max(st.base);
    rebase(st, top);
    st.s = warp_sum_f32(st.s);
    st.t = warp_sum_f32(st.t);
    if (kTeam > 1 && lane == 0) {
        sm.part_base[warp] = top;
        sm.part_s[warp] = st.s;
        sm.part_t[warp] = st.t;
    }

    // the k-th largest of the lanes' maxima of parts (the two largest of each)
    // bounds the k-th best logit; the parts are dealt to the members
    constexpr uint32_t kStep = 32 * kTeam;
    const uint32_t* words = staged_max + team * staged;
    const uint16_t* column = p.part_max + row;
    const uint64_t rows_of = p.split.padded_rows();
    // parts 2 j and 2 j + 1; -inf past the last
    auto pair_of = [&](uint32_t j) -> uint32_t {
        if (j >= n_pair) return kNonePair;
        if (staged) return words[j];
        return column[2 * j * rows_of] |
               (2 * j + 1 < n_part ? static_cast<uint32_t>(column[(2 * j + 1) * rows_of]) << 16 : kNonePair << 16);
    };
    float a = -CUDART_INF_F, b = -CUDART_INF_F, bound = -CUDART_INF_F;
    if (k) {
        uint32_t a2 = kNonePair, b2 = kNonePair;
#pragma unroll 1
        for (uint32_t j = member * 32 + lane; j < n_pair; j += 4 * kStep) {
            uint32_t v[4];
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) v[u] = pair_of(j + u * kStep);
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) {
                b2 = max_pairs(b2, min_pairs(a2, v[u]));
                a2 = max_pairs(a2, v[u]);
            }
        }
        a = half_float(a2);
        b = half_float(b2);
        two_largest(a, b, half_float(a2 >> 16));
        two_largest(a, b, half_float(b2 >> 16));
        if (member == 0 && lane == 0) sm.pick_count[team] = 0;
        if (kTeam > 1) {
            sm.pairs[warp][0][lane] = a;
            sm.pairs[warp][1][lane] = b;
        }
    }
    team_sync();
    if (kTeam > 1) {
        st = lane < kRowWarps ? RowStats{sm.part_base[lane], sm.part_s[lane], sm.part_t[lane]} : RowStats{-CUDART_INF_F, 0.f, 0.f};
        top = lanes_max(st.base);
        rebase(st, top);
        st.s = warp_sum_f32(st.s);
        st.t = warp_sum_f32(st.t);
    }
    const RowResult r = row_result(top, st.s, st.t);
    if (member == 0 && lane == 0) store_row(p.out, row, r);
    for (uint32_t i = first_target; i < targets; i += kTeam) {
        if (i != first_target) target_x = target_logit(i, target);
        if (lane == 0) p.out.logprobs[row * targets + i] = given_logprob(r, target, p.vocab, target_x);
    }
    if (!k) return;
    if (kTeam > 1) {
        a = b = -CUDART_INF_F;
#pragma unroll
        for (uint32_t w = 0; w < kRowWarps; ++w) {
            two_largest(a, b, sm.pairs[w][0][lane]);
            two_largest(a, b, sm.pairs[w][1][lane]);
        }
    }
    bound = kth_largest_of_pairs(a, b, k, lane);
    // no logit below `least` rounds to it, no group's byte is below group_bound.  (A
    // bound of zero counts as -0, what logits just below zero round to: the zeros
    // compare equal, so that its sign may be that of another maximum.)
    const uint16_t bits = bound == 0.f ? 0x8000u : __half_as_ushort(__float2half_rz(bound));
    const float least = bits >= 0x8000u && bits < 0xFC00u ? half_float(bits + 1u) : bound;
    const float group_bound = half_float(bits & 0xFF00u);
    auto group_reaches = [&](uint32_t part, uint32_t b) {
        const uint8_t* at = reinterpret_cast<const uint8_t*>(p.group_max + p.split.slot(part, static_cast<uint32_t>(row)));
        const float y = half_float(static_cast<uint32_t>(at[b]) << 8);
        return y >= group_bound && y > -CUDART_INF_F;
    };
    // the groups that reach it
    uint32_t n = 0;
#pragma unroll 1
    for (uint32_t j0 = member * 32; j0 < n_pair; j0 += 2 * kStep) {
        const uint32_t v[2] = {pair_of(j0 + lane), pair_of(j0 + kStep + lane)};
        const uint32_t both = max_pairs(v[0], v[1]);
        const float m = fmaxf(half_float(both), half_float(both >> 16));
        if (__any_sync(kFullMask, m >= bound && m > -CUDART_INF_F)) {
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) {
                const float y = half_float(v[u / 2] >> (u % 2 * 16));
                const uint32_t who = __ballot_sync(kFullMask, y >= bound && y > -CUDART_INF_F);
                if ((who >> lane) & 1u)
                    sm.parts[warp][n + __popc(who & ((1u << lane) - 1u))] = 2 * (j0 + kStep * (u / 2) + lane) + u % 2;
                n += __popc(who);
            }
        }
        if (n > 32 || j0 + 2 * kStep >= n_pair) {
            __syncwarp();
            // the 8 groups of 4 parts at a time
#pragma unroll 1
            for (uint32_t j = lane / 8; j < n + lane / 8; j += 4) {
                const uint32_t part = j < n ? sm.parts[warp][j] : 0u;
                const uint32_t in = __ballot_sync(kFullMask, j < n && group_reaches(part, lane % 8));
                uint32_t to = 0;
                if (lane == 0 && in) to = atomicAdd(&sm.pick_count[team], __popc(in));
                to = __shfl_sync(kFullMask, to, 0) + __popc(in & ((1u << lane) - 1u));
                if (((in >> lane) & 1u) && to < kPicks) sm.picks[team][to] = part * kGroupsPerPart + group_at(lane % 8, row);
            }
            n = 0;
            __syncwarp();
        }
    }
    team_sync();
    // their logits, two groups at a time
    const bool all = sm.pick_count[team] > kPicks;
    const uint32_t n_pick = all ? n_part * kGroupsPerPart : sm.pick_count[team];
    TopList best(sm.keys[warp], k, lane);
#pragma unroll 1
    for (uint32_t i = 2 * member; i < n_pick; i += 2 * kTeam) {
        const bool two = i + 1 < n_pick;
        const uint32_t ga = all ? i : sm.picks[team][i], gb = all ? i + 1 : sm.picks[team][two ? i + 1 : i];
        if (all) {
            const uint32_t part = i / kGroupsPerPart, pair = pair_of(part / 2);
            if (!(half_float(part % 2 ? pair >> 16 : pair) >= bound) ||
                !(group_reaches(part, group_at(ga % kGroupsPerPart, row)) ||
                  group_reaches(part, group_at(gb % kGroupsPerPart, row))))
                continue;
        }
        // lanes with lane % 4 < 2 answer for token lane / 4 of a group each
        const uint32_t c = group_token(lane % 4 & 1u ? gb : ga, lane / 4);
        const bool in = lane % 4 < (two ? 2u : 1u) && c < p.vocab && c != p.mask_id;
        const float w = in ? __ldg(p.w_scale + c) : 0.f, b = in && p.bias ? __ldg(p.bias + c) : 0.f;
        const int2 acc = group_sums<kPerSM == 2 ? 6 : 3>(h, p.weights, p.ld_weights, ga, gb, p.vocab, p.k, lane);
        const float x = score_logit<kWide>(lane % 4 ? acc.y : acc.x, ab, w, b);
        best.add(in && x >= least && x > -CUDART_INF_F ? token_key(x, c) : 0ull);
    }
    best.flush();
    if (kTeam > 1) {
        sm.lists[warp][lane] = best.list;
        __syncthreads();
        if (member != 0) return;
        uint64_t least_of = 0;
        for (uint32_t w = 0; w < kTeam; ++w) least_of = sm.lists[w][k - 1] > least_of ? sm.lists[w][k - 1] : least_of;
        TopList all(sm.keys[warp], k, lane);
        for (uint32_t w = 0; w < kTeam; ++w) all.add(sm.lists[w][lane] >= least_of ? sm.lists[w][lane] : 0ull);
        all.flush();
        best.list = all.list;
    }
    store_top(p.out, row, r, best.list, lane);
}

constexpr uint64_t align256(uint64_t v) { return (v + 255) / 256 * 256; }

uint64_t tiles_of(uint32_t rows, uint32_t vocab, uint32_t cols) {
    return static_cast<uint64_t>((rows + kBM - 1) / kBM) * ((vocab + cols - 1) / cols);
}

// Tiles of 256 columns, or of 192 where the longest span of a CTA becomes shorter by
// more than they cost: 32 x 50258 (2 of 192 or 2 of 256) 19.5 against 23.5 us, 32768
// rows (454 or 341) 963 against 888.
HeadSplit split_of(uint32_t rows, uint32_t vocab, uint32_t sms) {
    auto columns = [&](uint32_t cols) { return (tiles_of(rows, vocab, cols) + sms - 1) / sms * cols; };
    HeadSplit s{};
    s.rows = rows;
    s.cols = columns(192) * 10 < columns(256) * 9 ? 192 : 256;
    s.n_tiles = (vocab + s.cols - 1) / s.cols;
    s.parts = s.cols / kPartCols;
    const uint32_t total = static_cast<uint32_t>(tiles_of(rows, vocab, s.cols));
    s.grid = total < sms ? total : sms;
    s.each = total / s.grid;
    s.more = total % s.grid;
    // a span of that many tiles touches at most this many row tiles
    s.max_segs = (s.each + (s.more ? 1 : 0) + s.n_tiles - 2) / s.n_tiles + 1;
    return s;
}

uint64_t partial_bytes(const HeadSplit& s) {
    return align256(static_cast<uint64_t>(s.grid) * s.max_segs * s.parts * kBM * sizeof(float4));
}

uint64_t group_bytes(const HeadSplit& s) {
    return align256(s.padded_rows() * s.all_parts() * sizeof(uint2));
}
uint64_t part_max_bytes(const HeadSplit& s) {
    return align256(s.padded_rows() * s.all_parts() * sizeof(uint16_t));
}

template <uint32_t kBN, bool kWide, bool kResident, bool kTop>
cudaError_t launch_stats(const CUtensorMap& ta, const CUtensorMap& tb, HeadScoreParams p, cudaStream_t s) {
    using Tile = HeadTile<kBN>;
    static std::atomic<uint64_t> configured{0};
    auto kernel = head_stats_kernel<kWide, kResident, kTop, kBN>;
    const cudaError_t e = smem_optin_once(kernel, kSmemLimit, configured);
    if (e != cudaSuccess) return e;
    const uint32_t k_blocks = (p.k + kBK - 1) / kBK;
    p.stages = kResident ? Tile::resident_stages(k_blocks) : kStreamedStages;
    const uint32_t smem = Tile::kFixed + (kResident ? k_blocks : p.stages) * kABytes + p.stages * Tile::kBBytes;
    kernel<<<p.split.grid, Tile::kThreads, smem, s>>>(ta, tb, p);
    return cudaGetLastError();
}

template <uint32_t kBN>
cudaError_t launch_stats(const CUtensorMap& ta, const CUtensorMap& tb, const HeadScoreParams& p, bool wide, cudaStream_t s) {
    if (wide) return p.group_max ? launch_stats<kBN, true, false, true>(ta, tb, p, s)
                                 : launch_stats<kBN, true, false, false>(ta, tb, p, s);
    if (p.k <= kResidentK) return p.group_max ? launch_stats<kBN, false, true, true>(ta, tb, p, s)
                                              : launch_stats<kBN, false, true, false>(ta, tb, p, s);
    return p.group_max ? launch_stats<kBN, false, false, true>(ta, tb, p, s)
                       : launch_stats<kBN, false, false, false>(ta, tb, p, s);
}

}  // namespace
}  // namespace dh

using namespace dh;

extern "C" size_t dh_head_logprobs_workspace_size(uint32_t rows, uint32_t vocabulary_size, uint32_t top_k) {
    if (rows == 0 || vocabulary_size == 0 || tiles_of(rows, vocabulary_size, 192) > kMaxTiles) return 0;
    const HeadSplit s = split_of(rows, vocabulary_size, device_sms());
    return partial_bytes(s) + (top_k ? group_bytes(s) + part_max_bytes(s) : 0u);
}

extern "C" uint32_t dh_head_logprobs_i8(const int8_t* hidden, uint64_t ld_hidden, const float* a_scale,
                                        const int8_t* weights, uint64_t ld_weights, const float* w_scale,
                                        const float* bias, uint32_t rows, uint32_t hidden_size,
                                        uint32_t vocabulary_size, uint32_t mask_token_id, const void* targets,
                                        uint32_t target_bytes, uint32_t targets_per_row, uint32_t top_k,
                                        float* logprobs, float* entropy, float* logsumexp, int32_t* top_ids,
                                        float* top_logprobs, void* workspace, size_t workspace_bytes,
                                        void* stream) {
    if (rows == 0) return DH_HEAD_INVALID_POSITION_COUNT;
    if (hidden_size == 0) return DH_HEAD_INVALID_HIDDEN_SIZE;
    if (vocabulary_size == 0) return DH_HEAD_INVALID_VOCABULARY_SIZE;
    if (mask_token_id != DH_NO_TOKEN && mask_token_id >= vocabulary_size) return DH_HEAD_INVALID_MASK_TOKEN;
    // (first of these, as the workspace query has no size for such shapes)
    if (top_k > kMaxTopK || hidden_size > 131071 || rows > (1u << 24) || vocabulary_size > (1u << 24) ||
        tiles_of(rows, vocabulary_size, 192) > kMaxTiles)
        return DH_ERR_UNSUPPORTED_SHAPE;
    if (!hidden || !a_scale || !weights || !w_scale || !workspace) return DH_ERR_NULL_POINTER;
    const ScoreOutputs out{logprobs, entropy, logsumexp, top_ids, top_logprobs, targets,
                           targets_per_row, target_bytes, top_k};
    uint32_t st = check_score_outputs(out);
    if (st != DH_OK) return st;
    const HeadSplit split = split_of(rows, vocabulary_size, device_sms());
    if (((reinterpret_cast<uintptr_t>(a_scale) | reinterpret_cast<uintptr_t>(w_scale) |
          reinterpret_cast<uintptr_t>(bias)) & 3u) || (reinterpret_cast<uintptr_t>(workspace) & 255u))
        return DH_ERR_ALIGNMENT;
    if (workspace_bytes < dh_head_logprobs_workspace_size(rows, vocabulary_size, top_k)) return DH_ERR_WORKSPACE;
    CUtensorMap ta, tb;
    st = make_i8_operand_maps(&ta, &tb, hidden, ld_hidden, weights, ld_weights, rows, vocabulary_size,
                              hidden_size, split.cols);
    if (st != DH_OK) return st;
    const bool wide = hidden_size > kExactK;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    float4* partials = static_cast<float4*>(workspace);
    uint8_t* maxima = static_cast<uint8_t*>(workspace) + partial_bytes(split);
    uint2* group_max = top_k ? reinterpret_cast<uint2*>(maxima) : nullptr;
    uint16_t* part_max = top_k ? reinterpret_cast<uint16_t*>(maxima + group_bytes(split)) : nullptr;
    const HeadScoreParams sp{split, vocabulary_size, mask_token_id, hidden_size, 0, a_scale, w_scale, bias,
                             partials, group_max, part_max};
    const cudaError_t e = split.cols == 192 ? launch_stats<192>(ta, tb, sp, wide, s) : launch_stats<256>(ta, tb, sp, wide, s);
    if (e != cudaSuccess) return DH_ERR_CUDA;
    const HeadRowParams rp{split, vocabulary_size, mask_token_id, hidden_size, hidden, ld_hidden, weights,
                           ld_weights, a_scale, w_scale, bias, partials, group_max, part_max, out};
    const bool team = rows < kTeamRows;
    const bool deep = rows <= 2 * device_sms();
    auto rows_kernel =
        wide ? (team ? (deep ? head_rows_kernel<true, kRowWarps, 2> : head_rows_kernel<true, kRowWarps, 4>)
                     : head_rows_kernel<true, 1, 4>)
             : (team ? (deep ? head_rows_kernel<false, kRowWarps, 2> : head_rows_kernel<false, kRowWarps, 4>)
                     : head_rows_kernel<false, 1, 4>);
    // the part maxima of 8 rows, each row's 1 mod 2 words apart, where they fit
    uint32_t staged = ((split.all_parts() + 1) / 2) | 1u;
    if (!top_k || team || staged > kMaxStaged) staged = 0;
    // (its launch and its given tokens' logits overlap the first kernel's end: 32 rows
    // 21.5 against 23.5 us, 1001 rows and 8 alternatives 64.5 against 66.6)
    cudaLaunchAttribute overlap{};
    overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    overlap.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t launch{};
    launch.gridDim = team ? rows : (rows + kRowWarps - 1) / kRowWarps;
    launch.blockDim = 32 * kRowWarps;
    launch.dynamicSmemBytes = staged * kRowWarps * sizeof(uint32_t);
    launch.stream = s;
    launch.attrs = &overlap;
    launch.numAttrs = 1;
    return cudaLaunchKernelEx(&launch, rows_kernel, rp, staged) == cudaSuccess ? DH_OK : DH_ERR_CUDA;
}
