// head_scores.cu -- the int8 output head fused with the scores of its rows
// (log probabilities of given tokens, entropy, logsumexp, the k best tokens);
// logits never reach HBM.  Two kernels:
//
// 1. head_stats_kernel: the persistent, warp-specialised int8 GEMM of
//    gemm_tc.cuh's structure (TMA ring, one MMA thread, accumulators double
//    buffered in TMEM), whose epilogue threads each own a row and turn its
//    accumulators into logits x = fp32(acc * fp32(a_scale w_scale) + bias) and
//    these into running softmax statistics (row_scores.cuh).  A CTA walks a
//    contiguous span of tiles in (row tile, column tile) order, so that a
//    thread's statistics stay in registers until the row tile changes.  For
//    the k best tokens it stores only maxima: of each group of 16 logits and
//    of each 128 (half a tile).  The k best lie in the k groups of largest
//    maximum (earlier group first among equals), since each of those holds a
//    logit at least as good.
// 2. head_rows_kernel: joins a row's partial statistics, picks the k groups
//    through the larger maxima, and computes their 16 logits again (the same
//    fp32 expression of the same integer sum, so the same bits), like the given
//    tokens' logits.
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

constexpr uint32_t kBM = 128, kBN = 256, kBK = 128;
constexpr uint32_t kHeadStages = 4;
constexpr uint32_t kABytes = kBM * kBK, kBBytes = kBN * kBK;
constexpr uint32_t kEpiWarps = 16;                      // two groups of 8, one per TMEM buffer
constexpr uint32_t kHeadThreads = 64 + 32 * kEpiWarps;
constexpr uint32_t kHalfCols = kBN / 2;                 // columns of an epilogue warp
constexpr uint32_t kGroup = 16;                         // logits per stored maximum
constexpr uint32_t kGroupsPerTile = kBN / kGroup;
constexpr uint32_t kGroupsPerHalf = kHalfCols / kGroup;
constexpr uint32_t kBarBytes = 1024;
constexpr uint32_t kStagePerWarp = kHalfCols * 8;       // bias and w_scale of the warp's columns
constexpr uint32_t kHeadSmem =
    1024 + kHeadStages * (kABytes + kBBytes) + kBarBytes + kEpiWarps * kStagePerWarp;
// float(acc) is exact up to 2^24: k products of magnitude 127 * 127 (128 * 128)
constexpr uint32_t kExactK = 1024;

// How a launch splits the work: shared by the two kernels.
struct HeadSplit {
    uint32_t rows, n_tiles, grid, max_segs;
    uint64_t total;  // row tiles * n_tiles
    __host__ __device__ uint64_t first_tile(uint32_t cta) const { return total * cta / grid; }
    // the CTA that holds tile t: the last with first_tile <= t
    __host__ __device__ uint32_t cta_of(uint64_t t) const {
        return static_cast<uint32_t>(((t + 1) * grid - 1) / total);
    }
};

struct HeadScoreParams {
    HeadSplit split;
    uint32_t vocab, mask_id, k;
    const float* a_scale;
    const float* w_scale;
    const float* bias;   // or null
    float4* partials;    // [grid][max_segs][4][128]: base, s, t of a row's part
    float* group_max;    // [rows][n_tiles * 16], or null: none asked for
    float* half_max;     // [rows][n_tiles * 2]
};

// The logit of one accumulator.  kWide: k > kExactK, where float(acc) would
// round and the expression is evaluated in float64.
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

// 32 accumulators of one row: add to the statistics, return the maxima of
// the two groups.  kClamp: some logit may be -inf (or NaN).
template <bool kWide, bool kClamp>
DH_DEVINL float2 add_chunk(RowStats& st, bool& seen, const uint32_t* v, float ab, const float* ws, const float* bs) {
    float2 x[16];
    const float2 ab2 = make_float2(ab, ab);
#pragma unroll
    for (uint32_t j = 0; j < 16; j += 2) {
        const float4 w = *reinterpret_cast<const float4*>(ws + 2 * j);
        const float4 b = *reinterpret_cast<const float4*>(bs + 2 * j);
        if (kWide) {
            x[j] = make_float2(ref_logit(static_cast<int32_t>(v[2 * j]), ab, w.x, b.x),
                               ref_logit(static_cast<int32_t>(v[2 * j + 1]), ab, w.y, b.y));
            x[j + 1] = make_float2(ref_logit(static_cast<int32_t>(v[2 * j + 2]), ab, w.z, b.z),
                                   ref_logit(static_cast<int32_t>(v[2 * j + 3]), ab, w.w, b.w));
        } else {
            const float2 a0 = make_float2(static_cast<float>(static_cast<int32_t>(v[2 * j])),
                                          static_cast<float>(static_cast<int32_t>(v[2 * j + 1])));
            const float2 a1 = make_float2(static_cast<float>(static_cast<int32_t>(v[2 * j + 2])),
                                          static_cast<float>(static_cast<int32_t>(v[2 * j + 3])));
            x[j] = __ffma2_rn(a0, __fmul2_rn(ab2, make_float2(w.x, w.y)), make_float2(b.x, b.y));
            x[j + 1] = __ffma2_rn(a1, __fmul2_rn(ab2, make_float2(w.z, w.w)), make_float2(b.z, b.w));
        }
    }
    float gm[2];
#pragma unroll
    for (uint32_t g = 0; g < 2; ++g) {
        float a = fmaxf(x[8 * g].x, x[8 * g].y), b = fmaxf(x[8 * g + 1].x, x[8 * g + 1].y);
#pragma unroll
        for (uint32_t j = 2; j < 8; j += 2) {
            a = max3(a, x[8 * g + j].x, x[8 * g + j].y);
            b = max3(b, x[8 * g + j + 1].x, x[8 * g + j + 1].y);
        }
        gm[g] = fmaxf(a, b);
    }
    const float cm = fmaxf(gm[0], gm[1]);
    if (cm > st.base + kBaseSlack || (!seen && cm > -CUDART_INF_F)) {
        rebase(st, cm);
        seen = true;
    }
    // the chunk's own sums first: a thread adds thousands of logits, and one
    // long chain of fp32 additions would lose two digits
    const float2 nb = make_float2(-st.base, -st.base);
    const float2 c2 = make_float2(kLog2E, kLog2E);
    float2 s = make_float2(0.f, 0.f), t = make_float2(0.f, 0.f);
#pragma unroll
    for (uint32_t j = 0; j < 16; ++j) {
        float2 d = __fadd2_rn(x[j], nb);
        if (kClamp) d = make_float2(max_nan(d.x, -1e30f), max_nan(d.y, -1e30f));
        const float2 z = __fmul2_rn(d, c2);
        const float2 e = make_float2(exp2_fast(z.x), exp2_fast(z.y));
        s = __fadd2_rn(s, e);
        t = __ffma2_rn(e, d, t);
    }
    st.s += s.x + s.y;
    st.t += t.x + t.y;
    return make_float2(gm[0], gm[1]);
}

template <bool kWide>
__global__ void __launch_bounds__(kHeadThreads, 1)
head_stats_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                  const __grid_constant__ HeadScoreParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~static_cast<uintptr_t>(1023));
    uint8_t* a_smem = smem;
    uint8_t* b_smem = smem + kHeadStages * kABytes;
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(b_smem + kHeadStages * kBBytes);
    uint64_t* empty_bar = full_bar + kHeadStages;
    uint64_t* accf_bar = empty_bar + kHeadStages;  // [2]
    uint64_t* acce_bar = accf_bar + 2;             // [2]
    uint64_t* drain_bar = acce_bar + 2;            // [1]
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain_bar + 1);
    uint8_t* staging = reinterpret_cast<uint8_t*>(full_bar) + kBarBytes;

    const uint32_t warp = warp_id(), lane = lane_id();
    if (warp == 0 && lane == 0) {
        for (uint32_t s = 0; s < kHeadStages; ++s) {
            tc::mbar_init(&full_bar[s], 1);
            tc::mbar_init(&empty_bar[s], 1);
        }
        for (uint32_t b = 0; b < 2; ++b) {
            tc::mbar_init(&accf_bar[b], 1);
            tc::mbar_init(&acce_bar[b], 8 * 32);  // one group of 8 warps drains a buffer
        }
        tc::mbar_init(drain_bar, 1);
        tc::fence_barrier_init();
        tc::prefetch_tmap(&tmap_a);
        tc::prefetch_tmap(&tmap_b);
    }
    if (warp == 1) tc::tmem_alloc(tmem_holder, 2 * kBN);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem_base = *tmem_holder;

    const uint32_t n_tiles = p.split.n_tiles;
    const uint32_t k_blocks = (p.k + kBK - 1) / kBK;
    const uint32_t tile0 = static_cast<uint32_t>(p.split.first_tile(blockIdx.x));
    const uint32_t tile1 = static_cast<uint32_t>(p.split.first_tile(blockIdx.x + 1));

    if (warp == 0) {
        // ------------------------------------------------------ TMA producer
        if (tc::elect_one()) {
            uint32_t stage = 0, phase = 0, issued = 0;
            uint32_t issued_parity[kHeadStages];
            bool ok = true;
            for (uint32_t tile = tile0; tile < tile1 && ok; ++tile) {
                const uint32_t m0 = (tile / n_tiles) * kBM, n0 = (tile % n_tiles) * kBN;
                for (uint32_t kb = 0; kb < k_blocks; ++kb) {
                    if (!tc::mbar_wait(&empty_bar[stage], phase ^ 1, tc::kErrTimeoutEmpty)) {
                        ok = false;
                        break;
                    }
                    tc::mbar_arrive_expect_tx(&full_bar[stage], kABytes + kBBytes);
                    tc::tma_load_2d(a_smem + stage * kABytes, &tmap_a, &full_bar[stage],
                                    static_cast<int32_t>(kb * kBK), static_cast<int32_t>(m0));
                    tc::tma_load_2d(b_smem + stage * kBBytes, &tmap_b, &full_bar[stage],
                                    static_cast<int32_t>(kb * kBK), static_cast<int32_t>(n0));
                    issued_parity[stage] = phase;
                    ++issued;
                    if (++stage == kHeadStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            // Drain: every copy this CTA issued has landed before it may exit.
            const uint32_t last = issued < kHeadStages ? issued : kHeadStages;
            for (uint32_t i = 0; i < last; ++i) {
                const uint32_t s = (stage + kHeadStages - 1 - i) % kHeadStages;
                tc::mbar_wait(&full_bar[s], issued_parity[s], tc::kErrTimeoutFull);
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------- MMA issuer
        if (tc::elect_one()) {
            constexpr uint32_t idesc = tc::idesc_i8_s32<kBM, kBN>();
            uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
            bool ok = true;
            for (uint32_t tile = tile0; tile < tile1 && ok; ++tile) {
                if (!tc::mbar_wait(&acce_bar[acc], acc_phase ^ 1, tc::kErrTimeoutAccEmpty)) break;
                tc::tc_fence_after();
                const uint32_t d_tmem = tmem_base + acc * kBN;
                for (uint32_t kb = 0; kb < k_blocks; ++kb) {
                    if (!tc::mbar_wait(&full_bar[stage], phase, tc::kErrTimeoutFull)) {
                        ok = false;
                        break;
                    }
                    tc::tc_fence_after();
                    const uint64_t a_desc = tc::smem_desc_sw128(a_smem + stage * kABytes);
                    const uint64_t b_desc = tc::smem_desc_sw128(b_smem + stage * kBBytes);
#pragma unroll
                    for (uint32_t kk = 0; kk < kBK / 32; ++kk)
                        tc::mma_i8(d_tmem, tc::desc_advance(a_desc, kk * 32), tc::desc_advance(b_desc, kk * 32),
                                   idesc, (kb | kk) != 0u);
                    tc::mma_commit(&empty_bar[stage]);
                    if (++stage == kHeadStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (!ok) break;
                tc::mma_commit(&accf_bar[acc]);
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
        const uint32_t ew = warp - 2, group = ew / 8u, quad = warp & 3u, half = (ew >> 2) & 1u;
        float* bs = reinterpret_cast<float*>(staging + ew * kStagePerWarp);
        float* ws = bs + kHalfCols;
        const uint32_t mt0 = tile0 / n_tiles;
        const uint64_t pitch = static_cast<uint64_t>(n_tiles) * kGroupsPerTile;
        RowStats st{0.f, 0.f, 0.f};
        bool seen = false;
        uint32_t seg = 0;
        auto flush = [&]() {
            float4* dst = p.partials +
                          ((static_cast<uint64_t>(blockIdx.x) * p.split.max_segs + seg) * 4 + group * 2 + half) * kBM +
                          quad * 32 + lane;
            *dst = make_float4(seen ? st.base : -CUDART_INF_F, st.s, st.t, 0.f);
            st = RowStats{0.f, 0.f, 0.f};
            seen = false;
            ++seg;
        };
        uint32_t phase = 0;
        for (uint32_t tile = tile0 + group; tile < tile1; tile += 2) {
            const uint32_t mt = tile / n_tiles, nt = tile % n_tiles;
            while (seg < mt - mt0) flush();
            const uint32_t row = mt * kBM + quad * 32 + lane;
            const bool row_ok = row < p.split.rows;
            const float ab = row_ok ? __ldg(p.a_scale + row) : 0.f;
            // this warp's columns: excluded ones (past the vocabulary, the
            // masked token) get a logit of -inf from a scale of 0 and that bias
            __syncwarp();
            bool odd = !(fabsf(ab) < 1e11f);
#pragma unroll
            for (uint32_t i = 0; i < kHalfCols; i += 32) {
                const uint32_t c = nt * kBN + half * kHalfCols + i + lane;
                float w = 0.f, b = -CUDART_INF_F;
                if (c < p.vocab && c != p.mask_id) {
                    w = __ldg(p.w_scale + c);
                    b = p.bias ? __ldg(p.bias + c) : 0.f;
                }
                bs[i + lane] = b;
                ws[i + lane] = w;
                // within these no logit overflows, so no difference of two is
                // infinite or NaN
                odd = odd || !(fabsf(b) < 1e37f && fabsf(w) < 1e18f);
            }
            odd = __any_sync(kFullMask, odd);
            if (!tc::mbar_wait(&accf_bar[group], phase, tc::kErrTimeoutAccFull)) break;
            tc::tc_fence_after();
            float* gm = p.group_max && row_ok
                            ? p.group_max + row * pitch + nt * kGroupsPerTile + half * (kHalfCols / kGroup)
                            : nullptr;
            float hm = -CUDART_INF_F;
            const uint32_t taddr = tmem_base + ((quad * 32u) << 16) + group * kBN + half * kHalfCols;
#pragma unroll 1
            for (uint32_t c = 0; c < kHalfCols; c += 32) {
                uint32_t v[32];
                tc::tmem_ld_32x32b_x32(taddr + c, v);
                tc::tmem_ld_wait();
                const float2 g = odd ? add_chunk<kWide, true>(st, seen, v, ab, ws + c, bs + c)
                                     : add_chunk<kWide, false>(st, seen, v, ab, ws + c, bs + c);
                hm = fmaxf(hm, fmaxf(g.x, g.y));
                if (gm) *reinterpret_cast<float2*>(gm + c / kGroup) = g;
            }
            if (gm) p.half_max[row * static_cast<uint64_t>(n_tiles * 2) + nt * 2 + half] = hm;
            tc::tc_fence_before();
            tc::mbar_arrive(&acce_bar[group]);
            phase ^= 1;
        }
        const uint32_t segs = tile1 > tile0 ? (tile1 - 1) / n_tiles - mt0 + 1 : 0u;
        while (seg < segs) flush();
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem_base, 2 * kBN);
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
    const float* group_max;
    const float* half_max;
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

// Integer sums of the 16 tokens of a group with the hidden row, by a warp: a
// 16 x 8 x 32 MMA whose 16 rows are the tokens and whose first column is the
// hidden row (the other 7 are 0).  Any order of the k dimension serves as long
// as both operands share it, so a lane loads 16 consecutive bytes of token
// lane / 4 and of the one 8 further on, and feeds them to two MMAs.  Lanes with
// lane % 4 == 0 return the sums of tokens lane / 4 (x) and lane / 4 + 8 (y).
DH_DEVINL int2 group_sums(const int8_t* h, const int8_t* w, uint64_t ldw, uint32_t first, uint32_t vocab, uint32_t k,
                          uint32_t lane) {
    const uint32_t g = lane / 4, t = lane % 4;
    const int8_t* wa = w + min(first + g, vocab - 1) * ldw;
    const int8_t* wb = w + min(first + g + 8, vocab - 1) * ldw;
    const int4 none = make_int4(0, 0, 0, 0);
    int32_t c[4] = {0, 0, 0, 0};
    const uint32_t whole = k & ~15u;
    constexpr uint32_t kUnroll = 4;  // of 64 bytes a row: 8 loads a lane in flight
#pragma unroll 1
    for (uint32_t at = t * 16; at < whole + t * 16; at += 64 * kUnroll) {
        int4 a[kUnroll], b[kUnroll], x[kUnroll];
#pragma unroll
        for (uint32_t u = 0; u < kUnroll; ++u) {
            const uint32_t o = at + 64 * u;
            const bool in = o < whole;
            a[u] = in ? __ldg(reinterpret_cast<const int4*>(wa + o)) : none;
            b[u] = in ? __ldg(reinterpret_cast<const int4*>(wb + o)) : none;
            x[u] = in && g == 0 ? __ldg(reinterpret_cast<const int4*>(h + o)) : none;
        }
#pragma unroll
        for (uint32_t u = 0; u < kUnroll; ++u) {
            mma_s8(c, a[u].x, b[u].x, a[u].y, b[u].y, x[u].x, x[u].y);
            mma_s8(c, a[u].z, b[u].z, a[u].w, b[u].w, x[u].z, x[u].w);
        }
    }
    if (whole < k) {  // the bytes past the last whole 16
        int4 a = none, b = none, x = none;
        if (t == 0) {
#pragma unroll 1
            for (uint32_t o = whole; o < k; ++o) {
                const uint32_t sh = 8 * (o % 4), i = (o - whole) / 4;
                const int32_t va = static_cast<int32_t>(static_cast<uint8_t>(wa[o])) << sh;
                const int32_t vb = static_cast<int32_t>(static_cast<uint8_t>(wb[o])) << sh;
                const int32_t vx = g == 0 ? static_cast<int32_t>(static_cast<uint8_t>(h[o])) << sh : 0;
                if (i == 0) { a.x |= va; b.x |= vb; x.x |= vx; }
                else if (i == 1) { a.y |= va; b.y |= vb; x.y |= vx; }
                else if (i == 2) { a.z |= va; b.z |= vb; x.z |= vx; }
                else { a.w |= va; b.w |= vb; x.w |= vx; }
            }
        }
        mma_s8(c, a.x, b.x, a.y, b.y, x.x, x.y);
        mma_s8(c, a.z, b.z, a.w, b.w, x.z, x.w);
    }
    return make_int2(c[0], c[2]);
}

constexpr uint32_t kRowWarps = 8;
constexpr uint32_t kTeamRows = 2048;  // fewer rows: a CTA each

// kTeam warps a row: 1 when there are rows enough for every warp of the GPU,
// all of a CTA's when there are few.
template <bool kWide, uint32_t kTeam>
__global__ void __launch_bounds__(32 * kRowWarps, 3)
head_rows_kernel(const __grid_constant__ HeadRowParams p) {
    constexpr uint32_t kTeams = kRowWarps / kTeam;
    __shared__ float part_base[kRowWarps], part_s[kRowWarps], part_t[kRowWarps];
    __shared__ uint64_t keys[kRowWarps][32], lists[kRowWarps][32];
    __shared__ uint64_t groups[kTeams][32];
    __shared__ uint32_t halves[kTeams][64];

    const uint32_t warp = warp_id(), lane = lane_id();
    const uint32_t team = warp / kTeam, member = warp % kTeam;
    auto team_sync = [] {
        if (kTeam == 1) __syncwarp();
        else __syncthreads();
    };
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * kTeams + team;
    if (kTeam == 1 && row >= p.split.rows) return;  // (otherwise the grid is the rows)
    const uint32_t k = p.out.top_k, targets = p.out.targets_per_row;
    const int8_t* h = p.hidden + row * p.ld_hidden;
    const float ab = __ldg(p.a_scale + row);

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
    if (first_target < targets) target_x = target_logit(first_target, target);

    // the row's partial statistics
    const uint32_t mt = static_cast<uint32_t>(row / kBM), r_in = static_cast<uint32_t>(row % kBM);
    const uint64_t t0 = static_cast<uint64_t>(mt) * p.split.n_tiles;
    const uint32_t c_lo = p.split.cta_of(t0), c_hi = p.split.cta_of(t0 + p.split.n_tiles - 1);
    RowStats st{-CUDART_INF_F, 0.f, 0.f};
#pragma unroll 4
    for (uint32_t i = member * 32 + lane; i < (c_hi - c_lo + 1) * 4; i += kTeam * 32) {
        const uint32_t c = c_lo + i / 4;
        const uint32_t seg = mt - static_cast<uint32_t>(p.split.first_tile(c) / p.split.n_tiles);
        const float4 q = __ldg(p.partials + ((static_cast<uint64_t>(c) * p.split.max_segs + seg) * 4 + i % 4) * kBM + r_in);
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
        part_base[warp] = top;
        part_s[warp] = st.s;
        part_t[warp] = st.t;
    }

    if (k && member == 0) {
        // the k best groups: those of the half tiles that reach the k-th
        // largest of the lanes' maxima (the two largest of each)
        const uint32_t n_half = p.split.n_tiles * 2;
        const float* hm = p.half_max + row * n_half;
        const float* gm = p.group_max + row * n_half * kGroupsPerHalf;
        float a = -CUDART_INF_F, b = -CUDART_INF_F;
#pragma unroll 8
        for (uint32_t i = lane; i < n_half; i += 32) two_largest(a, b, __ldg(hm + i));
        const float bound = kth_largest_of_pairs(a, b, k, lane);
        TopList best(keys[warp], k, lane);
        uint32_t n = 0;
#pragma unroll 1
        for (uint32_t i0 = 0; i0 < n_half; i0 += 32) {
            const float v = i0 + lane < n_half ? __ldg(hm + i0 + lane) : -CUDART_INF_F;
            const uint32_t who = __ballot_sync(kFullMask, v >= bound && v > -CUDART_INF_F);
            if ((who >> lane) & 1u) halves[team][n + __popc(who & ((1u << lane) - 1u))] = i0 + lane;
            n += __popc(who);
            if (n > 32 || i0 + 32 >= n_half) {
                __syncwarp();
                // 8 groups of 4 half tiles at a time
#pragma unroll 1
                for (uint32_t j = lane / 8; j < n + lane / 8; j += 4) {
                    const uint32_t id = j < n ? halves[team][j] * kGroupsPerHalf + lane % 8 : 0u;
                    const float y = j < n ? __ldg(gm + id) : -CUDART_INF_F;
                    best.add(y >= bound && y > -CUDART_INF_F ? token_key(y, id) : 0ull);
                }
                n = 0;
                __syncwarp();
            }
        }
        best.flush();
        groups[team][lane] = best.list;
    }
    team_sync();
    if (kTeam > 1) {
        st = lane < kRowWarps ? RowStats{part_base[lane], part_s[lane], part_t[lane]} : RowStats{-CUDART_INF_F, 0.f, 0.f};
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
    // the groups' logits; the k-th group's maximum bounds the k-th best
    const uint64_t least = groups[team][k - 1];
    const float bound = least ? key_logit(least) : -CUDART_INF_F;
    TopList best(keys[warp], k, lane);
    for (uint32_t i = member; i < k && groups[team][i]; i += kTeam) {
        const uint32_t first = packed_id(groups[team][i]) * kGroup;
        const int2 acc = group_sums(h, p.weights, p.ld_weights, first, p.vocab, p.k, lane);
#pragma unroll
        for (uint32_t e = 0; e < 2; ++e) {
            const uint32_t c = first + lane / 4 + 8 * e;
            const float x = lane % 4 == 0 && c < p.vocab ? token_logit(c, e ? acc.y : acc.x) : -CUDART_INF_F;
            best.add(x >= bound && x > -CUDART_INF_F ? token_key(x, c) : 0ull);
        }
    }
    best.flush();
    if (kTeam > 1) {
        lists[warp][lane] = best.list;
        __syncthreads();
        if (member != 0) return;
        uint64_t least_of = 0;
        for (uint32_t w = 0; w < kTeam; ++w) least_of = lists[w][k - 1] > least_of ? lists[w][k - 1] : least_of;
        TopList all(keys[warp], k, lane);
        for (uint32_t w = 0; w < kTeam; ++w) all.add(lists[w][lane] >= least_of ? lists[w][lane] : 0ull);
        all.flush();
        best.list = all.list;
    }
    store_top(p.out, row, r, best.list, lane);
}

constexpr uint64_t align256(uint64_t v) { return (v + 255) / 256 * 256; }

HeadSplit split_of(uint32_t rows, uint32_t vocab, uint32_t sms) {
    HeadSplit s{};
    s.rows = rows;
    s.n_tiles = (vocab + kBN - 1) / kBN;
    s.total = static_cast<uint64_t>((rows + kBM - 1) / kBM) * s.n_tiles;
    s.grid = static_cast<uint32_t>(std::min<uint64_t>(s.total, sms));
    // a span of ceil(total / grid) tiles touches at most this many row tiles
    s.max_segs = static_cast<uint32_t>(((s.total + s.grid - 1) / s.grid + s.n_tiles - 2) / s.n_tiles + 1);
    return s;
}

uint64_t partial_bytes(const HeadSplit& s) {
    return align256(static_cast<uint64_t>(s.grid) * s.max_segs * 4 * kBM * sizeof(float4));
}

uint64_t group_bytes(const HeadSplit& s) {
    return align256(static_cast<uint64_t>(s.rows) * s.n_tiles * kGroupsPerTile * sizeof(float));
}
uint64_t half_bytes(const HeadSplit& s) {
    return align256(static_cast<uint64_t>(s.rows) * s.n_tiles * 2 * sizeof(float));
}

}  // namespace
}  // namespace dh

using namespace dh;

extern "C" size_t dh_head_logprobs_workspace_size(uint32_t rows, uint32_t vocabulary_size, uint32_t top_k) {
    if (rows == 0 || vocabulary_size == 0) return 0;
    const HeadSplit s = split_of(rows, vocabulary_size, device_sms());
    return partial_bytes(s) + (top_k ? group_bytes(s) + half_bytes(s) : 0u);
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
    if (!hidden || !a_scale || !weights || !w_scale || !workspace) return DH_ERR_NULL_POINTER;
    const ScoreOutputs out{logprobs, entropy, logsumexp, top_ids, top_logprobs, targets,
                           targets_per_row, target_bytes, top_k};
    uint32_t st = check_score_outputs(out);
    if (st != DH_OK) return st;
    if (top_k > kMaxTopK || hidden_size > 131071 || rows > (1u << 24) || vocabulary_size > (1u << 24))
        return DH_ERR_UNSUPPORTED_SHAPE;
    const HeadSplit split = split_of(rows, vocabulary_size, device_sms());
    if (split.total > 0x7FFFFFFFull) return DH_ERR_UNSUPPORTED_SHAPE;
    if (((reinterpret_cast<uintptr_t>(a_scale) | reinterpret_cast<uintptr_t>(w_scale) |
          reinterpret_cast<uintptr_t>(bias)) & 3u) || (reinterpret_cast<uintptr_t>(workspace) & 255u))
        return DH_ERR_ALIGNMENT;
    if (workspace_bytes < dh_head_logprobs_workspace_size(rows, vocabulary_size, top_k)) return DH_ERR_WORKSPACE;
    CUtensorMap ta, tb;
    st = make_i8_operand_maps(&ta, &tb, hidden, ld_hidden, weights, ld_weights, rows, vocabulary_size,
                              hidden_size, kBN);
    if (st != DH_OK) return st;
    const bool wide = hidden_size > kExactK;
    auto stats = wide ? head_stats_kernel<true> : head_stats_kernel<false>;
    static std::atomic<uint64_t> configured[2];
    if (smem_optin_once(stats, kHeadSmem, configured[wide]) != cudaSuccess) return DH_ERR_CUDA;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    float4* partials = static_cast<float4*>(workspace);
    uint8_t* maxima = static_cast<uint8_t*>(workspace) + partial_bytes(split);
    float* group_max = top_k ? reinterpret_cast<float*>(maxima) : nullptr;
    float* half_max = top_k ? reinterpret_cast<float*>(maxima + group_bytes(split)) : nullptr;
    const HeadScoreParams sp{split, vocabulary_size, mask_token_id, hidden_size, a_scale, w_scale, bias,
                             partials, group_max, half_max};
    stats<<<split.grid, kHeadThreads, kHeadSmem, s>>>(ta, tb, sp);
    DH_LAUNCH_CHECK();
    const HeadRowParams rp{split, vocabulary_size, mask_token_id, hidden_size, hidden, ld_hidden, weights,
                           ld_weights, a_scale, w_scale, bias, partials, group_max, half_max, out};
    const bool team = rows < kTeamRows;
    auto rows_kernel = wide ? (team ? head_rows_kernel<true, kRowWarps> : head_rows_kernel<true, 1>)
                            : (team ? head_rows_kernel<false, kRowWarps> : head_rows_kernel<false, 1>);
    rows_kernel<<<team ? rows : (rows + kRowWarps - 1) / kRowWarps, 32 * kRowWarps, 0, s>>>(rp);
    DH_LAUNCH_CHECK();
    return DH_OK;
}
