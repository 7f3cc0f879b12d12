// gemm_scaled.cu -- the W8A8 linear of any width: the int8 matrix product
// with a scale for each token (row of A) and each channel (row of W),
//
//   y[r, c] = (sum_k A[r, k] W[c, k]) * fp32(a_scale[r] * w_scale[c]) + bias[c]
//
// as fp32, bf16 or f16 (fixed_mlp.quantized_linear, fixed_mlp.py:65-136), on
// the tcgen05 kernel of gemm_tc.cuh.  The integer sum is exact (int32 holds
// k <= 133,152 products of +-127), so the only roundings are those of the
// epilogue:
//   fp32 outputs  the sum, scale and bias meet in float64 and are rounded
//                 once (dequant.cuh): the reference's own logits, bit for bit.
//   16-bit        float(acc) rounds sums past 2^24 and the fp32 FMA rounds
//                 again, each by 2^-24 of a value that then keeps 8 or 11 bits;
//                 float64 would cost the epilogue twice the time for nothing
//                 a 16-bit output can show.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dequant.cuh"
#include "gemm_tc.cuh"
#include "tmap.h"

namespace dh {

uint32_t make_i8_operand_maps(CUtensorMap* ta, CUtensorMap* tb, const int8_t* a, uint64_t lda,
                              const int8_t* w, uint64_t ldw, uint32_t m, uint32_t n, uint32_t k,
                              uint32_t bn);

namespace {

struct ScaledParams {
    const float* a_scale;  // [m]
    const float* w_scale;  // [n]
    const float* bias;     // [n] or null
    void* out;             // [m, n], rows ldo elements apart
    uint64_t ldo;
    uint32_t n;
    bool vec;              // out and its row pitch are multiples of 16 bytes
    bool tma;              // and so are its rows
};

constexpr uint32_t kFull = 0xFFFFFFFFu;

DH_DEVINL uint16_t to_bits16(float v, __nv_bfloat16) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
DH_DEVINL uint16_t to_bits16(float v, __half) { return __half_as_ushort(__float2half_rn(v)); }

// ---------------------------------------------------- small and tall products
//
// 128 x 64 tiles on the kernel of gemm_tc.cuh, mostly one a CTA.  Latency of the
// k-blocks bounds it: 1 x 2304 x 768 4.7 us from a graph, 32 x 768 x 3072 7.3.
template <class T>
struct EpiScaled : EpiBase {
    static constexpr uint32_t kHalf = 32;  // columns of an epilogue warp, half the tile
    static constexpr bool kF32 = sizeof(T) == 4;
    static constexpr uint32_t kStages = 6;
    static constexpr uint32_t kChunk = 32;
    // per warp: the 32 x 32 outputs on their way to whole row segments (4 KB),
    // then its columns' biases (double for fp32 outputs) and w_scale
    static constexpr uint32_t kStagingPerWarp = 4096 + kHalf * 8 + kHalf * 4;
    using Params = ScaledParams;
    struct TileState {
        float ab;
    };
    static DH_DEVINL bool tile_begin(const Params& p, TileState& st, const EpiCtx& ctx, uint32_t col_start) {
        st.ab = ctx.row_ok ? __ldg(p.a_scale + ctx.row) : 0.f;
        __syncwarp();  // the previous tile's chunks finished reading the slots
        double* bias = reinterpret_cast<double*>(ctx.stage + 4096);
        float* ws = reinterpret_cast<float*>(ctx.stage + 4096 + kHalf * 8);
#pragma unroll
        for (uint32_t i = 0; i < kHalf; i += 32) {
            const uint32_t c = col_start + ctx.lane + i;
            const float b = p.bias && c < p.n ? __ldg(p.bias + c) : 0.f;
            if (kF32) bias[ctx.lane + i] = static_cast<double>(b);
            else reinterpret_cast<float*>(bias)[ctx.lane + i] = b;
            ws[ctx.lane + i] = c < p.n ? __ldg(p.w_scale + c) : 0.f;
        }
        __syncwarp();
        return true;
    }
    static DH_DEVINL void chunk(const Params& p, TileState& st, const EpiCtx& ctx, uint32_t col0,
                                const uint32_t* v) {
        const uint32_t lane = ctx.lane, cw = col0 % kHalf;
        const float* ws = reinterpret_cast<const float*>(ctx.stage + 4096 + kHalf * 8) + cw;
        if constexpr (kF32) {
            const double* bias = reinterpret_cast<const double*>(ctx.stage + 4096) + cw;
#pragma unroll
            for (uint32_t j = 0; j < 32; j += 4) {
                float y[4];
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e)
                    y[e] = ref_logit_bits(static_cast<int32_t>(v[j + e]), st.ab, ws[j + e], bias[j + e]);
                *reinterpret_cast<float4*>(ctx.stage + lane * 128 + (((j / 4) ^ (lane & 7u)) << 4)) =
                    make_float4(y[0], y[1], y[2], y[3]);
            }
        } else {
            const float* bias = reinterpret_cast<const float*>(ctx.stage + 4096) + cw;
#pragma unroll
            for (uint32_t j = 0; j < 32; j += 8) {
                uint32_t pk[4];
#pragma unroll
                for (uint32_t e = 0; e < 8; e += 2) {
                    const float y0 = __fmaf_rn(static_cast<float>(static_cast<int32_t>(v[j + e])),
                                               __fmul_rn(st.ab, ws[j + e]), bias[j + e]);
                    const float y1 = __fmaf_rn(static_cast<float>(static_cast<int32_t>(v[j + e + 1])),
                                               __fmul_rn(st.ab, ws[j + e + 1]), bias[j + e + 1]);
                    pk[e / 2] = to_bits16(y0, T()) | (static_cast<uint32_t>(to_bits16(y1, T())) << 16);
                }
                *reinterpret_cast<uint4*>(ctx.stage + lane * 64 + (((j / 8) ^ ((lane >> 1) & 3u)) << 4)) =
                    make_uint4(pk[0], pk[1], pk[2], pk[3]);
            }
        }
        __syncwarp();
        constexpr uint32_t kRowBytes = 32 * sizeof(T);
        T* out = static_cast<T*>(p.out);
        if (p.vec && col0 + 32 <= p.n) {
            // 16 bytes a lane: whole 64- or 128-byte row segments
            constexpr uint32_t kPieces = kRowBytes / 16, kRows = 32 / kPieces;
#pragma unroll
            for (uint32_t i = 0; i < kPieces; ++i) {
                const uint32_t rr = i * kRows + lane / kPieces, c = lane % kPieces;
                const uint32_t sw = kF32 ? (c ^ (rr & 7u)) : (c ^ ((rr >> 1) & 3u));
                if (ctx.row0 + rr < ctx.m_eff)
                    *reinterpret_cast<uint4*>(out + (ctx.row0 + rr) * p.ldo + col0 + c * (16 / sizeof(T))) =
                        *reinterpret_cast<const uint4*>(ctx.stage + rr * kRowBytes + sw * 16);
            }
        } else if (col0 < p.n) {
            // any pitch: one element a lane, one row an instruction
            const uint32_t c = lane / (16 / sizeof(T)), o = lane % (16 / sizeof(T)) * sizeof(T);
            const bool in = col0 + lane < p.n;
#pragma unroll 8
            for (uint32_t rr = 0; rr < 32; ++rr) {
                const uint32_t sw = kF32 ? (c ^ (rr & 7u)) : (c ^ ((rr >> 1) & 3u));
                if (in && ctx.row0 + rr < ctx.m_eff)
                    out[(ctx.row0 + rr) * p.ldo + col0 + lane] =
                        *reinterpret_cast<const T*>(ctx.stage + rr * kRowBytes + sw * 16 + o);
            }
        }
        __syncwarp();
    }
    static DH_DEVINL void tile_end(const Params&, TileState&, const EpiCtx&) {}
};

// ------------------------------------------------------------ large products
//
// Tiles of 128 x 192 or 256, the TMA ring, MMA thread and double-buffered
// accumulators of gemm_tc.cuh, but an epilogue of 12 or 16 warps that all drain the
// same tile (none idles while its accumulators are made) and whose threads hold 4
// rows and 2 of every 8 columns, so that a column's scale and bias are read from
// shared memory once for 4 outputs.  Outputs leave through shared memory as whole
// row segments: TMA stores where the row pitch allows them (512 x 50264 x 768 to
// bf16 35 us, 512 x 50257 through registers 44).
//
// What bounds it: with k = 768 the outputs' way to memory beside the MMAs (512 x 50260
// x 768 to fp32 47 us, where a kernel that only stores, in the same tiles, takes 27;
// 50258 columns 54 and 31; 32768 x 3072 x 768 to bf16 80 us, 61 without the stores,
// which alone take 37); with k = 8192 the tensor cores (8192^3 423 us, 2.6 Pop/s under
// the power cap).
constexpr uint32_t kBM = 128, kBK = 128;
constexpr uint32_t kABytes = kBM * kBK;
constexpr uint32_t kPartCols = 64;             // columns of an epilogue warp
constexpr uint32_t kOutBytes = 4096;           // its outputs on their way
constexpr uint32_t kColBytes = kPartCols * 8;  // and its columns' scales and biases
template <uint32_t kBN>
struct BigTile {
    static constexpr uint32_t kBBytes = kBN * kBK;
    static constexpr uint32_t kEpiWarps = 4 * (kBN / kPartCols);
    static constexpr uint32_t kThreads = 64 + 32 * kEpiWarps;
    static constexpr uint32_t kFixed = 2048 + kEpiWarps * (kOutBytes + kColBytes);
    static constexpr uint32_t kStages = (227 * 1024 - kFixed) / (kABytes + kBBytes);
    static constexpr uint32_t kSmem = kFixed + kStages * (kABytes + kBBytes);
    static_assert(kBN % kPartCols == 0 && kStages >= 3 && kSmem <= 227 * 1024, "shared memory of a CTA");
};

struct BigParams {
    CUtensorMap out_map;  // with Out::kTma: out, box 32 rows x 128 bytes, 128-byte swizzle
    const float* a_scale;
    const float* w_scale;
    const float* bias;
    void* out;
    uint64_t ldo;
    uint32_t m, n, k;
};

// acc * combined + bias for positive normal `combined`, as ref_logit_bits.
DH_DEVINL float scaled_f32(uint32_t acc, float combined, double bias) {
    const double acc_d = __hiloint2double(0x43300000, static_cast<int32_t>(acc ^ 0x80000000u)) - 4503601774854144.0;
    const uint32_t cb = __float_as_uint(combined);
    const double comb_d =
        __hiloint2double(static_cast<int32_t>((cb >> 3) + 0x38000000u), static_cast<int32_t>(cb << 29));
    return __double2float_rn(__fma_rn(acc_d, comb_d, bias));
}

// Where 16-byte piece c of row r lies in a buffer of 128-byte rows under the
// 128-byte swizzle of the TMA stores.
DH_DEVINL uint32_t swz128(uint32_t r, uint32_t c) { return r * 128 + ((c ^ (r & 7u)) << 4); }

// How outputs leave the warp's buffer: by TMA (start, row pitch and the rows' own
// bytes multiples of 16), or through the registers, 8, 4 or 2 bytes a lane.
enum class Out { kTma, k8, k4, k2 };

// The warp's buffer, 32 rows x 128 bytes, to rows of any pitch: the first `cols`
// elements of the first `rows`, sizeof(V) bytes a lane.
template <class T, class V>
DH_DEVINL void store_rows(const uint8_t* buf, T* out, uint64_t ldo, uint32_t rows, uint32_t cols, uint32_t lane) {
    constexpr uint32_t kLanes = 128 / sizeof(V), kE = sizeof(V) / sizeof(T);  // lanes a row needs
    constexpr uint32_t kRows = kLanes < 32 ? 32 / kLanes : 1;                 // rows an instruction covers
    constexpr uint32_t kRounds = kLanes > 32 ? kLanes / 32 : 1;               // instructions a row needs
    const uint32_t sub = lane / kLanes * (kLanes < 32), at = lane % kLanes;
    out += sub * ldo + at * kE;
    const uint32_t piece = at * sizeof(V) / 16, in = at * sizeof(V) % 16;
    const bool whole = rows == 32 && cols * sizeof(T) == 128;
#pragma unroll 4
    for (uint32_t r0 = 0; r0 < 32; r0 += kRows) {
#pragma unroll
        for (uint32_t o = 0; o < kRounds; ++o) {
            // piece c of row r lies at c ^ (r & 7)
            const uint32_t c = piece + o * (32 * sizeof(V) / 16);
            const V v = *reinterpret_cast<const V*>(buf + (r0 + sub) * 128 + ((c ^ sub ^ (r0 & 7u)) << 4) + in);
            const uint32_t e = (at + 32 * o) * kE;
            if (whole || (r0 + sub < rows && e + kE <= cols)) {
                *reinterpret_cast<V*>(out + 32 * o * kE) = v;
            } else if (kE > 1 && r0 + sub < rows) {
#pragma unroll
                for (uint32_t i = 0; i < kE; ++i)
                    if (e + i < cols) out[32 * o * kE + i] = reinterpret_cast<const T*>(&v)[i];
            }
        }
        out += kRows * ldo;
    }
}

template <class T, Out kOut, uint32_t kBN>
__global__ void __launch_bounds__(BigTile<kBN>::kThreads, 1)
gemm_scaled_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                   const __grid_constant__ BigParams p) {
    constexpr bool kF32 = sizeof(T) == 4;
    constexpr uint32_t kSegCols = 128 / sizeof(T);  // columns of the buffer's 128-byte rows
    constexpr uint32_t kStages = BigTile<kBN>::kStages, kBBytes = BigTile<kBN>::kBBytes;
    constexpr uint32_t kEpiWarps = BigTile<kBN>::kEpiWarps;
    constexpr uint32_t kTmemCols = 512;  // two accumulators, a power of two
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~static_cast<uintptr_t>(1023));
    uint8_t* a_smem = smem;
    uint8_t* b_smem = smem + kStages * kABytes;
    uint8_t* out_smem = b_smem + kStages * kBBytes;
    uint8_t* col_smem = out_smem + kEpiWarps * kOutBytes;
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(col_smem + kEpiWarps * kColBytes);
    uint64_t* empty_bar = full_bar + kStages;
    uint64_t* accf_bar = empty_bar + kStages;  // [2]
    uint64_t* acce_bar = accf_bar + 2;            // [2]
    uint64_t* drain_bar = acce_bar + 2;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain_bar + 1);

    const uint32_t warp = warp_id(), lane = lane_id();
    if (warp == 0 && lane == 0) {
        for (uint32_t s = 0; s < kStages; ++s) {
            tc::mbar_init(&full_bar[s], 1);
            tc::mbar_init(&empty_bar[s], 1);
        }
        for (uint32_t b = 0; b < 2; ++b) {
            tc::mbar_init(&accf_bar[b], 1);
            tc::mbar_init(&acce_bar[b], kEpiWarps);
        }
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

    const uint32_t n_tiles = (p.n + kBN - 1) / kBN, total = (p.m + kBM - 1) / kBM * n_tiles;
    const uint32_t k_blocks = (p.k + kBK - 1) / kBK;

    if (warp == 0) {
        // ------------------------------------------------------ TMA producer
        if (tc::elect_one()) {
            uint32_t stage = 0, phase = 0, issued = 0, issued_parity = 0;
            bool ok = true;
            for (uint32_t tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
                const uint32_t m0 = tile / n_tiles * kBM, n0 = tile % n_tiles * kBN;
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
                    issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
                    ++issued;
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            // Drain: every copy this CTA issued has landed before it may exit.
            for (uint32_t s = 0; s < kStages && s < issued; ++s)
                tc::mbar_wait(&full_bar[s], (issued_parity >> s) & 1u, tc::kErrTimeoutFull);
        }
    } else if (warp == 1) {
        // ------------------------------------------------------- MMA issuer
        if (tc::elect_one()) {
            constexpr uint32_t idesc = tc::idesc_i8_s32<kBM, kBN>();
            uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
            bool ok = true;
            for (uint32_t tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
                if (!tc::mbar_wait(&acce_bar[acc], acc_phase ^ 1, tc::kErrTimeoutAccEmpty)) break;
                tc::tc_fence_after();
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
                        tc::mma_i8(tmem_base + acc * kBN, tc::desc_advance(a_desc, kk * 32),
                                   tc::desc_advance(b_desc, kk * 32), idesc, (kb | kk) != 0u);
                    tc::mma_commit(&empty_bar[stage]);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (!ok) break;
                tc::mma_commit(&accf_bar[acc]);
                acc ^= 1;
                acc_phase ^= acc == 0;
            }
            // Drain: all MMAs issued by this thread complete before TMEM is freed.
            tc::mma_commit(drain_bar);
            tc::mbar_wait(drain_bar, 0, tc::kErrTimeoutAccFull);
        }
    } else {
        // --------------------------------------------------------- epilogue
        const uint32_t ew = warp - 2, quad = warp & 3u, part = ew >> 2, quarter = lane % 4;
        uint8_t* buf = out_smem + ew * kOutBytes;
        float* bs = reinterpret_cast<float*>(col_smem + ew * kColBytes);
        float* ws = bs + kPartCols;
        // the next tile's scales and biases, fetched while one is stored
        float w_next[kPartCols / 32], b_next[kPartCols / 32], a_next[4];
        auto fetch = [&](uint32_t tile) {
            const uint32_t row = tile / n_tiles * kBM + quad * 32 + lane / 4, col = tile % n_tiles * kBN + part * kPartCols;
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) a_next[r] = row + 8 * r < p.m ? __ldg(p.a_scale + row + 8 * r) : 1.f;
#pragma unroll
            for (uint32_t i = 0; i < kPartCols / 32; ++i) {
                const uint32_t c = col + i * 32 + lane;
                w_next[i] = c < p.n ? __ldg(p.w_scale + c) : 1.f;
                b_next[i] = c < p.n && p.bias ? __ldg(p.bias + c) : 0.f;
            }
        };
        // scales whose products are positive normal numbers
        auto usual = [](float x) { return x > 1e-18f && x < 1e18f; };
        if (blockIdx.x < total) fetch(blockIdx.x);
        uint32_t acc = 0, phase = 0;
        for (uint32_t tile = blockIdx.x; tile < total; tile += gridDim.x) {
            const uint32_t row0 = tile / n_tiles * kBM + quad * 32, col0 = tile % n_tiles * kBN + part * kPartCols;
            __syncwarp();
            bool plain = true;
            float ab[4];
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                ab[r] = a_next[r];
                plain = plain && usual(ab[r]);
            }
#pragma unroll
            for (uint32_t i = 0; i < kPartCols / 32; ++i) {
                bs[i * 32 + lane] = b_next[i];
                ws[i * 32 + lane] = w_next[i];
                plain = plain && usual(w_next[i]);
            }
            if (kF32) plain = __all_sync(kFull, plain);
            __syncwarp();
            if (tile + gridDim.x < total) fetch(tile + gridDim.x);
            if (!tc::mbar_wait(&accf_bar[acc], phase, tc::kErrTimeoutAccFull)) break;
            tc::tc_fence_after();
            const uint32_t taddr = tmem_base + ((quad * 32u) << 16) + acc * kBN + part * kPartCols;
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {  // 32 columns at a time
                float2 w[4], b[4];
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    w[j] = *reinterpret_cast<const float2*>(ws + 32 * h + 8 * j + 2 * quarter);
                    b[j] = *reinterpret_cast<const float2*>(bs + 32 * h + 8 * j + 2 * quarter);
                }
                if (kOut == Out::kTma && (kF32 || h == 0)) {
                    // the last store has read the buffer
                    if (lane == 0) tc::tma_store_wait_read<0>();
                    __syncwarp();
                }
                // 16 rows at a time (fp32's float64 temporaries leave no registers for
                // both halves), or 32
                constexpr uint32_t kHalves = kF32 ? 1 : 2;
#pragma unroll
                for (uint32_t q = 0; q < 2; q += kHalves) {
                    uint32_t v[kHalves][16];
#pragma unroll
                    for (uint32_t i = 0; i < kHalves; ++i)
                        tc::tmem_ld_16x256b_x4(taddr + 32 * h + ((16u * (q + i)) << 16), v[i]);
                    tc::tmem_ld_wait();
                    if (h == 1 && q + kHalves == 2) {
                        // the accumulators are read: their buffer may be filled again
                        tc::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(&acce_bar[acc]);
                    }
#pragma unroll
                    for (uint32_t i = 0; i < 2 * kHalves; ++i) {
                        const uint32_t r = 2 * q + i, row = lane / 4 + 8 * r;
#pragma unroll
                        for (uint32_t j = 0; j < 4; ++j) {
                            const uint32_t v0 = v[i / 2][4 * j + i % 2 * 2], v1 = v[i / 2][4 * j + i % 2 * 2 + 1];
                            if constexpr (kF32) {
                                float2 y;
                                if (plain) {
                                    y.x = scaled_f32(v0, __fmul_rn(ab[r], w[j].x), static_cast<double>(b[j].x));
                                    y.y = scaled_f32(v1, __fmul_rn(ab[r], w[j].y), static_cast<double>(b[j].y));
                                } else {
                                    y.x = ref_logit(static_cast<int32_t>(v0), ab[r], w[j].x, b[j].x);
                                    y.y = ref_logit(static_cast<int32_t>(v1), ab[r], w[j].y, b[j].y);
                                }
                                *reinterpret_cast<float2*>(buf + swz128(row, 2 * j + quarter / 2) + quarter % 2 * 8) = y;
                            } else {
                                const float2 y = __ffma2_rn(make_float2(static_cast<float>(static_cast<int32_t>(v0)),
                                                                        static_cast<float>(static_cast<int32_t>(v1))),
                                                            __fmul2_rn(make_float2(ab[r], ab[r]), w[j]), b[j]);
                                *reinterpret_cast<uint32_t*>(buf + swz128(row, 4 * h + j) + quarter * 4) =
                                    to_bits16(y.x, T()) | (static_cast<uint32_t>(to_bits16(y.y, T())) << 16);
                            }
                        }
                    }
                }
                if (!kF32 && h == 0) continue;  // 64 columns of 2 bytes make a row of the buffer
                const uint32_t col = col0 + (kF32 ? 32 * h : 0u);
                if (kOut == Out::kTma) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0 && col < p.n && row0 < p.m) {
                        tc::tma_store_2d(&p.out_map, buf, static_cast<int32_t>(col), static_cast<int32_t>(row0));
                        tc::tma_store_commit();
                    }
                } else {
                    __syncwarp();
                    if (col < p.n && row0 < p.m) {
                        T* out = static_cast<T*>(p.out) + row0 * p.ldo + col;
                        const uint32_t rows = min(32u, p.m - row0), cols = min(kSegCols, p.n - col);
                        if constexpr (kOut == Out::k8) store_rows<T, uint2>(buf, out, p.ldo, rows, cols, lane);
                        else if constexpr (kOut == Out::k4) store_rows<T, uint32_t>(buf, out, p.ldo, rows, cols, lane);
                        else if constexpr (!kF32) store_rows<T, uint16_t>(buf, out, p.ldo, rows, cols, lane);
                    }
                    __syncwarp();
                }
            }
            acc ^= 1;
            phase ^= acc == 0;
        }
        if (kOut == Out::kTma && lane == 0) tc::tma_store_wait_all();
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem_base, kTmemCols);
    }
}

template <class T, Out kOut, uint32_t kBN>
cudaError_t launch_big(const CUtensorMap& ta, const CUtensorMap& tb, const BigParams& p, uint32_t tiles, cudaStream_t s) {
    using Tile = BigTile<kBN>;
    static std::atomic<uint64_t> configured{0};
    const cudaError_t e = smem_optin_once(gemm_scaled_kernel<T, kOut, kBN>, Tile::kSmem, configured);
    if (e != cudaSuccess) return e;
    const uint32_t sms = device_sms();
    gemm_scaled_kernel<T, kOut, kBN><<<tiles < sms ? tiles : sms, Tile::kThreads, Tile::kSmem, s>>>(ta, tb, p);
    return cudaGetLastError();
}

template <class T, Out kOut>
cudaError_t launch_big(const CUtensorMap& ta, const CUtensorMap& tb, const BigParams& p, uint32_t bn, uint32_t tiles,
                       cudaStream_t s) {
    return bn == 192 ? launch_big<T, kOut, 192>(ta, tb, p, tiles, s) : launch_big<T, kOut, 256>(ta, tb, p, tiles, s);
}

template <class T>
cudaError_t launch_scaled(const CUtensorMap& ta, const CUtensorMap& tb, const GemmShape& shape,
                          const ScaledParams& p, uint32_t bn, uint32_t tiles, cudaStream_t s) {
    if (bn == 64) return launch_gemm_i8<64, EpiScaled<T>>(ta, tb, shape, p, tiles, s);
    BigParams q{};
    q.a_scale = p.a_scale;
    q.w_scale = p.w_scale;
    q.bias = p.bias;
    q.out = p.out;
    q.ldo = p.ldo;
    q.m = shape.M;
    q.n = shape.N;
    q.k = shape.K;
    if (p.tma) {
        if (!make_tmap_2d(&q.out_map, p.out,
                          sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, sizeof(T),
                          shape.M, shape.N, p.ldo * sizeof(T), 32, 128 / sizeof(T)))
            return cudaErrorInvalidValue;
        return launch_big<T, Out::kTma>(ta, tb, q, bn, tiles, s);
    }
    const uint64_t at = reinterpret_cast<uintptr_t>(p.out) | (p.ldo * sizeof(T));
    if (at % 8 == 0) return launch_big<T, Out::k8>(ta, tb, q, bn, tiles, s);
    if (at % 4 == 0) return launch_big<T, Out::k4>(ta, tb, q, bn, tiles, s);
    if constexpr (sizeof(T) == 2) return launch_big<T, Out::k2>(ta, tb, q, bn, tiles, s);
    return cudaErrorInvalidValue;
}

}  // namespace
}  // namespace dh

using namespace dh;

extern "C" uint32_t dh_gemm_i8_scaled(const int8_t* a, uint64_t lda, const float* a_scale, const int8_t* w,
                                      uint64_t ldw, const float* w_scale, const float* bias, void* out,
                                      uint64_t ldo, uint32_t out_type, uint32_t m, uint32_t n, uint32_t k,
                                      void* stream) {
    if (!a || !w || !a_scale || !w_scale || !out) return DH_ERR_NULL_POINTER;
    if (out_type > DH_TYPE_F16 || m == 0 || n == 0 || k == 0 || ldo < n) return DH_ERR_INVALID_ARGUMENT;
    // int32 holds every sum of k products of magnitude 127 * 127 (128 * 128 for a value of -128)
    if (k > 131071) return DH_ERR_UNSUPPORTED_SHAPE;
    const uint32_t es = out_type == DH_TYPE_F32 ? 4 : 2;
    const uintptr_t f32s = reinterpret_cast<uintptr_t>(a_scale) | reinterpret_cast<uintptr_t>(w_scale) |
                           reinterpret_cast<uintptr_t>(bias);
    if ((f32s & 3u) || (reinterpret_cast<uintptr_t>(out) & (es - 1))) return DH_ERR_ALIGNMENT;
    const uint32_t m_tiles = (m + 127) / 128;
    const bool vec = ((reinterpret_cast<uintptr_t>(out) | (ldo * es)) & 15u) == 0;
    // (a store that ends inside 16 bytes writes all 16, beside the outputs; no map
    // holds a pitch of 2^40 bytes)
    const bool tma = vec && n * static_cast<uint64_t>(es) % 16 == 0 && ldo < (1ull << 38);
    const uint32_t sms = device_sms();
    // Wide tiles of the width whose rounds over the SMs take fewer columns in all: 4096
    // x 4096 x 4096 to bf16 (5 rounds of 192 or 4 of 256) 58 against 63 us, 1024 x 8192 x
    // 8192 (3 or 2) 76 against 68, 512 x 50258 x 768 to fp32 (8 or 6: as many) 53 against
    // 59.  Tiles of 64 columns where each gets an SM of its own (launched from a graph,
    // 256 x 4736 x 768 to bf16 4.9 against 6.7 us), or where they take fewer columns at
    // one and a half times the price: 32768 x 64 x 768 to bf16 7.5 against 12.0 us, 32768
    // x 128 x 4096 (4 rounds or 2 of 192) 32.9 against 31.2.
    auto columns = [&](uint32_t cols) {
        const uint64_t t = static_cast<uint64_t>(m_tiles) * ((n + cols - 1) / cols);
        return (t + sms - 1) / sms * cols;
    };
    const uint32_t wide = columns(192) <= columns(256) ? 192u : 256u;
    const uint32_t bn = columns(64) == 64 || columns(64) * 3 < columns(wide) * 2 ? 64u : wide;
    const uint64_t tiles = static_cast<uint64_t>(m_tiles) * ((n + bn - 1) / bn);
    if (tiles > 0x7FFFFFFFull || m > 0x7FFFFF00u || n > 0x7FFFFF00u) return DH_ERR_UNSUPPORTED_SHAPE;
    CUtensorMap ta, tb;
    const uint32_t st = make_i8_operand_maps(&ta, &tb, a, lda, w, ldw, m, n, k, bn);
    if (st != DH_OK) return st;
    const ScaledParams p{a_scale, w_scale, bias, out, ldo, n, vec, tma};
    const GemmShape shape{m, n, k, nullptr};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (out_type == DH_TYPE_F32) e = launch_scaled<float>(ta, tb, shape, p, bn, static_cast<uint32_t>(tiles), s);
    else if (out_type == DH_TYPE_BF16)
        e = launch_scaled<__nv_bfloat16>(ta, tb, shape, p, bn, static_cast<uint32_t>(tiles), s);
    else e = launch_scaled<__half>(ta, tb, shape, p, bn, static_cast<uint32_t>(tiles), s);
    return e == cudaSuccess ? DH_OK : DH_ERR_CUDA;
}
