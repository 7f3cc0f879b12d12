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
};

DH_DEVINL uint16_t to_bits16(float v, __nv_bfloat16) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
DH_DEVINL uint16_t to_bits16(float v, __half) { return __half_as_ushort(__float2half_rn(v)); }

// kHalf: columns of an epilogue warp, half the tile.
template <class T, uint32_t kHalf_>
struct EpiScaled : EpiBase {
    static constexpr uint32_t kHalf = kHalf_;
    static constexpr bool kF32 = sizeof(T) == 4;
    static constexpr uint32_t kStages = kHalf == 128 ? 3 : 6;
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

template <class T>
cudaError_t launch_scaled(const CUtensorMap& ta, const CUtensorMap& tb, const GemmShape& shape,
                          const ScaledParams& p, uint32_t bn, uint32_t tiles, cudaStream_t s) {
    if (bn == 64) return launch_gemm_i8<64, EpiScaled<T, 32>>(ta, tb, shape, p, tiles, s);
    return launch_gemm_i8<256, EpiScaled<T, 128>>(ta, tb, shape, p, tiles, s);
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
    const uint32_t bn = static_cast<uint64_t>(m_tiles) * ((n + 63) / 64) <= kNumSMs ? 64u : 256u;
    const uint64_t tiles = static_cast<uint64_t>(m_tiles) * ((n + bn - 1) / bn);
    if (tiles > 0x7FFFFFFFull || m > 0x7FFFFF00u || n > 0x7FFFFF00u) return DH_ERR_UNSUPPORTED_SHAPE;
    CUtensorMap ta, tb;
    const uint32_t st = make_i8_operand_maps(&ta, &tb, a, lda, w, ldw, m, n, k, bn);
    if (st != DH_OK) return st;
    const bool vec = ((reinterpret_cast<uintptr_t>(out) | (ldo * es)) & 15u) == 0;
    const ScaledParams p{a_scale, w_scale, bias, out, ldo, n, vec};
    const GemmShape shape{m, n, k, nullptr};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (out_type == DH_TYPE_F32) e = launch_scaled<float>(ta, tb, shape, p, bn, static_cast<uint32_t>(tiles), s);
    else if (out_type == DH_TYPE_BF16)
        e = launch_scaled<__nv_bfloat16>(ta, tb, shape, p, bn, static_cast<uint32_t>(tiles), s);
    else e = launch_scaled<__half>(ta, tb, shape, p, bn, static_cast<uint32_t>(tiles), s);
    return e == cudaSuccess ? DH_OK : DH_ERR_CUDA;
}
