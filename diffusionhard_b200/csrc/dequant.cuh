// dequant.cuh -- the W8A8 output of one int32 accumulator,
//   y = fp32(acc * fp32(a_scale * w_scale) + bias)
// evaluated in float64 and rounded once to fp32: exactly the reference's
// fixed_mlp.quantized_linear (fixed_mlp.py:98-106).  Shared by the fused argmax
// head, the fp32 outputs of the scaled matrix product and the scoring head above
// its fp32 sizes, so that their logits are the same bits.
#pragma once

#include "dh_common.cuh"

namespace dh {

DH_DEVINL float ref_logit(int32_t acc, float a_scale, float w_scale, float bias) {
    const float combined = __fmul_rn(a_scale, w_scale);
    // double(acc) * double(combined) is exact (24 x 24 bits), so one DFMA equals
    // the reference's separate multiply and add in float64.
    const double v = __fma_rn(static_cast<double>(acc), static_cast<double>(combined),
                              static_cast<double>(bias));
    return __double2float_rn(v);
}

// The same logit with the int and float to double conversions done on the
// integer and FP64 pipes instead of the conversion unit:
//   double(acc): the double 2^52 + 2^31 + acc assembled from bits, minus
//   2^52 + 2^31 (exact for any int32);
//   double(combined): for a positive normal float the double's bits are the
//   float's re-biased (exact); other values take the converting path.
DH_DEVINL float ref_logit_bits(int32_t acc, float a_scale, float w_scale, double bias) {
    const float combined = __fmul_rn(a_scale, w_scale);
    const double acc_d = __hiloint2double(0x43300000, static_cast<int32_t>(static_cast<uint32_t>(acc) ^ 0x80000000u)) -
                         4503601774854144.0;  // 2^52 + 2^31
    const uint32_t cb = __float_as_uint(combined);
    double comb_d;
    if (cb - 0x00800000u < 0x7F000000u)  // positive, normal, finite
        comb_d = __hiloint2double(static_cast<int32_t>((cb >> 3) + 0x38000000u), static_cast<int32_t>(cb << 29));
    else
        comb_d = static_cast<double>(combined);
    return __double2float_rn(__fma_rn(acc_d, comb_d, bias));
}

}  // namespace dh
