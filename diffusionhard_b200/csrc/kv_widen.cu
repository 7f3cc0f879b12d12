// kv_widen.cu -- an int8 K/V cache as f16 rows, for attention with many tiles of rows.
//
// The tensor-core kernel over int8 turns codes into f16 tiles as it goes, once for
// every 128 rows: 32 canvases of 1024 queries and keys take 237 us that way and 154 us
// over 16-bit keys.  Where every key is visited by at least four tiles of rows, the
// codes are turned once, here, into the workspace (together 198 us).  Bound by HBM:
// 136 bytes in and 256 out for each position and K/V head (f16 queries: 512, see
// FineFactor; 260 us).
//
// A line is an (entry, head).  Its K becomes code * scale * 2^-(E + 9) with E the
// exponent of the line's largest scale, rounded once to f16 (its factor scale 2^(15 -
// E) is rounded before, see convert16), its V likewise with an E that is at least that
// of the sequence's prefix; both exponents go to `exps`.  Rows behind the last key
// become zeros up to the end of its tile.
#include "kv_kernels.h"

#include <algorithm>

namespace dh {
namespace kv {
namespace {

constexpr uint32_t kThreads = 256;

struct WidenArgs {
    Segment prefix, own;
    WideKeys out_prefix, out_own;
    uint32_t sequences, prefixes, prefix_chunks, own_chunks, with_prefix;
    FastDiv kv_heads, queries, per_prefix;
    const uint32_t* run_rows;
};

// The largest magnitude (as bits) among the first n scales, for all threads.
DH_DEVINL uint32_t largest(const float* scale, uint32_t n, uint32_t* smem) {
    float peak = 0.f;  // (of the numbers among them)
    for (uint32_t i = threadIdx.x * 4; i < n; i += kThreads * 4) {
        const float4 x = *reinterpret_cast<const float4*>(scale + i);  // (lines start at 256 bytes)
        peak = fmaxf(peak, fabsf(x.x));
        if (i + 1 < n) peak = fmaxf(peak, fabsf(x.y));
        if (i + 2 < n) peak = fmaxf(peak, fabsf(x.z));
        if (i + 3 < n) peak = fmaxf(peak, fabsf(x.w));
    }
    const uint32_t m = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(peak));
    if (lane_id() == 0) smem[warp_id()] = m;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (uint32_t i = 0; i < kThreads / 32; ++i) all = max(all, smem[i]);
    __syncthreads();
    return all;
}

DH_DEVINL int32_t exponent_in_range(uint32_t bits) { return min(max(exponent_of(bits), -100), 126); }

// FINE: see FineFactor.
template <bool FINE>
__global__ void __launch_bounds__(kThreads) kv_widen_kernel(const __grid_constant__ WidenArgs a) {
    __shared__ uint32_t smem[kThreads / 32];
    grid_launch_dependents();
    const uint32_t prefix_ctas = a.with_prefix ? a.prefixes * a.kv_heads.d * a.prefix_chunks : 0u;
    const bool own = blockIdx.x >= prefix_ctas;
    const uint32_t chunks = own ? a.own_chunks : a.prefix_chunks;
    const uint32_t index = own ? blockIdx.x - prefix_ctas : blockIdx.x;
    const uint32_t line = index / chunks, chunk = index % chunks;
    uint32_t head = line;
    const uint32_t entry = a.kv_heads.split(head);
    const uint32_t live = a.run_rows ? min(a.sequences, a.queries.of(min(*a.run_rows, 0x7FFFFFFFu))) : a.sequences;
    if ((own ? entry : entry * a.per_prefix.d) >= live) return;
    const Segment& s = own ? a.own : a.prefix;
    const WideKeys& to = own ? a.out_own : a.out_prefix;
    const uint32_t len = length_of(s, entry);
    const uint64_t at = static_cast<uint64_t>(line) * s.pitch, to_at = static_cast<uint64_t>(line) * s.capacity;
    const int32_t ek = exponent_in_range(largest(s.k_scale + at, len, smem));
    int32_t ev = exponent_in_range(largest(s.v_scale + at, len, smem));
    if (own && a.with_prefix) {
        const uint32_t p = a.per_prefix.of(entry);
        const uint64_t line0 = static_cast<uint64_t>(p) * a.kv_heads.d + head;
        ev = max(ev, exponent_in_range(
                         largest(a.prefix.v_scale + line0 * a.prefix.pitch, length_of(a.prefix, p), smem)));
    }
    if (chunk == 0 && threadIdx.x == 0)
        to.exps[line] = make_float2(pow2(min(ek + 9, 128)), __int_as_float(ev + 9));
    const float fk = pow2(15 - ek), fv = pow2(15 - ev);
    const uint32_t tiles = (len + kKT - 1) / kKT;
    // 8 codes of a row a thread, so that a warp writes whole lines; the loads of four
    // half tiles of K and V are under way together
    const uint32_t row = threadIdx.x / 8, c = threadIdx.x & 7u;
    constexpr uint32_t kAhead = 4;
    for (uint32_t t0 = chunk; t0 < tiles; t0 += kAhead / 2 * chunks) {
        uint2 codes[kAhead][2];
        float scale[kAhead][2];
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) {
            const uint32_t t = t0 + i / 2 * chunks, key = t * kKT + (i & 1u) * 32 + row;
#pragma unroll
            for (uint32_t side = 0; side < 2; ++side) {
                codes[i][side] = make_uint2(0, 0);
                if (t < tiles)
                    codes[i][side] = __ldcs(reinterpret_cast<const uint2*>((side ? s.v : s.k) + (at + key) * kDh) + c);
                scale[i][side] = t < tiles && key < len ? (side ? s.v_scale : s.k_scale)[at + key] : 0.f;
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) {
            const uint32_t t = t0 + i / 2 * chunks, key = t * kKT + (i & 1u) * 32 + row;
            if (t >= tiles) break;
#pragma unroll
            for (uint32_t side = 0; side < 2; ++side) {
                const float by = scale[i][side] * (side ? fv : fk);
                const uint2 w = codes[i][side];
                uint4 x;
                __half* dst = (side ? to.v : to.k) + (to_at + key) * kDh;
                if constexpr (FINE) {
                    const FineFactor f = fine_factor(by);
                    convert4(w.x, f.lo, f.off_lo, x.x, x.y);
                    convert4(w.y, f.lo, f.off_lo, x.z, x.w);
                    reinterpret_cast<uint4*>(dst + to.lo)[c] = x;
                    convert4(w.x, f.hi, f.off_hi, x.x, x.y);
                    convert4(w.y, f.hi, f.off_hi, x.z, x.w);
                } else {
                    const __half2 f = __float2half2_rn(by);
                    const __half2 off = __hmul2(f, __half2half2(__ushort_as_half(0x8080)));
                    convert4(w.x, f, off, x.x, x.y);
                    convert4(w.y, f, off, x.z, x.w);
                }
                reinterpret_cast<uint4*>(dst)[c] = x;
            }
        }
    }
}

}  // namespace

uint32_t launch_widen(const Args& a, const WideKeys& prefix, const WideKeys& own, uint32_t prefixes, cudaStream_t st) {
    WidenArgs w{};
    w.prefix = a.prefix, w.own = a.own, w.out_prefix = prefix, w.out_own = own;
    w.sequences = a.sequences, w.prefixes = prefixes, w.with_prefix = prefixes != 0;
    w.kv_heads = a.kv_heads, w.queries = a.queries, w.per_prefix = a.per_prefix;
    w.run_rows = a.run_rows;
    // eight CTAs an SM (196.5 us for 32 canvases, 198 with four, 199.5 with 16): every one
    // reads all scales of its line
    const auto chunks = [](uint64_t lines, uint32_t capacity) {
        return static_cast<uint32_t>(std::min<uint64_t>((8 * device_sms() + lines - 1) / lines, capacity / kKT));
    };
    const uint64_t own_lines = static_cast<uint64_t>(a.sequences) * a.kv_heads.d;
    const uint64_t prefix_lines = static_cast<uint64_t>(prefixes) * a.kv_heads.d;
    w.own_chunks = chunks(own_lines, a.own.capacity);
    w.prefix_chunks = prefixes ? chunks(prefix_lines, a.prefix.capacity) : 1;
    const uint64_t ctas = own_lines * w.own_chunks + prefix_lines * w.prefix_chunks;
    if (own.lo)
        kv_widen_kernel<true><<<static_cast<uint32_t>(ctas), kThreads, 0, st>>>(w);
    else
        kv_widen_kernel<false><<<static_cast<uint32_t>(ctas), kThreads, 0, st>>>(w);
    DH_LAUNCH_CHECK();
    return DH_OK;
}

}  // namespace kv
}  // namespace dh
