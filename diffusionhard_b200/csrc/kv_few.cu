// kv_few.cu -- attention over K/V caches for few rows (queries times query heads of
// a K/V head): single tokens and short blocks.  The operator is described in
// kv_attention.cu; this kernel has the items with at most 16 rows.
//
// With 1 to 16 rows a key costs at most 4,096 FLOP for its 136 (int8) or 256
// (16-bit) bytes, so the cache's bytes bound it, and the kernel is built around
// their flow: every warp streams tiles of 64 (16 bits: 32) keys of its own through two buffers
// in shared memory (one bulk copy for each array of codes and scales, or a TMA
// tile), and computes on the warp's matrix instruction (16 x 8 x 16) from
// registers: no barrier between warps, no trip of converted values through shared
// memory.  A tensor-core tile of 128 rows, almost all of them empty, needs ~2,100
// cycles per 64 keys and CTA for the same (16 single tokens over 24,000 keys on
// average: 289 us).
//
// Both products are transposed, S^T = K Q^T and O^T = V^T P^T: keys and the values'
// dimensions fill the 16 rows of the instruction, and the queries its 8 columns.
// (With the queries in the 16 rows the same case took 149 us: twice the
// instructions for the softmax and the products.)  P^T gets from the layout of a
// result to that of an operand by movmatrix.
//
// int8: scores are (q . codes) * scale of the key, by the integer instruction on the
// codes as they are, with the query in two int8 parts (15 bits of its row's largest
// value).  The weights enter the second product as f16(p * v_scale 2^-E), E an
// exponent that only grows (one for a warp), the codes of V exact as f16; for f16
// queries as two f16 (16 long caches 101 us in bf16 and 112 in f16; error of the
// result 3.0e-4 with one, 2.2e-4 with two, 2.0e-4 of that its own rounding).
//
// An item's keys are shared by the four warps of a CTA and the CTAs of a cluster, which
// join their sums through shared memory in a fixed order.  Where there are items
// enough, every warp has its own instead, and loads the next one's first tiles while
// it works on the last ones of the one before (`solo`).
#include <cuda.h>

#include "kv_kernels.h"
#include "row_quant.cuh"

#include <algorithm>

namespace dh {
namespace kv {
namespace {

constexpr uint32_t kWarps = 4;
constexpr uint32_t kThreads = 32 * kWarps;
constexpr uint32_t kStages = 2;
// The weights are relative to 2^m with m the maximum less this: f16 holds them down to
// 2^-32 of the largest.
constexpr float kHeadroom = 8.f;
constexpr int32_t kShift = 0x4B400000;  // 1.5 * 2^23 as fp32

enum Kind : int { kV16 = 0, kVBf16 = 1, kInt8 = 2 };

// Keys of a tile (16 bits: 3 CTAs of 64 KB an SM; with 64 keys 1 of 128 KB, and 128
// single tokens over up to 320 keys took 18.5 us instead of 14.4).
template <int KIND>
constexpr uint32_t kKeys = KIND == kInt8 ? kKT : kFewKeys16;
template <int KIND>
constexpr uint32_t kStageBytes = KIND == kInt8 ? kRawBytes : 2 * kKeys<KIND> * kDh * 2;
template <int KIND>
constexpr uint32_t kSmem = 1024 + kWarps * kStages * kStageBytes<KIND> + 128 + kOrdered * 6;

template <bool BF16>
DH_DEVINL void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// int8, 32 deep
DH_DEVINL void mma_16832(int32_t (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

DH_DEVINL void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
DH_DEVINL void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

// 8 x 8 transposed: a thread's pair (row g, columns 2 c and 2 c + 1) becomes (row
// 2 c and 2 c + 1, column g)
DH_DEVINL uint32_t transposed(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// Bytes 0 and 1 (HI: 2 and 3) of a word of codes plus 128 as an exact f16 pair of
// the codes: with 0x64 above it a byte is 1024 + its value.
template <bool HI>
DH_DEVINL uint32_t codes_f16(uint32_t u) {
    const uint32_t p = __byte_perm(u, 0x64646464u, HI ? 0x4342u : 0x4140u);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&p), __float2half2_rn(1152.0f));
    return *reinterpret_cast<const uint32_t*>(&x);
}

// Where key n (0..7) of an operand lies in its group of 8, int8: neighbours differ in
// parity, and so do 0, 2, 4, 6, so that neither the 16-byte reads of K nor the 8-byte
// reads of V pile up on banks.
DH_DEVINL uint32_t key_of(uint32_t n) { return n ^ ((n >> 1) & 1u); }

// NT: groups of 8 rows.
template <int KIND, bool QBF16, int NT>
__global__ void __launch_bounds__(kThreads, 3)
kv_few_kernel(const __grid_constant__ CUtensorMap tpk, const __grid_constant__ CUtensorMap tpv,
              const __grid_constant__ CUtensorMap tok, const __grid_constant__ CUtensorMap tov,
              const __grid_constant__ Args a, const uint32_t cls, const uint32_t cluster) {
    constexpr bool kI8 = KIND == kInt8;
    constexpr uint32_t kN = kKeys<KIND>, kSteps = kN / 16;
    constexpr uint32_t kTile16 = kN * kDh * 2;  // bytes of a 16-bit tile of K
    constexpr bool kFine = kI8 && !QBF16;  // weights in two f16
    constexpr bool kQB = QBF16 && !kI8;  // type of the first product's operands
    const uint32_t live = a.run_rows ? min(a.sequences, a.queries.of(min(*a.run_rows, 0x7FFFFFFFu))) : a.sequences;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~static_cast<uintptr_t>(1023));
    uint64_t* all_bars = reinterpret_cast<uint64_t*>(smem + kWarps * kStages * kStageBytes<KIND>);
    const uint32_t warp = warp_id(), lane = lane_id(), g = lane >> 2, c = lane & 3u;
    const Class& cl = a.cls[cls];
    grid_launch_dependents();
    const bool solo = cluster == 0;
    uint32_t* lengths = reinterpret_cast<uint32_t*>(all_bars + 16);
    uint16_t* order = reinterpret_cast<uint16_t*>(lengths + kOrdered);
    if (cl.ordered) order_sequences(a, lengths, order);
    const uint32_t rank = cluster > 1 ? cluster_rank() : 0u;

    uint8_t* ring = smem + warp * kStages * kStageBytes<KIND>;
    uint64_t* bars = all_bars + warp * kStages;
    if (lane == 0) {
        for (uint32_t i = 0; i < kStages; ++i) tc::mbar_init(&bars[i], 1);
        tc::fence_barrier_init();
    }
    __syncwarp();

    // This warp's tiles: of its items all, one after the other (solo), or of the
    // CTA's one item every kWarps-th of the CTA's part.
    const uint32_t first_item = solo ? blockIdx.x * kWarps + warp : blockIdx.x / cluster;
    const uint32_t next_item = solo ? gridDim.x * kWarps : cl.items;
    const uint32_t step = solo ? 1u : kWarps;
    auto item_at = [&](uint32_t w) {
        Item it = item_of<kN>(a, cl, w, live, order);
        if (!solo) {
            const uint32_t n = it.t1 - it.t0;
            it.t1 = it.t0 + n * (rank + 1) / cluster;
            it.t0 += n * rank / cluster + warp;
        }
        return it;
    };
    // The next tile that is not yet loaded, into buffer `st`.
    uint32_t ahead_w = first_item, ahead_j = 0, issued = 0;
    Item ahead;
    if (ahead_w < cl.items) {
        ahead = item_at(ahead_w);
        ahead_j = ahead.t0;
    }
    auto load_next = [&](uint32_t st) {
        while (ahead_w < cl.items && ahead_j >= ahead.t1) {
            ahead_w += next_item;
            if (ahead_w >= cl.items) break;
            ahead = item_at(ahead_w);
            ahead_j = ahead.t0;
        }
        if (ahead_w >= cl.items) return;
        const bool own = ahead_j >= ahead.n0;
        const uint32_t key = (own ? ahead_j - ahead.n0 : ahead_j) * kN;
        const uint32_t entry = own ? ahead.own : ahead.prefix;
        uint8_t* dst = ring + st * kStageBytes<KIND>;
        uint64_t* bar = &bars[st];
        if (lane == 0) tc::mbar_arrive_expect_tx(bar, kStageBytes<KIND>);
        __syncwarp();
        // a lane a copy, in one instruction
        if constexpr (kI8) {
            if (lane < 4) {
                const Segment& s = own ? a.own : a.prefix;
                const uint64_t at = (static_cast<uint64_t>(entry) * a.kv_heads.d + ahead.kv_head) * s.pitch + key;
                const bool is_v = lane & 1u, is_scale = lane & 2u;
                const void* codes = (is_v ? s.v : s.k) + at * kDh;
                const void* scales = (is_v ? s.v_scale : s.k_scale) + at;
                tc::bulk_load(dst + (is_scale ? 2 * kKT * kDh : 0) + (is_v ? (is_scale ? kKT * 4 : kKT * kDh) : 0),
                              is_scale ? scales : codes, is_scale ? kKT * 4 : kKT * kDh, bar);
            }
        } else if (lane < 2) {
            const bool turned = lane && a.v_transposed;
            const CUtensorMap* map = lane ? (own ? &tov : &tpv) : (own ? &tok : &tpk);
            tc::tma_load_4d(dst + lane * kTile16, map, bar, turned ? key : 0, turned ? 0 : key, ahead.kv_head, entry);
        }
        ++issued;
        ahead_j += step;
    };
#pragma unroll
    for (uint32_t i = 0; i < kStages; ++i) load_next(i);

    uint32_t n = 0;  // tiles done
    bool ok = true;
    // (one round if not solo; the CTAs of a cluster leave together or not at all)
    for (uint32_t w = first_item; w < cl.items && ok; w += next_item) {
    const Item it = item_at(w);
    if (it.rows == 0) continue;

    // the query rows 8 t + g as operands of the first product; the factors of the
    // scores of rows 8 t + 2 c and 8 t + 2 c + 1
    uint32_t qb[NT][4][2];
    float cr[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const uint32_t r = t * 8 + g;
        const uint8_t* q = nullptr;
        if (r < it.rows) row_index(a, it, r, &q);
        if constexpr (kI8) {
            // 16 values from 16 c on: values 4 s .. 4 s + 3 of them in step s
            uint32_t x[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) x[i] = 0;
            if (q) {
                const uint4 lo = __ldg(reinterpret_cast<const uint4*>(q + 32 * c));
                const uint4 hi = __ldg(reinterpret_cast<const uint4*>(q + 32 * c + 16));
                x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w;
                x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w;
            }
            float2 f[8];
            uint32_t peak = 0;
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                f[i] = QBF16 ? make_float2(__uint_as_float(x[i] << 16), __uint_as_float(x[i] & 0xFFFF0000u))
                             : __half22float2(*reinterpret_cast<const __half2*>(&x[i]));
                peak = max(peak, max(__float_as_uint(f[i].x) & 0x7FFFFFFFu, __float_as_uint(f[i].y) & 0x7FFFFFFFu));
            }
            peak = max(peak, __shfl_xor_sync(0xFFFFFFFFu, peak, 1));
            peak = max(peak, __shfl_xor_sync(0xFFFFFFFFu, peak, 2));
            // a value is (128 hi + lo) amax / 16256, hi and lo int8
            const bool live = peak >= 0x0D800000u;  // 2^-100
            const float amax = __uint_as_float(peak);
            const float by = live ? __fdiv_rn(16256.0f, amax) : 0.f;
            const float factor = peak >= 0x7F800000u ? __uint_as_float(0x7FC00000u)
                                                     : fmaxf(a.c * (live ? amax * (1.0f / 16256.0f) : 0.f), kLeastFactor);
            cr[t][0] = __shfl_sync(0xFFFFFFFFu, factor, 8 * c);
            cr[t][1] = __shfl_sync(0xFFFFFFFFu, factor, 8 * c + 4);
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {  // four values
                int32_t v[4], hi[4];
                v[0] = __float2int_rn(f[2 * k].x * by), v[1] = __float2int_rn(f[2 * k].y * by);
                v[2] = __float2int_rn(f[2 * k + 1].x * by), v[3] = __float2int_rn(f[2 * k + 1].y * by);
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) hi[i] = (v[i] + 64) >> 7, v[i] -= hi[i] * 128;
                qb[t][k][0] = pack4_i8(hi[0], hi[1], hi[2], hi[3]);
                qb[t][k][1] = pack4_i8(v[0], v[1], v[2], v[3]);
            }
        } else {
            cr[t][0] = cr[t][1] = a.c;
#pragma unroll
            for (uint32_t s = 0; s < 4; ++s) {
                qb[t][s][0] = q ? __ldg(reinterpret_cast<const uint32_t*>(q + 32 * s + 4 * c)) : 0u;
                qb[t][s][1] = q ? __ldg(reinterpret_cast<const uint32_t*>(q + 32 * s + 4 * c + 16)) : 0u;
            }
        }
    }

    float o[NT][4][4] = {};  // O^T: d = 16 i + g and 16 i + g + 8, rows 2 c and 2 c + 1
    float m[NT][2], l[NT][2];
    int32_t ev = -100;  // exponent of O (int8)
#pragma unroll
    for (int t = 0; t < NT; ++t) m[t][0] = m[t][1] = kNoMax, l[t][0] = l[t][1] = 0.f;

    for (uint32_t j = it.t0; j < it.t1; j += step, ++n) {
        const uint32_t st = n % kStages;
        if (!tc::mbar_wait(&bars[st], (n / kStages) & 1u, tc::kErrTimeoutFull)) {
            ok = false;
            break;
        }
        uint8_t* tile = ring + st * kStageBytes<KIND>;
        const float* scales = reinterpret_cast<const float*>(tile + 2 * kKT * kDh);
        const uint32_t left = keys_left<kN>(it, j);

        // scores of keys 16 i + g (x[0], x[1]) and 16 i + 8 + g (x[2], x[3]), the last
        // index through key_of for int8
        float s[NT][kSteps][4] = {};
#pragma unroll
        for (uint32_t i = 0; i < kSteps; ++i) {
            if constexpr (kI8) {
                const uint8_t* row = tile + (16 * i + key_of(g)) * kDh + 16 * c;
                const uint4 w0 = *reinterpret_cast<const uint4*>(row);
                const uint4 w1 = *reinterpret_cast<const uint4*>(row + 8 * kDh);
                const uint32_t ka[2][4] = {{w0.x, w1.x, w0.y, w1.y}, {w0.z, w1.z, w0.w, w1.w}};
                const float k0 = scales[16 * i + key_of(g)], k1 = scales[16 * i + 8 + key_of(g)];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    // integers below 2^22 on top of 1.5 2^23: the sums' bits are floats
                    int32_t hi[4] = {kShift, kShift, kShift, kShift}, lo[4] = {kShift, kShift, kShift, kShift};
#pragma unroll
                    for (uint32_t k = 0; k < 2; ++k) {
                        mma_16832(hi, ka[k], qb[t][2 * k][0], qb[t][2 * k + 1][0]);
                        mma_16832(lo, ka[k], qb[t][2 * k][1], qb[t][2 * k + 1][1]);
                    }
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) {
                        const float2 m2 = make_float2(-__int_as_float(kShift), -__int_as_float(kShift));
                        const float2 a2 = __fadd2_rn(make_float2(__int_as_float(hi[2 * h]), __int_as_float(hi[2 * h + 1])), m2);
                        const float2 b2 = __fadd2_rn(make_float2(__int_as_float(lo[2 * h]), __int_as_float(lo[2 * h + 1])), m2);
                        const float ks = h ? k1 : k0;
                        const float2 x = __fmul2_rn(__ffma2_rn(a2, make_float2(128.f, 128.f), b2), make_float2(ks, ks));
                        s[t][i][2 * h] = x.x, s[t][i][2 * h + 1] = x.y;
                    }
                }
            } else {
                const uint32_t key = 16 * i + ((lane >> 3) & 1u) * 8 + (lane & 7u);
                const uint32_t row = smem_u32(tile) + key * 128;
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) {
                    uint32_t ka[4];
                    ldmatrix4(ka, row + (((2 * k + (lane >> 4)) ^ (lane & 7u)) * 16));
#pragma unroll
                    for (int t = 0; t < NT; ++t) mma_16816<kQB>(s[t][i], ka, qb[t][k][0], qb[t][k][1]);
                }
            }
        }
        float vs[kSteps][2];  // v_scale 2^-E of this thread's keys
        float fe = 1.f;
        if constexpr (kI8) {
            float peak = 0.f;  // (of the numbers among them)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) vs[i][h] = scales[kKT + 16 * i + 8 * h + key_of(g)];
            if (left < kKT) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h)
                        if (16 * i + 8 * h + key_of(g) >= left) vs[i][h] = 0.f;
            }
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) peak = fmaxf(peak, fmaxf(fabsf(vs[i][0]), fabsf(vs[i][1])));
            const int32_t et =
                max(ev, min(exponent_of(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(peak))), 126));
            const float by = pow2(-et);
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) vs[i][0] *= by, vs[i][1] *= by;
            fe = pow2(max(ev - et, -126));
            ev = et;
        }
        if (left < kN) {
            // keys behind the last one: whatever was read scores -inf; V there is zero
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (uint32_t i = 0; i < kSteps; ++i)
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h)
                        if (16 * i + 8 * h + (kI8 ? key_of(g) : g) >= left) s[t][i][2 * h] = s[t][i][2 * h + 1] = -INFINITY;
            if constexpr (!kI8) {
                if (a.v_transposed) {
                    for (uint32_t i = lane; i < kDh * kN; i += 32) {  // (64-byte swizzle)
                        const uint32_t d = i / kN, key = i % kN;
                        if (key >= left)
                            *reinterpret_cast<uint16_t*>(tile + kTile16 + d * 64 +
                                                         (((key >> 3) ^ ((d >> 1) & 3u)) * 16) + (key & 7u) * 2) = 0;
                    }
                } else {
                    for (uint32_t i = left * 8 + lane; i < kN * 8; i += 32)
                        *reinterpret_cast<uint4*>(tile + kTile16 + i * 16) = make_uint4(0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (before the next load here)
                __syncwarp();
            }
        }
        // weights, in place
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float next[2], alpha[2];
#pragma unroll
            for (uint32_t e = 0; e < 2; ++e) {
                float top = max_nan(max_nan(s[t][0][e], s[t][0][e + 2], s[t][1][e]), s[t][1][e + 2]);
                if constexpr (kSteps == 4)
                    top = max_nan(top, max_nan(max_nan(s[t][2][e], s[t][2][e + 2], s[t][kSteps - 1][e]),
                                               s[t][kSteps - 1][e + 2]));
                top = max_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
                top = max_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
                top = max_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
                // finite, or NaN for a score that is infinite or NaN: the row is NaN
                const float top2 = top * cr[t][e];
                next[e] = max_nan(max_nan(top2 - (fabsf(top2) < kFar ? kHeadroom : 0.f), kNoMax), m[t][e]);
                next[e] = __fmaf_rn(next[e], -0.f, next[e]);
                alpha[e] = growth(m[t][e], next[e]);
                m[t][e] = next[e];
                l[t][e] *= alpha[e];
                alpha[e] *= fe;
            }
            const float damp[2] = {damping(next[0]), damping(next[1])};
            const float2 cr2 = make_float2(fmaxf(cr[t][0] * damp[0], kLeastFactor), fmaxf(cr[t][1] * damp[1], kLeastFactor));
            const float2 nm2 = make_float2(-next[0] * damp[0], -next[1] * damp[1]);
            float2 sum = make_float2(l[t][0], l[t][1]);
#pragma unroll
            for (uint32_t i = 0; i < kSteps; ++i) {
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    const float2 x = __ffma2_rn(make_float2(s[t][i][2 * h], s[t][i][2 * h + 1]), cr2, nm2);
                    float2 p = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                    sum = __fadd2_rn(sum, p);
                    if constexpr (kI8) p = __fmul2_rn(p, make_float2(vs[i][h], vs[i][h]));
                    s[t][i][2 * h] = p.x, s[t][i][2 * h + 1] = p.y;
                }
            }
            l[t][0] = sum.x, l[t][1] = sum.y;
            if (__any_sync(0xFFFFFFFFu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    o[t][i][0] *= alpha[0], o[t][i][2] *= alpha[0];
                    o[t][i][1] *= alpha[1], o[t][i][3] *= alpha[1];
                }
            }
        }
        // O^T += V^T P^T, 16 keys at a time
#pragma unroll
        for (uint32_t k = 0; k < kSteps; ++k) {
            uint32_t pb[NT][2], pl[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h)
                    pb[t][h] = transposed(KIND == kVBf16 ? pack_bf16x2(s[t][k][2 * h], s[t][k][2 * h + 1])
                                                         : pack_f16x2(s[t][k][2 * h], s[t][k][2 * h + 1]));
            if constexpr (kFine) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) {
                        const float x = s[t][k][2 * h], y = s[t][k][2 * h + 1];
                        const __half2 p = __floats2half2_rn(x, y);
                        pl[t][h] = transposed(pack_f16x2(x - __low2float(p), y - __high2float(p)));
                    }
            }
            if constexpr (kI8) {
                // row g of part i is d = 8 g + 2 i, row g + 8 the next one: a thread reads
                // d = 8 g .. 8 g + 7 of its four keys and pairs them up byte by byte
                uint2 w[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t key = 16 * k + 8 * (i >> 1) + key_of(2 * c + (i & 1u));
                    w[i] = *reinterpret_cast<const uint2*>(tile + kKT * kDh + key * kDh + 8 * g);
                    w[i].x ^= 0x80808080u, w[i].y ^= 0x80808080u;
                }
#pragma unroll
                for (uint32_t hw = 0; hw < 2; ++hw) {
                    const uint32_t k0 = hw ? w[0].y : w[0].x, k1 = hw ? w[1].y : w[1].x;
                    const uint32_t k2 = hw ? w[2].y : w[2].x, k3 = hw ? w[3].y : w[3].x;
                    const uint32_t lo01 = __byte_perm(k0, k1, 0x5140), hi01 = __byte_perm(k0, k1, 0x7362);
                    const uint32_t lo23 = __byte_perm(k2, k3, 0x5140), hi23 = __byte_perm(k2, k3, 0x7362);
                    const uint32_t va[4] = {codes_f16<false>(lo01), codes_f16<true>(lo01), codes_f16<false>(lo23),
                                            codes_f16<true>(lo23)};
                    const uint32_t vb[4] = {codes_f16<false>(hi01), codes_f16<true>(hi01), codes_f16<false>(hi23),
                                            codes_f16<true>(hi23)};
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        mma_16816<false>(o[t][2 * hw], va, pb[t][0], pb[t][1]);
                        mma_16816<false>(o[t][2 * hw + 1], vb, pb[t][0], pb[t][1]);
                        if constexpr (kFine) {
                            mma_16816<false>(o[t][2 * hw], va, pl[t][0], pl[t][1]);
                            mma_16816<false>(o[t][2 * hw + 1], vb, pl[t][0], pl[t][1]);
                        }
                    }
                }
            } else {
                const uint32_t row = lane & 7u, low = (lane >> 3) & 1u, high = lane >> 4;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    uint32_t va[4];
                    if (a.v_transposed)  // rows d, their keys contiguous
                        ldmatrix4(va, smem_u32(tile) + kTile16 + (16 * i + 8 * low + row) * 64 +
                                          (((2 * k + high) ^ (row >> 1)) * 16));
                    else
                        ldmatrix4_trans(va, smem_u32(tile) + kTile16 + (16 * k + 8 * high + row) * 128 +
                                                (((2 * i + low) ^ row) * 16));
#pragma unroll
                    for (int t = 0; t < NT; ++t) mma_16816<KIND == kVBf16>(o[t][i], va, pb[t][0], pb[t][1]);
                }
            }
        }
        __syncwarp();
        load_next(st);
    }
    if (!ok)  // every copy of this warp has landed before its buffers are used again
        for (uint32_t x = n; x < issued; ++x)
            tc::mbar_wait(&bars[x % kStages], (x / kStages) & 1u, tc::kErrTimeoutFull);
    const float fo = kI8 ? pow2(ev) : 1.f;
    if (solo) {
        // ---- the rows leave from the registers
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (uint32_t e = 0; e < 2; ++e) {
                const uint32_t r = 8 * t + 2 * c + e;
                float total = l[t][e];
                total += __shfl_xor_sync(0xFFFFFFFFu, total, 4);
                total += __shfl_xor_sync(0xFFFFFFFFu, total, 8);
                total += __shfl_xor_sync(0xFFFFFFFFu, total, 16);
                if (r >= it.rows) continue;
                const uint64_t row = row_index(a, it, r, nullptr);
                if (a.part_ml) {
                    const uint64_t at = it.slot * a.total_rows + row;
                    if (g == 0) a.part_ml[at] = make_float2(m[t][e], total);
                    float* dst = a.part_o + at * kDh;
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        if constexpr (kI8) {
                            *reinterpret_cast<float2*>(dst + 8 * g + 2 * i) =
                                make_float2(o[t][i][e] * fo, o[t][i][e + 2] * fo);
                        } else {
                            dst[16 * i + g] = o[t][i][e];
                            dst[16 * i + 8 + g] = o[t][i][e + 2];
                        }
                    }
                } else {
                    const float f = total == 0.f ? 0.f : fo / total;
                    if (a.lse && g == 0)
                        a.lse[row] = total == 0.f ? -INFINITY : (m[t][e] + log2f(total)) * 0.6931471805599453f;
                    uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + row * kDh;
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        const float x = o[t][i][e] * f, y = o[t][i][e + 2] * f;
                        const uint32_t p = a.q_bf16 ? pack_bf16x2(x, y) : pack_f16x2(x, y);
                        if constexpr (kI8) {
                            *reinterpret_cast<uint32_t*>(dst + 8 * g + 2 * i) = p;
                        } else {
                            dst[16 * i + g] = static_cast<uint16_t>(p);
                            dst[16 * i + 8 + g] = static_cast<uint16_t>(p >> 16);
                        }
                    }
                }
            }
        continue;
    }

    // ---- join the warps: [warp][row][64] sums and [warp][row] (m, l) over the rings
    constexpr uint32_t kRowsMax = 8 * NT;
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem);
    float2* ml = reinterpret_cast<float2*>(smem + kWarps * kRowsMax * kSumPitch * 4);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (uint32_t e = 0; e < 2; ++e) {
            const uint32_t r = 8 * t + 2 * c + e;
            float total = l[t][e];
            total += __shfl_xor_sync(0xFFFFFFFFu, total, 4);
            total += __shfl_xor_sync(0xFFFFFFFFu, total, 8);
            total += __shfl_xor_sync(0xFFFFFFFFu, total, 16);
            if (r >= it.rows) continue;
            if (g == 0) ml[warp * kRowsMax + r] = make_float2(m[t][e], total);
            float* dst = sums + (warp * kRowsMax + r) * kSumPitch;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                if constexpr (kI8) {
                    *reinterpret_cast<float2*>(dst + 8 * g + 2 * i) = make_float2(o[t][i][e] * fo, o[t][i][e + 2] * fo);
                } else {
                    dst[16 * i + g] = o[t][i][e];
                    dst[16 * i + 8 + g] = o[t][i][e + 2];
                }
            }
        }
    __syncthreads();
    // four values of a row at a time
    const uint32_t parts = it.rows * (kDh / 4);
    float2* joined_ml = ml + kWarps * kRowsMax;
    for (uint32_t i = threadIdx.x; i < parts; i += kThreads) {
        const uint32_t r = i / (kDh / 4), part = i % (kDh / 4);
        float top = kNoMax, total = 0.f;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        float2 x[kWarps];
#pragma unroll
        for (uint32_t p = 0; p < kWarps; ++p) {
            x[p] = ml[p * kRowsMax + r];
            top = max_nan(top, x[p].x);
        }
#pragma unroll
        for (uint32_t p = 0; p < kWarps; ++p) {
            const float f = growth(x[p].x, top);
            total = __fmaf_rn(f, x[p].y, total);
            add(sum, f, *reinterpret_cast<const float4*>(sums + (p * kRowsMax + r) * kSumPitch + 4 * part));
        }
        if (cluster == 1) {
            write_part(a, it, r, part, top, total, sum);
        } else {
            // (only this thread reads these values of the warps' sums)
            *reinterpret_cast<float4*>(sums + r * kSumPitch + 4 * part) = sum;
            if (part == 0) joined_ml[r] = make_float2(top, total);
        }
    }
    if (cluster == 1) break;
    join_cluster(a, it, smem_u32(sums), smem_u32(joined_ml), cluster, rank, kThreads);
    }
    grid_wait();  // (what waits for this kernel waits for one that it may run beside, too)
}

template <int KIND, bool QBF16, int NT>
uint32_t launch(const CUtensorMap (&maps)[4], const Args& a, uint32_t cls, uint32_t cluster, bool beside,
                uint32_t taken, cudaStream_t st) {
    const auto kernel = kv_few_kernel<KIND, QBF16, NT>;
    static std::atomic<uint64_t> configured{0};
    if (all_shared_once(kernel, kSmem<KIND>, configured) != cudaSuccess) return DH_ERR_CUDA;
    cudaLaunchConfig_t config{};
    // solo: as many CTAs as run at once, their warps walk the items (one CTA an SM beside
    // tensor-core tiles, with room for two, cost 40.3 us instead of 37.4)
    const uint32_t fit = device_sms() * std::max((227u * 1024u - taken) / (kSmem<KIND> + 1024u), 1u);
    const uint32_t items = a.cls[cls].items;
    config.gridDim = dim3(cluster ? items * cluster : std::min((items + kWarps - 1) / kWarps, fit));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = kSmem<KIND>;
    config.stream = st;
    cudaLaunchAttribute attrs[2] = {};
    config.attrs = attrs;
    if (cluster > 1) {
        attrs[config.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attrs[config.numAttrs].val.clusterDim.x = cluster;
        attrs[config.numAttrs].val.clusterDim.y = attrs[config.numAttrs].val.clusterDim.z = 1;
        ++config.numAttrs;
    }
    if (beside) {
        attrs[config.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attrs[config.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cudaLaunchKernelEx(&config, kernel, maps[0], maps[1], maps[2], maps[3], a, cls, cluster) != cudaSuccess) {
        cudaGetLastError();
        return DH_ERR_CUDA;
    }
    return DH_OK;
}

template <int KIND, bool QBF16>
uint32_t launch_rows(const CUtensorMap (&maps)[4], const Args& a, uint32_t cls, uint32_t cluster, bool beside,
                uint32_t taken, cudaStream_t st) {
    return a.cls[cls].tile_rows <= 8 ? launch<KIND, QBF16, 1>(maps, a, cls, cluster, beside, taken, st)
                                     : launch<KIND, QBF16, 2>(maps, a, cls, cluster, beside, taken, st);
}

template <int KIND>
uint32_t launch_type(const CUtensorMap (&maps)[4], const Args& a, uint32_t cls, uint32_t cluster, bool beside,
                uint32_t taken, cudaStream_t st) {
    return a.q_bf16 ? launch_rows<KIND, true>(maps, a, cls, cluster, beside, taken, st)
                    : launch_rows<KIND, false>(maps, a, cls, cluster, beside, taken, st);
}

}  // namespace

uint32_t launch_few(const CUtensorMap (&maps)[4], const Args& a, uint32_t cls, uint32_t cluster, bool int8, bool v_bf16,
                    bool beside, uint32_t taken, cudaStream_t st) {
    return int8 ? launch_type<kInt8>(maps, a, cls, cluster, beside, taken, st)
                : (v_bf16 ? launch_type<kVBf16>(maps, a, cls, cluster, beside, taken, st) : launch_type<kV16>(maps, a, cls, cluster, beside, taken, st));
}

}  // namespace kv
}  // namespace dh
