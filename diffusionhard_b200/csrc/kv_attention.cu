// kv_attention.cu -- attention over K/V caches: softmax(scale Q K^T) V where a
// sequence's keys are [the prefix of its group ; its own rows], either part in
// 16 bits or as int8 codes with a scale for each (head, position), every
// sequence with its own number of keys, several query heads for each K/V head,
// any number of queries from one up.
//
// For a query i: s_j = scale (q_i . k_j), m = max_j s_j, p_j = e^(s_j - m),
// out = sum_j p_j v_j / sum_j p_j, lse = m + log sum_j p_j; without keys out = 0
// and lse = -inf.
//
// Work items.  A row is a (query, query head of the K/V head) pair; 128 rows
// make a tile of the tensor core.  An item is (row tile, K/V head, a range of
// key tiles of 64).  Rows of one sequence walk its prefix and its own keys.  With
// few rows a sequence, those of all sequences of a group are stacked over the prefix,
// which is then read once for all of them, and the sequences' own keys are items of
// their own (see plan_of).  Items of at most 16 rows are kv_few.cu's.  Where keys of
// a row fall to several items, the CTAs of a cluster join their sums through shared
// memory, or each item leaves its unnormalised sums and maximum in the workspace and
// a further kernel joins them, both in a fixed order.
//
// One persistent kernel, two CTAs per SM, 6 warps (int8: 8):
//   warp 0    loads: TMA tiles of K and V (16 bits), or the contiguous codes and
//             scales of 64 keys (int8)
//   warp 1    tcgen05 MMAs: S = Q K^T, Q from TMEM; [O | l] += P [V | 1], P from
//             TMEM, where a column of ones beside V sums P
//   warps 2-3 int8 alone: codes to f16 tiles, see convert_rows
//   four more softmax, a thread a row: P = 2^(s c - m) over S in TMEM; O in TMEM
//             is rescaled only when the maximum grew by more than 2^15
//
// Bound by the softmax: 128 x 512 queries over 1024 16-bit keys take 305 us in a burst
// (676 TFLOP/s; 350 us under the power cap), exponentials 47%, issue slots 47% and the
// tensor pipe 34% of the time busy, with eight warps an SM that wait for one another in
// turn.  Tried and slower:
// exponentials of f16 pairs (360 then, where this took 338), four CTAs an SM with
// 128 columns of TMEM each (365), registers moved between the warps (no change).
#include <cuda.h>

#include "kv_kernels.h"
#include "tmap.h"

#include <algorithm>
#include <cmath>

namespace dh {
namespace {

using namespace kv;

constexpr uint32_t kRows = 128;                  // rows per item
constexpr uint32_t kOnesBytes = 2048;            // 16 rows of 128 bytes
constexpr uint32_t kVPitch = kTileBytes + kOnesBytes;  // (a fine V's second tile behind it)
constexpr uint32_t kTmemCols = 256;
constexpr uint32_t kOCol = 128;                  // S/P buffers at 0 and 64, O at 128, l at 192
constexpr uint32_t kQCol = 224;
constexpr uint32_t kPvN = kDh + 16;
constexpr uint32_t kExpRing = 8;                 // tiles whose exponents are kept

constexpr uint32_t kMaxSplits = 64;              // parts of an item's keys

// kWide: int8 keys that kv_widen.cu has turned into f16.  The fine forms, for queries in
// f16, whose results show more: codes times a scale as the sum of two f16, and so the
// products (600 f16 queries over 1000 keys: off by 1.0e-3 of the result's norm with one
// f16, 2.4e-4 with two, 2.1e-4 of that the result's own rounding).
enum Kind : int { kV16 = 0, kVBf16 = 1, kInt8 = 2, kWide = 3, kInt8Fine = 4, kWideFine = 5 };

template <int KIND>
struct Cfg {
    static constexpr bool int8 = KIND == kInt8 || KIND == kInt8Fine;
    static constexpr bool wide = KIND == kWide || KIND == kWideFine;
    static constexpr bool scaled = int8 || wide;  // keys carry exponents
    static constexpr bool fine = KIND == kInt8Fine || KIND == kWideFine;
    static constexpr uint32_t k_bytes = fine ? 2 * kTileBytes : kTileBytes;
    static constexpr uint32_t v_bytes = fine ? kVPitch + kTileBytes : kVPitch;
    static constexpr uint32_t threads = int8 ? 256 : 192;
    static constexpr uint32_t raw_stages = int8 ? (fine ? 2 : 4) : 0;
    // (16 bits: 4 of K and 3 of V 305 us where 2 and 2 took 302.5)
    static constexpr uint32_t k_stages = 2;
    static constexpr uint32_t v_stages = 2;
    static constexpr uint32_t q_at = 0;
    static constexpr uint32_t k_at = kRows * 128;
    static constexpr uint32_t v_at = k_at + k_stages * k_bytes;
    static constexpr uint32_t ones_at = v_at + v_stages * v_bytes;
    static constexpr uint32_t raw_at = ones_at + kOnesBytes;
    static constexpr uint32_t bars_at = raw_at + raw_stages * kRawBytes;
    static constexpr uint32_t order_at = bars_at + 512;  // lengths, then their order
    static constexpr uint32_t bytes = 1024 + order_at + kOrdered * 6;
};

enum Bar : uint32_t {
    kRawFull = 0, kRawEmpty = kRawFull + 4, kKFull = kRawEmpty + 4, kKEmpty = kKFull + 4, kVFull = kKEmpty + 4,
    kVEmpty = kVFull + 4, kSFull = kVEmpty + 4, kPFull = kSFull + 2, kSPFree = kPFull + 2, kOFull = kSPFree + 2,
    kOFree, kQReady, kDrain, kNumBars
};
static_assert(kNumBars * 8 + 8 + 2 * kExpRing * 4 <= 512, "barrier area");
static_assert(Cfg<0>::bars_at >= kRows * (kSumPitch * 4 + 8) && Cfg<2>::bars_at >= kRows * (kSumPitch * 4 + 8),
              "a CTA's sums lie below the barriers");

DH_DEVINL void fence_proxy_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 2^x of two values on the FMA pipe (x < 100): x = n + f with n = rint(x) by the
// 1.5 * 2^23 shifter, 2^f on [-0.5, 0.5] by a cubic (largest relative error
// 7.8e-5, a third of an f16 half step), 2^n into the exponent field.  Takes a
// quarter of the exponentials off the MUFU.
constexpr float kExp2C0 = 0.99992895f, kExp2C1 = 0.69327623f, kExp2C2 = 0.24260406f, kExp2C3 = 0.05508874f;
DH_DEVINL float2 exp2_poly2(float2 x) {
    x = make_float2(fmaxf(x.x, -120.f), fmaxf(x.y, -120.f));
    const float2 t = __fadd2_rn(x, make_float2(12582912.f, 12582912.f));
    const float2 n = __fadd2_rn(t, make_float2(-12582912.f, -12582912.f));
    const float2 f = __ffma2_rn(n, make_float2(-1.f, -1.f), x);
    float2 p = __ffma2_rn(make_float2(kExp2C3, kExp2C3), f, make_float2(kExp2C2, kExp2C2));
    p = __ffma2_rn(p, f, make_float2(kExp2C1, kExp2C1));
    p = __ffma2_rn(p, f, make_float2(kExp2C0, kExp2C0));
    return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(t.x) << 23)),
                       __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(t.y) << 23)));
}
// The maximum that P is relative to stays until it grew by more than this power of
// two, P's largest value meanwhile (f16 ends at 2^16).  32 canvases over int8, scores
// of a few: 245 us at 8, 237 at 15; 128 x 512 queries over 1024 16-bit keys 325 and 305 then.
constexpr float kMaxGrowth = 15.f;
// f16 loses weights below 2^-25 of the one it is relative to: together up to 2^-11 of
// all over 2^14 keys, which is a rounding of the result.  Longer parts set the maximum
// lower, by the headroom, and keep them down to 2^-33 (their maximum settles early:
// with a headroom of 4 everywhere the 16 tiles of the cases above took 1.5% longer).
constexpr uint32_t kLongTiles = 256;
constexpr float kHeadroom = 8.f;
constexpr uint32_t kPolyPairMask = 0x11u;  // pairs e with bit e % 8 set

// Half of a tile's 64 rows of codes (those of this warp) into a 128-byte swizzled f16
// tile; `factor`: of row `lane` of that half.  FINE: what it lacks into the tile `lo`
// bytes behind it.
template <bool FINE>
DH_DEVINL void convert_rows(const uint8_t* raw, uint8_t* tile, uint32_t lo_at, uint32_t warp_half, uint32_t lane,
                            float factor) {
    const uint32_t c = lane & 3u;
    uint4 codes[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t row = warp_half * 32 + i * 8 + (lane >> 2);
        codes[i] = *reinterpret_cast<const uint4*>(raw + row * kDh + c * 16);
    }
    const uint32_t mine = __half_as_ushort(__float2half_rn(factor));
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t row = warp_half * 32 + i * 8 + (lane >> 2), from = i * 8 + (lane >> 2);
        const auto turn = [&](uint8_t* to, __half2 f, __half2 off) {
            uint4 lo, hi;
            convert16(codes[i], f, off, lo, hi);
            *reinterpret_cast<uint4*>(to + row * 128 + (((2 * c) ^ (row & 7u)) * 16)) = lo;
            *reinterpret_cast<uint4*>(to + row * 128 + (((2 * c + 1) ^ (row & 7u)) * 16)) = hi;
        };
        if constexpr (FINE) {
            const FineFactor f = fine_factor(__shfl_sync(0xFFFFFFFFu, factor, from));
            turn(tile, f.hi, f.off_hi);
            turn(tile + lo_at, f.lo, f.off_lo);
        } else {
            const __half2 f = __half2half2(__ushort_as_half(static_cast<uint16_t>(__shfl_sync(0xFFFFFFFFu, mine, from))));
            turn(tile, f, __hmul2(f, __half2half2(__ushort_as_half(0x8080))));  // (-2^-17)
        }
    }
}

// Zeros over the rows of a V tile from `left` on, by the 128 softmax threads.
DH_DEVINL void zero_rows(uint8_t* tile, uint32_t left, uint32_t transposed, uint32_t thread) {
    if (transposed) {
        for (uint32_t i = thread; i < kDh * kKT; i += 128) {
            const uint32_t d = i / kKT, key = i % kKT;
            if (key >= left)
                *reinterpret_cast<uint16_t*>(tile + d * 128 + (((key >> 3) ^ (d & 7u)) * 16) + (key & 7u) * 2) = 0;
        }
    } else {
        for (uint32_t i = left * 8 + thread; i < kKT * 8; i += 128)
            *reinterpret_cast<uint4*>(tile + i * 16) = make_uint4(0, 0, 0, 0);
    }
}

// Item w of both classes, `first` the number of the first class's (0: they are not
// this kernel's).
DH_DEVINL Item item_at(const Args& a, uint32_t first, uint32_t w, uint32_t live, const uint16_t* order) {
    return w < first ? item_of(a, a.cls[0], w, live, order) : item_of(a, a.cls[1], w - first, live, order);
}

// CLUSTER: the CTAs of a cluster (`cluster` of them) have an item's parts and join them.
template <int KIND, bool CLUSTER>
__global__ void __launch_bounds__(Cfg<KIND>::threads, 2)
kv_attention_kernel(const __grid_constant__ CUtensorMap tpk, const __grid_constant__ CUtensorMap tpv,
                    const __grid_constant__ CUtensorMap tok, const __grid_constant__ CUtensorMap tov,
                    const __grid_constant__ Args a, const uint32_t first, const uint32_t total,
                    const uint32_t cluster) {
    using C = Cfg<KIND>;
    const uint32_t live = a.run_rows ? min(a.sequences, a.queries.of(min(*a.run_rows, 0x7FFFFFFFu))) : a.sequences;
    if (live == 0) {
        if constexpr (C::wide) grid_wait();  // (what waits for this kernel waits for that one)
        return;
    }
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~static_cast<uintptr_t>(1023));
    uint8_t* q_s = smem + C::q_at;
    // (a cluster's CTAs join their sums through shared memory, which is theirs alone
    // once a CTA's one item is done)
    float* sums_s = reinterpret_cast<float*>(smem);
    float2* ml_s = reinterpret_cast<float2*>(smem + kRows * kSumPitch * 4);
    uint8_t* k_ring = smem + C::k_at;
    uint8_t* v_ring = smem + C::v_at;
    uint8_t* ones = smem + C::ones_at;
    uint8_t* raw_ring = smem + C::raw_at;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::bars_at);
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + kNumBars);
    int32_t* exps = reinterpret_cast<int32_t*>(tmem_holder + 2);  // [kExpRing][2]: K, V of a tile

    uint16_t* order = reinterpret_cast<uint16_t*>(smem + C::order_at + kOrdered * 4);
    const uint32_t warp = warp_id(), lane = lane_id();
    grid_launch_dependents();
    if (a.cls[1].ordered) order_sequences(a, reinterpret_cast<uint32_t*>(smem + C::order_at), order);

    if (warp == 0 && lane == 0) {
        for (uint32_t i = 0; i < kNumBars; ++i) {
            uint32_t count = 1;
            if ((i >= kPFull && i < kPFull + 2) || i == kOFree || i == kQReady) count = 128;
            if (C::int8 && ((i >= kRawEmpty && i < kRawEmpty + 4) || (i >= kKFull && i < kKFull + 4) ||
                            (i >= kVFull && i < kVFull + 4)))
                count = 2;
            tc::mbar_init(&bars[i], count);
        }
        tc::fence_barrier_init();
        if (!C::int8) {
            tc::prefetch_tmap(&tok);
            tc::prefetch_tmap(&tov);
            if (a.cls[0].with_prefix | a.cls[1].with_prefix) {
                tc::prefetch_tmap(&tpk);
                tc::prefetch_tmap(&tpv);
            }
        }
    }
    // The column of ones.  V as it is stored ([key][64]): 16 rows (keys) whose
    // first element is 1, the same for every 16 keys.  Transposed V ([64][key]): 16
    // further rows under every tile, the first of them ones.
    const uint32_t one2 = KIND == kVBf16 ? 0x3F803F80u : 0x3C003C00u;
    if (a.v_transposed) {
        for (uint32_t i = threadIdx.x; i < C::v_stages * 512; i += C::threads) {
            const uint32_t st = i / 512, w = i % 512;
            reinterpret_cast<uint32_t*>(v_ring + st * C::v_bytes + kTileBytes)[w] = w < 32 ? one2 : 0u;
        }
    } else {
        for (uint32_t i = threadIdx.x; i < 512; i += C::threads) {
            const uint32_t r = i / 32, w = i % 32;
            reinterpret_cast<uint32_t*>(ones)[i] = w == (r & 7u) * 4 ? (one2 & 0xFFFFu) : 0u;
        }
    }
    fence_proxy_async_smem();
    if (warp == 1) tc::tmem_alloc(tmem_holder, kTmemCols);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_holder;
    if constexpr (C::wide) grid_wait();  // (the keys are another kernel's)

    if (warp == 0) {
        // ---------------------------------------------------------- loads
        if (tc::elect_one()) {
            uint32_t g = 0;
            bool ok = true;
            for (uint32_t w = blockIdx.x; w < total && ok; w += gridDim.x) {
                const Item it = item_at(a, first, w, live, order);
                for (uint32_t j = it.t0; j < it.t1; ++j, ++g) {
                    const bool own = j >= it.n0;
                    const uint32_t key = (own ? j - it.n0 : j) * kKT;
                    const uint32_t entry = own ? it.own : it.prefix;
                    if constexpr (C::int8) {
                        const uint32_t rs = g % C::raw_stages;
                        if (!tc::mbar_wait_suspend(&bars[kRawEmpty + rs], ((g / C::raw_stages) & 1u) ^ 1u,
                                                   tc::kErrTimeoutEmpty)) {
                            ok = false;
                            break;
                        }
                        const Segment& s = own ? a.own : a.prefix;
                        const uint64_t at = (static_cast<uint64_t>(entry) * a.kv_heads.d + it.kv_head) * s.pitch + key;
                        uint8_t* dst = raw_ring + rs * kRawBytes;
                        uint64_t* bar = &bars[kRawFull + rs];
                        tc::mbar_arrive_expect_tx(bar, kRawBytes);
                        tc::bulk_load(dst, s.k + at * kDh, kKT * kDh, bar);
                        tc::bulk_load(dst + 2 * kKT * kDh, s.k_scale + at, kKT * 4, bar);
                        tc::bulk_load(dst + kKT * kDh, s.v + at * kDh, kKT * kDh, bar);
                        tc::bulk_load(dst + 2 * kKT * kDh + kKT * 4, s.v_scale + at, kKT * 4, bar);
                    } else {
                        const uint32_t ks = g % C::k_stages, vs = g % C::v_stages;
                        if (!tc::mbar_wait_suspend(&bars[kKEmpty + ks], ((g / C::k_stages) & 1u) ^ 1u,
                                                   tc::kErrTimeoutEmpty)) {
                            ok = false;
                            break;
                        }
                        tc::mbar_arrive_expect_tx(&bars[kKFull + ks], C::k_bytes);
                        tc::tma_load_4d(k_ring + ks * C::k_bytes, own ? &tok : &tpk, &bars[kKFull + ks], 0, key,
                                        it.kv_head, entry);
                        // (what they lack lies behind all entries)
                        const uint32_t lo_entry = C::fine ? entry + (own ? a.sequences : a.prefixes) : 0u;
                        if constexpr (C::fine)
                            tc::tma_load_4d(k_ring + ks * C::k_bytes + kTileBytes, own ? &tok : &tpk,
                                            &bars[kKFull + ks], 0, key, it.kv_head, lo_entry);
                        if (!tc::mbar_wait_suspend(&bars[kVEmpty + vs], ((g / C::v_stages) & 1u) ^ 1u,
                                                   tc::kErrTimeoutEmpty)) {
                            ++g;  // (the K tile is on its way)
                            ok = false;
                            break;
                        }
                        tc::mbar_arrive_expect_tx(&bars[kVFull + vs], C::fine ? 2 * kTileBytes : kTileBytes);
                        tc::tma_load_4d(v_ring + vs * C::v_bytes, own ? &tov : &tpv, &bars[kVFull + vs],
                                        a.v_transposed ? key : 0, a.v_transposed ? 0 : key, it.kv_head, entry);
                        if constexpr (C::fine)
                            tc::tma_load_4d(v_ring + vs * C::v_bytes + kVPitch, own ? &tov : &tpv, &bars[kVFull + vs],
                                            0, key, it.kv_head, lo_entry);
                    }
                }
            }
            // every copy this CTA issued has landed before it may exit
            if constexpr (C::int8) {
                for (uint32_t x = g > C::raw_stages ? g - C::raw_stages : 0; x < g; ++x)
                    tc::mbar_wait_suspend(&bars[kRawFull + x % C::raw_stages], (x / C::raw_stages) & 1u,
                                          tc::kErrTimeoutFull);
            } else {
                for (uint32_t x = g > C::k_stages ? g - C::k_stages : 0; x < g; ++x)
                    tc::mbar_wait_suspend(&bars[kKFull + x % C::k_stages], (x / C::k_stages) & 1u,
                                          tc::kErrTimeoutFull);
                for (uint32_t x = g > C::v_stages ? g - C::v_stages : 0; x < g; ++x)
                    tc::mbar_wait_suspend(&bars[kVFull + x % C::v_stages], (x / C::v_stages) & 1u,
                                          tc::kErrTimeoutFull);
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA
        if (tc::elect_one()) {
            const uint32_t o_tmem = tmem + kOCol;
            constexpr uint32_t kIdescLo = tc::idesc_f16_f32<kRows, kDh>() | tc::kIdescBMnMajor;
            auto issue_s = [&](uint32_t g) -> bool {
                const uint32_t ks = g % C::k_stages, sb = g & 1u;
                if (!tc::mbar_wait_suspend(&bars[kKFull + ks], (g / C::k_stages) & 1u, tc::kErrTimeoutFull) ||
                    !tc::mbar_wait_suspend(&bars[kSPFree + sb], ((g >> 1) & 1u) ^ 1u, tc::kErrTimeoutAccEmpty))
                    return false;
                tc::tc_fence_after();
                const uint64_t k_desc = tc::smem_desc_sw128(k_ring + ks * C::k_bytes);
#pragma unroll
                for (uint32_t kk = 0; kk < C::k_bytes / kTileBytes * (kDh / 16); ++kk)
                    tc::mma_f16_ts(tmem + sb * kKT, tmem + kQCol + (kk % 4) * 8,
                                   tc::desc_advance(k_desc, kk / 4 * kTileBytes + (kk % 4) * 32), a.idesc_s, kk != 0);
                tc::mma_commit(&bars[kSFull + sb]);
                tc::mma_commit(&bars[kKEmpty + ks]);
                return true;
            };
            uint32_t g = 0, n_items = 0;
            bool ok = true;
            for (uint32_t w = blockIdx.x; w < total && ok; w += gridDim.x) {
                const Item it = item_at(a, first, w, live, order);
                if (it.t0 == it.t1) continue;
                if (!tc::mbar_wait_suspend(&bars[kQReady], n_items & 1u, tc::kErrTimeoutFull)) break;
                tc::tc_fence_after();
                if (!issue_s(g)) break;
                for (uint32_t j = it.t0; j < it.t1; ++j, ++g) {
                    if (j + 1 < it.t1 && !issue_s(g + 1)) {
                        ok = false;
                        break;
                    }
                    const uint32_t vs = g % C::v_stages, sb = g & 1u;
                    ok = tc::mbar_wait_suspend(&bars[kPFull + sb], (g >> 1) & 1u, tc::kErrTimeoutFull) &&
                         tc::mbar_wait_suspend(&bars[kVFull + vs], (g / C::v_stages) & 1u, tc::kErrTimeoutFull) &&
                         (j != it.t0 ||
                          tc::mbar_wait_suspend(&bars[kOFree], (n_items & 1u) ^ 1u, tc::kErrTimeoutAccEmpty));
                    if (!ok) break;
                    tc::tc_fence_after();
                    const uint8_t* v_tile = v_ring + vs * C::v_bytes;
                    if (a.v_transposed) {
                        const uint64_t v_desc = tc::smem_desc_sw128(v_tile);
#pragma unroll
                        for (uint32_t kk = 0; kk < kKT / 16; ++kk)
                            tc::mma_f16_ts(o_tmem, tmem + sb * kKT + kk * 8, tc::desc_advance(v_desc, kk * 32),
                                           a.idesc_o, kk != 0 || j != it.t0);
                    } else {
#pragma unroll
                        for (uint32_t kk = 0; kk < kKT / 16; ++kk) {
                            const uint8_t* at = v_tile + kk * 2048;
                            tc::mma_f16_ts(o_tmem, tmem + sb * kKT + kk * 8,
                                           tc::smem_desc_mn_sw128(at, static_cast<uint32_t>(ones - at)), a.idesc_o,
                                           kk != 0 || j != it.t0);
                            if constexpr (C::fine)
                                tc::mma_f16_ts(o_tmem, tmem + sb * kKT + kk * 8,
                                               tc::smem_desc_mn_sw128(at + kVPitch, kTileBytes), kIdescLo, true);
                        }
                    }
                    tc::mma_commit(&bars[kVEmpty + vs]);
                    tc::mma_commit(&bars[kSPFree + sb]);
                    if (j + 1 == it.t1) tc::mma_commit(&bars[kOFull]);
                }
                ++n_items;
            }
            tc::mma_commit(&bars[kDrain]);
            tc::mbar_wait_suspend(&bars[kDrain], 0, tc::kErrTimeoutAccFull);
        }
    } else if (C::int8 && warp < 4) {
        uint32_t g = 0;
        bool ok = true;
        if constexpr (C::int8) {
            // ---------------------------------------------------- conversion
            const uint32_t half = warp - 2;
            for (uint32_t w = blockIdx.x; w < total && ok; w += gridDim.x) {
                const Item it = item_at(a, first, w, live, order);
                int32_t ev = -1000;
                for (uint32_t j = it.t0; j < it.t1; ++j, ++g) {
                    const uint32_t rs = g % C::raw_stages, ks = g % C::k_stages, vs = g % C::v_stages;
                    if (!tc::mbar_wait_suspend(&bars[kRawFull + rs], (g / C::raw_stages) & 1u, tc::kErrTimeoutFull)) {
                        ok = false;
                        break;
                    }
                    const uint8_t* raw = raw_ring + rs * kRawBytes;
                    const float* scales = reinterpret_cast<const float*>(raw + 2 * kKT * kDh);
                    const uint32_t left = keys_left(it, j);
                    // scales of rows lane and lane + 32, 0 behind the last key (what lies
                    // there is anything); the tile's exponents, from the finite ones
                    float sc[2][2];
                    int32_t e[2];
#pragma unroll
                    for (uint32_t side = 0; side < 2; ++side) {
                        uint32_t peak = 0;
#pragma unroll
                        for (uint32_t h = 0; h < 2; ++h) {
                            const uint32_t row = lane + 32 * h;
                            const float f = row < left ? scales[side * kKT + row] : 0.f;
                            sc[side][h] = f;
                            const uint32_t bits = __float_as_uint(f) & 0x7FFFFFFFu;
                            if (bits < 0x7F800000u) peak = max(peak, bits);
                        }
                        e[side] = max(exponent_of(__reduce_max_sync(0xFFFFFFFFu, peak)), -100);
                    }
                    // O keeps one exponent of V for all tiles of an item, four times what
                    // it has to be when it is set: it only grows, and O is rescaled when
                    // it does
                    ev = e[1] > ev ? min(e[1] + 2, 126) : ev;
                    const float fk = pow2(15 - min(e[0], 126)), fv = pow2(15 - ev);
                    if (!tc::mbar_wait_suspend(&bars[kKEmpty + ks], ((g / C::k_stages) & 1u) ^ 1u,
                                               tc::kErrTimeoutEmpty)) {
                        ok = false;
                        break;
                    }
                    if (half == 0 && lane == 0) {
                        exps[(g % kExpRing) * 2] = min(e[0], 126) + 9;
                        exps[(g % kExpRing) * 2 + 1] = ev + 9;
                    }
                    convert_rows<C::fine>(raw, k_ring + ks * C::k_bytes, kTileBytes, half, lane, (half ? sc[0][1] : sc[0][0]) * fk);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&bars[kKFull + ks]);
                    if (!tc::mbar_wait_suspend(&bars[kVEmpty + vs], ((g / C::v_stages) & 1u) ^ 1u,
                                               tc::kErrTimeoutEmpty)) {
                        ok = false;
                        break;
                    }
                    convert_rows<C::fine>(raw + kKT * kDh, v_ring + vs * C::v_bytes, kVPitch, half, lane, (half ? sc[1][1] : sc[1][0]) * fv);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tc::mbar_arrive(&bars[kVFull + vs]);
                        tc::mbar_arrive(&bars[kRawEmpty + rs]);
                    }
                }
            }
        }
    } else {
        // ----------------------------------------------------------- softmax
        const uint32_t quad = warp & 3u;
        const uint32_t r = quad * 32 + lane;
        const uint32_t lane_base = (quad * 32u) << 16;
        uint8_t* my_q = q_s + r * 128;

        // Row `row` of slot `slot` has no keys.  (Sums in shared memory: see below.)
        auto write_empty = [&](uint64_t row, uint32_t slot) {
            if constexpr (CLUSTER) {
                ml_s[r] = make_float2(kNoMax, 0.f);
#pragma unroll
                for (uint32_t i = 0; i < kDh / 4; ++i)
                    reinterpret_cast<float4*>(sums_s + r * kSumPitch)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                return;
            }
            if (a.part_ml) {
                a.part_ml[slot * a.total_rows + row] = make_float2(0.f, 0.f);
                return;
            }
            uint4* dst = reinterpret_cast<uint4*>(a.out + row * (kDh * 2));
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) dst[i] = make_uint4(0, 0, 0, 0);
            if (a.lse) a.lse[row] = -INFINITY;
        };
        // From item w on: rows of items without keys are answered at once; the
        // first item with keys (w >= total: none), its query row on its way to
        // shared memory.
        auto next_item = [&](uint32_t& w, Item& it) {
            for (; w < total; w += gridDim.x) {
                it = item_at(a, first, w, live, order);
                if (it.t0 != it.t1) break;
                if (r < it.rows) write_empty(row_index(a, it, r, nullptr), it.slot);
            }
            if (w < total && r < it.rows) {
                const uint8_t* q;
                row_index(a, it, r, &q);
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                                     smem_u32(my_q + ((i ^ (r & 7u)) * 16))),
                                 "l"(__cvta_generic_to_global(q + i * 16)));
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        // This thread's query row from shared memory into TMEM.  Returns the
        // factor of its scores.  int8 keys: the row as f16 between 1/2 and 1 in
        // magnitude, its exponent in the factor.
        auto copy_q = [&]() -> float {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            uint32_t qv[32];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                const uint4 v = *reinterpret_cast<const uint4*>(my_q + ((i ^ (r & 7u)) * 16));
                qv[4 * i] = v.x, qv[4 * i + 1] = v.y, qv[4 * i + 2] = v.z, qv[4 * i + 3] = v.w;
            }
            float c = a.c;
            if constexpr (C::scaled) {
                uint32_t peak = 0;
                if (a.q_bf16) {
#pragma unroll
                    for (uint32_t i = 0; i < 32; ++i)
                        peak = max(peak, max((qv[i] << 16) & 0x7FFF0000u, qv[i] & 0x7FFF0000u));
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < 32; ++i) {
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&qv[i]));
                        peak = max(peak, max(__float_as_uint(f.x) & 0x7FFFFFFFu, __float_as_uint(f.y) & 0x7FFFFFFFu));
                    }
                }
                const int32_t e = min(max(exponent_of(peak), -100), 126);
                const float f = pow2(-e);
#pragma unroll
                for (uint32_t i = 0; i < 32; ++i) {
                    float2 x;
                    if (a.q_bf16)
                        x = make_float2(__uint_as_float(qv[i] << 16), __uint_as_float(qv[i] & 0xFFFF0000u));
                    else
                        x = __half22float2(*reinterpret_cast<const __half2*>(&qv[i]));
                    qv[i] = pack_f16x2(x.x * f, x.y * f);
                }
                c *= pow2(e);
            }
            tc::tmem_st_32x32b_x32(tmem + lane_base + kQCol, qv);
            tc::tmem_st_wait();
            tc::tc_fence_before();
            tc::mbar_arrive(&bars[kQReady]);
            return c;
        };

        uint32_t g = 0, n_items = 0;
        bool ok = true;
        Item it;
        uint32_t w = blockIdx.x;
        next_item(w, it);
        float c = 0.f;
        if (w < total) c = copy_q();
        while (w < total && ok) {
            Item next;
            uint32_t next_w = w + gridDim.x;
            next_item(next_w, next);
            const bool active = quad * 32 < it.rows;  // the warp has rows
            float m = -INFINITY;
            int32_t ev = -1000;  // exponent of O (int8 keys)
            float2 ex0 = make_float2(1.f, 0.f), ex1 = ex0;  // of the prefix, of its own keys
            if constexpr (C::wide) {
                if (it.len0) ex0 = a.prefix_exps[it.prefix * a.kv_heads.d + it.kv_head];
                if (it.len1) ex1 = a.own_exps[it.own * a.kv_heads.d + it.kv_head];
            }
            for (uint32_t j = it.t0; j < it.t1; ++j, ++g) {
                const uint32_t sb = g & 1u;
                if (!tc::mbar_wait_suspend(&bars[kSFull + sb], (g >> 1) & 1u, tc::kErrTimeoutAccFull)) {
                    ok = false;
                    break;
                }
                tc::tc_fence_after();
                if (active) {
                    uint32_t sv[64];
                    tc::tmem_ld_32x32b_x32(tmem + lane_base + sb * kKT, *reinterpret_cast<uint32_t(*)[32]>(&sv[0]));
                    tc::tmem_ld_32x32b_x32(tmem + lane_base + sb * kKT + 32,
                                           *reinterpret_cast<uint32_t(*)[32]>(&sv[32]));
                    float ct = C::scaled ? c : a.c;
                    int32_t et = 0;
                    if constexpr (C::int8) {
                        ct = fmaxf(c * pow2(min(exps[(g % kExpRing) * 2], 128)), kLeastFactor);
                        et = exps[(g % kExpRing) * 2 + 1];
                    } else if constexpr (C::scaled) {
                        const float2 ex = j < it.n0 ? ex0 : ex1;
                        ct = fmaxf(c * ex.x, kLeastFactor);
                        et = __float_as_int(ex.y);
                    }
                    const uint32_t left = keys_left(it, j);
                    tc::tmem_ld_wait();
                    if (left < kKT) {
#pragma unroll
                        for (uint32_t e = 0; e < 64; ++e)
                            if (e >= left) sv[e] = 0xFF800000u;
                    }
                    float pm[8];
#pragma unroll
                    for (uint32_t q = 0; q < 8; ++q) pm[q] = __uint_as_float(sv[q]);
#pragma unroll
                    for (uint32_t e = 8; e < 56; e += 16) {
#pragma unroll
                        for (uint32_t q = 0; q < 8; ++q)
                            pm[q] = max_nan(pm[q], __uint_as_float(sv[e + q]), __uint_as_float(sv[e + 8 + q]));
                    }
#pragma unroll
                    for (uint32_t q = 0; q < 8; ++q) pm[q] = max_nan(pm[q], __uint_as_float(sv[56 + q]));
                    const float tmax = max_nan(max_nan(max_nan(pm[0], pm[1]), pm[2], pm[3]),
                                               max_nan(max_nan(pm[4], pm[5]), pm[6], pm[7]));
                    // finite (a row of -inf would give inf - inf), or NaN for an infinite
                    // score, as for one that is NaN: the row is NaN
                    float mt = max_nan(tmax * ct, kNoMax);
                    mt = __fmaf_rn(mt, -0.f, mt);
                    float alpha = 1.f, alpha_o = 1.f;
                    bool need = false;
                    // (far maxima without room: 32 canvases over int8 195 us without this
                    // and 198 with it, 128 x 512 queries 304 and 305.5; other forms to 311)
                    if (!(max_nan(mt - kMaxGrowth, fabsf(mt) < kFar ? m : mt) <= m)) {
                        need = true;
                        mt -= fabsf(mt) < kFar && it.t1 - it.t0 > kLongTiles ? kHeadroom : 0.f;
                        alpha = growth(m, mt);
                        m = mt;
                    }
                    alpha_o = alpha;
                    if (C::scaled && et > ev) {
                        need = true;
                        alpha_o = alpha * pow2(max(ev - et, -126));
                        ev = et;
                    }
                    need = need && j != it.t0;
                    const float damp = damping(m), cd = fmaxf(ct * damp, kLeastFactor), nm = -m * damp;
                    const float2 c2 = make_float2(cd, cd), nm2 = make_float2(nm, nm);
                    uint32_t pk[32];
#pragma unroll
                    for (uint32_t e = 0; e < 32; ++e) {
                        const float2 s2 = make_float2(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1]));
                        const float2 x = __ffma2_rn(s2, c2, nm2);
                        float2 y;
                        if ((kPolyPairMask >> (e & 7u)) & 1u)
                            y = exp2_poly2(x);
                        else
                            y = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                        pk[e] = KIND == kVBf16 ? pack_bf16x2(y.x, y.y) : pack_f16x2(y.x, y.y);
                    }
                    tc::tmem_st_32x32b_x32(tmem + lane_base + sb * kKT, pk);
                    // (rows behind the last hold anything: they ask for nothing)
                    if (__any_sync(0xFFFFFFFFu, need && r < it.rows)) {
                        // PV of the tile before (the only one that may still run) finished
                        if (!tc::mbar_wait_suspend(&bars[kSPFree + (sb ^ 1u)], ((g - 1) >> 1) & 1u,
                                                   tc::kErrTimeoutEmpty)) {
                            ok = false;
                            break;
                        }
                        tc::tc_fence_after();
#pragma unroll
                        for (uint32_t h2 = 0; h2 < 2; ++h2) {
                            uint32_t ov[32];
                            tc::tmem_ld_32x32b_x32(tmem + lane_base + kOCol + 32 * h2, ov);
                            tc::tmem_ld_wait();
#pragma unroll
                            for (uint32_t d = 0; d < 32; ++d)
                                ov[d] = __float_as_uint(__uint_as_float(ov[d]) * alpha_o);
                            tc::tmem_st_32x32b_x32(tmem + lane_base + kOCol + 32 * h2, ov);
                        }
                        const uint32_t lv = tc::tmem_ld_32x32b_x1(tmem + lane_base + kOCol + kDh);
                        tc::tmem_ld_wait();
                        tc::tmem_st_32x32b_x1(tmem + lane_base + kOCol + kDh,
                                              __float_as_uint(__uint_as_float(lv) * alpha));
                    }
                    tc::tmem_st_wait();
                    tc::tc_fence_before();
                }
                if (!C::int8 && keys_left(it, j) < kKT) {
                    // V behind the last key: 0 * NaN must not reach O.  (The stage is
                    // not loaded again before this tile's PV, which waits for this.)
                    const uint32_t vs = g % C::v_stages;
                    if (!tc::mbar_wait_suspend(&bars[kVFull + vs], (g / C::v_stages) & 1u, tc::kErrTimeoutFull)) {
                        ok = false;
                        break;
                    }
                    zero_rows(v_ring + vs * C::v_bytes, keys_left(it, j), a.v_transposed, r);
                    fence_proxy_async_smem();
                }
                tc::mbar_arrive(&bars[kPFull + sb]);
            }
            if (!ok) break;
            // the next item's Q before this item's result, so that its S can start
            float next_c = 0.f;
            if (next_w < total) next_c = copy_q();
            if (!tc::mbar_wait_suspend(&bars[kOFull], n_items & 1u, tc::kErrTimeoutAccFull)) break;
            tc::tc_fence_after();
            const float l = __uint_as_float(tc::tmem_ld_32x32b_x1(tmem + lane_base + kOCol + kDh));
            const uint64_t row = row_index(a, it, r, nullptr);
            const bool mine = r < it.rows;
            tc::tmem_ld_wait();
            float f = C::scaled ? pow2(min(ev, 128)) : 1.f;
            float4* part = nullptr;
            if constexpr (CLUSTER) {
                ml_s[r] = make_float2(m, l);
                part = reinterpret_cast<float4*>(sums_s + r * kSumPitch);
            } else if (a.part_ml) {
                const uint64_t at = it.slot * a.total_rows + row;
                if (mine) a.part_ml[at] = make_float2(m, l);
                part = reinterpret_cast<float4*>(a.part_o + at * kDh);
            } else {
                f = l == 0.f ? 0.f : f / l;
                if (mine && a.lse) a.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
            }
            uint4* dst = reinterpret_cast<uint4*>(a.out + row * (kDh * 2));
            // (a loop: code that runs once an item is mostly time to fetch it)
#pragma unroll 1
            for (uint32_t h = 0; h < 4; ++h) {
                uint32_t v[16];
                tc::tmem_ld_32x32b_x16(tmem + lane_base + kOCol + 16 * h, v);
                tc::tmem_ld_wait();
                if (!mine) continue;
                float x[16];
#pragma unroll
                for (uint32_t i = 0; i < 16; ++i) x[i] = __uint_as_float(v[i]) * f;
                if (part) {
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i)
                        part[4 * h + i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < 2; ++i) {
                        const float* y = x + 8 * i;
                        dst[2 * h + i] = a.q_bf16 ? make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]),
                                                               pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]))
                                                  : make_uint4(pack_f16x2(y[0], y[1]), pack_f16x2(y[2], y[3]),
                                                               pack_f16x2(y[4], y[5]), pack_f16x2(y[6], y[7]));
                    }
                }
            }
            tc::tc_fence_before();
            tc::mbar_arrive(&bars[kOFree]);
            ++n_items;
            w = next_w;
            it = next;
            c = next_c;
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, kTmemCols);
    }
    if constexpr (CLUSTER)
        join_cluster(a, item_at(a, first, blockIdx.x, live, order), smem_u32(sums_s), smem_u32(ml_s), cluster,
                     cluster_rank(), C::threads);
}

// Joins the parts of a row, 8 lanes a row: with M = max m, w_s = 2^(m_s - M),
// out = sum w_s O_s / sum w_s l_s over the slots in their order.  A lane holds the
// weights of every 8th slot and 8 values of the row.
constexpr uint32_t kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads) kv_join_kernel(const float2* ml, const float* part, uint32_t slots,
                                                               uint64_t rows, FastDiv queries, uint32_t heads,
                                                               uint32_t bf16, uint8_t* out, float* lse,
                                                               const uint32_t* run_rows) {
    grid_wait();  // (the parts are other kernels')
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * (kJoinThreads / 8) + threadIdx.x / 8;
    const uint32_t c = threadIdx.x & 7u;
    uint64_t live = rows;
    if (run_rows)
        live = min(rows, static_cast<uint64_t>(queries.of(min(*run_rows, 0x7FFFFFFFu))) * queries.d * heads);
    const bool mine = row < live;  // (lanes of other rows stay for the exchanges)
    // (all loads before their use, the first eight parts' before the maximum is known;
    // what an empty part holds is dropped, not added)
    const float4* from = reinterpret_cast<const float4*>(part + row * kDh) + c;
    float4 xs[8], ys[8];
    const auto load = [&](uint32_t s0) {
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) {
            xs[k] = ys[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (mine && s0 + k < slots) {
                const float4* at = from + (s0 + k) * rows * (kDh / 4);
                xs[k] = at[0], ys[k] = at[8];
            }
        }
    };
    const auto stats = [&](uint32_t s) { return mine && s < slots ? ml[s * rows + row] : make_float2(0.f, 0.f); };
    float2 x = stats(c);
    load(0);
    float top = x.y != 0.f ? x.x : -INFINITY;
    for (uint32_t s = c + 8; s < slots; s += 8) {
        const float2 other = stats(s);
        if (other.y != 0.f) top = max_nan(top, other.x);
    }
#pragma unroll
    for (uint32_t o = 1; o < 8; o <<= 1) top = max_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    float l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    for (uint32_t s0 = 0; s0 < slots; s0 += 8) {
        if (s0) {
            x = stats(s0 + c);
            load(s0);
        }
        const float w = x.y != 0.f ? growth(x.x, top) : 0.f;
        l = __fmaf_rn(w, x.y, l);
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) {
            const float f = __shfl_sync(0xFFFFFFFFu, w, (threadIdx.x & 24u) + k);
            if (f == 0.f) continue;
            add(a, f, xs[k]);
            add(b, f, ys[k]);
        }
    }
#pragma unroll
    for (uint32_t o = 1; o < 8; o <<= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
    if (!mine) return;
    const float f = l == 0.f ? 0.f : 1.f / l;
    uint2* dst = reinterpret_cast<uint2*>(out) + row * (kDh / 4) + c;
    dst[0] = bf16 ? make_uint2(pack_bf16x2(a.x * f, a.y * f), pack_bf16x2(a.z * f, a.w * f))
                  : make_uint2(pack_f16x2(a.x * f, a.y * f), pack_f16x2(a.z * f, a.w * f));
    dst[8] = bf16 ? make_uint2(pack_bf16x2(b.x * f, b.y * f), pack_bf16x2(b.z * f, b.w * f))
                  : make_uint2(pack_f16x2(b.x * f, b.y * f), pack_f16x2(b.z * f, b.w * f));
    if (lse && c == 0) lse[row] = l == 0.f ? -INFINITY : (top + log2f(l)) * 0.6931471805599453f;
}

// ------------------------------------------------------------------ plan

// Visits of every tile of int8 keys from which they are turned into f16 first.
constexpr uint32_t kWidenFrom = 4;

struct Plan {
    Class cls[2];         // prefix of stacked rows, and each sequence's own keys
    bool widen;           // int8 keys are turned into f16 first
    bool few[2];          // items of the kernel for few rows, on `cluster` CTAs each
    uint32_t cluster[2];
    uint32_t many_cluster;  // CTAs an item of tensor-core tiles, 0: none share one
    uint32_t slots;
    uint64_t estimate;    // of tensor-core tiles alone, in tiles
};

uint32_t ceil_div(uint64_t a, uint64_t b) { return static_cast<uint32_t>((a + b - 1) / b); }

// Few rows: a warp an item where there are items enough with few tiles (single tokens,
// 12 heads, int8, such warps and the other way: 40 x 128 keys 8.3 and 10.3 us, 64 x 256
// 12.4 and 14.5, 64 x 1024 28.8 and 26.8, 100 x 1024 31.9 and 37.9, 128 x 1024 36.5 and
// 45.3, 128 x 4096 111 and 98).  Else parts of at least a tile a warp, up to eight in a
// cluster until the GPU has four CTAs an SM, then as many clusters as that still takes.
void split_few(Class& c, uint32_t& cluster, uint64_t items, uint32_t tiles, uint32_t sms) {
    if (items >= 3ull * sms && tiles <= (items >= 8ull * sms ? 32u : 8u)) {
        cluster = 0;
        return;
    }
    cluster = 1;
    while (cluster < kMaxCluster && cluster * 8 <= tiles && items * cluster < 4ull * sms) cluster *= 2;
    const uint64_t ctas = items * cluster;
    if (ctas < 2ull * sms)
        c.splits = FastDiv(static_cast<uint32_t>(
            std::min<uint64_t>({kMaxSplits, std::max<uint64_t>(tiles / (cluster * 8), 1),
                                std::max<uint64_t>(3ull * sms / ctas, 1)})));
}

// Tensor-core tiles: 1 to 64 parts of the keys, by the shortest estimated time, in
// tiles: full rounds of items on the CTAs that run at once, two tiles of start and end
// for each item, six for a kernel that joins the parts, one for a join in a cluster
// (at most eight parts, and an eighth of the CTAs are lost to SMs that a cluster's
// shape leaves over: 24 x 4 items of 74 tiles took 65 us in 96 clusters of three, of
// which not all run at once, and 47 with the kernel; 8 x 12 items of 16 tiles 17.2 us
// in clusters of two and 16.5 with the kernel and three parts, which is another launch).
// Returns the size of the clusters, 0: none.
uint32_t split_many(Class* cls, const uint64_t* items, const uint32_t* tiles, uint32_t ctas, bool joined,
                    uint64_t& best) {
    best = ~0ull;
    uint32_t best_splits[2] = {1, 1}, best_cluster = 0;
    const uint32_t most = std::max(std::max(items[0] ? tiles[0] : 0, items[1] ? tiles[1] : 0), 1u);
    for (uint32_t n = 1; n <= kMaxSplits; ++n) {
        const uint32_t chunk = ceil_div(most, n);
        uint64_t work = 0, longest = 0;
        uint32_t splits[2];
        for (int i = 0; i < 2; ++i) {
            splits[i] = std::min(std::max(ceil_div(tiles[i], chunk), 1u), kMaxSplits);
            const uint64_t each = ceil_div(tiles[i], splits[i]) + 2;
            if (!items[i]) continue;
            work += items[i] * splits[i] * each;
            longest = std::max(longest, each);
        }
        const uint64_t count = items[0] * splits[0] + items[1] * splits[1];
        const auto rounds = [&](uint32_t at_once) {
            return std::max<uint64_t>(ceil_div(count, at_once) * longest, ceil_div(work, at_once));
        };
        const bool split = joined || splits[1] > 1;
        const bool may_cluster = !joined && split && splits[1] <= kMaxCluster;
        const uint64_t alone = rounds(ctas) + (split ? 6 : 0);
        const uint64_t clustered = may_cluster ? rounds(ctas * 7 / 8) + 1 : ~0ull;
        if (std::min(alone, clustered) < best) {
            best = std::min(alone, clustered);
            best_cluster = clustered < alone ? splits[1] : 0;
            best_splits[0] = splits[0];
            best_splits[1] = splits[1];
        }
        if (chunk == 1) break;
    }
    for (int i = 0; i < 2; ++i)
        if (items[i]) cls[i].splits = FastDiv(best_splits[i]);
    return best_cluster;
}

// stacked: a group's rows are stacked over its prefix.
Plan plan_with(bool stacked, uint32_t sequences, uint32_t rows, uint32_t kv_heads, uint32_t prefixes,
               uint32_t prefix_keys, uint32_t own_keys, bool int8, bool ragged, uint32_t sms) {
    Plan p{};
    const uint32_t per = prefixes ? sequences / prefixes : sequences;
    const uint32_t t0 = ceil_div(prefix_keys, kKT), t1 = ceil_div(own_keys, kKT);
    const uint32_t tiles[2] = {stacked ? t0 : 0, t1 + (stacked || !prefixes ? 0 : t0)};
    uint64_t items[2] = {0, 0}, many[2] = {0, 0};
    for (int i = stacked ? 0 : 1; i < 2; ++i) {
        Class& c = p.cls[i];
        c.groups = i ? sequences : prefixes;
        c.seqs = i ? 1 : per;
        c.with_prefix = prefixes && (!i || !stacked);
        c.with_own = i;
        const uint64_t all = static_cast<uint64_t>(c.seqs) * rows;
        const bool few = all <= kFewRows;
        c.tile_rows = few ? (all > 8 ? 16 : 8) : kRows;
        c.row_tiles = FastDiv(ceil_div(all, c.tile_rows));
        items[i] = static_cast<uint64_t>(c.groups) * kv_heads * c.row_tiles.d;
        p.few[i] = few;
        if (few)
            split_few(c, p.cluster[i], items[i], tiles[i], sms);
        else
            many[i] = items[i];
    }
    // (beside the kernel for few rows one CTA fits an SM)
    // Turned or not, 32 sequences of 1024 keys: 82 and 63 us with 1 visit, 95 and 97
    // with 3, 124 and 126 with 4, 197 and 237 with 8; 4 of 8192 keys: 96 and 93 with 3,
    // 120 and 125 with 4.
    const uint64_t visits = many[0] * tiles[0] + many[1] * tiles[1];
    const uint64_t tiles_held = static_cast<uint64_t>(kv_heads) * (static_cast<uint64_t>(sequences) * t1 +
                                                                  static_cast<uint64_t>(prefixes) * t0);
    p.widen = int8 && !p.few[0] && !p.few[1] && visits >= kWidenFrom * tiles_held;
    if (many[0] || many[1]) p.many_cluster = split_many(p.cls, many, tiles, p.few[1] ? sms : 2 * sms, stacked, p.estimate);
    for (int i = 0; i < 2; ++i) {
        if (!items[i]) continue;
        Class& c = p.cls[i];
        // (where all items start at once their order does not matter)
        const uint64_t ctas = p.few[i] ? (p.cluster[i] ? items[i] * c.splits.d * p.cluster[i] : ~0ull) : items[i] * c.splits.d;
        c.ordered = i && ragged && sequences <= kOrdered && ctas > (p.few[i] ? 3ull : 2ull) * sms;
        c.items = static_cast<uint32_t>(items[i] * c.splits.d);
        c.slot = p.slots;
        p.slots += i && p.many_cluster ? 1 : c.splits.d;
    }
    return p;
}

// Rows of a group are stacked over its prefix where that saves more than the parts of
// rows and their joining cost.  Up to 16 rows a sequence: from 17 visits an SM of the
// prefix's tiles saved (8 single tokens behind 512 keys 10.3 us either way, behind 4000
// 23.1 and 12.5; 16 x 4 behind 1000 20.6 and 16.8, 16 x 16 behind 500 14.4 and 16.8).
// Else by the estimates, with a tile's time for 4000 rows of parts (64 x 32 rows behind 1000 keys 53.2 and 73.7, 8 x 96
// behind 4000 39.1 and 53.2, 8 x 32 behind 4000 32.6 and 24.7, 2 x 20 behind 8000 26.7
// and 20.6).
Plan plan_of(uint32_t sequences, uint32_t rows, uint32_t kv_heads, uint32_t prefixes, uint32_t prefix_keys,
             uint32_t own_keys, bool int8, bool ragged, uint32_t sms) {
    const Plan p = plan_with(false, sequences, rows, kv_heads, prefixes, prefix_keys, own_keys, int8, ragged, sms);
    if (!prefixes || sequences == prefixes) return p;
    const Plan s = plan_with(true, sequences, rows, kv_heads, prefixes, prefix_keys, own_keys, int8, ragged, sms);
    if (p.few[1])
        return static_cast<uint64_t>(sequences - prefixes) * kv_heads * ceil_div(prefix_keys, kKT) >= 17ull * sms ? s : p;
    const uint64_t all = static_cast<uint64_t>(sequences) * rows * kv_heads;
    const auto cost = [&](const Plan& x) { return x.estimate + (x.slots > 1 ? all * x.slots / 4000 : 0); };
    return cost(s) < cost(p) ? s : p;
}

bool fits(uint32_t sequences, uint32_t queries, uint32_t heads, uint32_t kv_heads, uint32_t prefixes) {
    // items and rows stay below 2^31: at most 64 splits of 128-row tiles
    const uint64_t rows = static_cast<uint64_t>(sequences) * queries;
    if (rows > (1ull << 31)) return false;
    const uint64_t per_seq = ceil_div(static_cast<uint64_t>(queries) * (heads / kv_heads), kRows);
    return rows * heads <= (1ull << 31) && per_seq * sequences * kv_heads <= (1ull << 24) && prefixes <= sequences;
}

bool misaligned(const void* p, uint32_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

// The workspace: parts of rows, then keys as f16.
struct Layout {
    size_t ml, exps[2], wide[2], bytes;  // [0] of the prefixes, [1] of the sequences
};

Layout layout_of(const Plan& p, uint64_t rows, uint32_t kv_heads, const uint32_t (&entries)[2],
                 const uint32_t (&capacity)[2], bool fine) {
    const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    Layout l{};
    if (p.slots > 1) {
        l.ml = static_cast<size_t>(p.slots) * rows * kDh * sizeof(float);
        l.bytes = up(l.ml + static_cast<size_t>(p.slots) * rows * sizeof(float2));
    }
    if (p.widen) {
        for (int i = 0; i < 2; ++i) {
            const size_t lines = static_cast<size_t>(entries[i]) * kv_heads;
            l.exps[i] = l.bytes;
            l.wide[i] = up(l.exps[i] + lines * sizeof(float2));
            l.bytes = l.wide[i] + (fine ? 4 : 2) * lines * capacity[i] * kDh * 2;
        }
    }
    return l;
}

uint32_t check_view(const dh_kv_view& v) {
    if (!v.k || !v.v) return DH_ERR_NULL_POINTER;
    if (v.capacity == 0 || v.capacity > 0x7FFFFFFFu || (!v.lengths && v.length > v.capacity))
        return DH_ERR_INVALID_ARGUMENT;
    if (v.k_type == DH_TYPE_I8 && v.v_type == DH_TYPE_I8) {
        if (!v.k_scale || !v.v_scale) return DH_ERR_NULL_POINTER;
        const uint64_t pitch = v.k_strides[1];
        if (v.capacity % kKT || pitch != v.v_strides[1] || pitch % (kKT * kDh) || pitch >> 37 ||
            (pitch && pitch < static_cast<uint64_t>(v.capacity) * kDh))
            return DH_ERR_UNSUPPORTED_SHAPE;
        if (misaligned(v.k, 16) || misaligned(v.v, 16) || misaligned(v.k_scale, 16) || misaligned(v.v_scale, 16) ||
            misaligned(v.lengths, 4))
            return DH_ERR_ALIGNMENT;
        return DH_OK;
    }
    if ((v.k_type != DH_TYPE_BF16 && v.k_type != DH_TYPE_F16) || (v.v_type != DH_TYPE_BF16 && v.v_type != DH_TYPE_F16))
        return DH_ERR_INVALID_ARGUMENT;
    const bool rows = v.v_strides[3] == 1, turned = v.v_strides[2] == 1;
    if (v.k_strides[3] != 1 || (!rows && !turned)) return DH_ERR_UNSUPPORTED_SHAPE;
    const uint64_t all = v.k_strides[0] | v.k_strides[1] | v.k_strides[2] | v.v_strides[0] | v.v_strides[1] |
                         v.v_strides[rows ? 2 : 3];
    if (misaligned(v.k, 16) || misaligned(v.v, 16) || all % 8 || misaligned(v.lengths, 4)) return DH_ERR_ALIGNMENT;
    if (all >> 38) return DH_ERR_UNSUPPORTED_SHAPE;  // (a tensor map's strides lie below 2^40 bytes)
    return DH_OK;
}

// Tiles of `keys` (32 or 64) rows of K and V with `times` the entries.
bool view_maps(CUtensorMap* k, CUtensorMap* v, const dh_kv_view& s, uint32_t entries, uint32_t heads, uint32_t keys,
               uint32_t times = 1) {
    const auto type = [](uint32_t t) {
        return t == DH_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    };
    const bool rows = s.v_strides[3] == 1;
    return make_tmap_4d(k, s.k, type(s.k_type), kDh, s.capacity, heads, times * entries, s.k_strides[2] * 2,
                        s.k_strides[1] * 2, s.k_strides[0] * 2, kDh, keys) &&
           make_tmap_4d(v, s.v, type(s.v_type), rows ? kDh : s.capacity, rows ? s.capacity : kDh, heads, times * entries,
                        s.v_strides[rows ? 2 : 3] * 2, s.v_strides[1] * 2, s.v_strides[0] * 2, rows ? kDh : keys,
                        rows ? keys : kDh);
}

// Launch that may begin while the kernel before it in the stream still runs
// (`beside`; that one lets it, and the kernel itself waits before it needs or ends).
template <class Kernel, class... A>
uint32_t launch_beside(Kernel kernel, uint32_t grid, uint32_t threads, uint32_t smem, uint32_t cluster, bool beside,
                       cudaStream_t st, const A&... args) {
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
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
    if (cudaLaunchKernelEx(&config, kernel, args...) != cudaSuccess) {
        cudaGetLastError();
        return DH_ERR_CUDA;
    }
    return DH_OK;
}

template <int KIND, bool CLUSTER>
uint32_t launch_one(const CUtensorMap (&maps)[4], const Args& a, uint32_t first, uint32_t total, uint32_t cluster,
                    bool beside, cudaStream_t st) {
    const auto kernel = kv_attention_kernel<KIND, CLUSTER>;
    static std::atomic<uint64_t> configured{0};
    if (all_shared_once(kernel, Cfg<KIND>::bytes, configured) != cudaSuccess) return DH_ERR_CUDA;
    const uint32_t grid = CLUSTER ? total : std::min(total, 2 * device_sms());  // (a cluster has one item)
    return launch_beside(kernel, grid, Cfg<KIND>::threads, Cfg<KIND>::bytes, cluster, beside, st, maps[0], maps[1],
                         maps[2], maps[3], a, first, total, cluster);
}

template <int KIND>
uint32_t launch(const CUtensorMap (&maps)[4], const Args& a, uint32_t first, uint32_t total, uint32_t cluster,
                bool beside, cudaStream_t st) {
    return cluster ? launch_one<KIND, true>(maps, a, first, total, cluster, beside, st)
                   : launch_one<KIND, false>(maps, a, first, total, 0, beside, st);
}

}  // namespace
}  // namespace dh

using namespace dh;

extern "C" size_t dh_kv_attention_workspace_size(uint32_t sequences, uint32_t queries, uint32_t heads,
                                                 uint32_t kv_heads, uint32_t prefixes, uint32_t prefix_capacity,
                                                 uint32_t own_capacity, uint32_t k_type, uint32_t q_type) {
    if (!sequences || !queries || !heads || !kv_heads || heads % kv_heads || (prefixes && sequences % prefixes) ||
        !fits(sequences, queries, heads, kv_heads, prefixes))
        return 0;
    const Plan p = plan_of(sequences, queries * (heads / kv_heads), kv_heads, prefixes, prefix_capacity, own_capacity,
                           k_type == DH_TYPE_I8, false, device_sms());
    return layout_of(p, static_cast<uint64_t>(sequences) * queries * heads, kv_heads, {prefixes, sequences},
                     {prefix_capacity, own_capacity}, q_type == DH_TYPE_F16)
        .bytes;
}

extern "C" uint32_t dh_kv_attention_launches(uint32_t sequences, uint32_t queries, uint32_t heads, uint32_t kv_heads,
                                             uint32_t prefixes, uint32_t prefix_capacity, uint32_t own_capacity,
                                             uint32_t k_type) {
    if (!sequences || !queries || !heads || !kv_heads || heads % kv_heads || (prefixes && sequences % prefixes) ||
        !fits(sequences, queries, heads, kv_heads, prefixes))
        return 0;
    const Plan p = plan_of(sequences, queries * (heads / kv_heads), kv_heads, prefixes, prefix_capacity, own_capacity,
                           k_type == DH_TYPE_I8, false, device_sms());
    const bool many = (p.cls[0].items && !p.few[0]) || !p.few[1];
    return p.widen + many + p.few[0] + p.few[1] + (p.slots > 1);
}

extern "C" uint32_t dh_kv_attention(const void* q, uint32_t q_type, const uint64_t* q_strides, uint32_t sequences,
                                    uint32_t queries, uint32_t heads, uint32_t kv_heads, const dh_kv_view* own,
                                    const dh_kv_view* prefix, uint32_t prefixes, float scale, void* out, float* lse,
                                    const uint32_t* run_rows, void* workspace, size_t workspace_bytes, void* stream) {
    if (!q || !q_strides || !own || !out || (prefixes && !prefix)) return DH_ERR_NULL_POINTER;
    if ((q_type != DH_TYPE_BF16 && q_type != DH_TYPE_F16) || !sequences || !queries || !heads || !kv_heads ||
        heads % kv_heads || (prefixes && sequences % prefixes))
        return DH_ERR_INVALID_ARGUMENT;
    const float c = scale * 1.4426950408889634f;  // log2(e)
    if (!(c >= kLeastFactor && std::isfinite(c))) return DH_ERR_INVALID_ARGUMENT;
    if (!fits(sequences, queries, heads, kv_heads, prefixes)) return DH_ERR_UNSUPPORTED_SHAPE;
    if (uint32_t st = check_view(*own)) return st;
    const bool int8 = own->k_type == DH_TYPE_I8;
    if (!int8 && own->k_type != q_type) return DH_ERR_INVALID_ARGUMENT;
    if (prefixes) {
        if (uint32_t st = check_view(*prefix)) return st;
        if (prefix->k_type != own->k_type || prefix->v_type != own->v_type) return DH_ERR_INVALID_ARGUMENT;
        if (!int8 && (prefix->v_strides[3] == 1) != (own->v_strides[3] == 1)) return DH_ERR_INVALID_ARGUMENT;
    }
    if (misaligned(q, 16) || (q_strides[0] | q_strides[1] | q_strides[2]) % 8 || misaligned(out, 16) ||
        misaligned(lse, 4) || misaligned(run_rows, 4))
        return DH_ERR_ALIGNMENT;
    const uint32_t ratio = heads / kv_heads;
    const uint64_t rows = static_cast<uint64_t>(sequences) * queries * heads;
    const Plan p = plan_of(sequences, queries * ratio, kv_heads, prefixes, prefixes ? prefix->capacity : 0,
                           own->capacity, int8, own->lengths != nullptr, device_sms());
    const bool fine = q_type == DH_TYPE_F16;  // (int8 keys)
    const Layout l = layout_of(p, rows, kv_heads, {prefixes, sequences},
                               {prefixes ? prefix->capacity : 0, own->capacity}, fine);
    const size_t need = l.bytes;
    if (need && !workspace) return DH_ERR_NULL_POINTER;
    if (need > workspace_bytes) return DH_ERR_WORKSPACE;
    if (misaligned(workspace, 256)) return DH_ERR_ALIGNMENT;

    Args a{};
    a.cls[0] = p.cls[0], a.cls[1] = p.cls[1];
    const auto segment = [](const dh_kv_view& v) {
        return Segment{static_cast<const int8_t*>(v.k), static_cast<const int8_t*>(v.v), v.k_scale, v.v_scale,
                       v.lengths, v.length, v.capacity,
                       v.k_type == DH_TYPE_I8 && v.k_strides[1] ? static_cast<uint32_t>(v.k_strides[1] / kDh) : v.capacity};
    };
    a.own = segment(*own);
    if (prefixes) a.prefix = segment(*prefix);
    a.q = static_cast<const uint8_t*>(q);
    a.q_seq = q_strides[0] * 2, a.q_head = q_strides[1] * 2, a.q_row = q_strides[2] * 2;
    a.q_bf16 = q_type == DH_TYPE_BF16;
    a.sequences = sequences, a.prefixes = prefixes, a.heads = heads;
    a.queries = FastDiv(queries), a.kv_heads = FastDiv(kv_heads), a.ratio = FastDiv(ratio);
    a.per_prefix = FastDiv(prefixes ? sequences / prefixes : sequences);
    a.v_transposed = !int8 && own->v_strides[3] != 1;
    a.idesc_s = int8 || q_type == DH_TYPE_F16 ? tc::idesc_f16_f32<kRows, kKT>() : tc::idesc_bf16_f32<kRows, kKT>();
    const bool v_bf16 = own->v_type == DH_TYPE_BF16;
    a.idesc_o = (v_bf16 ? tc::idesc_bf16_f32<kRows, kPvN>() : tc::idesc_f16_f32<kRows, kPvN>()) |
                (a.v_transposed ? 0u : tc::kIdescBMnMajor);
    a.c = c;
    a.out = static_cast<uint8_t*>(out);
    a.lse = lse;
    a.total_rows = rows;
    a.run_rows = run_rows;
    if (p.slots > 1) {
        a.part_o = static_cast<float*>(workspace);
        a.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + l.ml);
    }
    const bool any_many = p.cls[0].items && !p.few[0] ? true : !p.few[1];
    CUtensorMap maps[4] = {}, few_maps[4] = {};
    for (int kind = 0; kind < 2 && !int8; ++kind) {
        if (kind ? !(p.few[0] || p.few[1]) : !any_many) continue;
        CUtensorMap* m = kind ? few_maps : maps;
        const uint32_t keys = kind ? kFewKeys16 : kKT;
        if (!view_maps(&m[2], &m[3], *own, sequences, kv_heads, keys)) return DH_ERR_CUDA;
        if (prefixes && !view_maps(&m[0], &m[1], *prefix, prefixes, kv_heads, keys)) return DH_ERR_CUDA;
    }
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p.widen) {
        WideKeys to[2];
        for (int i = prefixes ? 0 : 1; i < 2; ++i) {
            const uint32_t entries = i ? sequences : prefixes, capacity = i ? own->capacity : prefix->capacity;
            uint8_t* base = static_cast<uint8_t*>(workspace);
            to[i].exps = reinterpret_cast<float2*>(base + l.exps[i]);
            to[i].k = reinterpret_cast<__half*>(base + l.wide[i]);
            const size_t each = static_cast<size_t>(entries) * kv_heads * capacity * kDh;
            to[i].lo = fine ? each : 0;
            to[i].v = to[i].k + (fine ? 2 : 1) * each;
            dh_kv_view f{};
            f.k = to[i].k, f.v = to[i].v, f.k_type = f.v_type = DH_TYPE_F16, f.capacity = capacity;
            f.k_strides[2] = f.v_strides[2] = kDh, f.k_strides[3] = f.v_strides[3] = 1;
            f.k_strides[1] = f.v_strides[1] = static_cast<uint64_t>(capacity) * kDh;
            f.k_strides[0] = f.v_strides[0] = static_cast<uint64_t>(capacity) * kDh * kv_heads;
            if (!view_maps(&maps[2 * i], &maps[2 * i + 1], f, entries, kv_heads, kKT, fine ? 2 : 1)) return DH_ERR_CUDA;
        }
        a.prefix_exps = to[0].exps, a.own_exps = to[1].exps;
        if (uint32_t status = launch_widen(a, to[0], to[1], prefixes, st)) return status;
    }
    // Tensor-core tiles first: their few CTAs take long, and the others run beside them.
    uint32_t status = DH_OK, first = 0, total = 0;
    for (uint32_t i = 0; i < 2; ++i)
        if (!p.few[i]) total += a.cls[i].items, first += i ? 0 : a.cls[0].items;
    if (total) {
        const auto go = !int8 ? (v_bf16 ? launch<kVBf16> : launch<kV16>)
                        : p.widen ? (fine ? launch<kWideFine> : launch<kWide>) : (fine ? launch<kInt8Fine> : launch<kInt8>);
        status = go(maps, a, first, total, p.many_cluster, p.widen, st);
    }
    bool beside = total;
    const uint32_t taken = total ? (!int8 ? Cfg<kV16>::bytes : fine ? Cfg<kInt8Fine>::bytes : Cfg<kInt8>::bytes) + 1024 : 0;
    for (uint32_t i = 0; i < 2 && !status; ++i) {
        if (!p.few[i]) continue;
        status = launch_few(few_maps, a, i, p.cluster[i], int8, v_bf16, beside, taken, st);
        beside = true;
    }
    if (status || p.slots < 2) return status;
    return launch_beside(kv_join_kernel, ceil_div(rows, kJoinThreads / 8), kJoinThreads, 0, 1, true, st,
                         static_cast<const float2*>(a.part_ml), static_cast<const float*>(a.part_o), p.slots, rows,
                         a.queries, heads, a.q_bf16, a.out, lse, run_rows);
}
