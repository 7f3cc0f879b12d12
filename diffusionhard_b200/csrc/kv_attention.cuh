// kv_attention.cuh -- what the kernels of attention over K/V caches share: the
// arguments, which rows and keys a work item has, and small arithmetic.  The
// operator is described in kv_attention.cu.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fast_div.cuh"
#include "tc_ptx.cuh"

namespace dh {
namespace kv {

constexpr uint32_t kDh = 64;
constexpr uint32_t kKT = 64;                                 // keys per tile
constexpr uint32_t kTileBytes = kKT * kDh * 2;               // 8 KB: a 16-bit K or V tile
constexpr uint32_t kRawBytes = 2 * kKT * kDh + 2 * kKT * 4;  // codes and scales of 64 keys
// Factors of scores stay above zero: keys behind the last one score -inf, and
// -inf * 0 would be NaN.
constexpr float kLeastFactor = 1.17549435e-38f;

// Rows and keys of one class of items.
struct Class {
    uint32_t groups, seqs;               // groups of consecutive sequences whose rows are stacked
    uint32_t tile_rows, items, slot;     // rows of an item; all items; the first part's slot
    FastDiv row_tiles, splits;           // items a group and K/V head; parts of the keys
    uint32_t with_prefix, with_own;
    uint32_t ordered;                    // the longest sequences' items come first
};

struct Segment {
    const int8_t* k;
    const int8_t* v;
    const float* k_scale;
    const float* v_scale;
    const int32_t* lengths;
    uint32_t length, capacity;
    uint32_t pitch;                      // int8: positions from one head's rows to the next's
};

struct Args {
    Class cls[2];
    Segment prefix, own;
    const uint8_t* q;                        // 16-bit elements
    uint64_t q_seq, q_head, q_row;           // strides in bytes
    uint32_t q_bf16;
    uint32_t sequences, prefixes, heads;
    FastDiv queries, kv_heads, ratio, per_prefix;  // ratio: query heads of a K/V head
    uint32_t v_transposed, idesc_s, idesc_o;
    float c;                                 // scale * log2(e)
    uint8_t* out;                            // [sequences, queries, heads, 64], of q's type
    float* lse;                              // [sequences, queries, heads], or null
    float2* part_ml;                         // [slots][rows], or null: one slot
    float* part_o;                           // [slots][rows][64]
    uint64_t total_rows;
    const uint32_t* run_rows;
    const float2* prefix_exps;               // of keys turned into f16: factor of K, exponent of V
    const float2* own_exps;
};

// Programmatic dependent launch: the next kernel may begin; all before this one have
// ended and their writes are seen.
DH_DEVINL void grid_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;"); }
DH_DEVINL void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

DH_DEVINL float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// maxima that are NaN if an operand is
DH_DEVINL float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
DH_DEVINL float max_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
DH_DEVINL uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
DH_DEVINL uint32_t pack_bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// 2^n, -126 <= n <= 127; infinite for 128
DH_DEVINL float pow2(int32_t n) { return __uint_as_float(static_cast<uint32_t>(n + 127) << 23); }
// e with 2^(e - 1) <= x < 2^e for the normal fp32 with these bits
DH_DEVINL int32_t exponent_of(uint32_t bits) { return static_cast<int32_t>((bits >> 23) & 0xFFu) - 126; }

// 4 codes -> 4 f16 of code * ratio * 2^-9, where f = f16(ratio * 2^15): a code plus
// 128 as the bits of a subnormal f16 is (code + 128) 2^-24, so one FMA with f and off =
// -f 2^-17 (exact, a power of two) takes the 128 off and scales, with one rounding.
DH_DEVINL void convert4(uint32_t codes, __half2 f, __half2 off, uint32_t& lo, uint32_t& hi) {
    const uint32_t u = codes ^ 0x80808080u;
    const uint32_t p = __byte_perm(u, 0u, 0x4140u), q = __byte_perm(u, 0u, 0x4342u);
    const __half2 x = __hfma2(*reinterpret_cast<const __half2*>(&p), f, off);
    const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&q), f, off);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
}
DH_DEVINL void convert16(const uint4& codes, __half2 f, __half2 off, uint4& lo, uint4& hi) {
    convert4(codes.x, f, off, lo.x, lo.y);
    convert4(codes.y, f, off, lo.z, lo.w);
    convert4(codes.z, f, off, hi.x, hi.y);
    convert4(codes.w, f, off, hi.z, hi.w);
}

// The same with f = hi + lo and hi of 4 bits, so that code * hi is exact: 4 f16 of code *
// hi 2^-24 and of code * lo 2^-24, whose sum is off by 2^-15.
struct FineFactor {
    __half2 hi, lo, off_hi, off_lo;
};
DH_DEVINL FineFactor fine_factor(float f) {
    const float hi = __uint_as_float((__float_as_uint(f) + (1u << 19)) & 0xFFF00000u);
    const __half2 shift = __half2half2(__ushort_as_half(0x8080));  // -2^-17
    FineFactor r;
    r.hi = __float2half2_rn(hi), r.lo = __float2half2_rn(f - hi);
    r.off_hi = __hmul2(r.hi, shift), r.off_lo = __hmul2(r.lo, shift);
    return r;
}
struct Item {
    uint32_t seq0, kv_head, row0, rows, slot;  // rows: live rows of the tile (may be 0)
    uint32_t prefix, own;                      // cache entries
    uint32_t len0, len1, n0, t0, t1;           // keys and tiles of the two parts, tile range
};

DH_DEVINL uint32_t length_of(const Segment& s, uint32_t entry) {
    const int32_t n = s.lengths ? __ldg(s.lengths + entry) : static_cast<int32_t>(s.length);
    return static_cast<uint32_t>(min(max(n, 0), static_cast<int32_t>(s.capacity)));
}

// Sequences by falling length (the lower index first among equals) into order[],
// by the CTA's first kOrdered threads; all threads call it.  Items of long sequences
// that start last would run alone (16 single tokens over up to 32768 keys 111 us as they
// come, 101 in this order).  kOrdered: what shared memory is set aside for.
constexpr uint32_t kOrdered = 128;
DH_DEVINL void order_sequences(const Args& a, uint32_t* lengths, uint16_t* order) {
    const uint32_t n = a.sequences, t = threadIdx.x;
    uint32_t mine = 0;
    if (t < n) lengths[t] = mine = length_of(a.own, t);
    __syncthreads();
    if (t < n) {
        uint32_t rank = 0;
        for (uint32_t u = 0; u < n; ++u) {
            const uint32_t other = lengths[u];
            rank += other > mine || (other == mine && u < t);
        }
        order[rank] = static_cast<uint16_t>(t);
    }
    __syncthreads();
}

// Item w of a class, of the first `live` sequences, in tiles of KT keys.
template <uint32_t KT = kKT>
DH_DEVINL Item item_of(const Args& a, const Class& c, uint32_t w, uint32_t live, const uint16_t* order) {
    Item it;
    uint32_t split = w, tile, head;
    tile = c.splits.split(split);
    head = c.row_tiles.split(tile);
    uint32_t group = a.kv_heads.split(head);
    if (c.ordered) group = order[group];
    it.kv_head = head;
    it.seq0 = group * c.seqs;
    it.slot = c.slot + split;
    it.row0 = tile * c.tile_rows;
    const uint32_t seqs = live > it.seq0 ? min(live - it.seq0, c.seqs) : 0u;
    const uint32_t rows = seqs * a.queries.d * a.ratio.d;
    it.rows = rows > it.row0 ? min(rows - it.row0, c.tile_rows) : 0u;
    it.own = it.seq0;
    it.prefix = a.per_prefix.of(it.seq0);
    it.len0 = c.with_prefix ? length_of(a.prefix, it.prefix) : 0u;
    it.len1 = c.with_own ? length_of(a.own, it.own) : 0u;
    it.n0 = (it.len0 + KT - 1) / KT;
    const uint32_t n = it.n0 + (it.len1 + KT - 1) / KT;
    if (c.splits.d == 1) {
        it.t0 = 0, it.t1 = n;
    } else {
        uint32_t more = n;  // `more` parts have a tile more than the others
        const uint32_t each = c.splits.split(more);
        it.t0 = each * split + c.splits.of(more * split);
        it.t1 = each * (split + 1) + c.splits.of(more * (split + 1));
    }
    if (it.rows == 0) it.t1 = it.t0;
    return it;
}
// keys left from tile j on in its part (a full tile: KT or more)
template <uint32_t KT = kKT>
DH_DEVINL uint32_t keys_left(const Item& it, uint32_t j) {
    return j < it.n0 ? it.len0 - j * KT : it.len1 - (j - it.n0) * KT;
}

// Row r of an item: its query, as an index of [sequences, queries, heads].
DH_DEVINL uint64_t row_index(const Args& a, const Item& it, uint32_t r, const uint8_t** q) {
    uint32_t in_kv = it.row0 + r;
    uint32_t s = a.ratio.split(in_kv);  // the token among the group's, then in its sequence
    const uint32_t head = it.kv_head * a.ratio.d + in_kv;
    const uint32_t seq = it.seq0 + a.queries.split(s);
    if (q) *q = a.q + seq * a.q_seq + head * a.q_head + s * a.q_row;
    return (static_cast<uint64_t>(seq) * a.queries.d + s) * a.heads + head;
}

DH_DEVINL uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
DH_DEVINL void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
DH_DEVINL uint32_t map_to(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
DH_DEVINL float2 load_remote2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
DH_DEVINL float4 load_remote4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}
DH_DEVINL void add(float4& s, float f, const float4& v) {
    s = make_float4(__fmaf_rn(f, v.x, s.x), __fmaf_rn(f, v.y, s.y), __fmaf_rn(f, v.z, s.z), __fmaf_rn(f, v.w, s.w));
}

// A weight's exponent is one FMA, s c - m, with m the maximum rounded to fp32.  That
// rounding is the same for all weights of a row and their sum: it cancels, and only the
// range of the weights sees it.  From kFar on a maximum is taken as it is, without room
// above or below it, so that the largest weight lies within 2^-8 .. 2^8 up to |m| = 2^28.
constexpr float kFar = 4194304.f;  // 2^22
// From there on differences to m are taken by this power of two, which keeps it below
// 2^28 (1 for all others): what is 33 2^-27 of m below it, 2^-21 and less, is still 2^-33
// of it.  Maxima are compared by the same measure wherever sums meet.
DH_DEVINL float damping(float top) {
    constexpr uint32_t kFrom = (127u + 27u) << 23;
    return __uint_as_float(0x3F800000u + kFrom - max(__float_as_uint(top) & 0x7F800000u, kFrom));
}
// Sums relative to 2^m as ones relative to 2^top: their factor.
DH_DEVINL float growth(float m, float top) { return ex2_approx((m - top) * damping(top)); }
constexpr float kNoMax = -3.0e38f;  // below every maximum, and finite

// Four values (part 0..15) of row r of an item from its sums: relative to 2^top, the
// weights' sum is `total`.
DH_DEVINL void write_part(const Args& a, const Item& it, uint32_t r, uint32_t part, float top, float total,
                          const float4& sum) {
    const uint64_t row = row_index(a, it, r, nullptr);
    if (a.part_ml) {
        const uint64_t at = it.slot * a.total_rows + row;
        if (part == 0) a.part_ml[at] = make_float2(top, total);
        reinterpret_cast<float4*>(a.part_o + at * kDh)[part] = sum;
        return;
    }
    const float f = total == 0.f ? 0.f : 1.f / total;
    reinterpret_cast<uint2*>(a.out)[row * (kDh / 4) + part] =
        a.q_bf16 ? make_uint2(pack_bf16x2(sum.x * f, sum.y * f), pack_bf16x2(sum.z * f, sum.w * f))
                 : make_uint2(pack_f16x2(sum.x * f, sum.y * f), pack_f16x2(sum.z * f, sum.w * f));
    if (a.lse && part == 0) a.lse[row] = total == 0.f ? -INFINITY : (top + log2f(total)) * 0.6931471805599453f;
}

// An item's rows from the sums [row][kSumPitch] and (m, l) [row] that every CTA of the
// cluster has at these addresses of its shared memory, in the order of the CTAs; each
// writes its share.  All threads of all of them call it.
constexpr uint32_t kMaxCluster = 8;
constexpr uint32_t kSumPitch = kDh + 4;
DH_DEVINL void join_cluster(const Args& a, const Item& it, uint32_t sums_at, uint32_t ml_at, uint32_t cluster,
                            uint32_t rank, uint32_t threads) {
    cluster_sync();
    for (uint32_t i = rank * threads + threadIdx.x; i < it.rows * (kDh / 4); i += cluster * threads) {
        const uint32_t r = i / (kDh / 4), part = i % (kDh / 4);
        float top = kNoMax, total = 0.f;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        float2 x[kMaxCluster];
#pragma unroll
        for (uint32_t p = 0; p < kMaxCluster; ++p) {
            if (p >= cluster) break;
            x[p] = load_remote2(map_to(ml_at + r * 8, p));
            top = max_nan(top, x[p].x);
        }
#pragma unroll
        for (uint32_t p = 0; p < kMaxCluster; ++p) {
            if (p >= cluster) break;
            const float f = growth(x[p].x, top);
            total = __fmaf_rn(f, x[p].y, total);
            add(sum, f, load_remote4(map_to(sums_at + (r * kSumPitch + 4 * part) * 4, p)));
        }
        write_part(a, it, r, part, top, total, sum);
    }
    cluster_sync();  // (no CTA leaves while its sums are read)
}

}  // namespace kv
}  // namespace dh
