// kv_cache.cu -- K / V rows into an int8 cache as they are produced, and back.
//
// A cache holds, for each (entry, head, position), 64 int8 codes and one fp32
// scale of K and of V: [entries, heads, capacity, 64] and [entries, heads,
// capacity].  With amax = max |x| over the 64 values of a row,
//   scale = fp32(amax / 127), code = rint(fp32(x / scale)) within +-127,
// both quotients IEEE-rounded, as the framework's per-token quantiser has them
// (fixed_mlp._quantize_symmetric, fixed_mlp.py:11-35), but for the rows it
// cannot hold: amax < 2^-100 gives scale 0 and codes 0, a value that is not
// finite gives scale NaN and codes 0, so that whatever reads the row is NaN.
//
// Both directions are bound by HBM: a bf16 row is read once (128 bytes) and
// leaves as 68, or the other way round, with five operations a value.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fast_div.cuh"
#include "row_quant.cuh"

#include <type_traits>

namespace dh {
namespace {

constexpr uint32_t kDim = 64;
constexpr uint32_t kTileRows = 128;  // rows of one (entry, head) and side a CTA takes
constexpr uint32_t kSteps = kTileRows / 32;  // rows a group of 8 lanes takes
constexpr uint32_t kThreads = 256;
constexpr float kSmallest = 7.8886090522101181e-31f;  // 2^-100

struct WriteSide {
    const void* src;
    int8_t* codes;
    float* scale;
    uint64_t seq, head, row, dim;  // strides in elements
    uint32_t type;
    uint32_t wide;                 // rows, or columns, are contiguous and 16-byte aligned
};

struct WriteArgs {
    WriteSide side[2];
    uint32_t rows, capacity;
    FastDiv tiles, heads;
    const int32_t* starts;
    uint32_t start;
    const int32_t* counts;
    const uint32_t* run_rows;
};

// 8 consecutive elements of a row as they are stored (16-byte loads), and what the
// quantiser needs of them: the largest magnitude as the bits of an fp32 (NaN above
// infinity above every finite value) and pairs as fp32.
template <class T>
struct Row8;

template <>
struct Row8<float> {
    uint32_t w[8];
    DH_DEVINL void load(const float* p) {
        const uint4 a = *reinterpret_cast<const uint4*>(p), b = *reinterpret_cast<const uint4*>(p + 4);
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
    }
    DH_DEVINL void load(const float* p, uint64_t stride) {
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) w[e] = __float_as_uint(p[e * stride]);
    }
    DH_DEVINL void clear() {
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) w[e] = 0;
    }
    DH_DEVINL uint32_t peak() const {
        uint32_t m = 0;
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) m = max(m, w[e] & 0x7FFFFFFFu);
        return m;
    }
    static DH_DEVINL uint32_t peak_bits(uint32_t m) { return m; }
    DH_DEVINL float2 pair(uint32_t i) const { return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1])); }
};

// 16-bit types: magnitudes are ordered as their bits are
template <class T>
struct Row8 {
    uint32_t w[4];
    DH_DEVINL void load(const T* p) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    }
    DH_DEVINL void load(const T* p, uint64_t stride) {
        const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) w[i] = q[2 * i * stride] | static_cast<uint32_t>(q[(2 * i + 1) * stride]) << 16;
    }
    DH_DEVINL void clear() { w[0] = w[1] = w[2] = w[3] = 0; }
    DH_DEVINL uint32_t peak() const {
        uint32_t m = 0;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
        return max(m & 0xFFFFu, m >> 16);
    }
    static DH_DEVINL uint32_t peak_bits(uint32_t m) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) return m << 16;
        return __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(m))));
    }
    DH_DEVINL float2 pair(uint32_t i) const {
        if constexpr (std::is_same<T, __nv_bfloat16>::value)
            return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
        return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    }
};

// Codes of a pair in the low bytes of x and y.  The quotient is the IEEE-rounded one
// (see Divisor); |x| <= amax keeps it within 127 (1 + 2^-23), which rounds to 127, so
// nothing is clamped.
DH_DEVINL uint2 codes_of(float2 x, const Divisor& by) {
    const float2 r2 = make_float2(by.r, by.r), nb2 = make_float2(-by.b, -by.b);
    const float2 q0 = __fmul2_rn(x, r2);
    const float2 q = __ffma2_rn(__ffma2_rn(q0, nb2, x), r2, q0);
    const float2 t = __fadd2_rn(q, make_float2(12582912.0f, 12582912.0f));  // (see rint_bits)
    return make_uint2(__float_as_uint(t.x), __float_as_uint(t.y));
}

// Row pitch of the staged tile: odd in 4-byte words, so that neither side of the
// turn piles up on banks.
template <class T>
constexpr uint32_t kPitch = sizeof(T) == 4 ? kDim + 1 : kDim + 2;

// A tile whose positions are contiguous (a transposed V), turned in shared memory.
template <class T>
DH_DEVINL void stage_tile(const T* src, uint64_t dim, uint32_t rows, uint32_t wide, T* t) {
    const uint32_t warp = warp_id(), lane = lane_id();
    if (sizeof(T) == 2 && wide && rows == kTileRows) {
        // 8 positions of columns d and d + 1 a thread; 128 bytes of a column are read
        // by 8 neighbours
        const uint32_t d = (warp * 4 + (lane >> 3)) * 2;
#pragma unroll
        for (uint32_t h = 0; h < kTileRows / 64; ++h) {
            const uint32_t p = (lane & 7u) * 8 + 64 * h;
            const uint4 a = *reinterpret_cast<const uint4*>(src + d * dim + p);
            const uint4 b = *reinterpret_cast<const uint4*>(src + (d + 1) * dim + p);
            const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                *reinterpret_cast<uint32_t*>(t + (p + 2 * i) * kPitch<T> + d) = __byte_perm(x[i], y[i], 0x5410);
                *reinterpret_cast<uint32_t*>(t + (p + 2 * i + 1) * kPitch<T> + d) = __byte_perm(x[i], y[i], 0x7632);
            }
        }
        return;
    }
    for (uint32_t i = 0; i < kDim / 8; ++i) {
        const uint32_t d = warp * (kDim / 8) + i;
#pragma unroll
        for (uint32_t h = 0; h < kTileRows / 32; ++h) {
            const uint32_t r = lane + 32 * h;
            if (r < rows) t[r * kPitch<T> + d] = src[d * dim + r];
        }
    }
}

template <class T>
DH_DEVINL void write_tile(const WriteArgs& a, const WriteSide& s, uint32_t seq, uint32_t head, uint32_t row0,
                          uint32_t rows, int64_t at, uint8_t* smem) {
    const T* src = static_cast<const T*>(s.src) + seq * s.seq + head * s.head + row0 * s.row;
    const uint32_t warp = warp_id(), lane = lane_id();
    const uint64_t base = (static_cast<uint64_t>(seq) * a.heads.d + head) * a.capacity;
    const bool staged = s.row == 1 && s.dim != 1;
    T* t = reinterpret_cast<T*>(smem);
    if (staged) {
        stage_tile(src, s.dim, rows, s.wide, t);
        __syncthreads();
    }
    // 8 lanes a row, 8 values each; a warp takes rows 16 w .. 16 w + 15 in four steps
    const uint32_t c = lane & 7u, r0 = warp * (4 * kSteps) + (lane >> 3);
    Row8<T> x[kSteps];
#pragma unroll
    for (uint32_t i = 0; i < kSteps; ++i) {
        const uint32_t r = r0 + 4 * i;
        x[i].clear();
        if (r >= rows) continue;
        if (staged) {
            const uint32_t* p = reinterpret_cast<const uint32_t*>(t + r * kPitch<T> + c * 8);
#pragma unroll
            for (uint32_t e = 0; e < 2 * sizeof(T); ++e) x[i].w[e] = p[e];
        } else if (s.wide) {
            x[i].load(src + r * s.row + c * 8);
        } else {
            x[i].load(src + r * s.row + c * 8 * s.dim, s.dim);
        }
    }
    // largest magnitudes of the four rows over their 8 lanes, halving the rows that a
    // lane holds with every exchange: lane c is left with that of step c % 4, and
    // takes that row's scale and reciprocal for all of them
    static_assert(kSteps == 4, "four rows in two exchanges");
    const bool odd = c & 1u, high = c & 2u;
    uint32_t m[kSteps];
#pragma unroll
    for (uint32_t i = 0; i < kSteps; ++i) m[i] = x[i].peak();
    const uint32_t a01 = max(odd ? m[1] : m[0], __shfl_xor_sync(0xFFFFFFFFu, odd ? m[0] : m[1], 1));
    const uint32_t a23 = max(odd ? m[3] : m[2], __shfl_xor_sync(0xFFFFFFFFu, odd ? m[2] : m[3], 1));
    uint32_t top = max(high ? a23 : a01, __shfl_xor_sync(0xFFFFFFFFu, high ? a01 : a23, 2));
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
    const uint32_t peak = Row8<T>::peak_bits(top);
    const bool live = peak >= __float_as_uint(kSmallest) && peak < 0x7F800000u;
    const float scale = live ? divide(__uint_as_float(peak), make_divisor(127.0f))
                             : (peak >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : 0.f);
    const float inverse = __frcp_rn(live ? scale : 1.0f);
    // rows [from_row, to_row) of the tile lie inside the cache
    const uint32_t from_row = static_cast<uint32_t>(min(max(-at, int64_t{0}), static_cast<int64_t>(rows)));
    const uint32_t to_row = static_cast<uint32_t>(
        min(max(static_cast<int64_t>(a.capacity) - at, static_cast<int64_t>(from_row)), static_cast<int64_t>(rows)));
    int8_t* codes = s.codes + static_cast<int64_t>(base + at) * kDim + r0 * kDim + c * 8;
    float* scales = s.scale + static_cast<int64_t>(base + at) + r0;
#pragma unroll
    for (uint32_t i = 0; i < kSteps; ++i) {
        const uint32_t from = (lane & 24u) | i;
        const Divisor by = {__shfl_sync(0xFFFFFFFFu, scale, from), __shfl_sync(0xFFFFFFFFu, inverse, from)};
        uint32_t w[2];
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            const uint2 lo = codes_of(x[i].pair(2 * h), by), hi = codes_of(x[i].pair(2 * h + 1), by);
            w[h] = by.b > 0.f ? pack4_i8(lo.x, lo.y, hi.x, hi.y) : 0u;
        }
        if (r0 + 4 * i - from_row < to_row - from_row) {
            *reinterpret_cast<uint2*>(codes + 4 * i * kDim) = make_uint2(w[0], w[1]);
            if (c == i) scales[4 * i] = scale;
        }
    }
}

// F32: either side may be fp32, whose rows take twice the registers (5 CTAs an SM for
// 16 bits: 32 canvases with a transposed V 35.6 us, 37.8 with 4; fp32 blocks 12.3 with
// 4, 14.5 with 5).
template <bool F32>
__global__ void __launch_bounds__(kThreads, F32 ? 4 : 5) kv_write_kernel(const __grid_constant__ WriteArgs a) {
    __shared__ __align__(16) uint8_t smem[kTileRows * (F32 ? kPitch<float> * 4 : kPitch<__half> * 2)];
    uint32_t tile = blockIdx.x, head;
    head = a.tiles.split(tile);
    const uint32_t w = a.heads.split(head), seq = w >> 1;
    if (a.run_rows && static_cast<uint64_t>(seq + 1) * a.rows > *a.run_rows) return;
    uint32_t rows = a.rows;
    if (a.counts) rows = static_cast<uint32_t>(min(max(a.counts[seq], 0), static_cast<int32_t>(a.rows)));
    const uint32_t row0 = tile * kTileRows;
    if (row0 >= rows) return;
    rows = min(rows - row0, kTileRows);
    const int64_t at = (a.starts ? static_cast<int64_t>(a.starts[seq]) : static_cast<int64_t>(a.start)) + row0;
    const WriteSide& s = a.side[w & 1u];
    if (s.type == DH_TYPE_BF16)
        write_tile<__nv_bfloat16>(a, s, seq, head, row0, rows, at, smem);
    else if (s.type == DH_TYPE_F16)
        write_tile<__half>(a, s, seq, head, row0, rows, at, smem);
    else if constexpr (F32)
        write_tile<float>(a, s, seq, head, row0, rows, at, smem);
}

struct ReadArgs {
    const int8_t* codes[2];
    const float* scale[2];
    void* out[2];
    uint32_t rows, start, capacity;
    FastDiv tiles, heads;
};

DH_DEVINL void store8(float* p, const float (&x)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
DH_DEVINL void store8(__nv_bfloat16* p, const float (&x)[8]) {
    uint4 v;
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = v;
}
DH_DEVINL void store8(__half* p, const float (&x)[8]) {
    uint4 v;
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = v;
}

template <class T>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ ReadArgs a) {
    uint32_t tile = blockIdx.x, head;
    head = a.tiles.split(tile);
    const uint32_t w = a.heads.split(head), side = w & 1u;
    const uint64_t line = static_cast<uint64_t>(w >> 1) * a.heads.d + head;
    const uint32_t c = threadIdx.x & 7u;
    uint2 q[kSteps];
    float scale[kSteps];
#pragma unroll
    for (uint32_t i = 0; i < kSteps; ++i) {
        const uint32_t r = tile * kTileRows + i * 32 + (threadIdx.x >> 3);
        if (r >= a.rows) break;
        const uint64_t at = line * a.capacity + a.start + r;
        q[i] = __ldg(reinterpret_cast<const uint2*>(a.codes[side] + at * kDim + c * 8));
        scale[i] = __ldg(a.scale[side] + at);
    }
#pragma unroll
    for (uint32_t i = 0; i < kSteps; ++i) {
        const uint32_t r = tile * kTileRows + i * 32 + (threadIdx.x >> 3);
        if (r >= a.rows) break;
        float x[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            const uint32_t word = e < 4 ? q[i].x : q[i].y;
            x[e] = static_cast<float>(static_cast<int8_t>(word >> (8 * (e & 3u)))) * scale[i];
        }
        store8(static_cast<T*>(a.out[side]) + (line * a.rows + r) * kDim + c * 8, x);
    }
}

uint32_t type_bytes(uint32_t type) { return type == DH_TYPE_F32 ? 4u : 2u; }

bool misaligned(const void* p, uint32_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

WriteSide side_of(const void* src, uint32_t type, const uint64_t* strides, int8_t* codes, float* scale) {
    WriteSide s{src, codes, scale, strides[0], strides[1], strides[2], strides[3], type, 0};
    const uint32_t e = type_bytes(type);
    s.wide = (s.dim == 1 || s.row == 1) && !misaligned(src, 16) &&
             ((s.seq | s.head | (s.dim == 1 ? s.row : s.dim)) * e) % 16 == 0;
    return s;
}

}  // namespace
}  // namespace dh

using namespace dh;

extern "C" uint32_t dh_kv_write_i8(const void* k, uint32_t k_type, const uint64_t* k_strides, const void* v,
                                   uint32_t v_type, const uint64_t* v_strides, uint32_t sequences, uint32_t heads,
                                   uint32_t rows, const int32_t* starts, uint32_t start, const int32_t* counts,
                                   int8_t* k_codes, float* k_scale, int8_t* v_codes, float* v_scale,
                                   uint32_t capacity, const uint32_t* run_rows, void* stream) {
    if (!k || !v || !k_strides || !v_strides || !k_codes || !k_scale || !v_codes || !v_scale)
        return DH_ERR_NULL_POINTER;
    if (k_type > DH_TYPE_F16 || v_type > DH_TYPE_F16 || sequences == 0 || heads == 0 || rows == 0 || capacity == 0)
        return DH_ERR_INVALID_ARGUMENT;
    if (rows > 0x7FFFFFFFu || capacity > 0x7FFFFFFFu) return DH_ERR_UNSUPPORTED_SHAPE;
    if (!starts && (start > capacity || (!counts && rows > capacity - start))) return DH_ERR_INVALID_ARGUMENT;
    if (misaligned(k, type_bytes(k_type)) || misaligned(v, type_bytes(v_type)) || misaligned(k_codes, 8) ||
        misaligned(v_codes, 8) || misaligned(k_scale, 4) || misaligned(v_scale, 4) || misaligned(starts, 4) ||
        misaligned(counts, 4) || misaligned(run_rows, 4))
        return DH_ERR_ALIGNMENT;
    WriteArgs a{};
    a.side[0] = side_of(k, k_type, k_strides, k_codes, k_scale);
    a.side[1] = side_of(v, v_type, v_strides, v_codes, v_scale);
    a.rows = rows, a.capacity = capacity;
    a.tiles = FastDiv((rows - 1) / kTileRows + 1), a.heads = FastDiv(heads);
    a.starts = starts, a.start = start, a.counts = counts, a.run_rows = run_rows;
    const uint64_t lines = static_cast<uint64_t>(sequences) * heads;  // of K, and as many of V
    if (lines > 0x3FFFFFFFull || 2 * lines * a.tiles.d > 0x7FFFFFFFull) return DH_ERR_UNSUPPORTED_SHAPE;
    const uint32_t grid = static_cast<uint32_t>(2 * lines * a.tiles.d);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (k_type == DH_TYPE_F32 || v_type == DH_TYPE_F32)
        kv_write_kernel<true><<<grid, kThreads, 0, st>>>(a);
    else
        kv_write_kernel<false><<<grid, kThreads, 0, st>>>(a);
    DH_LAUNCH_CHECK();
    return DH_OK;
}

extern "C" uint32_t dh_kv_read_i8(const int8_t* k_codes, const float* k_scale, const int8_t* v_codes,
                                  const float* v_scale, uint32_t entries, uint32_t heads, uint32_t capacity,
                                  uint32_t start, uint32_t rows, void* k, void* v, uint32_t out_type, void* stream) {
    if (!k_codes || !k_scale || !v_codes || !v_scale || !k || !v) return DH_ERR_NULL_POINTER;
    if (out_type > DH_TYPE_F16 || entries == 0 || heads == 0 || rows == 0 || start > capacity ||
        rows > capacity - start)
        return DH_ERR_INVALID_ARGUMENT;
    if (misaligned(k_codes, 8) || misaligned(v_codes, 8) || misaligned(k_scale, 4) || misaligned(v_scale, 4) ||
        misaligned(k, 16) || misaligned(v, 16))
        return DH_ERR_ALIGNMENT;
    const uint32_t tiles = (rows - 1) / kTileRows + 1;
    const uint64_t lines = static_cast<uint64_t>(entries) * heads;
    if (lines > 0x3FFFFFFFull || 2 * lines * tiles > 0x7FFFFFFFull) return DH_ERR_UNSUPPORTED_SHAPE;
    const ReadArgs a{{k_codes, v_codes}, {k_scale, v_scale}, {k, v}, rows, start, capacity, FastDiv(tiles), FastDiv(heads)};
    const uint32_t grid = static_cast<uint32_t>(2 * lines * tiles);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (out_type == DH_TYPE_BF16)
        kv_read_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(a);
    else if (out_type == DH_TYPE_F16)
        kv_read_kernel<__half><<<grid, kThreads, 0, st>>>(a);
    else
        kv_read_kernel<float><<<grid, kThreads, 0, st>>>(a);
    DH_LAUNCH_CHECK();
    return DH_OK;
}
