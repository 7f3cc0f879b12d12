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

#include "row_quant.cuh"

namespace dh {
namespace {

constexpr uint32_t kDim = 64;
constexpr uint32_t kTileRows = 64;   // rows of one (entry, head) and side a CTA takes
constexpr uint32_t kThreads = 256;
constexpr float kSmallest = 7.8886090522101181e-31f;  // 2^-100

struct WriteSide {
    const void* src;
    int8_t* codes;
    float* scale;
    uint64_t seq, head, row, dim;  // strides in elements
    uint32_t type;
    uint32_t wide;                 // rows are contiguous and 16-byte aligned
};

struct WriteArgs {
    WriteSide side[2];
    uint32_t sequences, heads, rows, capacity, tiles;
    const int32_t* starts;
    uint32_t start;
    const int32_t* counts;
    const uint32_t* run_rows;
};

DH_DEVINL float to_float(float x) { return x; }
DH_DEVINL float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
DH_DEVINL float to_float(__half x) { return __half2float(x); }

// 8 consecutive elements of a row as fp32 (16-byte loads)
DH_DEVINL void load8(const float* p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
DH_DEVINL void load8(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
DH_DEVINL void load8(const __half* p, float (&x)[8]) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

// Row pitch of the staged tile: odd in 4-byte words, so that 32 rows' stores of
// one column fall into 32 banks.
template <class T>
constexpr uint32_t kPitch = sizeof(T) == 4 ? kDim + 1 : kDim + 2;

template <class T>
DH_DEVINL void write_tile(const WriteArgs& a, const WriteSide& s, uint32_t seq, uint32_t head, uint32_t row0,
                          uint32_t rows, int64_t at, uint8_t* smem) {
    const T* src = static_cast<const T*>(s.src) + seq * s.seq + head * s.head + row0 * s.row;
    const uint32_t warp = warp_id(), lane = lane_id();
    const uint64_t base = (static_cast<uint64_t>(seq) * a.heads + head) * a.capacity;
    const bool staged = s.row == 1 && s.dim != 1;
    if (staged) {
        // positions are contiguous (a transposed V): 64 of them at a time, one
        // column after the other, turned in shared memory
        T* t = reinterpret_cast<T*>(smem);
#pragma unroll
        for (uint32_t i = 0; i < kDim / 8; ++i) {
            const uint32_t d = warp * (kDim / 8) + i;
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                const uint32_t r = lane + 32 * h;
                if (r < rows) t[r * kPitch<T> + d] = src[d * s.dim + r];
            }
        }
        __syncthreads();
    }
    // 8 lanes a row, 8 values each; a warp takes rows 8 w .. 8 w + 7 in two steps
    const uint32_t c = lane & 7u;
    float x[2][8];
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t r = warp * 8 + i * 4 + (lane >> 3);
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) x[i][e] = 0.f;
        if (r >= rows) continue;
        if (staged) {
            const T* p = reinterpret_cast<const T*>(smem) + r * kPitch<T> + c * 8;
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) x[i][e] = to_float(p[e]);
        } else if (s.wide) {
            load8(src + r * s.row + c * 8, x[i]);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) x[i][e] = to_float(src[r * s.row + (c * 8 + e) * s.dim]);
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t r = warp * 8 + i * 4 + (lane >> 3);
        // |x| ordered by its bits: NaN above infinity above every finite value
        uint32_t peak = 0;
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) peak = max(peak, __float_as_uint(x[i][e]) & 0x7FFFFFFFu);
#pragma unroll
        for (uint32_t o = 1; o < 8; o <<= 1) peak = max(peak, __shfl_xor_sync(0xFFFFFFFFu, peak, o));
        const bool live = peak >= __float_as_uint(kSmallest) && peak < 0x7F800000u;
        const float scale = live ? __fdiv_rn(__uint_as_float(peak), 127.0f)
                                 : (peak >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : 0.f);
        const Divisor by = make_divisor(live ? scale : 1.0f);
        uint32_t q[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) q[e] = q8_div_bits(x[i][e], by);
        uint2 w = make_uint2(pack4_i8(q[0], q[1], q[2], q[3]), pack4_i8(q[4], q[5], q[6], q[7]));
        if (!live) w = make_uint2(0u, 0u);
        const int64_t pos = at + r;
        if (r < rows && pos >= 0 && pos < a.capacity) {
            *reinterpret_cast<uint2*>(s.codes + (base + pos) * kDim + c * 8) = w;
            if (c == 0) s.scale[base + pos] = scale;
        }
    }
}

__global__ void __launch_bounds__(kThreads) kv_write_kernel(const __grid_constant__ WriteArgs a) {
    __shared__ __align__(16) uint8_t smem[kTileRows * kPitch<float> * 4];
    uint32_t w = blockIdx.x;
    const uint32_t tile = w % a.tiles;
    w /= a.tiles;
    const uint32_t head = w % a.heads;
    w /= a.heads;
    const uint32_t seq = w >> 1;
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
    else
        write_tile<float>(a, s, seq, head, row0, rows, at, smem);
}

struct ReadArgs {
    const int8_t* codes[2];
    const float* scale[2];
    void* out[2];
    uint32_t heads, rows, start, capacity, tiles;
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
    uint32_t w = blockIdx.x;
    const uint32_t tile = w % a.tiles;
    w /= a.tiles;
    const uint32_t head = w % a.heads;
    w /= a.heads;
    const uint32_t side = w & 1u, entry = w >> 1;
    const uint64_t line = static_cast<uint64_t>(entry) * a.heads + head;
    const uint32_t c = threadIdx.x & 7u;
    uint2 q[2];
    float scale[2];
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t r = tile * kTileRows + i * 32 + (threadIdx.x >> 3);
        if (r >= a.rows) break;
        const uint64_t at = line * a.capacity + a.start + r;
        q[i] = __ldg(reinterpret_cast<const uint2*>(a.codes[side] + at * kDim + c * 8));
        scale[i] = __ldg(a.scale[side] + at);
    }
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
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
    s.wide = s.dim == 1 && !misaligned(src, 16) && ((s.seq * e) | (s.head * e) | (s.row * e)) % 16 == 0;
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
    a.sequences = sequences, a.heads = heads, a.rows = rows, a.capacity = capacity;
    a.tiles = (rows + kTileRows - 1) / kTileRows;
    a.starts = starts, a.start = start, a.counts = counts, a.run_rows = run_rows;
    const uint64_t lines = static_cast<uint64_t>(sequences) * heads;  // of K, and as many of V
    if (lines > 0x3FFFFFFFull || 2 * lines * a.tiles > 0x7FFFFFFFull) return DH_ERR_UNSUPPORTED_SHAPE;
    kv_write_kernel<<<static_cast<uint32_t>(2 * lines * a.tiles), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
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
    const ReadArgs a{{k_codes, v_codes}, {k_scale, v_scale}, {k, v}, heads, rows, start, capacity, tiles};
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
