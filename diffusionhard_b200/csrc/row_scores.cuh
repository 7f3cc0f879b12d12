// row_scores.cuh -- pieces of the scoring kernels (token_scores.cu,
// head_scores.cu): softmax statistics of a row that are gathered in one pass
// and joined across threads, the k best tokens of a row as a list held by one
// warp, and the outputs of a finished row.
//
// For logits x of a row, m = max x, s = sum e^(x - m), t = sum e^(x - m) (x - m):
//   logsumexp = m + log s,  log p[c] = (x[c] - m) - log s,  entropy = log s - t / s.
// entropy adds two terms of the same sign (t <= 0), so nothing cancels.  A NaN
// or +inf anywhere in the row makes s NaN, and with it every result; a row
// whose logits are all -inf keeps m = -inf, s = 0.
#pragma once

#include "dh_common.cuh"

#include <math_constants.h>

namespace dh {

constexpr uint32_t kMaxTopK = 32;  // a warp holds the list, one entry a lane
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kFullMask = 0xFFFFFFFFu;

DH_DEVINL float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The larger value; NaN if either is.
DH_DEVINL float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// Statistics of part of a row.  `base` is the value the exponentials are
// relative to: the largest logit seen, or one up to kBaseSlack below it (a
// new maximum then needs no rescaling), and 0 while every logit was -inf.
struct RowStats {
    float base, s, t;
};
constexpr float kBaseSlack = 4.f;

// A part's sums relative to `m`, the maximum of the whole row (-inf: the
// row is empty so far).  Two parts relative to the same m add.
DH_DEVINL void rebase(RowStats& p, float m) {
    if (p.s == 0.f) {  // nothing but -inf
        p.t = 0.f;
    } else {
        // bounded, and the vanishing factor first: from the lowest finite
        // value to a usual one, s d and d itself overflow while e^d is 0
        const float d = max_nan(p.base - m, -1e30f);
        const float f = exp2_fast(d * kLog2E);
        p.s *= f;
        p.t = __fmaf_rn(p.s, d, f * p.t);
    }
    p.base = m;
}

// ------------------------------------------------- the k best of a row

// (logit, token) as one word that orders like (logit, lower token first).
// -0 counts as +0; 0 is no entry.  -inf and NaN are no candidates.
DH_DEVINL uint64_t token_key(float x, uint32_t id) { return pack_float_id(x + 0.f, id); }
DH_DEVINL float key_logit(uint64_t key) {
    const uint32_t b = static_cast<uint32_t>(key >> 32);
    return __uint_as_float((b & 0x80000000u) ? (b & 0x7FFFFFFFu) : ~b);
}

DH_DEVINL uint64_t shfl_u64(uint64_t v, uint32_t src) {
    return (static_cast<uint64_t>(__shfl_sync(kFullMask, static_cast<uint32_t>(v >> 32), src)) << 32) |
           __shfl_sync(kFullMask, static_cast<uint32_t>(v), src);
}
DH_DEVINL uint64_t shfl_up1_u64(uint64_t v) {
    return (static_cast<uint64_t>(__shfl_up_sync(kFullMask, static_cast<uint32_t>(v >> 32), 1)) << 32) |
           __shfl_up_sync(kFullMask, static_cast<uint32_t>(v), 1);
}

// Insert each lane's candidate (0: none) into the warp's list (lane i holds
// the i-th largest key; lanes >= k stay 0).  Whole warp.
DH_DEVINL void list_insert(uint64_t& list, uint64_t cand, uint32_t k, uint32_t lane) {
    uint64_t kth = shfl_u64(list, k - 1);
    uint32_t todo = __ballot_sync(kFullMask, cand > kth);
    while (todo) {
        const uint64_t key = shfl_u64(cand, __ffs(todo) - 1);
        todo &= todo - 1;
        const uint32_t pos = __popc(__ballot_sync(kFullMask, list > key));
        const uint64_t up = shfl_up1_u64(list);
        if (lane < k && lane >= pos) list = lane == pos ? key : up;
        if (todo) {
            kth = shfl_u64(list, k - 1);
            todo &= __ballot_sync(kFullMask, cand > kth);
        }
    }
}

// The k best of the list and a batch of up to 32 keys in shared memory, which
// serves as scratch.  A first batch (`fresh`) is sorted: a key's place is the
// number of keys above it.  Out of line: a row's end runs once a row, and its
// code size costs more than the call.  Whole warp.
static __device__ __noinline__ uint64_t list_merge(uint64_t list, bool fresh, uint64_t* batch, uint32_t count,
                                                   uint32_t k, uint32_t lane) {
    __syncwarp();
    const uint64_t key = lane < count ? batch[lane] : 0ull;
    if (!fresh) {
        list_insert(list, key, k, lane);
        __syncwarp();
        return list;
    }
    uint32_t place = 0;
#pragma unroll 4
    for (uint32_t i = 0; i < count; ++i) place += batch[i] > key;
    __syncwarp();
    if (lane >= count) batch[lane] = 0;
    __syncwarp();
    if (key) batch[place] = key;
    __syncwarp();
    list = lane < k ? batch[lane] : 0ull;
    __syncwarp();
    return list;
}

// The k best of a stream of candidates, gathered 32 at a time.  Whole warp.
struct TopList {
    uint64_t list;       // lane i: the i-th best so far
    uint64_t* batch;     // 32 words of shared memory
    uint32_t count, k, lane;
    bool fresh;          // nothing merged yet
    DH_DEVINL TopList(uint64_t* batch, uint32_t k, uint32_t lane)
        : list(0), batch(batch), count(0), k(k), lane(lane), fresh(true) {}
    DH_DEVINL void flush() {
        list = list_merge(list, fresh, batch, count, k, lane);
        fresh = false;
        count = 0;
    }
    // each lane's candidate (0: none)
    DH_DEVINL void add(uint64_t key) {
        const uint32_t mask = __ballot_sync(kFullMask, key != 0);
        const uint32_t n = __popc(mask);
        if (count + n > 32) flush();
        if (key) batch[count + __popc(mask & ((1u << lane) - 1u))] = key;
        count += n;
    }
};

// The largest of the lanes' values (no NaN).  Whole warp.
DH_DEVINL float lanes_max(float v) {
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(v));
    return y;
}
// One step of a bitonic sort across the lanes: partners `stride` apart, the
// larger first where `desc`.
DH_DEVINL float sort_step(float v, uint32_t stride, bool desc, uint32_t lane) {
    const float o = __shfl_xor_sync(kFullMask, v, stride);
    return ((lane & stride) != 0) != desc ? fmaxf(v, o) : fminf(v, o);
}

// The k-th largest of the lanes' pairs a >= b (1 <= k <= 64, no NaN; of a zero the
// sign may be either): one maximum after the other for a small k (~115 clocks each),
// else a sort of the 64.
// Rolled up: code that runs once a row is fetched from afar each time, and
// unrolled loops took longer to fetch than to run.  Whole warp.
DH_DEVINL float kth_largest_of_pairs(float a, float b, uint32_t k, uint32_t lane) {
    if (k <= 8) {
        float y = 0.f;
#pragma unroll 1
        for (uint32_t i = 0; i < k; ++i) {
            y = lanes_max(a);
            if (lane == __ffs(__ballot_sync(kFullMask, a == y)) - 1) {
                a = b;
                b = -CUDART_INF_F;
            }
        }
        return y;
    }
#pragma unroll 1
    for (uint32_t size = 2; size <= 64; size <<= 1) {
        if (size == 64) {
            const float hi = fmaxf(a, b);
            b = fminf(a, b);
            a = hi;
        }
#pragma unroll 1
        for (uint32_t stride = size == 64 ? 16 : size >> 1; stride > 0; stride >>= 1) {
            a = sort_step(a, stride, size >= 32 || (lane & size) == 0, lane);
            b = sort_step(b, stride, size == 64 || (size < 32 && (lane & size) == 0), lane);
        }
    }
    return __shfl_sync(kFullMask, k <= 32 ? a : b, (k - 1) % 32);
}
// v joins the two largest of a set, a >= b.
DH_DEVINL void two_largest(float& a, float& b, float v) {
    b = fmaxf(b, fminf(a, v));
    a = fmaxf(a, v);
}

// ------------------------------------------------------------- outputs

struct ScoreOutputs {
    float* logprobs;       // [rows, targets_per_row] or null
    float* entropy;        // [rows] or null
    float* logsumexp;      // [rows] or null
    int32_t* top_ids;      // [rows, top_k]
    float* top_logprobs;   // [rows, top_k]
    const void* targets;   // int32 or int64 [rows, targets_per_row]
    uint32_t targets_per_row, target_bytes, top_k;
};

DH_DEVINL int64_t target_of(const ScoreOutputs& o, uint64_t row, uint32_t i) {
    const uint64_t at = row * o.targets_per_row + i;
    return o.target_bytes == 8 ? __ldg(static_cast<const long long*>(o.targets) + at)
                               : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(o.targets) + at));
}

// What a finished row answers with.
struct RowResult {
    float m, log_s, entropy;
    bool bad, empty;  // NaN or +inf in the row; nothing above -inf
};
DH_DEVINL RowResult row_result(float m, float s, float t) {
    RowResult r;
    r.empty = s == 0.f;
    r.bad = !(s == s);
    r.m = m;
    r.log_s = logf(s);
    r.entropy = r.empty ? 0.f : r.log_s - t / s;
    return r;
}
DH_DEVINL float row_logprob(const RowResult& r, float x) {
    if (r.bad) return CUDART_NAN_F;
    if (r.empty) return -CUDART_INF_F;
    return (x - r.m) - r.log_s;
}
// The answer for given token t of a row (x: its logit).
DH_DEVINL float given_logprob(const RowResult& r, int64_t t, uint32_t vocab, float x) {
    return t < 0 ? 0.f : (t >= vocab ? CUDART_NAN_F : row_logprob(r, x));
}
DH_DEVINL void store_row(const ScoreOutputs& o, uint64_t row, const RowResult& r) {
    if (o.entropy) o.entropy[row] = r.entropy;
    if (o.logsumexp) o.logsumexp[row] = r.bad ? CUDART_NAN_F : (r.empty ? -CUDART_INF_F : r.m + r.log_s);
}
// Lane i holds the i-th best token's key (0: there is none).
DH_DEVINL void store_top(const ScoreOutputs& o, uint64_t row, const RowResult& r, uint64_t list, uint32_t lane) {
    if (lane >= o.top_k) return;
    const bool have = list != 0 && !r.bad;
    o.top_ids[row * o.top_k + lane] = have ? static_cast<int32_t>(packed_id(list)) : -1;
    o.top_logprobs[row * o.top_k + lane] =
        r.bad ? CUDART_NAN_F : (have ? row_logprob(r, key_logit(list)) : -CUDART_INF_F);
}

// Argument checks that the scoring entry points share.
inline uint32_t check_score_outputs(const ScoreOutputs& o) {
    if (o.targets_per_row && (!o.targets || !o.logprobs)) return DH_ERR_NULL_POINTER;
    if (o.top_k && (!o.top_ids || !o.top_logprobs)) return DH_ERR_NULL_POINTER;
    if (!o.targets_per_row && !o.top_k && !o.entropy && !o.logsumexp) return DH_ERR_NULL_POINTER;
    if (o.targets_per_row && o.target_bytes != 4 && o.target_bytes != 8) return DH_ERR_INVALID_ARGUMENT;
    const uintptr_t f = reinterpret_cast<uintptr_t>(o.logprobs) | reinterpret_cast<uintptr_t>(o.entropy) |
                        reinterpret_cast<uintptr_t>(o.logsumexp) | reinterpret_cast<uintptr_t>(o.top_ids) |
                        reinterpret_cast<uintptr_t>(o.top_logprobs);
    if ((f & 3u) || (o.targets_per_row && (reinterpret_cast<uintptr_t>(o.targets) & (o.target_bytes - 1))))
        return DH_ERR_ALIGNMENT;
    return DH_OK;
}

}  // namespace dh
