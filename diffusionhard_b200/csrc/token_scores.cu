// token_scores.cu -- log probabilities of given tokens, entropy, logsumexp and
// the k best tokens of rows of logits, in one pass over the row
// (row_scores.cuh has the formulas).  The SUBS parametrisation excludes the
// mask token (mdlm._mdlm_log_probabilities, mdlm.py:851-858): its logit counts
// as -inf.
//
// Persistent, warp-specialised CTAs take a row each.  One thread copies the row
// through a ring in shared memory (bulk copies, so that tens of KB are in flight
// whatever the other warps do); 8 warps add it up, each thread keeping its own
// maximum and sums; 2 warps take turns at what is left of a row (joining the
// threads' sums, the k best, the outputs) while the next row is already being
// added.
//
// The k best tokens: the k-th largest of any maxima of disjoint sets of logits
// is at most the k-th best logit.  The threads leave their maxima so far in
// shared memory after the first, third, 7th, 15th and so on stage of a row; each warp
// takes a bound from what it finds there and from then on notes each batch of a thread
// whose maximum, which the softmax needs anyway, reaches it.  At the end of the
// row the bound from all threads' maxima leaves about k batches of 64 bytes,
// which the finisher reads again, from L2.  Which batches are noted depends on
// the warps' timing, the result does not.  (Reading the whole shares of the
// threads that reach the final bound instead took 152 against 122 us for
// 4096 x 50258 bf16 logits and 8 alternatives, 80 us without any.)
//
// What bounds it: memory, with rows enough to fill the GPU (16384 x 50258 fp32
// logits without alternatives 486 us, 6.8 TB/s; 8880 x 50258 fp32 with 8
// alternatives 301 us, 5.9 TB/s); the end of the last rows with few (512 x 50258
// fp32 27 us, 35 with 5 alternatives, one row 12 and 18), which is latency of
// shared memory, shuffles and code that runs once a row.  A large k adds notes
// (8880 x 50258 fp32 with 32 alternatives 430 us; 645 with two bounds a row and room
// for 256 notes, where rows lost some and were read again).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "row_scores.cuh"
#include "tc_ptx.cuh"

namespace dh {
namespace {

constexpr uint32_t kScoreWarps = 8;
constexpr uint32_t kScoreThreads = 32 * kScoreWarps;
constexpr uint32_t kScoreUnroll = 4;  // 16-byte loads a thread has in flight
constexpr uint32_t kStageVecs = kScoreUnroll * kScoreThreads;  // 16 KB

DH_DEVINL float to_float(float v) { return v; }
DH_DEVINL float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
DH_DEVINL float to_float(__half v) { return __half2float(v); }

// The 16-byte vector's logits in pairs.
DH_DEVINL void unpack(const uint4& v, float2 (&x)[2], float) {
    x[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
    x[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
}
DH_DEVINL void unpack(const uint4& v, float2 (&x)[4], __nv_bfloat16) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
        x[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
}
DH_DEVINL void unpack(const uint4& v, float2 (&x)[4], __half) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) x[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
}

// The larger and the smaller of two (pairs of) logits as they are stored; a
// NaN is passed over.
DH_DEVINL uint32_t raw_max(uint32_t a, uint32_t b, float) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
}
DH_DEVINL uint32_t raw_min(uint32_t a, uint32_t b, float) {
    return __float_as_uint(fminf(__uint_as_float(a), __uint_as_float(b)));
}
DH_DEVINL uint32_t raw_max(uint32_t a, uint32_t b, __nv_bfloat16) {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}
DH_DEVINL uint32_t raw_min(uint32_t a, uint32_t b, __nv_bfloat16) {
    const __nv_bfloat162 m = __hmin2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}
DH_DEVINL uint32_t raw_max(uint32_t a, uint32_t b, __half) {
    const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}
DH_DEVINL uint32_t raw_min(uint32_t a, uint32_t b, __half) {
    const __half2 m = __hmin2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}
DH_DEVINL float2 raw_float(uint32_t a, float) { return make_float2(__uint_as_float(a), __uint_as_float(a)); }
DH_DEVINL float2 raw_float(uint32_t a, __nv_bfloat16) {
    return make_float2(__uint_as_float(a << 16), __uint_as_float(a & 0xFFFF0000u));
}
DH_DEVINL float2 raw_float(uint32_t a, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&a)); }

// A new maximum cm: move the base if it is too far below.
DH_DEVINL void raise(RowStats& st, float& m, float cm) {
    if (cm > st.base + kBaseSlack || (m == -CUDART_INF_F && cm > m)) rebase(st, cm);
    m = fmaxf(m, cm);
}

// N pairs of logits added to (s, t), relative to -nb.  kClamp: some may be
// -inf or far below: they add 0 to both sums, where 0 * -inf would be NaN.
template <bool kClamp, uint32_t N>
DH_DEVINL void add_pairs(float2& s, float2& t, const float2 (&x)[N], float nb) {
    const float2 nb2 = make_float2(nb, nb), c2 = make_float2(kLog2E, kLog2E);
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
        float2 d = __fadd2_rn(x[i], nb2);
        if (kClamp) d = make_float2(max_nan(d.x, -1e30f), max_nan(d.y, -1e30f));
        const float2 z = __fmul2_rn(d, c2);
        const float2 e = make_float2(exp2_fast(z.x), exp2_fast(z.y));
        s = __fadd2_rn(s, e);
        t = __ffma2_rn(e, d, t);
    }
}

template <class T, bool kClamp, uint32_t N>
DH_DEVINL void add_sums(RowStats& st, const uint4 (&v)[N]) {
    // two chains of additions each, and the vectors' own sums first
    float2 s[2] = {}, t[2] = {};
#pragma unroll
    for (uint32_t u = 0; u < N; ++u) {
        float2 x[8 / sizeof(T)];
        unpack(v[u], x, T());
        add_pairs<kClamp>(s[u & 1], t[u & 1], x, -st.base);
    }
    const float2 ss = __fadd2_rn(s[0], s[1]), tt = __fadd2_rn(t[0], t[1]);
    st.s += ss.x + ss.y;
    st.t += tt.x + tt.y;
}

// N 16-byte vectors of logits added to the thread's statistics.  Returns
// their maximum.
template <class T, uint32_t N>
DH_DEVINL float add_vectors(RowStats& st, float& m, const uint4 (&v)[N]) {
    uint32_t hi[N], lo[N];
#pragma unroll
    for (uint32_t u = 0; u < N; ++u) {
        hi[u] = raw_max(raw_max(v[u].x, v[u].y, T()), raw_max(v[u].z, v[u].w, T()), T());
        lo[u] = raw_min(raw_min(v[u].x, v[u].y, T()), raw_min(v[u].z, v[u].w, T()), T());
    }
#pragma unroll
    for (uint32_t u = 1; u < N; ++u) {
        hi[0] = raw_max(hi[0], hi[u], T());
        lo[0] = raw_min(lo[0], lo[u], T());
    }
    const float2 h = raw_float(hi[0], T()), l = raw_float(lo[0], T());
    const float top = fmaxf(h.x, h.y);
    raise(st, m, top);
    // (a NaN passes either way into both sums)
    if (fminf(l.x, l.y) > -1e30f && st.base < 1e30f) add_sums<T, false>(st, v);
    else add_sums<T, true>(st, v);
    return top;
}

struct LogitRows {
    const void* logits;
    uint64_t row_stride;  // elements
    uint32_t rows, vocab, mask_id;
    ScoreOutputs out;
};

// A row as 16-byte vectors from the boundary at or before its start: vector v
// holds elements v * VE - off ...; those in [v_lo, v_hi) lie inside the row,
// the up to 2 (VE - 1) elements around them ("edges") are read one by one.
template <class T>
struct RowView {
    static constexpr uint32_t VE = 16 / sizeof(T);
    const T* x;
    const uint4* vec;
    uint32_t off, v_lo, v_hi, head, tail_at, edges;
    uint32_t mask_id, mask_vec, mask_elt;  // the excluded token, and where it lies

    DH_DEVINL RowView(const LogitRows& p, uint64_t row) {
        x = static_cast<const T*>(p.logits) + row * p.row_stride;
        off = static_cast<uint32_t>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
        vec = reinterpret_cast<const uint4*>(x - off);
        v_lo = off ? 1u : 0u;
        v_hi = (off + p.vocab) / VE;
        if (v_hi < v_lo) v_hi = v_lo;
        const bool any = v_hi > v_lo;
        head = any ? (off ? VE - off : 0u) : p.vocab;
        tail_at = any ? v_hi * VE - off : p.vocab;
        edges = head + (p.vocab - tail_at);
        mask_id = p.mask_id;
        mask_vec = p.mask_id < p.vocab ? (p.mask_id + off) / VE : 0xFFFFFFFFu;
        mask_elt = (p.mask_id + off) % VE;
    }
    DH_DEVINL uint32_t edge_id(uint32_t i) const { return i < head ? i : tail_at + (i - head); }
    DH_DEVINL float element(uint32_t id) const { return id == mask_id ? -CUDART_INF_F : to_float(x[id]); }
    DH_DEVINL void exclude(uint4& r) const {
        T* e = reinterpret_cast<T*>(&r);
#pragma unroll
        for (uint32_t i = 0; i < VE; ++i)
            if (i == mask_elt) e[i] = static_cast<T>(-CUDART_INF_F);
    }
    DH_DEVINL uint4 vector(uint32_t v) const {
        uint4 r = __ldg(vec + v);
        if (v == mask_vec) exclude(r);
        return r;
    }
};

DH_DEVINL void add_one(RowStats& st, float& m, float x) {
    raise(st, m, x);
    const float d = max_nan(x - st.base, -1e30f), e = exp2_fast(d * kLog2E);
    st.s += e;
    st.t = __fmaf_rn(e, d, st.t);
}

// At most the k-th largest of the lanes' values (k <= 16, no NaN): the least maximum
// of k or more groups of lanes.  Lower than kth_largest_of_pairs, so that more is
// noted, but without its k steps one after the other, which every warp takes several
// times a row: 4096 x 50258 bf16 logits with 8 alternatives 116 against 123 us, 16000
// x 8000 fp32 174 against 187.  For more than 8 it would be too low.  Whole warp.
DH_DEVINL float least_of_groups(float v, uint32_t k) {
#pragma unroll 1
    for (uint32_t d = 1; d * k <= 16; d <<= 1) v = fmaxf(v, __shfl_xor_sync(kFullMask, v, d));
    return -lanes_max(-v);
}

// A batch: the kScoreUnroll vectors of one stage that one thread adds.
DH_DEVINL uint32_t batch_id(uint32_t stage, uint32_t thread) { return stage * kScoreThreads + thread; }

// The logits of n batches of a row that reach `bound`.  Whole warp.
template <class T>
DH_DEVINL void collect(TopList& best, const RowView<T>& r, float bound, const uint32_t* batches, uint32_t n,
                       uint32_t lane) {
    constexpr uint32_t VE = RowView<T>::VE;
    // (rolled up like all that runs once a row: see kth_largest_of_pairs)
#pragma unroll 1
    for (uint32_t i0 = 0; i0 < n * kScoreUnroll; i0 += 32) {
        const uint32_t i = i0 + lane;
        uint32_t reach = 0, at = 0;  // which of the lane's logits reach the bound
        float2 f[VE / 2];
        if (i < n * kScoreUnroll) {
            const uint32_t b = batches[i / kScoreUnroll];
            at = r.v_lo + b / kScoreThreads * kStageVecs + b % kScoreThreads + i % kScoreUnroll * kScoreThreads;
            if (at < r.v_hi) {
                unpack(r.vector(at), f, T());
#pragma unroll
                for (uint32_t e = 0; e < VE; ++e) {
                    const float y = e & 1 ? f[e / 2].y : f[e / 2].x;
                    if (y >= bound && y > -CUDART_INF_F) reach |= 1u << e;
                }
            }
        }
#pragma unroll 1
        while (__any_sync(kFullMask, reach != 0)) {
            uint64_t key = 0;
            if (reach) {
                const uint32_t e = __ffs(reach) - 1;
                reach &= reach - 1;
                float y = f[0].x;
#pragma unroll
                for (uint32_t j = 1; j < VE; ++j) y = j == e ? (j & 1 ? f[j / 2].y : f[j / 2].x) : y;
                key = token_key(y, at * VE - r.off + e);
            }
            best.add(key);
        }
    }
}

DH_DEVINL void bulk_load(void* smem, const void* gmem, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32(smem)),
                 "l"(gmem), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}

// --------------------------------------------------------------- the kernel

constexpr uint32_t kFinishers = 2;
constexpr uint32_t kThreads = kScoreThreads + 32 + 32 * kFinishers;
constexpr uint32_t kRingStages = 3;
constexpr uint32_t kCtasPerSM = 3;
constexpr uint32_t kNotes = 448;    // batches a row may note (more: its threads' whole shares are read again)
constexpr uint32_t kBatches = kScoreThreads + kNotes;

struct StreamSmem {
    uint4 ring[kRingStages][kStageVecs];
    // what a row's threads end with, and what a finisher needs for it
    float m[kFinishers][kScoreThreads], s[kFinishers][kScoreThreads], t[kFinishers][kScoreThreads];
    // the threads' maxima after the first stage of the row and a later one, -inf before
    float m_first[kFinishers][kScoreThreads], m_later[kFinishers][kScoreThreads];
    uint2 notes[kFinishers][kNotes];   // maximum and batch
    uint32_t note_count[kFinishers];
    uint32_t batches[kFinishers][kBatches];
    uint64_t keys[kFinishers][32];
    uint64_t full[kRingStages], empty[kRingStages];
    uint64_t done[kFinishers];    // a row's results are there
    uint64_t taken[kFinishers];   // and were read
};
constexpr uint32_t kStreamSmem = sizeof(StreamSmem) + 128;
static_assert(kCtasPerSM * (kStreamSmem + 1024) <= 228 * 1024, "shared memory of an SM");

template <class T, bool kTop>
__global__ void __launch_bounds__(kThreads, kCtasPerSM)
token_scores_kernel(const __grid_constant__ LogitRows p) {
    extern __shared__ uint8_t smem_raw[];
    StreamSmem& sm = *reinterpret_cast<StreamSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) &
                                                    ~static_cast<uintptr_t>(127));
    const uint32_t tid = threadIdx.x, warp = warp_id(), lane = lane_id();
    const uint64_t row0 = blockIdx.x, row_step = gridDim.x;
    if (tid == 0) {
        for (uint32_t s = 0; s < kRingStages; ++s) {
            tc::mbar_init(&sm.full[s], 1);
            tc::mbar_init(&sm.empty[s], kScoreWarps);
        }
        for (uint32_t f = 0; f < kFinishers; ++f) {
            tc::mbar_init(&sm.done[f], kScoreWarps);
            tc::mbar_init(&sm.taken[f], 1);
            sm.note_count[f] = 0;
        }
        tc::fence_barrier_init();
    }
    for (uint32_t i = tid; i < kFinishers * kScoreThreads; i += kThreads)
        (&sm.m_first[0][0])[i] = (&sm.m_later[0][0])[i] = -CUDART_INF_F;
    __syncthreads();

    if (warp < kScoreWarps) {
        // ------------------------------------------------------------ adders
        uint32_t stage = 0, phase = 0, f = 0, f_phase = 0;
        bool ok = true;
        for (uint64_t row = row0; row < p.rows && ok; row += row_step) {
            const RowView<T> x(p, row);
            RowStats st{0.f, 0.f, 0.f};
            float m = -CUDART_INF_F, bound = -CUDART_INF_F;
            if (tid < x.edges) add_one(st, m, x.element(x.edge_id(tid)));
            // this row's results go where the finisher's last row's were
            if (!tc::mbar_wait(&sm.taken[f], f_phase ^ 1, tc::kErrTimeoutEmpty)) break;
            uint32_t j = 0, take = 1;  // the row's stage, and the one that takes the next bound
            for (uint32_t v = x.v_lo; v < x.v_hi; v += kStageVecs, ++j) {
                if (!tc::mbar_wait(&sm.full[stage], phase, tc::kErrTimeoutFull)) {
                    ok = false;
                    break;
                }
                const uint4* in = sm.ring[stage];
                const uint32_t n = min(kStageVecs, x.v_hi - v);
                float h = -CUDART_INF_F;
                if (n == kStageVecs && x.mask_vec - v >= kStageVecs) {
                    uint4 r[kScoreUnroll];
#pragma unroll
                    for (uint32_t u = 0; u < kScoreUnroll; ++u) r[u] = in[tid + u * kScoreThreads];
                    h = add_vectors<T>(st, m, r);
                } else {
#pragma unroll 1
                    for (uint32_t i = tid; i < n; i += kScoreThreads) {
                        uint4 r[1] = {in[i]};
                        if (v + i == x.mask_vec) x.exclude(r[0]);
                        h = fmaxf(h, add_vectors<T>(st, m, r));
                    }
                }
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&sm.empty[stage]);
                if (++stage == kRingStages) {
                    stage = 0;
                    phase ^= 1;
                }
                if (kTop) {
                    if (j == take) {
                        const volatile float* held = j == 1 ? sm.m_first[f] : sm.m_later[f];
                        float a = -CUDART_INF_F, b = -CUDART_INF_F;
#pragma unroll
                        for (uint32_t w = 0; w < kScoreWarps; ++w) two_largest(a, b, held[w * 32 + lane]);
                        bound = p.out.top_k > 2 && p.out.top_k <= 8 ? least_of_groups(a, p.out.top_k)
                                                                    : kth_largest_of_pairs(a, b, p.out.top_k, lane);
                        take = 2 * j + 1;
                    }
                    if (j == 0) {
                        sm.m_first[f][tid] = m;
                    } else {
                        if (j + 1 == take) sm.m_later[f][tid] = m;
                        const bool note = h >= bound && h > -CUDART_INF_F;
                        const uint32_t who = __ballot_sync(kFullMask, note);
                        if (who) {
                            uint32_t at = 0;
                            if (lane == 0) at = atomicAdd(&sm.note_count[f], __popc(who));
                            at = __shfl_sync(kFullMask, at, 0) + __popc(who & ((1u << lane) - 1u));
                            if (note && at < kNotes)
                                sm.notes[f][at] = make_uint2(__float_as_uint(h), batch_id(j, tid));
                        }
                    }
                }
            }
            if (!ok) break;
            rebase(st, m);
            sm.m[f][tid] = m;
            sm.s[f][tid] = st.s;
            sm.t[f][tid] = st.t;
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&sm.done[f]);
            if (++f == kFinishers) {
                f = 0;
                f_phase ^= 1;
            }
        }
    } else if (warp == kScoreWarps) {
        // ------------------------------------------------------------ copies
        if (lane == 0) {
            uint32_t stage = 0, phase = 0, issued = 0, issued_parity = 0;
            bool ok = true;
            for (uint64_t row = row0; row < p.rows && ok; row += row_step) {
                const RowView<T> x(p, row);
                for (uint32_t v = x.v_lo; v < x.v_hi; v += kStageVecs) {
                    if (!tc::mbar_wait(&sm.empty[stage], phase ^ 1, tc::kErrTimeoutEmpty)) {
                        ok = false;
                        break;
                    }
                    const uint32_t bytes = min(kStageVecs, x.v_hi - v) * 16;
                    tc::mbar_arrive_expect_tx(&sm.full[stage], bytes);
                    bulk_load(sm.ring[stage], x.vec + v, bytes, &sm.full[stage]);
                    issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
                    ++issued;
                    if (++stage == kRingStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            // every copy has landed before this CTA may exit
            for (uint32_t s = 0; s < kRingStages && s < issued; ++s)
                tc::mbar_wait(&sm.full[s], (issued_parity >> s) & 1u, tc::kErrTimeoutFull);
        }
    } else {
        // --------------------------------------------------------- finishers
        const uint32_t f = warp - kScoreWarps - 1;
        uint32_t phase = 0;
        for (uint64_t row = row0 + f * row_step; row < p.rows; row += kFinishers * row_step, phase ^= 1) {
            const RowView<T> x(p, row);
            int64_t target = -1;
            float target_x = 0.f;
            if (lane < p.out.targets_per_row) {
                target = target_of(p.out, row, lane);
                if (target >= 0 && target < p.vocab) target_x = x.element(static_cast<uint32_t>(target));
            }
            const float edge = kTop && lane < x.edges ? x.element(x.edge_id(lane)) : 0.f;
            if (!tc::mbar_wait(&sm.done[f], phase, tc::kErrTimeoutFull)) break;
            float part = -CUDART_INF_F, second = -CUDART_INF_F;  // of the threads of this lane
#pragma unroll
            for (uint32_t w = 0; w < kScoreWarps; ++w) two_largest(part, second, sm.m[f][w * 32 + lane]);
            float top = lanes_max(part), s = 0.f, t = 0.f;
#pragma unroll
            for (uint32_t w = 0; w < kScoreWarps; ++w) {
                const uint32_t i = w * 32 + lane;
                RowStats st{sm.m[f][i], sm.s[f][i], sm.t[f][i]};
                rebase(st, top);
                s += st.s;
                t += st.t;
            }
            TopList best(sm.keys[f], p.out.top_k, lane);
            if (kTop) {
                const float bound = kth_largest_of_pairs(part, second, p.out.top_k, lane);
                // the first stage's batches, whose maxima are all kept, and the noted
                // ones; or, with notes lost, every batch of the threads that reach it
                const uint32_t notes = sm.note_count[f];
                const bool all = notes > kNotes;
                const uint32_t stages = all ? (x.v_hi - x.v_lo + kStageVecs - 1) / kStageVecs : 1u;
                uint32_t* batches = sm.batches[f];
                uint32_t n = 0;
                auto gather = [&](float h, uint32_t id) {
                    const uint32_t who = __ballot_sync(kFullMask, h >= bound && h > -CUDART_INF_F);
                    if ((who >> lane) & 1u) batches[n + __popc(who & ((1u << lane) - 1u))] = id;
                    n += __popc(who);
                };
#pragma unroll 1
                for (uint32_t j = 0; j < stages; ++j) {
                    n = 0;
#pragma unroll 2
                    for (uint32_t w = 0; w < kScoreWarps; ++w) {
                        const uint32_t i = w * 32 + lane;
                        gather(all ? sm.m[f][i] : sm.m_first[f][i], batch_id(j, i));
                    }
                    if (!all) {
#pragma unroll 1
                        for (uint32_t i = lane; i < notes + lane; i += 32) {
                            const uint2 note = i < notes ? sm.notes[f][i] : make_uint2(0xFF800000u, 0u);  // -inf
                            gather(__uint_as_float(note.x), note.y);
                        }
                    }
                    if (j + 1 == stages) {
                        // everything of this row was read
#pragma unroll
                        for (uint32_t w = 0; w < kScoreWarps; ++w)
                            sm.m_first[f][w * 32 + lane] = sm.m_later[f][w * 32 + lane] = -CUDART_INF_F;
                        if (lane == 0) sm.note_count[f] = 0;
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(&sm.taken[f]);
                    }
                    __syncwarp();
                    collect<T>(best, x, bound, batches, n, lane);
                    __syncwarp();
                }
                best.add(lane < x.edges && edge >= bound && edge > -CUDART_INF_F ? token_key(edge, x.edge_id(lane))
                                                                                 : 0ull);
                best.flush();
            } else {
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&sm.taken[f]);
            }
            s = warp_sum_f32(s);
            t = warp_sum_f32(t);
            const RowResult r = row_result(top, s, t);
            if (lane == 0) store_row(p.out, row, r);
            if (kTop) store_top(p.out, row, r, best.list, lane);
            for (uint32_t i = lane; i < p.out.targets_per_row; i += 32) {
                if (i != lane) {
                    target = target_of(p.out, row, i);
                    target_x = target >= 0 && target < p.vocab ? x.element(static_cast<uint32_t>(target)) : 0.f;
                }
                p.out.logprobs[row * p.out.targets_per_row + i] = given_logprob(r, target, p.vocab, target_x);
            }
        }
    }
}

template <class T, bool kTop>
cudaError_t launch_token_scores(const LogitRows& p, cudaStream_t stream) {
    static std::atomic<uint64_t> configured{0};
    const cudaError_t e = smem_optin_once(token_scores_kernel<T, kTop>, kStreamSmem, configured);
    if (e != cudaSuccess) return e;
    const uint32_t ctas = kCtasPerSM * device_sms();
    token_scores_kernel<T, kTop><<<p.rows < ctas ? p.rows : ctas, kThreads, kStreamSmem, stream>>>(p);
    return cudaGetLastError();
}

template <class T>
cudaError_t launch_token_scores(const LogitRows& p, cudaStream_t stream) {
    return p.out.top_k ? launch_token_scores<T, true>(p, stream) : launch_token_scores<T, false>(p, stream);
}

}  // namespace
}  // namespace dh

using namespace dh;

extern "C" uint32_t dh_token_logprobs(const void* logits, uint32_t logits_type, uint64_t row_stride, uint32_t rows,
                                      uint32_t vocabulary_size, uint32_t mask_token_id, const void* targets,
                                      uint32_t target_bytes, uint32_t targets_per_row, uint32_t top_k,
                                      float* logprobs, float* entropy, float* logsumexp, int32_t* top_ids,
                                      float* top_logprobs, void* stream) {
    if (!logits) return DH_ERR_NULL_POINTER;
    const ScoreOutputs out{logprobs, entropy, logsumexp, top_ids, top_logprobs, targets,
                           targets_per_row, target_bytes, top_k};
    const uint32_t st = check_score_outputs(out);
    if (st != DH_OK) return st;
    if (logits_type > DH_TYPE_F16 || rows == 0 || vocabulary_size == 0) return DH_ERR_INVALID_ARGUMENT;
    if (mask_token_id != DH_NO_TOKEN && mask_token_id >= vocabulary_size) return DH_ERR_INVALID_ARGUMENT;
    if (top_k > kMaxTopK || rows > (1u << 27) || vocabulary_size > (1u << 30)) return DH_ERR_UNSUPPORTED_SHAPE;
    if (reinterpret_cast<uintptr_t>(logits) & (logits_type == DH_TYPE_F32 ? 3u : 1u)) return DH_ERR_ALIGNMENT;
    const LogitRows p{logits, row_stride, rows, vocabulary_size, mask_token_id, out};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (logits_type == DH_TYPE_F32) e = launch_token_scores<float>(p, s);
    else if (logits_type == DH_TYPE_BF16) e = launch_token_scores<__nv_bfloat16>(p, s);
    else e = launch_token_scores<__half>(p, s);
    return e == cudaSuccess ? DH_OK : DH_ERR_CUDA;
}
