// token_scores.cu -- log probabilities of given tokens, entropy, logsumexp and
// the k best tokens of rows of logits, in one pass over the row
// (row_scores.cuh has the formulas).  The SUBS parametrisation excludes the
// mask token (mdlm._mdlm_log_probabilities, mdlm.py:851-858): its logit counts
// as -inf.
//
// One CTA, or a cluster of CTAs that split the row, per row.  Each thread
// streams 16-byte vectors of its CTA's slice and keeps its own maximum and
// sums.  The k best tokens then cost no work in the stream: the threads'
// maxima, taken over the warps, are the maxima of 32 disjoint parts of the
// slice, so the k-th largest of those 32 is at most the k-th best logit, and
// only the threads whose own maximum reaches it (about k of them) can hold one
// of the k best.  Those threads' vectors are read a second time, by whole
// warps, and what reaches the bound goes into the warp's list.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "row_scores.cuh"

namespace dh {
namespace {

constexpr uint32_t kScoreThreads = 256;
constexpr uint32_t kScoreWarps = kScoreThreads / 32;
constexpr uint32_t kScoreUnroll = 4;  // 16-byte loads a thread has in flight
constexpr uint32_t kMaxCluster = 8;

DH_DEVINL float to_float(float v) { return v; }
DH_DEVINL float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
DH_DEVINL float to_float(__half v) { return __half2float(v); }

DH_DEVINL void unpack(const uint4& v, float (&x)[4], float) {
    x[0] = __uint_as_float(v.x);
    x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z);
    x[3] = __uint_as_float(v.w);
}
DH_DEVINL void unpack(const uint4& v, float (&x)[8], __nv_bfloat16) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
DH_DEVINL void unpack(const uint4& v, float (&x)[8], __half) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

// Add N logits to the thread's statistics.
template <uint32_t N>
DH_DEVINL void add_logits(RowStats& st, float& m, const float (&x)[N]) {
    float cm = x[0];
#pragma unroll
    for (uint32_t i = 1; i < N; ++i) cm = fmaxf(cm, x[i]);
    if (cm > st.base + kBaseSlack || (m == -CUDART_INF_F && cm > m)) rebase(st, cm);
    m = fmaxf(m, cm);
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
        // a logit of -inf adds 0 to both sums: 0 * -inf would be NaN
        const float d = max_nan(x[i] - st.base, -1e30f);
        const float e = exp2_fast(d * kLog2E);
        st.s += e;
        st.t = __fmaf_rn(e, d, st.t);
    }
}

struct LogitRows {
    const void* logits;
    uint64_t row_stride;  // elements
    uint32_t vocab, mask_id;
    ScoreOutputs out;
};

DH_DEVINL uint32_t cluster_ctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
DH_DEVINL void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// This CTA's shared address as CTA `rank` of the cluster has it.
DH_DEVINL uint32_t peer_smem(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
DH_DEVINL uint64_t peer_load_u64(uint32_t a) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a));
    return v;
}
DH_DEVINL float peer_load_f32(uint32_t a) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a));
    return v;
}

template <class T>
__global__ void __launch_bounds__(kScoreThreads)
token_scores_kernel(const __grid_constant__ LogitRows p, uint32_t cluster) {
    constexpr uint32_t VE = 16 / sizeof(T);
    __shared__ float lane_max[kScoreWarps][32];
    __shared__ float sum_s[kScoreWarps], sum_t[kScoreWarps];
    __shared__ uint64_t lists[kScoreWarps][32];
    __shared__ uint64_t cta_list[32];
    __shared__ float cta_stats[3];

    const uint32_t tid = threadIdx.x, warp = warp_id(), lane = lane_id();
    const uint32_t rank = cluster > 1 ? cluster_ctarank() : 0u;
    const uint64_t row = blockIdx.x / cluster;
    const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
    // The row as 16-byte vectors from the boundary at or before its start:
    // vector v holds elements v * VE - off ...; those in [v_lo, v_hi) lie
    // inside the row, the up to 2 (VE - 1) elements around them are read one
    // by one, by the first CTA.
    const uint32_t off = static_cast<uint32_t>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
    const uint4* vec = reinterpret_cast<const uint4*>(x - off);
    const uint32_t v_lo = off ? 1u : 0u;
    const uint32_t v_hi = static_cast<uint32_t>((static_cast<uint64_t>(off) + p.vocab) / VE);
    const uint32_t n_vec = v_hi > v_lo ? v_hi - v_lo : 0u;
    const uint32_t per = (n_vec + cluster - 1) / cluster;
    const uint32_t begin = v_lo + min(n_vec, rank * per), end = v_lo + min(n_vec, (rank + 1) * per);
    const uint32_t head = n_vec ? (off ? VE - off : 0u) : p.vocab;
    const uint32_t tail_at = n_vec ? v_hi * VE - off : p.vocab;
    const uint32_t edges = rank == 0 ? head + (p.vocab - tail_at) : 0u;
    const uint64_t mask_at = static_cast<uint64_t>(p.mask_id) + off;  // past the row when there is none
    const uint32_t mask_vec = p.mask_id < p.vocab ? static_cast<uint32_t>(mask_at / VE) : 0xFFFFFFFFu;
    const uint32_t mask_elt = static_cast<uint32_t>(mask_at % VE);

    auto load = [&](uint32_t v, float (&f)[VE]) {
        unpack(__ldg(vec + v), f, T());
        if (v == mask_vec) {
#pragma unroll
            for (uint32_t e = 0; e < VE; ++e)
                if (e == mask_elt) f[e] = -CUDART_INF_F;
        }
    };
    auto edge_id = [&](uint32_t i) { return i < head ? i : tail_at + (i - head); };
    auto load_edge = [&](uint32_t id) { return id == p.mask_id ? -CUDART_INF_F : to_float(x[id]); };

    // the given tokens' logits, fetched while the row streams
    int64_t target = -1;
    float target_x = 0.f;
    if (rank == 0 && warp == 0 && lane < p.out.targets_per_row) {
        target = target_of(p.out, row, lane);
        if (target >= 0 && target < p.vocab) target_x = load_edge(static_cast<uint32_t>(target));
    }

    RowStats st{0.f, 0.f, 0.f};
    float m = -CUDART_INF_F;  // this thread's largest logit
    uint32_t v = begin + tid;
    for (; v + (kScoreUnroll - 1) * kScoreThreads < end; v += kScoreUnroll * kScoreThreads) {
        float f[kScoreUnroll][VE];
#pragma unroll
        for (uint32_t u = 0; u < kScoreUnroll; ++u) load(v + u * kScoreThreads, f[u]);
        add_logits(st, m, *reinterpret_cast<const float(*)[kScoreUnroll * VE]>(&f[0][0]));
    }
    for (; v < end; v += kScoreThreads) {
        float f[VE];
        load(v, f);
        add_logits(st, m, f);
    }
    if (tid < edges) {
        const float f[1] = {load_edge(edge_id(tid))};
        add_logits(st, m, f);
    }

    lane_max[warp][lane] = m;
    __syncthreads();
    float part = lane_max[0][lane];  // largest of the 8 threads of this lane
#pragma unroll
    for (uint32_t w = 1; w < kScoreWarps; ++w) part = fmaxf(part, lane_max[w][lane]);
    const float top = warp_max_f32(part);
    rebase(st, top);
    const float ws = warp_sum_f32(st.s), wt = warp_sum_f32(st.t);
    if (lane == 0) {
        sum_s[warp] = ws;
        sum_t[warp] = wt;
    }
    const uint32_t k = p.out.top_k;
    if (k) {
        const float bound = kth_largest_of_lanes(part, k, lane);
        uint64_t list = 0;
        for (uint32_t todo = __ballot_sync(kFullMask, m >= bound && m > -CUDART_INF_F); todo; todo &= todo - 1) {
            const uint32_t owner = warp * 32 + (__ffs(todo) - 1);  // whose vectors the warp reads again
            for (uint32_t v0 = begin + owner; v0 < end; v0 += 32 * kScoreThreads) {
                const uint64_t at = static_cast<uint64_t>(v0) + lane * kScoreThreads;
                float f[VE];
                const bool in = at < end;
                if (in) load(static_cast<uint32_t>(at), f);
#pragma unroll
                for (uint32_t e = 0; e < VE; ++e) {
                    const uint32_t id = static_cast<uint32_t>(at) * VE - off + e;
                    const bool c = in && f[e] >= bound && f[e] > -CUDART_INF_F;
                    if (__any_sync(kFullMask, c)) list_insert(list, c ? token_key(f[e], id) : 0ull, k, lane);
                }
            }
            if (owner < edges) {
                const uint32_t id = edge_id(owner);
                const float f = load_edge(id);
                const bool c = lane == 0 && f >= bound && f > -CUDART_INF_F;
                list_insert(list, c ? token_key(f, id) : 0ull, k, lane);
            }
        }
        lists[warp][lane] = list;
    }
    __syncthreads();
    if (warp == 0) {
        float s = warp_sum_f32(lane < kScoreWarps ? sum_s[lane] : 0.f);
        float t = warp_sum_f32(lane < kScoreWarps ? sum_t[lane] : 0.f);
        uint64_t list = 0;
        if (k) {
            list = lists[0][lane];
#pragma unroll
            for (uint32_t w = 1; w < kScoreWarps; ++w) list_insert(list, lists[w][lane], k, lane);
        }
        if (cluster > 1) {
            cta_list[lane] = list;
            if (lane == 0) {
                cta_stats[0] = top;
                cta_stats[1] = s;
                cta_stats[2] = t;
            }
        }
        sum_s[0] = s;
        sum_t[0] = t;
        lists[0][lane] = list;
    }
    if (cluster > 1) {
        cluster_sync();
        if (warp == 0 && rank == 0) {
            // join the CTAs' parts of the row
            RowStats o{-CUDART_INF_F, 0.f, 0.f};
            if (lane < cluster) {
                const uint32_t a = peer_smem(cta_stats, lane);
                o = RowStats{peer_load_f32(a), peer_load_f32(a + 4), peer_load_f32(a + 8)};
            }
            const float all = warp_max_f32(o.base);
            rebase(o, all);
            const float s = warp_sum_f32(o.s), t = warp_sum_f32(o.t);
            uint64_t list = cta_list[lane];
            for (uint32_t r = 1; r < cluster && k; ++r)
                list_insert(list, peer_load_u64(peer_smem(&cta_list[lane], r)), k, lane);
            lists[0][lane] = list;
            if (lane == 0) {
                lane_max[0][0] = all;
                sum_s[0] = s;
                sum_t[0] = t;
            }
        }
        cluster_sync();  // the peers' shared memory was read
        if (rank != 0) return;
    }
    if (warp != 0) return;
    __syncwarp();
    const float row_top = cluster > 1 ? lane_max[0][0] : top;
    const RowResult r = row_result(row_top, sum_s[0], sum_t[0]);
    if (lane == 0) store_row(p.out, row, r);
    if (k) store_top(p.out, row, r, lists[0][lane], lane);
    for (uint32_t i = lane; i < p.out.targets_per_row; i += 32) {
        if (i != lane) {
            target = target_of(p.out, row, i);
            target_x = target >= 0 && target < p.vocab ? load_edge(static_cast<uint32_t>(target)) : 0.f;
        }
        p.out.logprobs[row * p.out.targets_per_row + i] =
            target < 0 ? 0.f : (target >= p.vocab ? CUDART_NAN_F : row_logprob(r, target_x));
    }
}

template <class T>
cudaError_t launch_token_scores(const LogitRows& p, uint32_t rows, uint32_t cluster, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(rows * cluster);
    cfg.blockDim = dim3(kScoreThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, token_scores_kernel<T>, p, cluster);
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
    const LogitRows p{logits, row_stride, vocabulary_size, mask_token_id, out};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    // one CTA a row
    const uint32_t cluster = 1;
    cudaError_t e;
    if (logits_type == DH_TYPE_F32) e = launch_token_scores<float>(p, rows, cluster, s);
    else if (logits_type == DH_TYPE_BF16) e = launch_token_scores<__nv_bfloat16>(p, rows, cluster, s);
    else e = launch_token_scores<__half>(p, rows, cluster, s);
    return e == cudaSuccess ? DH_OK : DH_ERR_CUDA;
}
