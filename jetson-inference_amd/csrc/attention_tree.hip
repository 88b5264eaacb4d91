// Attention of drafted tokens over a K / V cache, and decode attention that
// adds up each position's attention weight (include/jinf/kv/kv_hip.h).
//
// A drafted token ("node") attends to its sequence's cached positions and to
// the drafted tokens of its mask row.  Scores are kept in units of log2: with
// c = scale * log2(e), the weight of a row is 2^(c q.k - m) / sum.
#include <hip/hip_runtime.h>
#include <math.h>

#include "attention_device.h"
#include "jinf_device.h"
#include "jinf_host.h"
#include "jinf/kv/kv_hip.h"

namespace jinf {
namespace {

// What the attention kernels work on.  A "row" is a (node, query head of the
// kv head) pair: row r of kv head j is node r / group, head j group + r % group.
struct TreeArgs {
    float* out;
    const float* q;
    const void *kc, *vc, *kd, *vd;
    const int32_t *lens, *n_nodes;
    const uint64_t* mask;  // null: no drafted tokens, one node a sequence
    int64_t ld_out, ld_out_seq, ld_q, ld_q_seq, ld_pos, ld_seq, ld_draft, ld_draft_seq;
    int max_nodes, words, max_ctx, head_dim, n_heads, n_kv, group;
    float c;  // scale * log2(e)
    float* scores;  // null, or the scores [n_seq][n_heads][ld_scores] wanted
    int64_t ld_scores;
    float* records;  // {O[head_dim], m, l} per (sequence, row, chunk), or null
    int draft_f16;
};

__device__ __forceinline__ float tree_exp2(float a) { return __builtin_amdgcn_exp2f(a); }

template <typename T>
__device__ __forceinline__ float tree_get(const T* p, int64_t i) {
    if constexpr (sizeof(T) == 2) return h2f(p[i]);
    else return p[i];
}

// A drafted value as the cache would hold it.
template <typename TC>
__device__ __forceinline__ float tree_draft(const void* p, int f16, int64_t i) {
    const float v = f16 ? h2f(static_cast<const uint16_t*>(p)[i]) : static_cast<const float*>(p)[i];
    return sizeof(TC) == 2 ? h2f(f2h(v)) : v;
}

// Any head_dim and alignment: one wave per (sequence, node, head), lane l
// holding dims l, l + 64, ...; one reduction per row attended to.
template <typename TC>
__global__ __launch_bounds__(64) void tree_any_kernel(TreeArgs a) {
    constexpr int kMax = 16;
    const int lane = threadIdx.x, h = blockIdx.x, i = blockIdx.y, s = blockIdx.z;
    const int nodes = a.n_nodes ? min(max(a.n_nodes[s], 0), a.max_nodes) : a.max_nodes;
    if (i >= nodes) return;
    const int len = min(max(a.lens[s], 0), a.max_ctx);
    const int j = h / a.group, hd = a.head_dim;
    const TC* kb = static_cast<const TC*>(a.kc) + (int64_t)s * a.ld_seq + (int64_t)j * hd;
    const TC* vb = static_cast<const TC*>(a.vc) + (int64_t)s * a.ld_seq + (int64_t)j * hd;
    const float* qh = a.q + (int64_t)s * a.ld_q_seq + (int64_t)i * a.ld_q + (int64_t)h * hd;
    const uint64_t* mask = a.mask ? a.mask + ((int64_t)s * a.max_nodes + i) * a.words : nullptr;
    float qv[kMax], acc[kMax];
#pragma unroll
    for (int e = 0; e < kMax; ++e) {
        const int d = lane + e * kWave;
        qv[e] = d < hd ? qh[d] * a.c : 0.0f;
        acc[e] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    int n = 0;
    auto step = [&](auto key, auto value) {
        float part = 0.0f;
#pragma unroll
        for (int e = 0; e < kMax; ++e) {
            const int d = lane + e * kWave;
            if (d < hd) part = fmaf(qv[e], key(d), part);
        }
        const float st = wave_sum_f32(part);
        const float mn = fmaxf(m, st), ref = softmax_ref(mn);
        const float corr = tree_exp2(m - ref), p = tree_exp2(st - ref);
        l = fmaf(l, corr, p);
        m = mn;
#pragma unroll
        for (int e = 0; e < kMax; ++e) {
            const int d = lane + e * kWave;
            if (d < hd) acc[e] = fmaf(p, value(d), acc[e] * corr);
        }
        ++n;
        return st;
    };
    for (int t = 0; t < len; ++t) {
        const int64_t at = (int64_t)t * a.ld_pos;
        const float st = step([&](int d) { return tree_get(kb, at + d); },
                              [&](int d) { return tree_get(vb, at + d); });
        if (a.scores && lane == 0) a.scores[((int64_t)s * a.n_heads + h) * a.ld_scores + t] = st;
    }
    if (mask)
        for (int jn = 0; jn < nodes; ++jn) {
            if (!((mask[jn >> 6] >> (jn & 63)) & 1)) continue;
            const int64_t at = (int64_t)s * a.ld_draft_seq + (int64_t)jn * a.ld_draft + (int64_t)j * hd;
            step([&](int d) { return tree_draft<TC>(a.kd, a.draft_f16, at + d); },
                 [&](int d) { return tree_draft<TC>(a.vd, a.draft_f16, at + d); });
        }
    float* oh = a.out + (int64_t)s * a.ld_out_seq + (int64_t)i * a.ld_out + (int64_t)h * hd;
#pragma unroll
    for (int e = 0; e < kMax; ++e) {
        const int d = lane + e * kWave;
        if (d < hd) oh[d] = n > 0 ? acc[e] / l : 0.0f;
    }
    if (a.records && lane == 0) {
        float* rec = a.records + ((int64_t)s * a.n_heads + h) * (hd + 2);
        rec[hd] = m;
        rec[hd + 1] = l;
    }
}

// weights[s, j, t] += sum over the group's heads of 2^(score - m) / l, from the
// scores and the chunk records' (m, l): grid (ceil(max_ctx / 256), n_kv, n_seq).
__global__ __launch_bounds__(256) void tree_weights_kernel(
    float* __restrict__ weights, int64_t ld_w, int64_t ld_w_seq, const float* __restrict__ scores,
    int64_t ld_scores, const float* __restrict__ records, const int32_t* __restrict__ lens,
    int max_ctx, int n_heads, int group, int hd) {
    const int t = blockIdx.x * 256 + threadIdx.x, j = blockIdx.y, s = blockIdx.z;
    const int len = min(max(lens[s], 0), max_ctx);
    if (t >= len) return;
    float sum = 0.0f;
    for (int g = 0; g < group; ++g) {
        const int64_t h = (int64_t)s * n_heads + (int64_t)j * group + g;
        const float* rec = records + h * (hd + 2);
        sum += tree_exp2(scores[h * ld_scores + t] - softmax_ref(rec[hd])) / rec[hd + 1];
    }
    weights[(int64_t)s * ld_w_seq + (int64_t)j * ld_w + t] += sum;
}

constexpr float kLog2e = 1.44269502162933349609375f;

int64_t scores_ld(int max_ctx) { return ((int64_t)max_ctx + 63) / 64 * 64; }

// Shared checks of the caches and the query; n_seq > 0.
int tree_check(const void* out, const float* q, const void* k, const void* v, int kv_type,
               int64_t ld_pos, int64_t ld_seq, const int32_t* lens, int n_seq, int max_ctx,
               int head_dim, int n_heads, int n_heads_kv, float scale) {
    if (kv_type != JINF_HIP_F32 && kv_type != JINF_HIP_F16) return JINF_HIP_ERR_INVALID;
    if (!out || !q || !lens || n_heads % n_heads_kv != 0) return JINF_HIP_ERR_INVALID;
    if (max_ctx > 0 && (!k || !v)) return JINF_HIP_ERR_INVALID;
    const uintptr_t es = kv_type == JINF_HIP_F16 ? 2 : 4;
    if (!aligned(out, 4) || !aligned(q, 4) || !aligned(lens, 4) || !aligned(k, es) || !aligned(v, es))
        return JINF_HIP_ERR_INVALID;
    if (head_dim > 1024 || max_ctx > (1 << 30) || n_seq > 65535 || n_heads > 65535)
        return JINF_HIP_ERR_INVALID;
    if (ld_pos < (int64_t)n_heads_kv * head_dim) return JINF_HIP_ERR_INVALID;
    if (n_seq > 1 && ld_seq != 0 && ld_seq < (int64_t)max_ctx * ld_pos) return JINF_HIP_ERR_INVALID;
    if (!(scale > 0.0f) || !(scale < INFINITY)) return JINF_HIP_ERR_INVALID;
    return JINF_HIP_OK;
}

int tree_any(const TreeArgs& a, int kv_type, int n_seq, hipStream_t stream) {
    const dim3 grid((unsigned)a.n_heads, (unsigned)a.max_nodes, (unsigned)n_seq);
    return kv_type == JINF_HIP_F16
               ? launch(tree_any_kernel<uint16_t>, grid, dim3(kWave), 0, stream, a)
               : launch(tree_any_kernel<float>, grid, dim3(kWave), 0, stream, a);
}

}  // namespace
}  // namespace jinf

extern "C" size_t jinf_attention_tree_workspace_bytes(int n_seq, int max_nodes, int n_heads,
                                                      int n_heads_kv, int head_dim, int max_ctx) {
    if (n_seq <= 0 || max_nodes <= 0 || n_heads <= 0 || n_heads_kv <= 0 || head_dim <= 0 || max_ctx < 0)
        return 0;
    return 256;
}

extern "C" int jinf_attention_tree(float* out, int ld_out, int64_t ld_out_seq, const float* q,
                                   int ld_q, int64_t ld_q_seq, const void* k_cache,
                                   const void* v_cache, int kv_type, int64_t ld_pos, int64_t ld_seq,
                                   const int32_t* lens, const void* k_draft, const void* v_draft,
                                   int draft_type, int ld_draft, int64_t ld_draft_seq,
                                   const uint64_t* mask, const int32_t* n_nodes, int max_nodes,
                                   int n_seq, int max_ctx, int head_dim, int n_heads,
                                   int n_heads_kv, float scale, void* workspace,
                                   size_t workspace_bytes, hipStream_t stream) {
    using namespace jinf;
    if (n_seq < 0 || max_nodes < 0 || max_nodes > JINF_HIP_MAX_NODES || max_ctx < 0 || head_dim <= 0 ||
        n_heads <= 0 || n_heads_kv <= 0)
        return JINF_HIP_ERR_INVALID;
    if (n_seq == 0 || max_nodes == 0) return JINF_HIP_OK;
    if (scale == 0.0f) scale = (float)(1.0 / sqrt((double)head_dim));
    const int rc = tree_check(out, q, k_cache, v_cache, kv_type, ld_pos, ld_seq, lens, n_seq, max_ctx,
                              head_dim, n_heads, n_heads_kv, scale);
    if (rc != JINF_HIP_OK) return rc;
    const int64_t qw = (int64_t)n_heads * head_dim, kvw = (int64_t)n_heads_kv * head_dim;
    if (draft_type != JINF_HIP_F32 && draft_type != JINF_HIP_F16) return JINF_HIP_ERR_INVALID;
    const uintptr_t ds = draft_type == JINF_HIP_F16 ? 2 : 4;
    if (!k_draft || !v_draft || !mask || !aligned(k_draft, ds) || !aligned(v_draft, ds) ||
        !aligned(mask, 8) || !aligned(n_nodes, 4))
        return JINF_HIP_ERR_INVALID;
    if (ld_q < qw || ld_out < qw || ld_draft < kvw) return JINF_HIP_ERR_INVALID;
    if (n_seq > 1 && (ld_q_seq < (int64_t)max_nodes * ld_q || ld_out_seq < (int64_t)max_nodes * ld_out ||
                      ld_draft_seq < (int64_t)max_nodes * ld_draft))
        return JINF_HIP_ERR_INVALID;
    if (workspace && !aligned(workspace, 16)) return JINF_HIP_ERR_INVALID;
    TreeArgs a{};
    a.out = out, a.q = q, a.kc = k_cache, a.vc = v_cache, a.kd = k_draft, a.vd = v_draft;
    a.lens = lens, a.n_nodes = n_nodes, a.mask = mask;
    a.ld_out = ld_out, a.ld_out_seq = ld_out_seq, a.ld_q = ld_q, a.ld_q_seq = ld_q_seq;
    a.ld_pos = ld_pos, a.ld_seq = ld_seq, a.ld_draft = ld_draft, a.ld_draft_seq = ld_draft_seq;
    a.max_nodes = max_nodes, a.words = (max_nodes + 63) / 64, a.max_ctx = max_ctx;
    a.head_dim = head_dim, a.n_heads = n_heads, a.n_kv = n_heads_kv, a.group = n_heads / n_heads_kv;
    a.c = scale * kLog2e, a.draft_f16 = draft_type == JINF_HIP_F16;
    (void)workspace_bytes;
    return tree_any(a, kv_type, n_seq, stream);
}

extern "C" size_t jinf_attention_scored_workspace_bytes(int n_seq, int n_heads, int n_heads_kv,
                                                        int head_dim, int max_ctx) {
    if (n_seq <= 0 || n_heads <= 0 || n_heads_kv <= 0 || head_dim <= 0 || max_ctx < 0) return 0;
    return (size_t)n_seq * n_heads * (jinf::scores_ld(max_ctx) + head_dim + 2) * sizeof(float);
}

extern "C" int jinf_attention_decode_scored(float* out, int ld_out, const float* q, int ld_q,
                                            const void* k_cache, const void* v_cache, int kv_type,
                                            int64_t ld_pos, int64_t ld_seq, float* weights,
                                            int64_t ld_w, int64_t ld_w_seq, const int32_t* lens,
                                            int n_seq, int max_ctx, int head_dim, int n_heads,
                                            int n_heads_kv, float scale, void* workspace,
                                            size_t workspace_bytes, hipStream_t stream) {
    using namespace jinf;
    if (n_seq < 0 || max_ctx < 0 || head_dim <= 0 || n_heads <= 0 || n_heads_kv <= 0)
        return JINF_HIP_ERR_INVALID;
    if (n_seq == 0) return JINF_HIP_OK;
    if (scale == 0.0f) scale = (float)(1.0 / sqrt((double)head_dim));
    int rc = tree_check(out, q, k_cache, v_cache, kv_type, ld_pos, ld_seq, lens, n_seq, max_ctx,
                        head_dim, n_heads, n_heads_kv, scale);
    if (rc != JINF_HIP_OK) return rc;
    const int64_t qw = (int64_t)n_heads * head_dim;
    if (ld_q < qw || ld_out < qw) return JINF_HIP_ERR_INVALID;
    if (max_ctx > 0 && (!weights || !aligned(weights, 4) || ld_w < max_ctx ||
                        (n_seq > 1 && ld_w_seq < n_heads_kv * ld_w)))
        return JINF_HIP_ERR_INVALID;
    if (!workspace || !aligned(workspace, 16) ||
        workspace_bytes < jinf_attention_scored_workspace_bytes(n_seq, n_heads, n_heads_kv, head_dim, max_ctx))
        return JINF_HIP_ERR_INVALID;
    TreeArgs a{};
    a.out = out, a.q = q, a.kc = k_cache, a.vc = v_cache;
    a.lens = lens;
    a.ld_out = ld_out, a.ld_out_seq = ld_out, a.ld_q = ld_q, a.ld_q_seq = ld_q;
    a.ld_pos = ld_pos, a.ld_seq = ld_seq;
    a.max_nodes = 1, a.max_ctx = max_ctx, a.head_dim = head_dim;
    a.n_heads = n_heads, a.n_kv = n_heads_kv, a.group = n_heads / n_heads_kv;
    a.c = scale * kLog2e;
    a.scores = static_cast<float*>(workspace), a.ld_scores = scores_ld(max_ctx);
    a.records = a.scores + (int64_t)n_seq * n_heads * a.ld_scores;
    rc = tree_any(a, kv_type, n_seq, stream);
    if (rc != JINF_HIP_OK || max_ctx == 0) return rc;
    return launch(tree_weights_kernel, dim3((unsigned)((max_ctx + 255) / 256), (unsigned)n_heads_kv,
                                            (unsigned)n_seq),
                  dim3(256), 0, stream, weights, ld_w, ld_w_seq, a.scores, a.ld_scores, a.records,
                  lens, max_ctx, n_heads, a.group, head_dim);
}
