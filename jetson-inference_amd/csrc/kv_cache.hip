// Rows into and out of the K / V caches (include/jinf/kv/kv_hip.h): the append
// of accepted tokens and the eviction by accumulated attention weight.
#include <hip/hip_runtime.h>

#include "jinf_device.h"
#include "jinf_host.h"
#include "jinf/kv/kv_hip.h"

namespace jinf {
namespace {

constexpr int kKvThreads = 256;
constexpr int kSelThreads = 1024;

// One value of a row as the cache stores it.
template <typename TC, typename TR>
__device__ __forceinline__ TC as_cached(TR v) {
    if constexpr (sizeof(TC) == sizeof(TR)) return v;
    else if constexpr (sizeof(TC) == 2) return f2h(v);
    else return h2f(v);
}

// grid (n_take, n_seq), one appended row a workgroup.
template <typename TC, typename TR>
__global__ __launch_bounds__(kKvThreads) void kv_append_kernel(
    TC* __restrict__ kc, TC* __restrict__ vc, int64_t ld_pos, int64_t ld_seq,
    float* __restrict__ weights, int64_t ld_w, int64_t ld_w_seq, const int32_t* __restrict__ lens,
    int32_t* __restrict__ lens_out, const TR* __restrict__ kr, const TR* __restrict__ vr,
    int64_t ld_rows, int64_t ld_rows_seq, int n_rows, const int32_t* __restrict__ index,
    const int32_t* __restrict__ counts, int n_take, int max_ctx, int kvw, int n_kv) {
    const int a = blockIdx.x, s = blockIdx.y;
    const int len = min(max(lens[s], 0), max_ctx);
    const int count = counts ? min(max(counts[s], 0), n_take) : n_take;
    if (a == 0 && threadIdx.x == 0 && lens_out) lens_out[s] = min(len + count, max_ctx);
    const int t = len + a;
    if (a >= count || t >= max_ctx) return;
    const int row = index ? index[(int64_t)s * n_take + a] : a;
    const bool live = row >= 0 && row < n_rows;
    const int64_t src = (int64_t)s * ld_rows_seq + (int64_t)(live ? row : 0) * ld_rows;
    const int64_t dst = (int64_t)s * ld_seq + (int64_t)t * ld_pos;
    for (int e = threadIdx.x; e < kvw; e += kKvThreads) {
        kc[dst + e] = live ? as_cached<TC, TR>(kr[src + e]) : TC(0);
        vc[dst + e] = live ? as_cached<TC, TR>(vr[src + e]) : TC(0);
    }
    if (weights)
        for (int j = threadIdx.x; j < n_kv; j += kKvThreads)
            weights[(int64_t)s * ld_w_seq + (int64_t)j * ld_w + t] = 0.0f;
}

// A weight as an unsigned number of the same order: NaN above everything, -0
// equal to +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The positions a (sequence, kv head) keeps: grid (n_kv, n_seq).  A radix
// select over the keys finds the smallest kept one and how many of its equals
// stay; an ordered pass then writes the kept positions and moves their weights
// (a weight moves to a lower place or stays, so within the pass a tile is read
// before it is written, and no later tile's weights are touched).
__global__ __launch_bounds__(kSelThreads) void kv_select_kernel(
    const float* weights, int64_t ld_w, int64_t ld_w_seq, float* weights_out, int64_t ld_wo,
    int64_t ld_wo_seq, const int32_t* __restrict__ lens, int32_t* __restrict__ list, int fill,
    int budget, int n_first, int n_recent, int max_ctx, int n_kv) {
    constexpr int kWaves = kSelThreads / kWave;
    __shared__ unsigned hist[256];
    __shared__ int wsum[2][kWaves];
    __shared__ unsigned s_digit, s_need;
    const int j = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
    const int wave = tid / kWave, lane = tid & (kWave - 1);
    const int len = min(max(lens[s], 0), max_ctx);
    const float* w = weights + (int64_t)s * ld_w_seq + (int64_t)j * ld_w;
    float* wo = weights_out + (int64_t)s * ld_wo_seq + (int64_t)j * ld_wo;
    int32_t* out = list + ((int64_t)s * n_kv + j) * budget;
    const int keep = min(len, budget);
    if (fill)
        for (int r = keep + tid; r < budget; r += kSelThreads) out[r] = -1;
    if (len <= budget) {
        for (int r = tid; r < len; r += kSelThreads) {
            out[r] = r;
            if (wo != w) wo[r] = w[r];
        }
        return;
    }
    const int lo = n_first, hi = len - n_recent;  // the positions that compete
    unsigned need = (unsigned)(budget - n_first - n_recent);  // of them, how many stay
    uint32_t prefix = 0;  // the threshold's digits found so far
    if (need > 0) {
#pragma unroll 1
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0;
            __syncthreads();
            for (int t = lo + tid; t < hi; t += kSelThreads) {
                const uint32_t k = weight_key(w[t]);
                if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)))
                    atomicAdd(&hist[(k >> shift) & 255], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                unsigned left = need;
                int d = 255;
                while (hist[d] < left) left -= hist[d--];
                s_digit = (unsigned)d;
                s_need = left;
            }
            __syncthreads();
            prefix |= s_digit << shift;
            need = s_need;
            __syncthreads();
        }
    }
    // need: how many positions whose key equals the threshold stay (0 when
    // none compete, and then nothing is above the threshold either)
    const bool none = budget == n_first + n_recent;
    int n_kept = 0, n_equal = 0;
    for (int t0 = 0; t0 < len; t0 += kSelThreads) {
        const int t = t0 + tid;
        float wt = 0.0f;
        bool above = false, equal = false;
        if (t < len) {
            wt = w[t];
            if (t < lo || t >= hi) {
                above = true;
            } else if (!none) {
                const uint32_t k = weight_key(wt);
                above = k > prefix;
                equal = k == prefix;
            }
        }
        const unsigned long long below = (1ull << lane) - 1;
        const unsigned long long eq = __ballot(equal);
        if (lane == 0) wsum[0][wave] = __popcll(eq);
        __syncthreads();
        int before = n_equal + __popcll(eq & below);
        for (int i = 0; i < kWaves; ++i) {
            if (i < wave) before += wsum[0][i];
            n_equal += wsum[0][i];
        }
        const bool stays = above || (equal && before < (int)need);
        const unsigned long long st = __ballot(stays);
        if (lane == 0) wsum[1][wave] = __popcll(st);
        __syncthreads();
        int r = n_kept + __popcll(st & below);
        for (int i = 0; i < kWaves; ++i) {
            if (i < wave) r += wsum[1][i];
            n_kept += wsum[1][i];
        }
        if (stays) {
            out[r] = t;
            wo[r] = wt;
        }
        __syncthreads();
    }
}

// The kept rows to their places: grid (n_kv, n_seq, 2 planes), rows in order.
// In place a row moves to a lower position or stays: a step's rows are all
// read before any is written, and no later step's rows are touched.
template <typename U>
__global__ __launch_bounds__(kKvThreads) void kv_move_kernel(
    U* ko, U* vo, int64_t ld_pos_out, int64_t ld_seq_out, const U* k, const U* v, int64_t ld_pos,
    int64_t ld_seq, const int32_t* __restrict__ lens, int32_t* __restrict__ lens_out,
    const int32_t* __restrict__ list, int budget, int max_ctx, int n_kv, int row_units) {
    const int j = blockIdx.x, s = blockIdx.y;
    const int len = min(max(lens[s], 0), max_ctx);
    const int keep = min(len, budget);
    const U* src = (blockIdx.z ? v : k) + (int64_t)s * ld_seq + (int64_t)j * row_units;
    U* dst = (blockIdx.z ? vo : ko) + (int64_t)s * ld_seq_out + (int64_t)j * row_units;
    const int32_t* at = list + ((int64_t)s * n_kv + j) * budget;
    const int64_t total = (int64_t)keep * row_units;
    for (int64_t i0 = 0; i0 < total; i0 += kKvThreads) {
        const int64_t i = i0 + threadIdx.x;
        const int r = (int)(i / row_units), u = (int)(i % row_units);
        U x{};
        if (i < total) x = src[(int64_t)at[r] * ld_pos + u];
        __syncthreads();
        if (i < total) dst[(int64_t)r * ld_pos_out + u] = x;
        __syncthreads();
    }
    (void)lens_out;
}

__global__ __launch_bounds__(kKvThreads) void kv_lens_kernel(const int32_t* lens, int32_t* lens_out,
                                                             int budget, int max_ctx, int n_seq) {
    const int s = blockIdx.x * kKvThreads + threadIdx.x;
    if (s < n_seq) lens_out[s] = min(min(max(lens[s], 0), max_ctx), budget);
}

bool kv_type_ok(int t) { return t == JINF_HIP_F32 || t == JINF_HIP_F16; }
int64_t kv_size(int t) { return t == JINF_HIP_F16 ? 2 : 4; }

// Bytes from the first to past the last element of n_seq caches of n_ctx positions.
int64_t kv_extent(int n_seq, int n_ctx, int64_t ld_seq, int64_t ld_pos, int64_t row, int64_t es) {
    if (n_seq <= 0 || n_ctx <= 0) return 0;
    return ((n_seq - 1) * ld_seq + (n_ctx - 1) * ld_pos + row) * es;
}

bool kv_overlap(const void* a, int64_t na, const void* b, int64_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return na > 0 && nb > 0 && x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}

template <typename U>
int kv_move(void* ko, void* vo, int64_t ld_pos_out, int64_t ld_seq_out, const void* k,
            const void* v, int64_t ld_pos, int64_t ld_seq, const int32_t* lens, int32_t* lens_out,
            const int32_t* list, int budget, int max_ctx, int n_seq, int n_kv, int64_t row_bytes,
            int64_t es, hipStream_t stream) {
    const int64_t n = (int64_t)sizeof(U) / es;  // elements of a unit (or units of an element: 1)
    return launch(kv_move_kernel<U>, dim3(n_kv, n_seq, 2), dim3(kKvThreads), 0, stream,
                  static_cast<U*>(ko), static_cast<U*>(vo), ld_pos_out / n, ld_seq_out / n,
                  static_cast<const U*>(k), static_cast<const U*>(v), ld_pos / n, ld_seq / n, lens,
                  lens_out, list, budget, max_ctx, n_kv, (int)(row_bytes / (int64_t)sizeof(U)));
}

}  // namespace
}  // namespace jinf

extern "C" int jinf_cache_append(void* k_cache, void* v_cache, int kv_type, int64_t ld_pos,
                                 int64_t ld_seq, float* weights, int64_t ld_w, int64_t ld_w_seq,
                                 const int32_t* lens, int32_t* lens_out, const void* k_rows,
                                 const void* v_rows, int rows_type, int ld_rows,
                                 int64_t ld_rows_seq, int n_rows, const int32_t* index,
                                 const int32_t* counts, int n_take, int n_seq, int max_ctx,
                                 int head_dim, int n_heads_kv, hipStream_t stream) {
    using namespace jinf;
    if (n_seq < 0 || n_take < 0 || n_rows < 0 || max_ctx < 0 || head_dim <= 0 || head_dim > 1024 ||
        n_heads_kv <= 0 || !kv_type_ok(kv_type) || !kv_type_ok(rows_type))
        return JINF_HIP_ERR_INVALID;
    if (n_seq == 0) return JINF_HIP_OK;
    const int64_t kvw = (int64_t)n_heads_kv * head_dim;
    if (n_seq > 65535 || max_ctx > (1 << 30) || kvw > 0x7FFFFFFF || !lens || lens_out == lens) return JINF_HIP_ERR_INVALID;
    if (!index && n_take > n_rows) return JINF_HIP_ERR_INVALID;
    if (ld_pos < kvw || (n_seq > 1 && ld_seq < (int64_t)max_ctx * ld_pos)) return JINF_HIP_ERR_INVALID;
    if (max_ctx > 0 && n_take > 0 && (!k_cache || !v_cache)) return JINF_HIP_ERR_INVALID;
    if (n_rows > 0 && n_take > 0 && (!k_rows || !v_rows || ld_rows < kvw || ld_rows_seq < 0))
        return JINF_HIP_ERR_INVALID;
    const uintptr_t ca = (uintptr_t)kv_size(kv_type), ra = (uintptr_t)kv_size(rows_type);
    if (!aligned(k_cache, ca) || !aligned(v_cache, ca) || !aligned(k_rows, ra) ||
        !aligned(v_rows, ra) || !aligned(weights, 4) || !aligned(lens, 4) || !aligned(lens_out, 4))
        return JINF_HIP_ERR_INVALID;
    if (weights && (ld_w < max_ctx || (n_seq > 1 && ld_w_seq < n_heads_kv * ld_w)))
        return JINF_HIP_ERR_INVALID;
    // (no rows: one workgroup a sequence still writes its length)
    const dim3 grid((unsigned)(n_take > 0 ? n_take : 1), (unsigned)n_seq);
#define JINF_KV_APPEND(TC, TR)                                                                     \
    launch(kv_append_kernel<TC, TR>, grid, dim3(kKvThreads), 0, stream, static_cast<TC*>(k_cache), \
           static_cast<TC*>(v_cache), ld_pos, ld_seq, weights, ld_w, ld_w_seq, lens, lens_out,     \
           static_cast<const TR*>(k_rows), static_cast<const TR*>(v_rows), ld_rows, ld_rows_seq,   \
           n_rows, index, counts, n_take, max_ctx, (int)kvw, n_heads_kv)
    if (kv_type == JINF_HIP_F16)
        return rows_type == JINF_HIP_F16 ? JINF_KV_APPEND(uint16_t, uint16_t)
                                         : JINF_KV_APPEND(uint16_t, float);
    return rows_type == JINF_HIP_F16 ? JINF_KV_APPEND(float, uint16_t) : JINF_KV_APPEND(float, float);
#undef JINF_KV_APPEND
}

extern "C" size_t jinf_cache_evict_workspace_bytes(int n_seq, int n_heads_kv, int budget) {
    if (n_seq <= 0 || n_heads_kv <= 0 || budget <= 0) return 0;
    return (size_t)n_seq * n_heads_kv * budget * sizeof(int32_t);
}

extern "C" int jinf_cache_evict(void* k_out, void* v_out, int64_t ld_pos_out, int64_t ld_seq_out,
                                const void* k_cache, const void* v_cache, int kv_type,
                                int64_t ld_pos, int64_t ld_seq, float* weights_out, int64_t ld_wo,
                                int64_t ld_wo_seq, const float* weights, int64_t ld_w,
                                int64_t ld_w_seq, const int32_t* lens, int32_t* lens_out,
                                int32_t* kept, int budget, int n_first, int n_recent, int n_seq,
                                int max_ctx, int head_dim, int n_heads_kv, void* workspace,
                                size_t workspace_bytes, hipStream_t stream) {
    using namespace jinf;
    if (n_seq < 0 || max_ctx < 0 || head_dim <= 0 || head_dim > 1024 || n_heads_kv <= 0 ||
        !kv_type_ok(kv_type) || budget < 0 || n_first < 0 || n_recent < 0 ||
        (int64_t)n_first + n_recent > budget)
        return JINF_HIP_ERR_INVALID;
    if (n_seq == 0) return JINF_HIP_OK;
    const int64_t kvw = (int64_t)n_heads_kv * head_dim, es = kv_size(kv_type);
    const int rows_out = budget < max_ctx ? budget : max_ctx;
    if (n_seq > 65535 || max_ctx > (1 << 30) || kvw > 0x7FFFFFFF || !lens || !aligned(lens, 4) || !aligned(lens_out, 4) ||
        !aligned(kept, 4))
        return JINF_HIP_ERR_INVALID;
    if (max_ctx > 0) {
        if (!k_cache || !v_cache || !weights || !k_out || !v_out || !weights_out)
            return JINF_HIP_ERR_INVALID;
        if (ld_pos < kvw || ld_pos_out < kvw || ld_w < max_ctx || ld_wo < rows_out)
            return JINF_HIP_ERR_INVALID;
        if (n_seq > 1 && (ld_seq < (int64_t)max_ctx * ld_pos || ld_w_seq < n_heads_kv * ld_w ||
                          ld_seq_out < (int64_t)rows_out * ld_pos_out ||
                          ld_wo_seq < n_heads_kv * ld_wo))
            return JINF_HIP_ERR_INVALID;
        if (!aligned(k_cache, es) || !aligned(v_cache, es) || !aligned(k_out, es) ||
            !aligned(v_out, es) || !aligned(weights, 4) || !aligned(weights_out, 4))
            return JINF_HIP_ERR_INVALID;
        // all in place, or apart from every input
        const bool in_place = k_out == k_cache;
        if (in_place != (v_out == v_cache) || in_place != (weights_out == weights))
            return JINF_HIP_ERR_INVALID;
        if (in_place) {
            if (ld_pos_out != ld_pos || ld_wo != ld_w ||
                (n_seq > 1 && (ld_seq_out != ld_seq || ld_wo_seq != ld_w_seq)))
                return JINF_HIP_ERR_INVALID;
        } else {
            const int64_t in = kv_extent(n_seq, max_ctx, ld_seq, ld_pos, kvw, es);
            const int64_t out = kv_extent(n_seq, rows_out, ld_seq_out, ld_pos_out, kvw, es);
            const int64_t wi = kv_extent(n_seq, n_heads_kv, ld_w_seq, ld_w, max_ctx, 4);
            const int64_t wo = kv_extent(n_seq, n_heads_kv, ld_wo_seq, ld_wo, rows_out, 4);
            if (kv_overlap(k_out, out, k_cache, in) || kv_overlap(v_out, out, v_cache, in) ||
                kv_overlap(weights_out, wo, weights, wi))
                return JINF_HIP_ERR_INVALID;
        }
    }
    if (!kept && budget > 0 &&
        (!workspace || !aligned(workspace, 16) ||
         workspace_bytes < jinf_cache_evict_workspace_bytes(n_seq, n_heads_kv, budget)))
        return JINF_HIP_ERR_INVALID;
    if (budget > 0) {
        int32_t* list = kept ? kept : static_cast<int32_t*>(workspace);
        int rc = launch(kv_select_kernel, dim3(n_heads_kv, n_seq), dim3(kSelThreads), 0, stream,
                        weights, ld_w, ld_w_seq, weights_out, ld_wo, ld_wo_seq, lens, list,
                        kept ? 1 : 0, budget, n_first, n_recent, max_ctx, n_heads_kv);
        if (rc != JINF_HIP_OK) return rc;
        // 16-byte units where everything is aligned to them, else single elements
        const int64_t row = (int64_t)head_dim * es;
        const bool wide = aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(k_out, 16) &&
                          aligned(v_out, 16) && row % 16 == 0 && ld_pos * es % 16 == 0 &&
                          ld_seq * es % 16 == 0 && ld_pos_out * es % 16 == 0 &&
                          ld_seq_out * es % 16 == 0;
#define JINF_KV_MOVE(U)                                                                          \
    kv_move<U>(k_out, v_out, ld_pos_out, ld_seq_out, k_cache, v_cache, ld_pos, ld_seq, lens, lens_out, \
               list, budget, max_ctx, n_seq, n_heads_kv, row, es, stream)
        if (max_ctx > 0)
            rc = wide ? JINF_KV_MOVE(u32x4) : es == 2 ? JINF_KV_MOVE(uint16_t) : JINF_KV_MOVE(uint32_t);
#undef JINF_KV_MOVE
        if (rc != JINF_HIP_OK) return rc;
    }
    if (lens_out)
        return launch(kv_lens_kernel, dim3((n_seq + kKvThreads - 1) / kKvThreads), dim3(kKvThreads),
                      0, stream, lens, lens_out, budget, max_ctx, n_seq);
    return JINF_HIP_OK;
}
