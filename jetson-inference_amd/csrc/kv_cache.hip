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

// Appended rows, V elements of K or V a thread: grid (ceil(n_take 2 kvw / V / 256), n_seq).
// What bounds it: the rows' bytes, read and written once (64 sequences x 76 rows of
// 1024 fp32 to fp16 on average: 17.4 us one element a thread at a time, 12.6 here).
template <typename TC, typename TR, int V>
__global__ __launch_bounds__(kKvThreads) void kv_append_kernel(
    TC* __restrict__ kc, TC* __restrict__ vc, int64_t ld_pos, int64_t ld_seq,
    float* __restrict__ weights, int64_t ld_w, int64_t ld_w_seq, const int32_t* __restrict__ lens,
    int32_t* __restrict__ lens_out, const TR* __restrict__ kr, const TR* __restrict__ vr,
    int64_t ld_rows, int64_t ld_rows_seq, int n_rows, const int32_t* __restrict__ index,
    const int32_t* __restrict__ counts, int n_take, int max_ctx, int units, int n_kv) {
    typedef TC VC __attribute__((ext_vector_type(V), aligned(V == 8 ? 16 : sizeof(TC))));
    typedef TR VR __attribute__((ext_vector_type(V), aligned(V == 8 ? 16 : sizeof(TR))));
    const int s = blockIdx.y;
    const int len = min(max(lens[s], 0), max_ctx);
    const int count = counts ? min(max(counts[s], 0), n_take) : n_take;
    if (blockIdx.x == 0 && threadIdx.x == 0 && lens_out) lens_out[s] = min(len + count, max_ctx);
    const int64_t x = (int64_t)blockIdx.x * kKvThreads + threadIdx.x;
    const int a = (int)(x / (2 * units)), u = (int)(x - (int64_t)a * 2 * units);
    const int t = len + a;
    if (a >= count || t >= max_ctx) return;
    const bool is_v = u >= units;
    const int e = (is_v ? u - units : u) * V;
    const int row = index ? index[(int64_t)s * n_take + a] : a;
    VC o = {};
    if (row >= 0 && row < n_rows) {
        const VR r = *reinterpret_cast<const VR*>((is_v ? vr : kr) + (int64_t)s * ld_rows_seq + (int64_t)row * ld_rows + e);
        if constexpr (sizeof(TC) == sizeof(TR)) {
            o = r;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = as_cached<TC, TR>(r[i]);
        }
    }
    *reinterpret_cast<VC*>((is_v ? vc : kc) + (int64_t)s * ld_seq + (int64_t)t * ld_pos + e) = o;
    if (weights && !is_v)
        for (int j = u; j < n_kv; j += units) weights[(int64_t)s * ld_w_seq + (int64_t)j * ld_w + t] = 0.0f;
}

// A weight as an unsigned number of the same order: -0 equal to +0, NaN above every
// number, and above it the positions that stay whatever their weight; 0 is no key.
constexpr uint32_t kKeyStays = 0xFFFFFFFFu, kKeyNan = 0xFFFFFFFEu;
__device__ __forceinline__ uint32_t weight_key(float w) {
    const uint32_t u = __float_as_uint(w + 0.0f);
    return w != w ? kKeyNan : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

// The positions a (sequence, kv head) keeps, those of the `budget` largest keys (the
// lowest first among equal ones), ascending: grid (n_kv, n_seq), one workgroup each.
// The keys are put into LDS once (for each pass, in segments of kSegMax, where there
// are more positions).  Three digits, 11, 11 and 10 bits from the top, each counted
// in LDS among the keys that share the digits before, give the smallest kept key and
// how many of its equals stay; a kept position's row is then the number of larger keys
// before it plus that of equals before it, at most as many as stay.
//
// What bounds it: instruction issue in the one workgroup, hence four keys a read and
// no range checks, and few keys left for the last digit; and code size, hence the
// rolled loops (weights in registers with unrolled passes, 50 KB of code, took 35 us at
// 8192 positions, fetching instructions).  Weights of one magnitude meet in few
// counters: a wave whose keys all share a digit adds once.
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
constexpr int kBins = 2048;
constexpr int kSelFew = 2048;  // keys that share the threshold's first digits, gathered if no more
constexpr int kSelStep = 4 * kSelThreads;
constexpr int kSegMax = 8 * kSelStep;  // positions held at once, 128 KiB
__global__ __launch_bounds__(kSelThreads) void kv_select_kernel(
    const float* __restrict__ weights, int64_t ld_w, int64_t ld_w_seq, const int32_t* __restrict__ lens,
    int32_t* __restrict__ list, int fill, int budget, int n_first, int n_recent, int max_ctx, int n_kv) {
    constexpr int kWaves = kSelThreads / kWave;
    extern __shared__ __attribute__((aligned(16))) uint32_t keys[];
    __shared__ unsigned hist[kBins];
    __shared__ unsigned counts[2][kSegMax / kSelStep * kWaves];  // larger, equal: per step and wave, then before
    __shared__ unsigned wsum[2][kWaves];
    __shared__ uint32_t few[kSelFew];
    __shared__ unsigned s_digit, s_need, s_here, s_few;
    const int j = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
    const int wave = tid / kWave, lane = tid & (kWave - 1);
    const int len = min(max(lens[s], 0), max_ctx);
    const float* w = weights + (int64_t)s * ld_w_seq + (int64_t)j * ld_w;
    int32_t* out = list + ((int64_t)s * n_kv + j) * budget;
    if (fill)
        for (int r = min(len, budget) + tid; r < budget; r += kSelThreads) out[r] = -1;
    if (len <= budget) {
        for (int r = tid; r < len; r += kSelThreads) out[r] = r;
        return;
    }
    const int n_seg = (len + kSegMax - 1) / kSegMax;
    // A segment's keys, 0 up to a whole step; steps in it.
    auto load = [&](int seg) {
        const int base = seg * kSegMax, n = min(kSegMax, len - base);
        const int steps = (n + kSelStep - 1) / kSelStep;
        if (n_seg > 1) __syncthreads();  // (the keys before have been read)
#pragma unroll 8
        for (int st = 0; st < steps; ++st) {
            const int at = st * kSelStep + 4 * tid, t = base + at;
            float x[4] = {0.f, 0.f, 0.f, 0.f};
            if (at + 4 <= n) {
                const f32x4u v = *reinterpret_cast<const f32x4u*>(w + t);
                x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (at + e < n) x[e] = w[t + e];
            }
            uint32_t k[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) k[e] = weight_key(x[e]);
            if (__ballot(t < n_first || t + 4 > len - n_recent)) {  // (past the end, too)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    k[e] = t + e >= len ? 0u : t + e < n_first || t + e >= len - n_recent ? kKeyStays : k[e];
            }
            *reinterpret_cast<uint4*>(keys + at) = make_uint4(k[0], k[1], k[2], k[3]);
        }
        __syncthreads();
        return steps;
    };
    int steps = load(0);
    auto key4 = [&](int st) { return *reinterpret_cast<const uint4*>(keys + st * kSelStep + 4 * tid); };
    // Sum of the threads' values before each thread, and of all.
    auto scan = [&](unsigned v, int which, unsigned& total) {
        unsigned x = v;
#pragma unroll
        for (int o = 1; o < kWave; o *= 2) {
            const unsigned y = __shfl_up(x, o, kWave);
            if (lane >= o) x += y;
        }
        if (lane == kWave - 1) wsum[which][wave] = x;
        __syncthreads();
        unsigned before = 0;
        total = 0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            if (i < wave) before += wsum[which][i];
            total += wsum[which][i];
        }
        return before + x - v;
    };
    uint32_t limit = 0;  // the threshold's digits found so far
    unsigned need = (unsigned)budget;
    unsigned here = 0, n_few = 0;  // keys that share the threshold's first digit, and those in `few`
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t digits = pass == 2 ? 1023u : 2047u;
        // keys whose digits before are the threshold's lie in [limit, limit + span] (0, no
        // key, is counted in the first pass, below every key, where nobody looks)
        const uint32_t span = pass == 0 ? 0xFFFFFFFFu : pass == 1 ? (1u << 21) - 1 : 1023u;
        hist[tid] = 0, hist[tid + kSelThreads] = 0;
        if (pass == 0 && tid == 0) s_few = 0;
        __syncthreads();
        const bool gather = pass == 1 && here <= kSelFew;  // this pass reads every key, the next these
        if (pass == 2 && here <= kSelFew && n_few > 0) {
            for (unsigned i = tid; i < n_few; i += kSelThreads) {
                const uint32_t k = few[i];
                if (k - limit <= span) atomicAdd(&hist[(k >> shift) & digits], 1u);
            }
        } else {
#pragma unroll 1
            for (int seg = 0; seg < n_seg; ++seg) {
                if (n_seg > 1) steps = load(seg);
#pragma unroll 1
                for (int st = 0; st < steps; ++st) {
                    const uint4 k4 = key4(st);
                    const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
                    bool in[4], any = false;
                    uint32_t d[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        in[e] = k[e] - limit <= span;
                        d[e] = (k[e] >> shift) & digits;
                        any |= in[e];
                    }
                    if (!__ballot(any)) continue;
                    const uint32_t d0 = __builtin_amdgcn_readfirstlane(d[0]);
                    if (!gather && !__ballot(!(in[0] && in[1] && in[2] && in[3] && d[0] == d0 && d[1] == d0 &&
                                               d[2] == d0 && d[3] == d0))) {
                        if (lane == 0) atomicAdd(&hist[d0], 4u * kWave);
                        continue;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (in[e]) atomicAdd(&hist[d[e]], 1u);
                    if (gather) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (in[e]) few[atomicAdd(&s_few, 1u)] = k[e];  // (at most `here` of them)
                    }
                }
            }
        }
        __syncthreads();
        // from the largest digit down: the one at which `need` are reached
        const unsigned h1 = hist[kBins - 1 - 2 * tid], h2 = hist[kBins - 2 - 2 * tid];
        unsigned total;
        const unsigned before = scan(h1 + h2, pass & 1, total);
        if (before < need && need <= before + h1 + h2) {
            const bool first = need <= before + h1;
            s_digit = (unsigned)(kBins - (first ? 1 : 2) - 2 * tid);
            s_need = need - before - (first ? 0 : h1);
            s_here = first ? h1 : h2;
        }
        __syncthreads();
        limit |= s_digit << shift;
        need = s_need;
        if (pass == 0) here = s_here;
        if (gather) n_few = s_few;
    }
    // `limit` is the smallest kept key now, and `need` of its equals stay
    unsigned n_larger = 0, n_equal = 0;  // in the segments before
#pragma unroll 1
    for (int seg = 0; seg < n_seg; ++seg) {
        if (n_seg > 1) steps = load(seg);
#pragma unroll 1
        for (int st = 0; st < steps; ++st) {
            const uint4 k = key4(st);
            const unsigned larger = __popcll(__ballot(k.x > limit)) + __popcll(__ballot(k.y > limit)) +
                                    __popcll(__ballot(k.z > limit)) + __popcll(__ballot(k.w > limit));
            unsigned equal = 0;  // (few keys equal the threshold)
            if (__ballot(k.x == limit || k.y == limit || k.z == limit || k.w == limit))
                equal = __popcll(__ballot(k.x == limit)) + __popcll(__ballot(k.y == limit)) +
                        __popcll(__ballot(k.z == limit)) + __popcll(__ballot(k.w == limit));
            if (lane == 0) counts[0][st * kWaves + wave] = larger, counts[1][st * kWaves + wave] = equal;
        }
        __syncthreads();
        unsigned total[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const unsigned v = tid < steps * kWaves ? counts[x][tid] : 0u;
            const unsigned before = scan(v, x, total[x]);
            if (tid < steps * kWaves) counts[x][tid] = before;
        }
        __syncthreads();
#pragma unroll 1
        for (int st = 0; st < steps; ++st) {
            const uint4 k4 = key4(st);
            const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
            unsigned a = n_larger + counts[0][st * kWaves + wave];
            unsigned b = n_equal + counts[1][st * kWaves + wave];
            // the lanes before, then this lane's own four in turn
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned long long x = __ballot(k[e] > limit);
                a = __builtin_amdgcn_mbcnt_hi((uint32_t)(x >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)x, a));
            }
            if (__ballot(k[0] == limit || k[1] == limit || k[2] == limit || k[3] == limit)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const unsigned long long y = __ballot(k[e] == limit);
                    b = __builtin_amdgcn_mbcnt_hi((uint32_t)(y >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)y, b));
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool larger = k[e] > limit, equal = k[e] == limit;
                if (larger || (equal && b < need)) out[a + min(b, need)] = seg * kSegMax + st * kSelStep + 4 * tid + e;
                a += larger;
                b += equal;
            }
        }
        n_larger += total[0], n_equal += total[1];
    }
}

// The kept rows to their places: grid (n_kv slices, n_seq, 2 planes x chunks + 1), rows in
// order, `w` units of a row a workgroup; the last of the third index move the weights
// (by the workgroups of slice 0).  A kept row moves to a lower position or stays.  In
// place, one workgroup therefore walks all rows of its slice, and a step's rows are all
// read before its first is written: rows that later steps read lie past them, so the
// next step's loads are under way meanwhile.  Into other caches, chunks of rows are
// independent.
//
// What bounds it: the rows' bytes, read and written once; with few sequences, how
// many of them one workgroup keeps in flight (64 KiB here), hence the slices.
constexpr int kMoveThreads = 1024;
constexpr int kMoveU = 4;  // units a thread holds per step
constexpr int kMoveItems = 256;  // workgroups that a call aims for, one a CU
// Rows r_begin .. r_end of one workgroup's slice: threads of lane-row rl < per take unit
// u (already in src and dst) of rows rl, rl + per, ...
template <typename U>
__device__ __forceinline__ void move_rows(U* dst, int64_t ld_dst, const U* src, int64_t ld_src,
                                          const int32_t* __restrict__ at, int r_begin, int r_end,
                                          int per, int rl, bool in_place) {
    const int step = per * kMoveU;
    int idx[kMoveU];  // the next step's positions
    U x[kMoveU];
    auto positions = [&](int r0) {
#pragma unroll
        for (int i = 0; i < kMoveU; ++i) {
            const int r = r0 + i * per + rl;
            idx[i] = rl < per && r < r_end ? at[r] : -1;
            if (in_place && idx[i] == r) idx[i] = -1;  // stays where it is
        }
    };
    bool moves[kMoveU];
    auto rows = [&]() {
#pragma unroll
        for (int i = 0; i < kMoveU; ++i) {
            moves[i] = idx[i] >= 0;
            if (moves[i]) x[i] = src[(int64_t)idx[i] * ld_src];
        }
    };
    positions(r_begin);
    rows();
    for (int r0 = r_begin; r0 < r_end; r0 += step) {
        U y[kMoveU];
        bool m[kMoveU];
        positions(r0 + step);
#pragma unroll
        for (int i = 0; i < kMoveU; ++i) y[i] = x[i], m[i] = moves[i];
        // every thread's rows of this step are in registers before any is written
        if (in_place) {
            __builtin_amdgcn_s_waitcnt(waitcnt_vm<0>());
            __syncthreads();
        }
        rows();
#pragma unroll
        for (int i = 0; i < kMoveU; ++i)
            if (m[i]) dst[(int64_t)(r0 + i * per + rl) * ld_dst] = y[i];
    }
}

template <typename U>
__global__ __launch_bounds__(kMoveThreads) void kv_move_kernel(
    U* ko, U* vo, int64_t ld_pos_out, int64_t ld_seq_out, const U* k, const U* v, int64_t ld_pos,
    int64_t ld_seq, float* weights_out, int64_t ld_wo, int64_t ld_wo_seq, const float* weights,
    int64_t ld_w, int64_t ld_w_seq, const int32_t* lens, int32_t* lens_out,
    const int32_t* __restrict__ list, int budget, int max_ctx, int n_kv, int row_units, int w,
    int chunk, int in_place) {
    const int j = blockIdx.x % n_kv, slice = blockIdx.x / n_kv, s = blockIdx.y;
    const bool is_weights = blockIdx.z == gridDim.z - 1;
    if (is_weights && slice > 0) return;
    const int len = min(max(lens[s], 0), max_ctx);
    const int keep = min(len, budget);
    // (lens_out may be lens: min(len, budget) is the same number before and after, len is
    // not, so what tells whether rows move is the last one's place: the list ascends)
    if (blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0 && lens_out) lens_out[s] = keep;
    const int32_t* at = list + ((int64_t)s * n_kv + j) * budget;
    if (in_place && (keep == 0 || at[keep - 1] == keep - 1)) return;
    if (is_weights) {
        move_rows(weights_out + (int64_t)s * ld_wo_seq + (int64_t)j * ld_wo, 1,
                  weights + (int64_t)s * ld_w_seq + (int64_t)j * ld_w, 1, at, 0, keep, kMoveThreads,
                  (int)threadIdx.x, in_place);
        return;
    }
    const int plane = blockIdx.z & 1, r_begin = (int)(blockIdx.z >> 1) * chunk;
    const int u = threadIdx.x % w, rl = threadIdx.x / w;
    const int64_t off = (int64_t)j * row_units + (int64_t)slice * w + u;
    move_rows((plane ? vo : ko) + (int64_t)s * ld_seq_out + off, ld_pos_out,
              (plane ? v : k) + (int64_t)s * ld_seq + off, ld_pos, at, r_begin,
              min(keep, r_begin + chunk), kMoveThreads / w, rl, in_place);
}

// No position stays: lengths of 0, and no kept one.
__global__ __launch_bounds__(kKvThreads) void kv_none_kernel(int32_t* __restrict__ lens_out, int n_seq,
                                                             int32_t* __restrict__ kept, int64_t n_kept) {
    const int64_t stride = (int64_t)gridDim.x * kKvThreads;
    for (int64_t i = (int64_t)blockIdx.x * kKvThreads + threadIdx.x; i < n_seq || i < n_kept; i += stride) {
        if (lens_out && i < n_seq) lens_out[i] = 0;
        if (i < n_kept) kept[i] = -1;
    }
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
            const void* v, int64_t ld_pos, int64_t ld_seq, float* weights_out, int64_t ld_wo,
            int64_t ld_wo_seq, const float* weights, int64_t ld_w, int64_t ld_w_seq,
            const int32_t* lens, int32_t* lens_out, const int32_t* list, int budget, int max_ctx,
            int n_seq, int n_kv, int64_t row_bytes, int64_t es, hipStream_t stream) {
    const int64_t n = (int64_t)sizeof(U) / es;  // elements of a unit
    const int row_units = (int)(row_bytes / (int64_t)sizeof(U));
    const bool in_place = ko == k;
    const int rows = budget < max_ctx ? budget : max_ctx;
    // In place with fewer (sequence, kv head, plane) than CUs, rows are cut into
    // slices of 128, then 64 bytes.
    int w = row_units;  // (at most 1024)
    if (in_place && sizeof(U) == 16)
        for (int cut = 8; cut >= 4; cut /= 2)
            if (row_units % cut == 0 && cut < w && (int64_t)n_seq * n_kv * 2 * (row_units / w) < kMoveItems) w = cut;
    // Into other caches: chunks of rows, of one step at least, for about four
    // workgroups a CU.
    const int step = kMoveThreads / w * kMoveU;
    int chunk = rows;
    if (!in_place) {
        const int64_t groups = (int64_t)n_seq * n_kv * 2 * (row_units / w);
        const int64_t nch = groups < 4 * kMoveItems ? 4 * kMoveItems / groups : 1;
        chunk = (int)(((int64_t)rows + nch - 1) / nch);
        chunk = (chunk + step - 1) / step * step;
    }
    const int64_t chunks = (rows + (int64_t)chunk - 1) / chunk;
    return launch(kv_move_kernel<U>,
                  dim3((unsigned)(n_kv * (row_units / w)), (unsigned)n_seq, (unsigned)(2 * chunks + 1)),
                  dim3(kMoveThreads), 0, stream, static_cast<U*>(ko), static_cast<U*>(vo),
                  ld_pos_out / n, ld_seq_out / n, static_cast<const U*>(k), static_cast<const U*>(v),
                  ld_pos / n, ld_seq / n, weights_out, ld_wo, ld_wo_seq, weights, ld_w, ld_w_seq, lens,
                  lens_out, list, budget, max_ctx, n_kv, row_units, w, chunk, in_place ? 1 : 0);
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
    // 8 elements a thread where every row starts at 16 bytes, else one
    const int64_t cs = kv_size(kv_type), rs = kv_size(rows_type);
    const bool wide = kvw % 8 == 0 && aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(k_rows, 16) &&
                      aligned(v_rows, 16) && ld_pos * cs % 16 == 0 && ld_seq * cs % 16 == 0 &&
                      ld_rows * rs % 16 == 0 && ld_rows_seq * rs % 16 == 0;
    const int64_t units = wide ? kvw / 8 : kvw;
    // (no rows: one workgroup a sequence still writes its length)
    const int64_t blocks = ((int64_t)n_take * 2 * units + kKvThreads - 1) / kKvThreads;
    if (blocks > 0x7FFFFFFF) return JINF_HIP_ERR_INVALID;
    const dim3 grid((unsigned)(blocks > 0 ? blocks : 1), (unsigned)n_seq);
#define JINF_KV_APPEND(TC, TR)                                                                       \
    launch(wide ? kv_append_kernel<TC, TR, 8> : kv_append_kernel<TC, TR, 1>, grid, dim3(kKvThreads), 0, \
           stream, static_cast<TC*>(k_cache), static_cast<TC*>(v_cache), ld_pos, ld_seq, weights, ld_w, \
           ld_w_seq, lens, lens_out, static_cast<const TR*>(k_rows), static_cast<const TR*>(v_rows),  \
           ld_rows, ld_rows_seq, n_rows, index, counts, n_take, max_ctx, (int)units, n_heads_kv)
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
    if (rows_out == 0) {  // (no budget, or caches of no positions)
        if (!lens_out && !kept) return JINF_HIP_OK;
        return launch(kv_none_kernel, dim3(64), dim3(kKvThreads), 0, stream, lens_out, n_seq, kept,
                      kept ? (int64_t)n_seq * n_heads_kv * budget : (int64_t)0);
    }
    int32_t* list = kept ? kept : static_cast<int32_t*>(workspace);
    const int held = max_ctx < kSegMax ? round_up(max_ctx, kSelStep) : kSegMax;
    const int rc = launch(kv_select_kernel, dim3(n_heads_kv, n_seq), dim3(kSelThreads), held * sizeof(uint32_t),
                          stream, weights, ld_w, ld_w_seq, lens, list, kept ? 1 : 0, budget, n_first,
                          n_recent, max_ctx, n_heads_kv);
    if (rc != JINF_HIP_OK) return rc;
    // 16-byte units where everything is aligned to them, else single elements
    const int64_t row = (int64_t)head_dim * es;
    const bool wide = aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(k_out, 16) &&
                      aligned(v_out, 16) && row % 16 == 0 && ld_pos * es % 16 == 0 &&
                      ld_seq * es % 16 == 0 && ld_pos_out * es % 16 == 0 && ld_seq_out * es % 16 == 0;
#define JINF_KV_MOVE(U)                                                                             \
    kv_move<U>(k_out, v_out, ld_pos_out, ld_seq_out, k_cache, v_cache, ld_pos, ld_seq,                 \
               weights_out, ld_wo, ld_wo_seq, weights, ld_w, ld_w_seq, lens, lens_out, list, budget, max_ctx, \
               n_seq, n_heads_kv, row, es, stream)
    return wide ? JINF_KV_MOVE(u32x4) : es == 2 ? JINF_KV_MOVE(uint16_t) : JINF_KV_MOVE(uint32_t);
#undef JINF_KV_MOVE
}
