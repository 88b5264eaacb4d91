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
    float* scores;  // null, or the scores wanted: [n_seq][n_kv][blocks][group][16], 16 positions a block
    int64_t blocks;
    int draft_f16;
    // Contexts in chunks of `chunk` positions, nch of them at most, the first of which also
    // takes the drafted tokens; each chunk of a row (s, j, r) has a record of partial sums
    // part[rec][head_dim] and {m, l} stats[rec] (TreeRecords).
    int chunk, nch;
    float* part;
    float2* stats;
    // Or, planned: chunks of `chunk` positions at least that the kernel divides itself
    // (tree_share) into nch places per kv head, each a row tile's chunk and 2^planned
    // records; a sequence's places follow each other, row tiles fastest.  It stores
    // {first place, chunks, row tiles} of each of the n_seq sequences in front of part.
    int n_seq, planned;
    __device__ __forceinline__ int4* plan() const { return reinterpret_cast<int4*>(part) - n_seq; }
};

// Where the records of a kv head's rows are: row r's first at at(r), `step` apart.
struct TreeRecords {
    int64_t first;
    int step, chunks, row_step, log;  // log: of the rows in a place
    __device__ __forceinline__ int64_t at(int r) const {
        return log < 0 ? first + (int64_t)r * row_step
                       : first + ((int64_t)(r >> log) << log) + (r & ((1 << log) - 1));
    }
};
__device__ __forceinline__ TreeRecords tree_records(const TreeArgs& a, int s, int j, int len) {
    if (a.planned) {
        const int4 p = a.plan()[s];
        return {((int64_t)j * a.nch + p.x) << a.planned, p.z << a.planned, p.y, 1, a.planned};
    }
    return {((int64_t)s * a.n_kv + j) * a.max_nodes * a.group * a.nch, 1, max(1, (len + a.chunk - 1) / a.chunk),
            a.nch, -1};
}

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
        if (a.scores && lane == 0)
            a.scores[((((int64_t)s * a.n_kv + j) * a.blocks + (t >> 4)) * a.group + h % a.group) * 16 + (t & 15)] = st;
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
    if (a.stats && lane == 0) a.stats[(int64_t)s * a.n_heads + h] = make_float2(m, l);
}

// ---- head_dim 64 and 128: matrix cores ----
//
// Per tile of positions, with the rows (node, head) of one kv head as columns:
//   S^T[t][r]  = sum_d K[t][d] Q'[d][r]       Q' = c q
//   O^T[d][r] += sum_t V^T[d][t] P'^T[t][r]   P' = 2^11 2^(S - m)
// Both products leave row r in lane r % 16 of every lane group, so the running
// maximum, the sum and the rescaling of O are one value a lane, and the scores'
// accumulators are the second product's operand as they stand.  The 2^11 keeps
// the probabilities of an fp16 product in its normal range; the sum l carries it
// too, so it cancels.
//   fp16 cache: v_mfma_f32_16x16x32_f16, Q' and P' as fp16 hi + lo in two products
//   into one accumulator (about 22 bits); V^T through transposing LDS reads.
//   fp32 cache: v_mfma_f32_16x16x4_f32, exact products.
//
// What bounds it: the K and V bytes while a kv head has few rows, the matrix
// cores and the softmax's vector work from about 64 rows on.  A workgroup's 4
// waves therefore share out rows and positions: RW waves take 16 R rows each,
// and 4 / RW groups of them the positions of a tile; every wave reads a tile's K
// and V from LDS once for its 16 R rows.
typedef _Float16 tr_h4 __attribute__((ext_vector_type(4)));
typedef _Float16 tr_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 tr_h2 __attribute__((ext_vector_type(2)));
typedef float tr_f2 __attribute__((ext_vector_type(2)));
typedef float tr_f4 __attribute__((ext_vector_type(4)));
typedef float tr_f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef short tr_s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) tr_s4 tr_lds_s4;

// Probabilities count 2^kTreeUnit in O and l.  A reference that lags the maximum by up
// to kTreeSlack keeps them below 2^15; the least that an fp16 hi + lo pair resolves,
// 2^-25, is then 2^-36 of the reference's.  (Following every new maximum cost 40
// vector operations in a quarter of the steps.)
constexpr float kTreeUnit = 11.0f, kTreeSlack = 4.0f;

__device__ __forceinline__ tr_h8 tr_cat(tr_h4 a, tr_h4 b) {
    return tr_h8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// x as fp16 hi and lo parts, four at a time.
// Of products: the conversion is kept apart from the multiply (f2h2), which the
// compiler otherwise merges into one instruction of another rounding for hi, but
// not for the hi that lo is the rest of.
__device__ __forceinline__ void tr_split_product(const float (&x)[4], tr_h4& hi, tr_h4& lo) {
    hi = __builtin_bit_cast(tr_h4, make_uint2(f2h2(x[0], x[1]), f2h2(x[2], x[3])));
    lo = __builtin_bit_cast(tr_h4, make_uint2(f2h2(x[0] - (float)hi[0], x[1] - (float)hi[1]),
                                              f2h2(x[2] - (float)hi[2], x[3] - (float)hi[3])));
}
// Of exponentials: plain conversions, since an instruction in inline assembly must
// not read v_exp's result without the wait that the compiler places for its own.
// minus_one is opaque to the compiler, so that the rest is one mixed-precision FMA.
__device__ __forceinline__ void tr_split_exp(const float (&x)[4], float minus_one, tr_h4& hi, tr_h4& lo) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const tr_h2 h = __builtin_convertvector((tr_f2{x[i], x[i + 1]}), tr_h2);
        const tr_f2 rest = {fmaf((float)h[0], minus_one, x[i]), fmaf((float)h[1], minus_one, x[i + 1])};
        const tr_h2 l = __builtin_convertvector(rest, tr_h2);
        hi[i] = h[0], hi[i + 1] = h[1];
        lo[i] = l[0], lo[i + 1] = l[1];
    }
}

template <typename TC, int HD, int R_, int RW_, bool ONCE>
struct TreeShape {
    static constexpr bool F16 = sizeof(TC) == 2;
    static constexpr int R = R_, RW = RW_, PW = 4 / RW_;
    static constexpr int ROWS = 16 * R * RW;               // rows per workgroup
    static constexpr int PITCH = HD * (int)sizeof(TC);     // LDS bytes per row
    // Positions per tile: 32 KiB of K and V, or 16 positions a wave where that is more.
    static constexpr int FIT = 16384 / PITCH, LEAST = 16 * PW;
    static constexpr int ST = RW == 4 ? (FIT < 64 ? FIT : 64) : FIT > LEAST ? FIT : LEAST;
    static constexpr int TP = ST / PW;                     // of them, a wave's
    static constexpr int SP = TP < 32 ? TP : 32;           // and those of one softmax step
    static constexpr int CH = PITCH / 16;                  // 16-byte pieces per row
    static constexpr int LD = ST * CH / 256;               // loads per lane per tile (K or V)
    static constexpr int BUF = 2 * ST * PITCH;             // K tile, V tile
    // Tiles in LDS, NS - 1 of them on their way.  Two workgroups a CU with two tiles each,
    // but one with four where few rows stream caches of many megabytes (64 sequences x
    // 8192 with scores: 353 against 389 us; 6 fp32 sequences x 3001: 29.6 against 19.5).
    static constexpr int NS = ONCE && RW == 1 && BUF <= 32768 ? 4 : 2;
    static constexpr int MERGE = PW > 1 ? PW * ROWS * (HD + 4) * 4 : 0;
    static constexpr int LDS = NS * BUF > MERGE ? NS * BUF : MERGE;
    static constexpr int WGS = 2 * LDS <= 159 * 1024 ? 2 : 1;  // workgroups per CU
};

// LDS place of a row's 16-byte piece c.  K: the 16 rows that a fragment read
// touches at one piece lie in distinct banks; V: so do the rows of a lane group's
// transposing read (fp16), and the rows 4 apart of a wave's read (fp32).
template <typename TC, int HD>
__device__ __forceinline__ int tree_k_at(int r, int c) {
    return c ^ (sizeof(TC) == 2 && HD == 64 ? (r >> 1) & 7 : r & 15);
}
template <typename TC>
__device__ __forceinline__ int tree_v_at(int r, int c) {
    return c ^ (sizeof(TC) == 2 ? 2 * (r & 3) : 4 * ((r >> 2) & 3));
}

// Equal shares of ragged work, one lane a sequence (at most 64): the sequences' chunks,
// of at most a common length, so that their row tiles' chunks fill the places.
// Drafted tokens count as positions in front of a context.  The host knows neither
// lengths nor node counts: chunks of the longest context possible leave workgroups
// without work and the others with too much (4 sequences x 64 nodes, 16384 to 32768
// positions: 403 -> 358 us; 64 x 1 with scores, 4096 to 8192: 373 -> 349).  Every
// workgroup comes to the same division at its start, about a microsecond.
struct TreeShare {
    int s, tile, cix, chunks, tiles, first, chunk, ahead;  // chunk: positions, of which `ahead` before the context
};
template <int ROWS, bool SCORE>
__device__ __forceinline__ bool tree_share(const TreeArgs& a, int place, TreeShare& w) {
    const int lane = threadIdx.x & (kWave - 1);
    const int at = min(lane, a.n_seq - 1);
    const int held = a.lens[at], given = a.n_nodes ? a.n_nodes[at] : a.max_nodes;
    const int len = min(max(held, 0), a.max_ctx);
    const int nodes = lane < a.n_seq ? min(max(given, 0), a.max_nodes) : 0;
    const int tiles = (nodes * a.group + ROWS - 1) / ROWS;
    // in blocks of 64 positions, at least one
    const int ahead = SCORE ? 0 : (nodes + 63) / 64;
    const int v = max((len + 63) / 64 + ahead, 1);
    // (guesses may round; the counts compared are whole numbers below 2^24)
    const float all = wave_sum_f32((float)tiles * (float)v), least = wave_sum_f32((float)tiles);
    int most = tiles ? v : 0;
#pragma unroll
    for (int o = 1; o < kWave; o *= 2) most = max(most, __shfl_xor(most, o, kWave));
    int c = max((int)ceilf(all / ((float)a.nch - 0.5f * least)), a.chunk / 64);
    int n;
    for (;;) {
        n = (v + c - 1) / c;
        // (one chunk each fits: the host counted places for the most row tiles)
        if (c >= most || wave_sum_f32((float)(tiles * n)) <= (float)a.nch) break;
        c += (c + 15) / 16;
    }
    const int chunk = (v + n - 1) / n;
    n = (v + chunk - 1) / chunk;
    int upto = tiles * n;  // places of the sequences before and this one
#pragma unroll
    for (int o = 1; o < kWave; o *= 2) {
        const int y = __shfl_up(upto, o, kWave);
        if (lane >= o) upto += y;
    }
    const int s = __popcll(__ballot(upto <= place));
    if (s >= a.n_seq) return false;
    w.s = s;
    w.chunks = __builtin_amdgcn_readlane(n, s);
    w.tiles = __builtin_amdgcn_readlane(tiles, s);
    w.first = __builtin_amdgcn_readlane(upto, s) - w.chunks * w.tiles;
    w.chunk = __builtin_amdgcn_readlane(chunk, s) * 64;
    w.ahead = __builtin_amdgcn_readlane(ahead, s) * 64;
    w.cix = (place - w.first) / w.tiles;
    w.tile = (place - w.first) % w.tiles;
    return true;
}

// grid (row tiles * n_kv, n_seq, chunks), or (n_kv, places) where the kernel divides the
// work (PLAN), 256 threads; the kv head is the fastest index, so that row tiles of one
// head, which read the same K and V, lie n_kv apart (on one XCD for 8 kv heads).  Heads, row tiles and sequences turn with the
// slower indices: workgroups go to XCDs, and in one of them to its 4 shader engines,
// by their number in the grid, so that otherwise an XCD reads one head's addresses
// alone (64 sequences x 8192, loads only: 335 -> 325 us) and the last, partly filled
// row tile of every sequence falls to the same shader engine (4 tiles: CUs busy 73% of
// the time).
// SCORE: one node a sequence, no drafted tokens, and the scores kept.
// ONCE: the caches are read once and are larger than what the Infinity Cache keeps.
template <typename TC, int HD, int R, int RW, bool SCORE, bool ONCE, bool PLAN>
__global__ __launch_bounds__(256, (TreeShape<TC, HD, R, RW, ONCE>::WGS)) void tree_mfma_kernel(TreeArgs a) {
    using Sh = TreeShape<TC, HD, R, RW, ONCE>;
    constexpr bool F16 = Sh::F16;
    constexpr int PW = Sh::PW, ST = Sh::ST, TP = Sh::TP, PITCH = Sh::PITCH, CH = Sh::CH, LD = Sh::LD;
    constexpr int NS = Sh::NS;
    constexpr int SP = Sh::SP;
    constexpr int NBK = SP / 16;   // 16-position blocks of a softmax step
    constexpr int NB = HD / 16;    // 16-dim blocks of the output
    constexpr int QV = F16 ? HD / 32 : HD / 4;  // q registers: h8 (hi and lo each) or floats
    extern __shared__ __attribute__((aligned(16))) uint8_t tree_lds[];
    __shared__ unsigned s_bad[4];  // drafted rows of the tile whose V has a non-finite value
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid & (kWave - 1);
    const int col = lane & 15, lg = lane >> 4;
    const int pw = wave / RW, rw = wave % RW;
    TreeShare w;
    if constexpr (PLAN) {
        if (!tree_share<Sh::ROWS, SCORE>(a, blockIdx.y, w)) return;
    } else {
        w.cix = blockIdx.z, w.s = (blockIdx.y + w.cix) % gridDim.y;
        w.tile = (blockIdx.x / a.n_kv + blockIdx.y + w.cix) % (gridDim.x / a.n_kv);
        w.chunk = a.chunk, w.ahead = 0;
    }
    const int s = w.s, cix = w.cix, tile = w.tile;
    const int j = (blockIdx.x + (PLAN ? s : blockIdx.y) + cix) % a.n_kv;
    const int len = min(max(a.lens[s], 0), a.max_ctx);
    if constexpr (!PLAN) w.chunks = max(1, (len + w.chunk - 1) / w.chunk);
    const int nodes = a.n_nodes ? min(max(a.n_nodes[s], 0), a.max_nodes) : a.max_nodes;
    const int rows = nodes * a.group, all_rows = a.max_nodes * a.group;
    const int row0 = tile * Sh::ROWS;
    // The lane's rows and their q.  (q's loads need neither lengths nor node counts,
    // and are used up before the tiles' loads: a wait for them is a wait for nothing else.)
    int node[R], head[R];
#pragma unroll
    for (int g = 0; g < R; ++g) {
        const int r = row0 + (rw * R + g) * 16 + col;
        node[g] = r < all_rows ? r / a.group : 0;
        head[g] = j * a.group + (r < all_rows ? r - node[g] * a.group : 0);
    }
    tr_h8 qh[R][F16 ? QV : 1], ql[R][F16 ? QV : 1];
    float qf[R][F16 ? 1 : QV];
#pragma unroll
    for (int g = 0; g < R; ++g) {
        const float* qp = a.q + (int64_t)s * a.ld_q_seq + (int64_t)node[g] * a.ld_q + (int64_t)head[g] * HD;
        if constexpr (F16) {
            // 32-deep k-step u: lane group lg holds dims HD / 4 lg + 8 u .. + 7, the
            // 16-byte piece HD / 32 lg + u of the K row
#pragma unroll
            for (int u = 0; u < QV; ++u) {
                tr_h4 hi[2], lo[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float4 v = *reinterpret_cast<const float4*>(qp + HD / 4 * lg + 8 * u + 4 * e);
                    const float x[4] = {v.x * a.c, v.y * a.c, v.z * a.c, v.w * a.c};
                    tr_split_product(x, hi[e], lo[e]);
                }
                qh[g][u] = tr_cat(hi[0], hi[1]);
                ql[g][u] = tr_cat(lo[0], lo[1]);
            }
        } else {
            // 4-deep k-step 4 u + i: lane group lg holds dim 16 u + 4 lg + i, element i
            // of the K row's 16-byte piece 4 u + lg
#pragma unroll
            for (int u = 0; u < HD / 16; ++u) {
                const float4 v = *reinterpret_cast<const float4*>(qp + 16 * u + 4 * lg);
                qf[g][4 * u] = v.x * a.c, qf[g][4 * u + 1] = v.y * a.c;
                qf[g][4 * u + 2] = v.z * a.c, qf[g][4 * u + 3] = v.w * a.c;
            }
        }
    }
    // (used up here, not further down)
#pragma unroll
    for (int g = 0; g < R; ++g)
#pragma unroll
        for (int u = 0; u < QV; ++u) {
            if constexpr (F16) asm volatile("" : "+v"(qh[g][u]), "+v"(ql[g][u]));
            else asm volatile("" : "+v"(qf[g][u]));
        }

    const int c0 = max(cix * w.chunk - w.ahead, 0), c1 = min(len, (cix + 1) * w.chunk - w.ahead);
    if (row0 >= rows || cix >= w.chunks) return;  // (workgroup-uniform, before any barrier)
    if (PLAN && tile == 0 && cix == 0 && j == 0 && tid == 0)
        a.plan()[s] = make_int4(w.first, w.chunks, w.tiles, 0);
    bool live[R];
#pragma unroll
    for (int g = 0; g < R; ++g) live[g] = row0 + (rw * R + g) * 16 + col < rows;
    const bool idle = row0 + rw * R * 16 >= rows;  // none of the wave's rows is live
    const int drafts = !SCORE && cix == 0 ? nodes : 0;
    const int n_dt = (drafts + ST - 1) / ST;
    const int n_it = n_dt + (max(c1 - c0, 0) + ST - 1) / ST;

    // The scores of one kv head's positions p0 .. lie together, block by block.
    auto scores_at = [&](int p0) {
        return a.scores + (((int64_t)s * a.n_kv + j) * a.blocks + (p0 >> 4)) * a.group * 16;
    };
    const char* kb = reinterpret_cast<const char*>(static_cast<const TC*>(a.kc) + (int64_t)s * a.ld_seq + (int64_t)j * HD);
    const char* vb = reinterpret_cast<const char*>(static_cast<const TC*>(a.vc) + (int64_t)s * a.ld_seq + (int64_t)j * HD);
    const uint32_t rowb = (uint32_t)a.ld_pos * (uint32_t)sizeof(TC);  // (the host keeps ST of them below 2^31)
    uint32_t koff[LD], voff[LD];
#pragma unroll
    for (int i = 0; i < LD; ++i) {
        const int slot = tid + 256 * i, r = slot / CH, p = slot % CH;
        koff[i] = (uint32_t)r * rowb + 16u * (uint32_t)tree_k_at<TC, HD>(r, p);
        voff[i] = (uint32_t)r * rowb + 16u * (uint32_t)tree_v_at<TC>(r, p);
    }
    // Positions t0 .. of the cache straight to LDS; rows at or past c1 read as zeros.
    auto load_cached = [&](int t0, int buf) {
        const int64_t at = (int64_t)t0 * rowb;
        const int nrec = (int)((uint32_t)min(ST, c1 - t0) * rowb);
        const __amdgpu_buffer_rsrc_t krs = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<char*>(kb + at), (short)0, nrec, 0x00020000);
        const __amdgpu_buffer_rsrc_t vrs = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<char*>(vb + at), (short)0, nrec, 0x00020000);
        uint8_t* base = tree_lds + buf * Sh::BUF + 1024 * wave;
        if constexpr (ONCE) {
#pragma unroll
            for (int i = 0; i < LD; ++i) lds_load16_buf_nt(krs, koff[i], 0, base + 4096 * i);
#pragma unroll
            for (int i = 0; i < LD; ++i) lds_load16_buf_nt(vrs, voff[i], 0, base + ST * PITCH + 4096 * i);
            return;
        }
#pragma unroll
        for (int i = 0; i < LD; ++i) lds_load16_buf(krs, koff[i], 0, base + 4096 * i);
#pragma unroll
        for (int i = 0; i < LD; ++i) lds_load16_buf(vrs, voff[i], 0, base + ST * PITCH + 4096 * i);
    };
    // Drafted tokens d0 .. as the cache would hold them; tokens past the sequence's
    // read as zeros, and so do non-finite V values (noted in s_bad, set up by the
    // caller): their probability is 0 in rows that do not see them, their product not.
    constexpr int EL = 16 / (int)sizeof(TC);  // elements per 16-byte piece
    const int64_t dbase = (int64_t)s * a.ld_draft_seq + (int64_t)j * HD;
    // K pieces, then V pieces: all of a lane's loads are under way before the first is used.
    auto load_draft = [&](int d0, int buf) {
        uint8_t* base = tree_lds + buf * Sh::BUF;
#pragma unroll 1
        for (int is_v = 0; is_v < 2; ++is_v) {
            const void* src = is_v ? a.vd : a.kd;
            float e[LD][EL];
#pragma unroll
            for (int i = 0; i < LD; ++i) {
                const int slot = tid + 256 * i, r = slot / CH, p = slot % CH;
                const int c = is_v ? tree_v_at<TC>(r, p) : tree_k_at<TC, HD>(r, p);
                const int64_t at = dbase + (int64_t)min(d0 + r, drafts - 1) * a.ld_draft + (int64_t)c * EL;
                if (a.draft_f16) {
                    typedef _Float16 row_h __attribute__((ext_vector_type(EL), aligned(2)));
                    const row_h h = *reinterpret_cast<const row_h*>(static_cast<const uint16_t*>(src) + at);
#pragma unroll
                    for (int x = 0; x < EL; ++x) e[i][x] = (float)h[x];
                } else {
#pragma unroll
                    for (int x = 0; x < EL; x += 4) {
                        const tr_f4u f = *reinterpret_cast<const tr_f4u*>(static_cast<const float*>(src) + at + x);
#pragma unroll
                        for (int y = 0; y < 4; ++y) e[i][x + y] = f[y];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < LD; ++i) {
                const int slot = tid + 256 * i, r = slot / CH;
                bool bad = false;
#pragma unroll
                for (int x = 0; x < EL; ++x) {
                    // as the cache would hold it: its type's range decides what is finite
                    const float f = F16 ? h2f(f2h(e[i][x])) : e[i][x];
                    const bool nf = !(fabsf(f) < INFINITY);
                    bad |= nf;
                    e[i][x] = (is_v && nf) || d0 + r >= drafts ? 0.0f : f;
                }
                if (is_v && bad && d0 + r < drafts) atomicOr(&s_bad[r >> 5], 1u << (r & 31));
                *reinterpret_cast<uint4*>(base + (is_v ? ST * PITCH : 0) + slot * 16) = Act<TC>::pack(e[i]);
            }
        }
    };

    // Tiles in order: the drafted tokens', then the cached positions'.  NS - 1 tiles
    // are under way; a tile of drafted tokens is read by ordinary loads, so the first
    // one is read after the cached tiles behind it have been asked for.
    auto stage = [&](int it) {
        if (it < n_dt) load_draft(it * ST, it % NS);
        else if (it < n_it) load_cached(c0 + (it - n_dt) * ST, it % NS);
    };
    if (n_dt > 0) {
        if (tid < 4) s_bad[tid] = 0u;
        if (n_dt == 1)
            for (int it = 1; it < NS - 1; ++it) stage(it);
        __syncthreads();  // s_bad
        load_draft(0, 0);
    } else {
        for (int it = 0; it < NS - 1; ++it) stage(it);
    }
    // (more tiles of drafted tokens, one by one as their buffers come free, below)
    const int ahead = n_dt > 1 ? 1 : NS - 1;  // tiles staged before the loop

    float m[R], lsum[R];
    tr_f4 O[R][NB];
    float minus_one;
    asm("s_mov_b32 %0, -1.0" : "=s"(minus_one));
#pragma unroll
    for (int g = 0; g < R; ++g) {
        m[g] = -INFINITY, lsum[g] = 0.0f;
#pragma unroll
        for (int n = 0; n < NB; ++n) O[g][n] = tr_f4{0.f, 0.f, 0.f, 0.f};
    }

    int staged = ahead;
#pragma unroll 1
    for (int it = 0; it < n_it; ++it) {
        const bool draft = it < n_dt;
        const int t0 = draft ? it * ST : c0 + (it - n_dt) * ST;
        const int buf = it % NS;
        // This tile has landed for every wave once at most the loads of the tiles behind
        // it are outstanding (they return in order), and every wave is done with the
        // buffer of the tile before it.
        const int behind = min(staged, n_it) - 1 - it;
        if (NS > 3 && behind >= 2) __builtin_amdgcn_s_waitcnt(waitcnt_vm<(NS > 3 ? 4 : 0) * LD>());
        else if (NS > 2 && behind == 1) __builtin_amdgcn_s_waitcnt(waitcnt_vm<(NS > 2 ? 2 : 0) * LD>());
        else __builtin_amdgcn_s_waitcnt(waitcnt_vm<0>());
        __syncthreads();
        unsigned long long bad = 0;
        if (draft) {
            const int b0 = pw * TP;  // the wave's bits (TP <= 64, within two words)
            bad = (unsigned long long)s_bad[b0 >> 5] | (TP > 32 ? (unsigned long long)s_bad[(b0 >> 5) + 1] << 32 : 0ull);
            if constexpr (TP < 32) bad = (bad >> (b0 & 31)) & ((1ull << TP) - 1);
            __syncthreads();
            if (tid < 4) s_bad[tid] = 0u;
            if (it + 1 < n_dt) __syncthreads();  // (the next tile sets bits)
        }
        // with several tiles of drafted tokens the next one is read now (its bits are
        // looked at before those of the one after it are set), cached tiles NS - 1 ahead
        for (const int to = it + 1 < n_dt ? it + 2 : it + NS; staged < to; ++staged) stage(staged);
        const int end = draft ? drafts : c1;
        if (idle) continue;  // (wave-uniform)
#pragma unroll 1
        for (int sub = pw * TP; sub < (pw + 1) * TP; sub += SP) {
            const int p0 = t0 + sub;    // the step's first position (or drafted token)
            const int left = end - p0;  // live ones from there
            if (left <= 0) break;
            const uint8_t* kst = tree_lds + buf * Sh::BUF + sub * PITCH;
            const uint8_t* vst = kst + ST * PITCH;
            tr_f4 S[R][NBK];
            if constexpr (F16) {
                // the small parts first: half as many roundings at a score's full size (16 x
                // 25 x 4096: error against 64 bits 7.0e-7 -> 5.4e-7, no slower)
#pragma unroll
                for (int lo = 1; lo >= 0; --lo)
#pragma unroll
                    for (int u = 0; u < QV; ++u)
#pragma unroll
                        for (int b = 0; b < NBK; ++b) {
                            const int r = 16 * b + col;
                            const tr_h8 kf = *reinterpret_cast<const tr_h8*>(
                                kst + r * PITCH + 16 * tree_k_at<TC, HD>(r, QV * lg + u));
#pragma unroll
                            for (int g = 0; g < R; ++g)
                                S[g][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                    kf, lo ? ql[g][u] : qh[g][u], lo && u == 0 ? tr_f4{0.f, 0.f, 0.f, 0.f} : S[g][b], 0, 0, 0);
                        }
            } else {
                // a score in NA sums of every NA-th step: each is shorter, and rounds less (6 x
                // 3001: error against 64 bits 8.7e-7 -> 4.1e-7, 18.3 -> 18.6 us)
                constexpr int NA = R == 1 ? 4 : 2;
#pragma unroll
                for (int b = 0; b < NBK; ++b) {
                    const int r = 16 * b + col;
                    tr_f4 A[R][NA];
#pragma unroll
                    for (int u = 0; u < HD / 16; ++u) {
                        const tr_f4 kf = *reinterpret_cast<const tr_f4*>(
                            kst + r * PITCH + 16 * tree_k_at<TC, HD>(r, 4 * u + lg));
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int g = 0; g < R; ++g)
                                A[g][i % NA] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                    kf[i], qf[g][4 * u + i],
                                    u || i >= NA ? A[g][i % NA] : tr_f4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                    }
#pragma unroll
                    for (int g = 0; g < R; ++g) {
                        S[g][b] = A[g][0] + A[g][1];
                        if constexpr (NA == 4) S[g][b] += A[g][2] + A[g][3];
                    }
                }
            }
            if (draft) {
                // bit 16 b + 4 lg + r: the lane's row sees drafted token p0 + 16 b + 4 lg + r
#pragma unroll
                for (int g = 0; g < R; ++g) {
                    unsigned bits = 0;
                    if (live[g])
                        bits = (unsigned)(a.mask[((int64_t)s * a.max_nodes + node[g]) * a.words + (p0 >> 6)] >> (p0 & 63));
                    if (left < 32) bits &= (1u << left) - 1;
                    bits >>= 4 * lg;
#pragma unroll
                    for (int b = 0; b < NBK; ++b)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (!((bits >> (16 * b + r)) & 1)) S[g][b][r] = -INFINITY;
                }
            } else {
                if (left < SP) {
#pragma unroll
                    for (int g = 0; g < R; ++g)
#pragma unroll
                        for (int b = 0; b < NBK; ++b)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (16 * b + 4 * lg + r >= left) S[g][b][r] = -INFINITY;
                }
                if constexpr (SCORE) {
                    // (Their 100 MB beside 1.6 GB read cost 64 x 8192 positions 40 us with loads past
                    // the Infinity Cache, whichever wave stores them and in whatever bursts.)
                    float* to = scores_at(p0);
#pragma unroll
                    for (int g = 0; g < R; ++g)
#pragma unroll
                        for (int b = 0; b < NBK; ++b)
                            if (live[g] && 16 * b < left)
                                *reinterpret_cast<tr_f4*>(to + (b * a.group + head[g] - j * a.group) * 16 + 4 * lg) = S[g][b];
                }
            }
            tr_h4 ph[R][F16 ? NBK : 1], pl[R][F16 ? NBK : 1];
#pragma unroll
            for (int g = 0; g < R; ++g) {
                float tmax = S[g][0][0];
#pragma unroll
                for (int b = 0; b < NBK; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r) tmax = fmaxf(tmax, S[g][b][r]);
                // The reference m follows the maximum only when it falls behind by more than
                // kTreeSlack (probabilities then stay below 2^15): some row's sums scale down.
                if (__ballot(tmax > m[g] + kTreeSlack)) {
                    tmax = fmaxf(tmax, __shfl_xor(tmax, 16, kWave));
                    tmax = xor32_max(tmax);
                    const float mn = fmaxf(m[g], tmax);
                    const float corr = tree_exp2(m[g] - softmax_ref(mn));
                    m[g] = mn;
                    lsum[g] *= corr;
#pragma unroll
                    for (int n = 0; n < NB; ++n) O[g][n] *= corr;
                }
                const float ref = softmax_ref(m[g]) - kTreeUnit;
                float psum;
#pragma unroll
                for (int b = 0; b < NBK; ++b) {
                    float x[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        x[r] = tree_exp2(S[g][b][r] - ref);
                        psum = b || r ? psum + x[r] : x[r];
                    }
                    if constexpr (F16) tr_split_exp(x, minus_one, ph[g][b], pl[g][b]);
                    else S[g][b] = tr_f4{x[0], x[1], x[2], x[3]};
                }
                lsum[g] += psum;
            }
            if constexpr (F16) {
                // V^T[16 n + col][16 b + 4 lg + i], i = 0..3, in one transposing read
                auto vfrag = [&](int b, int n) {
                    const int vr = 16 * b + 4 * lg + (col >> 2);
                    const int p = tree_v_at<TC>(vr, 2 * n + ((col & 3) >> 1));
                    return __builtin_bit_cast(tr_h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                         (tr_lds_s4*)(vst + vr * PITCH + 16 * p + 8 * (col & 1))));
                };
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    if constexpr (NBK == 1) {
                        const tr_h4 v = vfrag(0, n);
#pragma unroll
                        for (int g = 0; g < R; ++g) {
                            O[g][n] = __builtin_amdgcn_mfma_f32_16x16x16f16(v, ph[g][0], O[g][n], 0, 0, 0);
                            O[g][n] = __builtin_amdgcn_mfma_f32_16x16x16f16(v, pl[g][0], O[g][n], 0, 0, 0);
                        }
                    } else {
                        const tr_h8 v = tr_cat(vfrag(0, n), vfrag(1, n));
#pragma unroll
                        for (int g = 0; g < R; ++g) {
                            O[g][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, tr_cat(ph[g][0], ph[g][1]), O[g][n], 0, 0, 0);
                            O[g][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, tr_cat(pl[g][0], pl[g][1]), O[g][n], 0, 0, 0);
                        }
                    }
                }
            } else {
                // k-step r: lane group lg holds position 16 b + 4 lg + r
#pragma unroll
                for (int b = 0; b < NBK; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int vr = 16 * b + 4 * lg + r;
#pragma unroll
                        for (int n = 0; n < NB; ++n) {
                            const float v = *reinterpret_cast<const float*>(
                                vst + vr * PITCH + 16 * tree_v_at<TC>(vr, 4 * n + (col >> 2)) + 4 * (col & 3));
#pragma unroll
                            for (int g = 0; g < R; ++g)
                                O[g][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, S[g][b][r], O[g][n], 0, 0, 0);
                        }
                    }
            }
            // non-finite V values: NaN in their dims of the rows that see them
            unsigned step_bad = (unsigned)(bad >> (sub - pw * TP));
            if constexpr (SP < 32) step_bad &= (1u << SP) - 1;
#pragma unroll 1
            for (; step_bad; step_bad &= step_bad - 1) {
                const int d = p0 + __builtin_ctz(step_bad);
                const int64_t at = dbase + (int64_t)d * a.ld_draft;
#pragma unroll
                for (int g = 0; g < R; ++g) {
                    if (!live[g] || !((a.mask[((int64_t)s * a.max_nodes + node[g]) * a.words + (d >> 6)] >> (d & 63)) & 1))
                        continue;
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (!(fabsf(tree_draft<TC>(a.vd, a.draft_f16, at + 16 * n + 4 * lg + r)) < INFINITY))
                                O[g][n][r] = NAN;
                }
            }
        }
    }
#pragma unroll
    for (int g = 0; g < R; ++g) {
        lsum[g] += __shfl_xor(lsum[g], 16, kWave);
        lsum[g] = xor32_sum(lsum[g]);
    }
    const bool direct = w.chunks <= 1;
    // Whether a node sees nothing at all: its outputs are zeros.  (A node whose
    // scores are all -inf has no sum either, and gets NaN.)
    auto sees_none = [&](int nd) {
        if (len > 0) return false;
        uint64_t any = 0;
        for (int w = 0; 64 * w < drafts; ++w) {
            const uint64_t x = a.mask[((int64_t)s * a.max_nodes + nd) * a.words + w];
            any |= drafts - 64 * w < 64 ? x & ((1ull << (drafts - 64 * w)) - 1) : x;
        }
        return any == 0;
    };
    // row r's record of this chunk (TreeRecords)
    const int64_t rec0 = PLAN ? ((int64_t)j * a.nch + w.first + cix * w.tiles + tile) * Sh::ROWS - row0
                              : ((int64_t)s * a.n_kv + j) * all_rows;
    auto rec = [&](int r) { return PLAN ? rec0 + r : (rec0 + r) * a.nch + cix; };
    auto put = [&](int r, int nd, int hh, int d, tr_f4 o, float M, float L) {
        if (direct) {
            float* p = a.out + (int64_t)s * a.ld_out_seq + (int64_t)nd * a.ld_out + (int64_t)hh * HD + d;
            const bool none = L == 0.0f && sees_none(nd);
            *reinterpret_cast<tr_f4u*>(p) = none ? tr_f4{0.f, 0.f, 0.f, 0.f} : o / L;
        } else {
            *reinterpret_cast<tr_f4*>(a.part + rec(r) * HD + d) = o;
        }
        if (d == 0 && a.stats) a.stats[rec(r)] = make_float2(M, L);
    };
    if constexpr (PW == 1) {
#pragma unroll
        for (int g = 0; g < R; ++g) {
            if (!live[g]) continue;
#pragma unroll
            for (int n = 0; n < NB; ++n)
                put(row0 + (rw * R + g) * 16 + col, node[g], head[g], 16 * n + 4 * lg, O[g][n], m[g], lsum[g]);
        }
    } else {
        // the position groups' states through LDS, merged in their order
        constexpr int MS = HD + 4;
        float* mg = reinterpret_cast<float*>(tree_lds);
        __syncthreads();
#pragma unroll
        for (int g = 0; g < R; ++g) {
            float* e = mg + (pw * Sh::ROWS + (rw * R + g) * 16 + col) * MS;
#pragma unroll
            for (int n = 0; n < NB; ++n) *reinterpret_cast<tr_f4*>(e + 16 * n + 4 * lg) = O[g][n];
            if (lg == 0) e[HD] = m[g], e[HD + 1] = lsum[g];
        }
        __syncthreads();
        for (int x = tid; x < Sh::ROWS * (HD / 4); x += 256) {
            const int rl = x / (HD / 4), d = x % (HD / 4) * 4;
            const int r = row0 + rl;
            if (r >= rows) break;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < PW; ++w) M = fmaxf(M, mg[(w * Sh::ROWS + rl) * MS + HD]);
            const float ref = softmax_ref(M);
            tr_f4 o = {0.f, 0.f, 0.f, 0.f};
            float L = 0.0f;
#pragma unroll
            for (int w = 0; w < PW; ++w) {
                const float* e = mg + (w * Sh::ROWS + rl) * MS;
                const float f = tree_exp2(e[HD] - ref);
                L = fmaf(f, e[HD + 1], L);
                o += f * *reinterpret_cast<const tr_f4*>(e + d);
            }
            const int nd = r / a.group;
            put(r, nd, j * a.group + r - nd * a.group, d, o, M, L);
        }
    }
}

// The chunks' partial sums of every row whose context has more than one, in chunk
// order: grid (ceil(rows n_kv / RB), n_seq), HD / 4 lanes a row.
template <int HD>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a) {
    constexpr int LPR = HD / 4, RB = 256 / LPR;
    const int s = blockIdx.y, all_rows = a.max_nodes * a.group;
    // (no plan is stored for a sequence without nodes)
    const int len = min(max(a.lens[s], 0), a.max_ctx);
    const int nodes = a.n_nodes ? min(max(a.n_nodes[s], 0), a.max_nodes) : a.max_nodes;
    const int x = blockIdx.x * RB + threadIdx.x / LPR, d = threadIdx.x % LPR * 4;
    const int j = x / all_rows, r = x % all_rows;
    if (j >= a.n_kv || r >= nodes * a.group) return;
    const TreeRecords recs = tree_records(a, s, j, len);
    if (recs.chunks <= 1) return;
    const int64_t at = recs.at(r);
    const int step = recs.step;  // (all of a row's records lie within 2^18)
    // a row's lanes share its chunks' {m, l} (one after the other: 6.5 us for 5 x 13 nodes
    // x 12 chunks, 4.7 here)
    const float2* st = a.stats + at;
    const float* part = a.part + at * HD + d;
    const int l = threadIdx.x % LPR;
    float M = -INFINITY, L = 0.0f;
    for (int c = l; c < recs.chunks; c += LPR) M = fmaxf(M, st[c * step].x);
#pragma unroll
    for (int o = 1; o < LPR; o *= 2) M = fmaxf(M, __shfl_xor(M, o, kWave));
    const float ref = softmax_ref(M);
    for (int c = l; c < recs.chunks; c += LPR) {
        const float2 ml = st[c * step];
        L = fmaf(tree_exp2(ml.x - ref), ml.y, L);
    }
#pragma unroll
    for (int o = 1; o < LPR; o *= 2) L += __shfl_xor(L, o, kWave);
    tr_f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int c = 0; c < recs.chunks; ++c)
        o += tree_exp2(st[c * step].x - ref) * *reinterpret_cast<const tr_f4*>(part + c * step * HD);
    const int nd = r / a.group;
    float* p = a.out + (int64_t)s * a.ld_out_seq + (int64_t)nd * a.ld_out +
               (int64_t)(j * a.group + r - nd * a.group) * HD + d;
    *reinterpret_cast<tr_f4u*>(p) = o / L;
}

// The scored decode's end: weights[s, j, t] += sum over the group's heads of
// 2^(score - m) / l, from the scores and the chunks' (m, l), and the chunks' partial
// sums into out where a context has more than one.  grid (ceil(max_ctx / 1024), and one
// more where contexts are split, n_kv, n_seq); that last workgroup of each (sequence,
// kv head) joins the outputs.
// unit: what a probability of 1 counts in l.
constexpr int kWtHeads = 16;  // heads whose {reference, unit / l} are held at a time, 16 lanes each
__global__ __launch_bounds__(256) void tree_finish_kernel(float* __restrict__ weights, int64_t ld_w,
                                                          int64_t ld_w_seq, TreeArgs a, float unit) {
    __shared__ float2 ml[kWtHeads];
    const int tid = threadIdx.x, j = blockIdx.y, s = blockIdx.z;
    const int len = min(max(a.lens[s], 0), a.max_ctx);
    const int t0 = blockIdx.x * 1024;
    const TreeRecords recs = tree_records(a, s, j, len);
    const int used = recs.chunks;
    const int step = recs.step;
    if (a.part && blockIdx.x == gridDim.x - 1) {
        if (used <= 1) return;
        const int hd = a.head_dim;
        for (int x = 4 * tid; x < a.group * hd; x += 1024) {
            const int g = x / hd, d = x % hd;
            const float2* st = a.stats + recs.at(g);
            float M = -INFINITY;
#pragma unroll 4
            for (int c = 0; c < used; ++c) M = fmaxf(M, st[c * step].x);
            const float ref = softmax_ref(M);
            const float* part = a.part + recs.at(g) * hd + d;
            tr_f4 o = {0.f, 0.f, 0.f, 0.f};
            float L = 0.0f;
#pragma unroll 4
            for (int c = 0; c < used; ++c) {
                const float2 x2 = st[c * step];
                const float f = tree_exp2(x2.x - ref);
                L = fmaf(f, x2.y, L);
                o += f * *reinterpret_cast<const tr_f4*>(part + c * step * hd);
            }
            *reinterpret_cast<tr_f4u*>(a.out + (int64_t)s * a.ld_out_seq + ((int64_t)j * a.group + g) * hd + d) = o / L;
        }
        return;
    }
    if (t0 >= len) return;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    const int t = t0 + 4 * tid;
    for (int g0 = 0; g0 < a.group; g0 += kWtHeads) {
        const int n = min(kWtHeads, a.group - g0);
        // a head's lanes share its chunks
        const int g = tid >> 4, l = tid & 15;
        if (g < n) {
            const float2* st = a.stats + recs.at(g0 + g);
            float M = -INFINITY, L = 0.0f;
            for (int c = l; c < used; c += 16) M = fmaxf(M, st[c * step].x);
#pragma unroll
            for (int o = 1; o < 16; o *= 2) M = fmaxf(M, __shfl_xor(M, o, kWave));
            const float ref = softmax_ref(M);
            for (int c = l; c < used; c += 16) {
                const float2 x = st[c * step];
                L = fmaf(tree_exp2(x.x - ref), x.y, L);
            }
#pragma unroll
            for (int o = 1; o < 16; o *= 2) L += __shfl_xor(L, o, kWave);
            if (l == 0) ml[g] = make_float2(ref, unit / L);
        }
        __syncthreads();
        if (t < len) {
            const float* sc = a.scores + ((((int64_t)s * a.n_kv + j) * a.blocks + (t >> 4)) * a.group + g0) * 16 + (t & 15);
#pragma unroll 4
            for (int i = 0; i < n; ++i) {
                const tr_f4 x = *reinterpret_cast<const tr_f4*>(sc + 16 * i);
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] = fmaf(tree_exp2(x[e] - ml[i].x), ml[i].y, sum[e]);
            }
        }
        __syncthreads();
    }
    float* w = weights + (int64_t)s * ld_w_seq + (int64_t)j * ld_w + t;
    if (t + 4 <= len) {
        *reinterpret_cast<tr_f4u*>(w) = *reinterpret_cast<const tr_f4u*>(w) + tr_f4{sum[0], sum[1], sum[2], sum[3]};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (t + e < len) w[e] += sum[e];
    }
}

constexpr float kLog2e = 1.44269502162933349609375f;

// 16-position blocks that hold a context's scores
int64_t score_blocks(int max_ctx) { return ((int64_t)max_ctx + 15) / 16; }

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

// Rows a workgroup takes, by how many a kv head has: no more than there are to 16,
// 32 or 64, its waves then sharing out the positions; 128 beyond.
int tree_wg_rows(int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }

constexpr int kTreeItems = 512;     // workgroups that splits aim for, at most
constexpr int kTreeChunkMin = 128;  // positions per chunk, at least

// Fewest positions per chunk: twice a workgroup's rows, so that the K and V bytes of
// an fp16 chunk are at least twice those of its partial sums.  (4 times: 5 sequences
// x 13 nodes x 1999 fp32 positions 32.2 against 29.9 us.  256 positions at least: 7
// nodes x 333 positions 17.5 against 15.6 us.)
int tree_chunk_min(int wg_rows) { return wg_rows * 2 > kTreeChunkMin ? wg_rows * 2 : kTreeChunkMin; }

// Caches that hold more than this are not expected in the Infinity Cache (256 MB) when
// they are read again; where no two workgroups read the same rows either, K and V are
// loaded past it, which leaves it to the scores and partial sums (64 sequences x 8192
// positions with scores 396 -> 367 us).
constexpr int64_t kTreeOnceBytes = (int64_t)128 << 20;
bool tree_once(const TreeArgs& a, int kv_type, int n_seq) {
    const int64_t es = kv_type == JINF_HIP_F16 ? 2 : 4;
    return (int64_t)a.max_nodes * a.group <= 128 && a.ld_seq != 0 &&
           (int64_t)n_seq * a.max_ctx * a.n_kv * a.head_dim * es * 2 > kTreeOnceBytes;
}

// Chunks per context: as many as make kTreeItems workgroups, what the chip holds at
// once (more add their own starts and ends: 16 x 25 x 4096 70 us, 78 at twice as many;
// 4 x 64 x 32768 in even chunks 419 either way).  Four times as many where few rows stream large
// caches, whose ragged ends then even out (64 x 8192 with scores 418 -> 389 us).
constexpr int kTreeMany = 4 * kTreeItems;
int64_t tree_chunks(int64_t base, int wg_rows, bool stream_large, int max_ctx) {
    const int cmin = tree_chunk_min(wg_rows);
    const int64_t n = (stream_large ? kTreeMany : kTreeItems) / base;
    const int64_t most = (max_ctx + cmin - 1) / cmin;
    return n < most ? n : most;
}

// Records of partial sums that calls of up to these sizes need.
int64_t tree_part_rows(int n_seq, int max_nodes, int n_heads, int n_heads_kv, int max_ctx) {
    const int64_t rows = (int64_t)max_nodes * (n_heads / n_heads_kv);
    const int wr = tree_wg_rows(rows);
    const int64_t few = (int64_t)kTreeItems * wr, narrow = (int64_t)kTreeMany * (wr < 32 ? wr : 32);
    const int64_t a = few > narrow ? few : narrow;
    const int64_t b = (int64_t)n_seq * n_heads_kv * ((rows + wr - 1) / wr) * wr *
                      ((max_ctx + kTreeChunkMin - 1) / kTreeChunkMin + 1);
    return a < b ? a : b;
}

bool tree_split(const TreeArgs& a) { return a.planned || a.nch > 1; }

// Splits contexts into chunks, where the records fit into part_rows; records used.
// The kernel divides the work itself (planned) where even chunks would have eight times
// the fewest positions or more; below, its start costs what equal shares gain (16 x 25 x
// 4096 69 to 72 us either way; 5 x 13 x 1999 31.3 planned, 29.6 not).
int64_t tree_plan(TreeArgs& a, int kv_type, int n_seq, int64_t part_rows) {
    const int64_t rows = (int64_t)a.max_nodes * a.group;
    const int wr = tree_wg_rows(rows), cmin = tree_chunk_min(wr);
    const int64_t base = (int64_t)n_seq * a.n_kv * ((rows + wr - 1) / wr);
    const bool stream_large = rows <= 32 && tree_once(a, kv_type, n_seq);
    const int64_t nch = tree_chunks(base, wr, stream_large, a.max_ctx);
    const int items = stream_large ? kTreeMany : kTreeItems;
    const int64_t places = items / a.n_kv;
    a.n_seq = n_seq, a.chunk = a.max_ctx > 0 ? a.max_ctx : 1, a.nch = 1;
    if (n_seq <= kWave && base <= items && nch > 0 && 8 * nch <= (a.max_ctx + cmin - 1) / cmin) {
        if (places * a.n_kv * wr > part_rows) return 0;
        a.nch = (int)places, a.chunk = cmin;
        a.planned = wr == 16 ? 4 : wr == 32 ? 5 : wr == 64 ? 6 : 7;
        return places * a.n_kv * wr;
    }
    const int64_t whole = (int64_t)n_seq * a.n_heads * a.max_nodes;
    if (nch > 1) {
        const int chunk = (int)((a.max_ctx + nch - 1) / nch + 63) / 64 * 64;
        const int n = (a.max_ctx + chunk - 1) / chunk;
        if (n > 1 && whole * n <= part_rows) a.chunk = chunk, a.nch = n;
    }
    return tree_split(a) ? whole * a.nch : 0;
}

bool tree_fast(const TreeArgs& a, int kv_type) {
    const int64_t es = kv_type == JINF_HIP_F16 ? 2 : 4;
    return (a.head_dim == 64 || a.head_dim == 128) && aligned(a.q, 16) && aligned(a.kc, 16) &&
           aligned(a.vc, 16) && a.ld_q % 4 == 0 && a.ld_q_seq % 4 == 0 && a.ld_pos * es % 16 == 0 &&
           a.ld_seq * es % 16 == 0 &&
           a.ld_pos * es <= (1 << 23);  // a tile's positions within 32-bit offsets
}

template <typename TC, int HD, int R, int RW, bool SCORE, bool ONCE>
int tree_launch(const TreeArgs& a, int n_seq, hipStream_t stream) {
    using Sh = TreeShape<TC, HD, R, RW, ONCE>;
    if (a.planned)
        return launch(tree_mfma_kernel<TC, HD, R, RW, SCORE, ONCE, true>, dim3((unsigned)a.n_kv, (unsigned)a.nch),
                      dim3(256), Sh::LDS, stream, a);
    const int64_t rows = (int64_t)a.max_nodes * a.group;
    const dim3 grid((unsigned)((rows + Sh::ROWS - 1) / Sh::ROWS * a.n_kv), (unsigned)n_seq, (unsigned)a.nch);
    return launch(tree_mfma_kernel<TC, HD, R, RW, SCORE, ONCE, false>, grid, dim3(256), Sh::LDS, stream, a);
}

// SCORE: the scored decode, which joins the chunks' partial sums itself.
template <typename TC, int HD, bool SCORE>
int tree_rows_launch(const TreeArgs& a, int n_seq, bool once, hipStream_t stream) {
    const int wr = tree_wg_rows((int64_t)a.max_nodes * a.group);
#define JINF_TREE_LAUNCH(R, RW)                                       \
    (once ? tree_launch<TC, HD, R, RW, SCORE, true>(a, n_seq, stream) \
          : tree_launch<TC, HD, R, RW, SCORE, false>(a, n_seq, stream))
    const int rc = wr == 16   ? JINF_TREE_LAUNCH(1, 1)
                   : wr == 32 ? JINF_TREE_LAUNCH(2, 1)
                   : wr == 64 ? JINF_TREE_LAUNCH(2, 2)
                              : JINF_TREE_LAUNCH(2, 4);
#undef JINF_TREE_LAUNCH
    if (rc != JINF_HIP_OK || !tree_split(a) || SCORE) return rc;
    constexpr int RB = 256 / (HD / 4);
    const int64_t all = (int64_t)a.max_nodes * a.group * a.n_kv;
    return launch(tree_merge_kernel<HD>, dim3((unsigned)((all + RB - 1) / RB), (unsigned)n_seq), dim3(256), 0,
                  stream, a);
}

template <bool SCORE>
int tree_mfma(const TreeArgs& a, int kv_type, int n_seq, hipStream_t stream) {
    const bool once = tree_once(a, kv_type, n_seq);
    if (kv_type == JINF_HIP_F16)
        return a.head_dim == 64 ? tree_rows_launch<uint16_t, 64, SCORE>(a, n_seq, once, stream)
                                : tree_rows_launch<uint16_t, 128, SCORE>(a, n_seq, once, stream);
    return a.head_dim == 64 ? tree_rows_launch<float, 64, SCORE>(a, n_seq, once, stream)
                            : tree_rows_launch<float, 128, SCORE>(a, n_seq, once, stream);
}

}  // namespace
}  // namespace jinf

extern "C" size_t jinf_attention_tree_workspace_bytes(int n_seq, int max_nodes, int n_heads,
                                                      int n_heads_kv, int head_dim, int max_ctx) {
    if (n_seq <= 0 || max_nodes <= 0 || n_heads <= 0 || n_heads_kv <= 0 || head_dim <= 0 || max_ctx < 0)
        return 0;
    if (n_heads % n_heads_kv != 0 || max_nodes > JINF_HIP_MAX_NODES) return 0;
    // plan; sums and {m, l} of each record
    return (size_t)n_seq * sizeof(int4) + (size_t)jinf::tree_part_rows(n_seq, max_nodes, n_heads, n_heads_kv, max_ctx) *
           (head_dim + 2) * sizeof(float) + 16;
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
    if (!tree_fast(a, kv_type)) return tree_any(a, kv_type, n_seq, stream);
    // workspace: the plan, sums, {m, l}
    const size_t plan_bytes = (size_t)n_seq * sizeof(int4);
    const int64_t fit = workspace && workspace_bytes > plan_bytes
                            ? (int64_t)((workspace_bytes - plan_bytes) / ((head_dim + 2) * sizeof(float))) : 0;
    const int64_t used = tree_plan(a, kv_type, n_seq, fit);
    if (tree_split(a)) {
        a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan_bytes);
        a.stats = reinterpret_cast<float2*>(a.part + used * head_dim);
    }
    return tree_mfma<false>(a, kv_type, n_seq, stream);
}

extern "C" size_t jinf_attention_scored_workspace_bytes(int n_seq, int n_heads, int n_heads_kv,
                                                        int head_dim, int max_ctx) {
    if (n_seq <= 0 || n_heads <= 0 || n_heads_kv <= 0 || head_dim <= 0 || max_ctx < 0) return 0;
    if (n_heads % n_heads_kv != 0) return 0;
    // scores, plan, {m, l} of one chunk a context at least, or sums and {m, l}
    return ((size_t)n_seq * n_heads * 16 * jinf::score_blocks(max_ctx) + 4 * (size_t)n_seq +
            2 * (size_t)n_seq * n_heads +
            (size_t)jinf::tree_part_rows(n_seq, 1, n_heads, n_heads_kv, max_ctx) * (head_dim + 2)) *
               sizeof(float) + 16;
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
    a.scores = static_cast<float*>(workspace), a.blocks = score_blocks(max_ctx);
    float* part = a.scores + (int64_t)n_seq * n_heads * a.blocks * 16 + 4 * (int64_t)n_seq;  // (behind the plan)
    a.chunk = max_ctx > 0 ? max_ctx : 1, a.nch = 1;
    const bool fast = tree_fast(a, kv_type);
    int64_t used = 0;
    if (fast) used = tree_plan(a, kv_type, n_seq, tree_part_rows(n_seq, 1, n_heads, n_heads_kv, max_ctx));
    if (tree_split(a)) a.part = part;
    a.stats = reinterpret_cast<float2*>(part + (a.part ? used * head_dim : 0));
    rc = fast ? tree_mfma<true>(a, kv_type, n_seq, stream) : tree_any(a, kv_type, n_seq, stream);
    if (rc != JINF_HIP_OK || max_ctx == 0) return rc;
    return launch(tree_finish_kernel, dim3((unsigned)((max_ctx + 1023) / 1024 + (a.part ? 1 : 0)), (unsigned)n_heads_kv,
                                           (unsigned)n_seq),
                  dim3(256), 0, stream, weights, ld_w, ld_w_seq, a, fast ? exp2f(kTreeUnit) : 1.0f);
}
