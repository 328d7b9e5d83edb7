// The paged key/value cache: a step's block tables and slot map from the requests' lengths, the new rows'
// QK-norm + RoPE + write into the pages, and causal attention of the new rows over the pages (include/rbt2_hip.h).
// The engine's State (rabbit2/src/rabbit2.c:427-446) holds one sequence of a fixed context; the arithmetic per
// row is its own (:472-498).
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "paged.h"
#include "rbt2_internal.h"

namespace rbt {
namespace {

typedef __bf16 bf16_t;

// Inclusive prefix sum over the wave, by DPP: within rows of 16 lanes, then the rows' totals handed on.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
    return v;
}

// ---------------------------------------------------------------- plan
// One block: three prefix sums over the requests (new rows, blocks needed, blocks given back), then the blocks pushed
// and popped and the rows' slots, each by its place in those sums (a binary search in LDS), so that one long request
// costs no more than many short ones. It moves a few KB and computes next to nothing: what bounds it is latency, so the
// sums go by DPP, and a new row's block is taken from the free stack, not from the table entry that another thread is
// writing. Steps of many rows give those to a launch of their own (1024 requests, 32768 rows: 15 us against 27.5 in one
// launch; 32 requests take 4.1 us, about a launch's own time).
constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / kWave, kPlanPer = kPagedMaxReq / kPlanThreads;

struct PlanArgs {
    int n_req, max_blocks, n_blocks, max_tokens;
    PageDiv div;
    const int32_t *len, *new_len, *n_free;
    int32_t *tables, *free_list, *kv_len, *n_free_out, *q_start, *slots, *positions, *status;
};

__device__ __forceinline__ int pages_for(int n, const PageDiv &div) {
    const int p = (int)page_of((uint32_t)n, div);
    return p + (n - p * (int)div.d > 0);
}
__device__ __forceinline__ void plan_put(const PlanArgs &a, int t, int pos, int page, int b) {
    a.slots[t] = b >= 0 && b < a.n_blocks ? b * (int)a.div.d + (pos - page * (int)a.div.d) : -1;
    a.positions[t] = pos;
}

// rows: whether this launch fills slots and positions too (else plan_rows_kernel does).
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs a, int rows) {
    __shared__ int32_t s_start[kPagedMaxReq + 1], s_need[kPagedMaxReq], s_freed[kPagedMaxReq], s_len[kPagedMaxReq];
    __shared__ int s_sum[kPlanWaves][3];
    __shared__ float s_big[kPlanWaves];
    __shared__ int s_bad;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, bs = (int)a.div.d;
    const int count = a.n_free[0];
    const int per = (a.n_req + kPlanThreads - 1) / kPlanThreads;  // requests tid * per + i
    int len[kPlanPer], add[kPlanPer], need[kPlanPer], freed[kPlanPer];
    if (tid == 0) s_bad = count < 0 || count > a.n_blocks;
    bool bad = false;
    float big = 0.0f;
    int v[3] = {0, 0, 0}, inc[3], before[3], total[3];
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
        const int r = tid * per + i;
        len[i] = add[i] = need[i] = freed[i] = 0;
        if (i >= per || r >= a.n_req) continue;
        const int n = a.len[r], nl = a.new_len[r];
        len[i] = n;
        add[i] = max(nl, 0);
        const bool out = n < 0 || (long long)n + add[i] > (long long)a.max_blocks * bs;
        bad |= out;
        const int have = out ? 0 : pages_for(n, a.div);
        need[i] = out || nl < 0 ? 0 : pages_for(n + add[i], a.div) - have;
        freed[i] = nl < 0 ? have : 0;
        v[0] += add[i];
        v[1] += need[i];
        v[2] += freed[i];
        big += (float)add[i] + (float)need[i] + (float)freed[i];
    }
    // the 32-bit sums hold where their sum in floats, no part of which is negative, is below 2^30
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        inc[i] = wave_scan(v[i]);
        if (lane == kWave - 1) s_sum[wv][i] = inc[i];
    }
    big = wave_sum(big);
    if (lane == 0) s_big[wv] = big;
    __syncthreads();
    if (bad) s_bad = 1;
    big = 0.0f;
    for (int w = 0; w < kPlanWaves; ++w) big += s_big[w];
#pragma unroll
    for (int i = 0; i < 3; ++i) {  // the waves before this one, and all
        const int x = wave_scan(lane < kPlanWaves ? s_sum[lane][i] : 0);
        total[i] = __builtin_amdgcn_readlane(x, kPlanWaves - 1);
        before[i] = inc[i] - v[i] + (wv > 0 ? __builtin_amdgcn_readlane(x, max(wv - 1, 0)) : 0);
    }
    __syncthreads();
    const bool valid = !s_bad && big < 1073741824.0f && total[0] <= a.max_tokens && count + total[2] <= a.n_blocks;
    const int top = count + total[2], lack = valid ? max(total[1] - top, 0) : 0;
    const bool ok = valid && lack == 0;
    if (tid == 0) {
        a.status[0] = valid ? lack : -1;
        a.n_free_out[0] = ok ? top - total[1] : count;
        a.q_start[a.n_req] = s_start[a.n_req] = ok ? total[0] : 0;
    }
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
        const int r = tid * per + i;
        if (i >= per || r >= a.n_req) continue;
        s_start[r] = ok ? before[0] : 0;
        s_need[r] = ok ? before[1] : 0;
        s_freed[r] = ok ? before[2] : 0;
        s_len[r] = len[i];
        a.q_start[r] = s_start[r];
        a.kv_len[r] = !ok ? len[i] : a.new_len[r] < 0 ? 0 : len[i] + add[i];
        before[0] += add[i];
        before[1] += need[i];
        before[2] += freed[i];
    }
    __syncthreads();
    if (ok && total[2] > 0) {
        for (int i = tid; i < total[2]; i += kPlanThreads) {
            const int r = request_of(s_freed, a.n_req, i);
            a.free_list[count + i] = a.tables[(size_t)r * a.max_blocks + (i - s_freed[r])];
        }
        __syncthreads();  // they may be popped again
    }
    if (ok)
        for (int i = tid; i < total[1]; i += kPlanThreads) {
            const int r = request_of(s_need, a.n_req, i);
            a.tables[(size_t)r * a.max_blocks + pages_for(s_len[r], a.div) + (i - s_need[r])] = a.free_list[top - 1 - i];
        }
    if (!rows) return;
    const int T = s_start[a.n_req];
    for (int t = tid; t < a.max_tokens; t += kPlanThreads) {
        if (t >= T) {
            a.slots[t] = a.positions[t] = -1;
            continue;
        }
        const int r = request_of(s_start, a.n_req, t), pos = s_len[r] + (t - s_start[r]);
        const int page = (int)page_of((uint32_t)pos, a.div), have = pages_for(s_len[r], a.div);
        plan_put(a, t, pos, page,
                 page < have ? a.tables[(size_t)r * a.max_blocks + page] : a.free_list[top - 1 - (s_need[r] + page - have)]);
    }
}

__global__ __launch_bounds__(256) void plan_rows_kernel(PlanArgs a) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= a.max_tokens) return;
    const int t = (int)id;
    if (t >= a.q_start[a.n_req]) {
        a.slots[t] = a.positions[t] = -1;
        return;
    }
    const int r = request_of(a.q_start, a.n_req, t), pos = a.kv_len[r] - a.q_start[r + 1] + t;
    const int page = (int)page_of((uint32_t)pos, a.div);
    plan_put(a, t, pos, page, a.tables[(size_t)r * a.max_blocks + page]);
}

// ---------------------------------------------------------------- append
struct AppendArgs {
    PagedDims d;
    int n_heads, n_rope;
    const float *q, *k, *v;
    uint64_t q_stride, k_stride, v_stride;
    float *q_out;
    const float *q_norm, *k_norm;
    float eps;
    const float2 *rope;
    const int32_t *positions, *slots;
    void *kc, *vc;
};

template <int DT>
__device__ __forceinline__ void store_kv(void *p, uint64_t i, float v) {
    if constexpr (DT == RBT_DT_F32)
        static_cast<float *>(p)[i] = v;
    else
        static_cast<bf16_t *>(p)[i] = (bf16_t)v;  // to nearest even; NaN stays NaN
}

// grid (tokens), 256 threads: prompt_rope_kernel's arithmetic (prompt.hip) with the cache rows in pages. For any head dim
// and alignment; append_quads_kernel takes the others.
template <int DT>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    __shared__ float red[8];
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int hd = a.d.hd, half = hd / 2, qd = a.n_heads * hd, kvd = a.d.n_kv * hd;
    const int slot = a.slots[t], pos = a.rope ? a.positions[t] : 0;
    if (slot < 0 || slot >= a.d.n_blocks * a.d.block_size || (a.rope && (pos < 0 || pos >= a.n_rope))) return;
    const int b = (int)page_of((uint32_t)slot, a.d.div), off = slot - b * a.d.block_size;
    const float *q = a.q ? a.q + (size_t)t * a.q_stride : nullptr, *k = a.k + (size_t)t * a.k_stride,
                *v = a.v + (size_t)t * a.v_stride;
    float sq = 0.0f, sk = 0.0f;
    if (a.q && a.q_norm)
        for (int i = tid; i < qd; i += 256) sq += q[i] * q[i];
    if (a.k_norm)
        for (int i = tid; i < kvd; i += 256) sk += k[i] * k[i];
    sq = wave_sum(sq);
    sk = wave_sum(sk);
    if (lane == 0) {
        red[wv] = sq;
        red[4 + wv] = sk;
    }
    __syncthreads();
    sq = (red[0] + red[1]) + (red[2] + red[3]);
    sk = (red[4] + red[5]) + (red[6] + red[7]);
    const float inv_q = 1.0f / sqrtf(sq / (float)qd + a.eps), inv_k = 1.0f / sqrtf(sk / (float)kvd + a.eps);
    const float2 *cs = a.rope ? a.rope + (size_t)pos * half : nullptr;
    auto rows = [&](const float *src, const float *w, float inv, int n, auto put) {
        if (!cs) {
            for (int i = tid; i < n; i += 256) put(i, w ? src[i] * inv * w[i] : src[i]);
            return;
        }
        for (int u = tid; u < n / 2; u += 256) {  // pair u: elements i and i + half of one head
#pragma clang fp contract(off)
            const int h = u / half, i = u - h * half, lo = h * hd + i, hi = lo + half;
            float x = src[lo], y = src[hi];
            if (w) {
                x = x * inv * w[lo];
                y = y * inv * w[hi];
            }
            const float2 c = cs[i];
            put(lo, x * c.x - y * c.y);
            put(hi, y * c.x + x * c.y);
        }
    };
    if (q) rows(q, a.q_norm, inv_q, qd, [&](int i, float x) { a.q_out[(size_t)t * qd + i] = x; });
    auto at = [&](int i) { return paged_row(a.d, b, i / hd, off) + (uint64_t)(i % hd); };
    rows(k, a.k_norm, inv_k, kvd, [&](int i, float x) { store_kv<DT>(a.kc, at(i), x); });
    for (int i = tid; i < kvd; i += 256) store_kv<DT>(a.vc, at(i), v[i]);
}

// The same for head dims that are multiples of 8 and 16-byte aligned rows of up to 256 * 8 * kAppendQ floats of q and
// 256 * 8 * kAppendK of k: everything is asked for at once (the rows whether or not the token has a slot), held in
// registers through the norm, and each thread turns whole quads of pairs (elements 4 i .. 4 i + 3 of a head's halves).
// One pass over memory, which bounds it: 4096 tokens of 16 heads of 128 take 33.5 us, 5.1 TB/s (append_kernel 63 us).
// Rows of up to 2048 floats (the benchmark's model) take a quarter of the registers, so that four times the blocks share
// a CU (the same 4096 tokens on the larger rows' kernel: 45.8 us).
constexpr int kAppendQ = 4, kAppendK = 2;
__device__ __forceinline__ void store4(float *p, f32x4 v) { *reinterpret_cast<f32x4 *>(p) = v; }
template <int DT>
__device__ __forceinline__ void store_kv4(void *p, uint64_t i, f32x4 v) {
    if constexpr (DT == RBT_DT_F32) {
        store4(static_cast<float *>(p) + i, v);
    } else {
        typedef bf16_t bf16x4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<bf16x4 *>(static_cast<bf16_t *>(p) + i) = __builtin_convertvector(v, bf16x4);
    }
}
template <int N>
struct AppendRow {
    f32x4 lo[N], hi[N], wl[N], wh[N], c0[N], c1[N];  // halves, their norm weights, (cos, sin) of the four pairs
    __device__ __forceinline__ void load(const float *src, const float *w, int quads, int per_half, int hd) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = min((int)threadIdx.x + 256 * i, quads - 1), h = u / per_half, at = h * hd + 4 * (u - h * per_half);
            lo[i] = ld_f4(src + at);
            hi[i] = ld_f4(src + at + hd / 2);
            if (w) {
                wl[i] = ld_f4(w + at);
                wh[i] = ld_f4(w + at + hd / 2);
            }
        }
    }
    __device__ __forceinline__ void load_turns(const float *cs, int quads, int per_half) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = min((int)threadIdx.x + 256 * i, quads - 1), q = u % per_half;
            c0[i] = ld_f4(cs + 8 * q);
            c1[i] = ld_f4(cs + 8 * q + 4);
        }
    }
    __device__ __forceinline__ float squares(int quads) const {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if ((int)threadIdx.x + 256 * i < quads)
#pragma unroll
                for (int j = 0; j < 4; ++j) s += lo[i][j] * lo[i][j] + hi[i][j] * hi[i][j];
        return s;
    }
    // put(element, four values) of both halves, normed and turned
    template <typename Put>
    __device__ __forceinline__ void finish(bool norm, float inv, bool turn, int quads, int per_half, int hd, Put put) {
#pragma clang fp contract(off)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = (int)threadIdx.x + 256 * i;
            if (u >= quads) break;
            const int h = u / per_half, at = h * hd + 4 * (u - h * per_half);
            f32x4 x = lo[i], y = hi[i];
            if (norm) {
                x = x * inv * wl[i];
                y = y * inv * wh[i];
            }
            if (turn) {
                const f32x4 c = f32x4{c0[i].x, c0[i].z, c1[i].x, c1[i].z}, s = f32x4{c0[i].y, c0[i].w, c1[i].y, c1[i].w};
                const f32x4 a = x * c - y * s, b = y * c + x * s;
                x = a;
                y = b;
            }
            put(at, x);
            put(at + hd / 2, y);
        }
    }
};
template <int DT, int NQ, int NK>
__global__ __launch_bounds__(256) void append_quads_kernel(AppendArgs a) {
    __shared__ float red[8];
    const int t = blockIdx.x, lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int hd = a.d.hd, per_half = hd / 8, qd = a.n_heads * hd, kvd = a.d.n_kv * hd, q_quads = a.q ? qd / 8 : 0;
    const int slot = a.slots[t], pos = a.rope ? a.positions[t] : 0;
    AppendRow<NQ> q;
    AppendRow<NK> k;
    f32x4 v[2 * NK];
    if (a.q) q.load(a.q + (size_t)t * a.q_stride, a.q_norm, q_quads, per_half, hd);
    k.load(a.k + (size_t)t * a.k_stride, a.k_norm, kvd / 8, per_half, hd);
#pragma unroll
    for (int i = 0; i < 2 * NK; ++i)
        v[i] = ld_f4(a.v + (size_t)t * a.v_stride + 4 * min((int)threadIdx.x + 256 * i, kvd / 4 - 1));
    if (slot < 0 || slot >= a.d.n_blocks * a.d.block_size || (a.rope && (pos < 0 || pos >= a.n_rope))) return;
    if (a.rope) {
        const float *cs = reinterpret_cast<const float *>(a.rope + (size_t)pos * (hd / 2));
        if (a.q) q.load_turns(cs, q_quads, per_half);
        k.load_turns(cs, kvd / 8, per_half);
    }
    float inv_q = 1.0f, inv_k = 1.0f;
    if (a.q_norm || a.k_norm) {  // the same for all threads
        float sq = a.q && a.q_norm ? q.squares(q_quads) : 0.0f, sk = a.k_norm ? k.squares(kvd / 8) : 0.0f;
        sq = wave_sum(sq);
        sk = wave_sum(sk);
        if (lane == 0) {
            red[wv] = sq;
            red[4 + wv] = sk;
        }
        __syncthreads();
        sq = (red[0] + red[1]) + (red[2] + red[3]);
        sk = (red[4] + red[5]) + (red[6] + red[7]);
        inv_q = 1.0f / sqrtf(sq / (float)qd + a.eps);
        inv_k = 1.0f / sqrtf(sk / (float)kvd + a.eps);
    }
    const int b = (int)page_of((uint32_t)slot, a.d.div), off = slot - b * a.d.block_size;
    const bool turn = a.rope != nullptr;
    if (a.q)
        q.finish(a.q_norm != nullptr, inv_q, turn, q_quads, per_half, hd,
                 [&](int i, f32x4 x) { store4(a.q_out + (size_t)t * qd + i, x); });
    auto at = [&](int i) { return paged_row(a.d, b, i / hd, off) + (uint64_t)(i % hd); };
    k.finish(a.k_norm != nullptr, inv_k, turn, kvd / 8, per_half, hd, [&](int i, f32x4 x) { store_kv4<DT>(a.kc, at(i), x); });
#pragma unroll
    for (int i = 0; i < 2 * NK; ++i) {
        const int u = (int)threadIdx.x + 256 * i;
        if (u < kvd / 4) store_kv4<DT>(a.vc, at(4 * u), v[i]);
    }
}

// ---------------------------------------------------------------- attention
struct AttnArgs {
    PagedDims d;
    int n_req, max_blocks, T, n_heads, window;
    PageDiv group; // query heads to a key/value head
    int thin;      // whether requests of up to 16 rows are the thin blocks'
    int wide;      // whether there are wide blocks
    float scale2;  // scale * log2(e), into the query rows: the softmax runs in powers of two
    const int32_t *tables, *kv_len, *q_start;
    const void *kc, *vc;
    const float *q;
    float *out;
    uint64_t q_stride, out_stride;
    uint8_t *ws;
};

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Softmax state of a set of positions: the reference m (a power of two's exponent; -inf: none seen), the sum l of
// 2^(s - m) and their weighted values. What a state weighs against the reference M of several:
__device__ __forceinline__ float state_weight(float m, float M) { return m == -INFINITY ? 0.0f : exp2f(m - M); }

// One (row, head) over positions [j0, j1), by a block of 256 threads and in any head dim: 256 positions at a
// time, a thread per position for the scores and a thread per dim for the weighted sum. Returns the state, o in
// thread i < hd. Positions without a place in the cache are not seen, and what they are multiplied with is
// never read, so no value that is not finite enters from a position that is not seen.
struct RowShared {
    uint64_t row[256];
    float q[kPagedMaxHd], p[256], red[8];
};
template <int DT>
__device__ void row_any(const AttnArgs &a, RowShared &s, int r, int t, int h, int j0, int j1, float *m_out, float *l_out,
                        float *o_out) {
    constexpr uint64_t kNone = ~0ull;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, hd = a.d.hd, kvh = h / (int)a.group.d;
    __syncthreads();  // the shared values of a previous call have been read
    if (tid < hd) s.q[tid] = a.q[(size_t)t * a.q_stride + (size_t)h * hd + tid];
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (; j0 < j1; j0 += 256) {
        const int j = j0 + tid;
        float x = -INFINITY;
        uint64_t row = kNone;
        if (j < j1) {
            const int page = (int)page_of((uint32_t)j, a.d.div);
            const int b = a.tables[(size_t)r * a.max_blocks + page];
            if (b >= 0 && b < a.d.n_blocks) {
                row = paged_row(a.d, b, kvh, j - page * a.d.block_size);
                x = 0.0f;
                for (int i = 0; i < hd; ++i) x += s.q[i] * load_w<DT>(a.kc, row + i);
                x *= a.scale2;
            }
        }
        s.row[tid] = row;
        const float wm = wave_max(x);
        if (lane == 0) s.red[wv] = wm;
        __syncthreads();
        const float mn = fmaxf(fmaxf(m, fmaxf(s.red[0], s.red[1])), fmaxf(s.red[2], s.red[3]));
        const float ref = mn == -INFINITY ? 0.0f : mn;  // nothing seen yet: all weights 0
        const float p = row != kNone ? exp2f(x - ref) : 0.0f;
        s.p[tid] = p;
        const float ps = wave_sum(p);
        if (lane == 0) s.red[4 + wv] = ps;
        __syncthreads();
        const float alpha = exp2f(m - ref);
        l = l * alpha + ((s.red[4] + s.red[5]) + (s.red[6] + s.red[7]));
        o *= alpha;
        if (tid < hd)
            for (int jj = 0; jj < min(256, j1 - j0); ++jj)
                if (s.row[jj] != kNone) o += s.p[jj] * load_w<DT>(a.vc, s.row[jj] + tid);
        m = mn;
        __syncthreads();  // red, p and row are rewritten
    }
    *m_out = m;
    *l_out = l;
    *o_out = o;
}

// Request r of a step: its new rows m from row t0 on, positions n (p0 before the new ones; negative where the
// length is below the new rows). Rows outside the step's buffers: the request takes no part (m 0).
struct Request {
    int t0, m, n, p0;
};
__device__ __forceinline__ Request request(const AttnArgs &a, int r) {
    Request q;
    const int t0 = a.q_start[r], t1 = a.q_start[r + 1];
    q.t0 = t0;
    q.m = t0 < 0 || t1 > a.T || t1 <= t0 ? 0 : t1 - t0;
    q.n = min(max(a.kv_len[r], 0), a.max_blocks * a.d.block_size);
    q.p0 = q.n - q.m;
    return q;
}

// Any head dim and alignment: a block per (row, head).
template <int DT>
__global__ __launch_bounds__(256) void attn_any_kernel(AttnArgs a) {
    __shared__ RowShared s;
    for (uint64_t id = blockIdx.x; id < (uint64_t)a.T * a.n_heads; id += gridDim.x) {
        const int t = (int)(id / a.n_heads), h = (int)(id % a.n_heads);
        if (t < a.q_start[0]) continue;
        const int r = request_of(a.q_start, a.n_req, t);
        const Request q = request(a, r);
        if (t >= q.t0 + q.m) continue;
        const int pos = q.p0 + t - q.t0, first = a.window > 0 ? max(0, pos - a.window + 1) : 0;
        float m, l, o;
        row_any<DT>(a, s, r, t, h, first, pos + 1, &m, &l, &o);
        if ((int)threadIdx.x < a.d.hd)
            a.out[(size_t)t * a.out_stride + (size_t)h * a.d.hd + threadIdx.x] = l == 0.0f ? 0.0f : o / l;
    }
}

// ---- on the matrix cores (head dims that are multiples of 8, 16-byte aligned rows)
// Rows: a request's new tokens times the query heads of one key/value head, heads fastest. A tile of rows runs over
// its positions in tiles, staged in LDS as bf16 parts:
//   wide   128 rows, 32 to a wave; the block's waves share each tile of keys and values
//   thin   requests of up to 16 rows (a decoding token): each wave takes tiles of 32 positions of its own
// each kind by blocks of its own, and long ranges are cut into pieces that different blocks take, joined by
// attn_merge_kernel. (Joined by a tile's last block instead, thin tiles gain a microsecond and wide ones lose 20, whose
// few blocks then read what others wrote while the rest of the chip waits.)
//
// Products: v_mfma_f32_16x16x32_bf16, transposed so that nothing moves between lanes: S^T = K Q^T leaves lane
// (c = l % 16, g = l / 16) the scores of query c with keys 4 g + i of two 16-key groups, which as they stand are
// the B operand of O^T = V^T P^T whose k-slot (g, 4 t + i) is key 16 t + 4 g + i. V^T comes from the row-major
// tile by the transposing LDS read (ds_read_b64_tr_b16: lane c of group g gets column c of rows 4 g .. 4 g + 3).
//
// Precision: bf16 keys and values enter exactly. f32 operands are cut into three bf16 parts of 8 bits each (exact: 24
// bits), and the products of parts down to 2^-24 are taken: three for a bf16 cache, six for an f32 one. Sums, the softmax
// and its state are f32. Outputs are as far from 64 bits as f32 arithmetic leaves them (3e-7 of their size; two parts
// would leave 16 bits and save a third of the products).
//
// What bounds it: a prompt of 4096 tokens (16 heads of 128, bf16) takes 208 us, 206 GFLOP in its three products: 990
// TFLOP/s, where a large library product reaches 1200; the matrix units are busy 75% of the inner loop, items' starts
// and ends and the joining of pieces take 20 us each. 64 decoding sequences of up to 8192 positions take 218 us, 5.7
// TB/s of cache. Small steps are latency: the schedule, pages, queries and first keys one after the other, and two
// launches (one sequence: 16 us).
//
// Not finite: a position that a row does not see has weight 0, but 0 times an infinity is NaN, so rows whose
// result is not finite are computed again by row_any, which reads seen positions only. Rows past the positions
// repeat the last one's, with weight 0.
constexpr int kTabPages = 512;  // pages whose places are held in LDS at a time
// Workspace: for the wide and the thin blocks each a header (chunk length, blocks of the merge) and the prefix sums of
// those and of the partial units over the requests, then their partials: units of 16 rows, m [16], l [16],
// o [16][HDP].
struct AttnHeader {
    int32_t chunk, merge_blocks, pad[2];
    int32_t taken[8][16];  // items that each XCD's blocks took beyond their first, a line each; 0 between the calls
    int32_t merge[kPagedMaxReq + 4], units[kPagedMaxReq + 4];
};
constexpr size_t kWsThin = kPagedWsBytes / 4;  // of it, with its header
constexpr int unit_floats(int hdp) { return 16 * (hdp + 2); }
template <bool THIN>
struct AttnWs {
    static constexpr size_t kAt = THIN ? 0 : kWsThin, kBytes = THIN ? kWsThin : kPagedWsBytes - kWsThin;
    __device__ static AttnHeader *header(uint8_t *ws) { return reinterpret_cast<AttnHeader *>(ws + kAt); }
    __device__ static float *partials(uint8_t *ws) { return reinterpret_cast<float *>(ws + kAt + sizeof(AttnHeader)); }
    static constexpr int max_units(int hdp) { return (int)((kBytes - sizeof(AttnHeader)) / 4 / unit_floats(hdp)); }
};

template <bool THIN>
__device__ __forceinline__ Cut cut_of(const AttnArgs &a, const Request &q, int chunk) {
    int rows = q.m * (int)a.group.d;
    if (THIN != (a.thin && rows <= kThinRows)) rows = 0;
    return cut_rows<THIN>(rows, q.n, q.p0, (int)a.group.d, a.window, chunk);
}

// Rows that a block of attn_merge_kernel joins: a few per wave, or where many pieces have to be read, as many as one
// wave takes, the pieces dealt to the block's four.
constexpr int kMergeManyPieces = 16;
template <int HDP>
__device__ __forceinline__ int merge_rows(int nc) { return 256 / HDP * (nc >= kMergeManyPieces ? 1 : 4); }

// A kind's items (request, head, row tile, piece), by every block for itself: prefix sums over the requests into
// s_items [n_req + 1] and s_units. The chunk length is a little over a block's share of the positions, so that most
// blocks get one piece and the rests fill the gaps: 19 decoding, chunked and prompt steps take 82.6 us on average, and
// 85.0 with half of it for thin tiles (131072 positions 92 against 99 us, 64 long sequences 218 against 217); half of it
// for wide tiles: a windowed prompt of 2 x 2048 tokens 108 against 68, three prompts of 1500 141 against 164. It doubles
// until the partials fit, which ends at the latest at kMaxChunk, where no tile is cut. Returns 0 where no request is of
// this kind.
struct ScheduleShared {
    float work[4];
    int any[4], sum[4][3];
};
template <bool THIN, int HDP>
__device__ int schedule(const AttnArgs &a, int block, int blocks, int32_t *s_items, int32_t *s_units, ScheduleShared &s) {
    constexpr int tr = kTileRows<THIN>, kUnits = AttnWs<THIN>::max_units(HDP);
    const int per = (a.n_req + 255) / 256, r0 = min(a.n_req, (int)threadIdx.x * per), r1 = min(a.n_req, r0 + per);
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    AttnHeader *hdr = block == 0 ? AttnWs<THIN>::header(a.ws) : nullptr;  // one block tells attn_merge_kernel
    // the first request of a thread (all of them, up to 256 requests) stays in registers
    Request first{};
    if (r0 < r1) first = request(a, r0);
    auto req = [&](int r) { return r == r0 ? first : request(a, r); };
    float work = 0.0f;
    bool any = false;
    for (int r = r0; r < r1; ++r) {
        const Request q = req(r);
        if (!q.m) continue;
        const Cut c = cut_of<THIN>(a, q, kMaxChunk);
        any |= c.nt > 0;
        work += (float)c.nt * (float)(a.window > 0 ? min(q.n, min(a.window, q.n) + tr) : q.n - q.m / 2);
    }
    work = wave_sum(work);
    const bool wave_any = __any(any);
    if (lane == 0) {
        s.work[wv] = work;
        s.any[wv] = wave_any;
    }
    __syncthreads();
    if (!(s.any[0] | s.any[1] | s.any[2] | s.any[3])) {
        if (hdr && threadIdx.x == 0) hdr->merge_blocks = 0;
        return 0;
    }
    work = ((s.work[0] + s.work[1]) + (s.work[2] + s.work[3])) * (float)a.d.n_kv / (float)blocks;
    int chunk = max((int)fminf(1.025f * work, 1.0e9f), 0) / 128 * 128 + 128;
    for (;;) {
        int v[3] = {0, 0, 0}, inc[3], before[3], total[3];  // items, partial units, merge blocks
        for (int r = r0; r < r1; ++r) {
            const Request q = req(r);
            if (!q.m) continue;
            const Cut c = cut_of<THIN>(a, q, chunk);
            const int64_t n = pieces_before<THIN>(c, c.nt) * a.d.n_kv;
            v[0] += (int)min(n, (int64_t)1 << 30);
            if (c.nc > 1) {
                v[1] = (int)min(v[1] + n * (tr / 16), (int64_t)1 << 22);  // more than ever fit, and no sum of them wraps
                v[2] += (c.rows * a.d.n_kv + merge_rows<HDP>(c.nc) - 1) / merge_rows<HDP>(c.nc);
            }
        }
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            inc[i] = wave_scan(v[i]);
            if (lane == 63) s.sum[wv][i] = inc[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            before[i] = inc[i] - v[i];
            total[i] = 0;
            for (int w = 0; w < 4; ++w) {
                if (w < wv) before[i] += s.sum[w][i];
                total[i] += s.sum[w][i];
            }
        }
        if (total[1] > kUnits && chunk < kMaxChunk) {
            chunk = chunk < kMaxChunk / 2 ? 2 * chunk : kMaxChunk;
            __syncthreads();  // the sums have been read
            continue;
        }
        for (int r = r0; r < r1; ++r) {
            s_items[r] = before[0];
            s_units[r] = before[1];
            if (hdr) {
                hdr->merge[r] = before[2];
                hdr->units[r] = before[1];
            }
            const Request q = req(r);
            if (!q.m) continue;
            const Cut c = cut_of<THIN>(a, q, chunk);
            const int n = (int)pieces_before<THIN>(c, c.nt) * a.d.n_kv;
            before[0] += n;
            if (c.nc > 1) {
                before[1] += n * (tr / 16);
                before[2] += (c.rows * a.d.n_kv + merge_rows<HDP>(c.nc) - 1) / merge_rows<HDP>(c.nc);
            }
        }
        if (threadIdx.x == 0) {
            s_items[a.n_req] = total[0];
            if (hdr) {
                hdr->chunk = chunk;
                hdr->merge_blocks = total[2];
            }
        }
        __syncthreads();
        return chunk;
    }
}

// Two f32 as packed bf16, to nearest, and exactly what that leaves of them: x - hi(x) is one dot product of the pair with
// (-1, 0) instead of an unpack and a subtraction (the weights' parts are a third of a step's arithmetic). The
// constants stay in registers: as literals of the packed type the compiler encodes one of them as the other.
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
struct PartConsts {
    uint32_t lo = 0x0000BF80u, hi = 0xBF800000u;
    __device__ __forceinline__ PartConsts() { asm("" : "+v"(lo), "+v"(hi)); }
};
__device__ __forceinline__ uint32_t take_part(float &x, float &y, const PartConsts &pc) {
    const bf16x2 h = {(__bf16)x, (__bf16)y};
    x = __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, pc.lo), x, false);
    y = __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, pc.hi), y, false);
    return __builtin_bit_cast(uint32_t, h);
}
// Eight f32 in three parts.
__device__ __forceinline__ void split3(float (&x)[8], u32x4 (&part)[3], const PartConsts &pc) {
#pragma unroll
    for (int p = 0; p < 3; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[p][i] = take_part(x[2 * i], x[2 * i + 1], pc);
}

// max and sum over the four lanes of a query
__device__ __forceinline__ float group_max(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float group_sum(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// LDS layouts of a tile part, in which the same 16-byte chunk of 16 rows (a K operand) and the same 32 bytes of 16
// rows (V^T) lie in all banks evenly. k_at(t, st) and v_at(t, d): a lane's byte of the operands of key group t, k-step
// st and of dims 16 d.
// Rows of HDP bf16 and 16 bytes more: every operand at a fixed distance from a lane's first.
template <int HDP>
struct PaddedTile {
    static constexpr int ROW = HDP * 2 + 16;
    int k0, v0;
    __device__ __forceinline__ PaddedTile() {
        const int c = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
        k0 = c * ROW + 16 * g;
        v0 = (4 * g + (c >> 2)) * ROW + 8 * (c & 3);
    }
    __device__ __forceinline__ int k_at(int t, int st) const { return k0 + t * 16 * ROW + st * 64; }
    __device__ __forceinline__ int v_at(int t, int d) const { return v0 + t * 16 * ROW + d * 32; }
};
// Rows of HDP bf16 whose chunks are permuted by the row (chunk ^ key(row)): what direct copies can write, whose lanes
// each choose what they read but not where it lands.
template <int HDP>
struct SwizzledTile {
    static constexpr int ROW = HDP * 2, CH = HDP / 8, KN = CH < 16 ? CH / 4 : 4, VN = CH < 16 ? CH / 2 : 8;
    __device__ static __forceinline__ int key(int row) { return CH == 8 ? (row >> 1) & 7 : row & 15; }
    int k[KN], v[VN];
    __device__ __forceinline__ SwizzledTile() {
        const int c = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4, vr = 4 * g + (c >> 2);
#pragma unroll
        for (int i = 0; i < KN; ++i) k[i] = c * ROW + ((4 * i + g) ^ key(c)) * 16;
#pragma unroll
        for (int i = 0; i < VN; ++i) v[i] = vr * ROW + ((2 * i + ((c & 3) >> 1)) ^ key(vr)) * 16 + 8 * (c & 1);
    }
    __device__ __forceinline__ int k_at(int t, int st) const { return k[st % KN] + t * 16 * ROW + st / KN * 64 * KN; }
    __device__ __forceinline__ int v_at(int t, int d) const { return v[d % VN] + t * 16 * ROW + d / VN * 32 * VN; }
};

extern __shared__ __align__(16) uint8_t smem[];

// What a wave keeps of its NQ * 16 rows. QP: parts of the query rows in registers; the third may lie in LDS instead, from
// q_at on for this lane, laid out as a PaddedTile of the wave's rows.
template <int HDP, int NQ, int QP = 3>
struct WaveState {
    u32x4 q[NQ][HDP / 32][QP];
    int q_at;
    f32x4 o[NQ][HDP / 16];
    float m[NQ], l[NQ];
    int pos[NQ];  // this lane's query's position
    PartConsts pc;
};

// 32 positions, staged from byte k_off (keys) and v_off (values) of LDS on, parts `part` bytes apart; between(i) is
// called among the products, for i = 0 .. HDP / 16 NP - 1 in turn; seen(n): bit 4 t + i, whether query n of this lane
// sees key 16 t + 4 g + i of them (asked where !full).
// Mid: a call between the keys' last use and the values' first (and no value is read before it), or NoMid.
struct NoMid {};
template <int HDP, int NQ, int QP, int NP, int part, typename Tile, typename Between, typename Seen, typename Mid>
__device__ __forceinline__ void attn_step(WaveState<HDP, NQ, QP> &w, const Tile &tile, int k_off, int v_off, bool full,
                                          Between between, Seen seen, Mid mid) {
    constexpr bool kMid = !std::is_same_v<Mid, NoMid>;
    // Consecutive products go to different sums: a sum's next product waits for its last. The operands of the next
    // products are read from LDS before those of the last ones are used.
    constexpr int KI = HDP / 32 * NP, VI = HDP / 32 * NP;  // (k-step, part) and (pair of 16 dims, part)
    auto read_k = [&](int i, u32x4 (&k)[2]) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
            k[t] = *reinterpret_cast<const u32x4 *>(smem + (k_off + i % NP * part) + tile.k_at(t, i / NP));
    };
    auto read_v = [&](int i, u32x4 (&v)[2]) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const u32x2 h = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s16x4 *)(smem + (v_off + i % NP * part) +
                                                                tile.v_at(t, i / NP * 2 + e))));
                v[e][2 * t] = h[0];
                v[e][2 * t + 1] = h[1];
            }
    };
    f32x4 s[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) s[n][0] = s[n][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    u32x4 k[2][2], v[2][2];
    read_k(0, k[0]);
#pragma unroll
    for (int i = 0; i < KI; ++i) {
        if (i + 1 < KI)
            read_k(i + 1, k[(i + 1) & 1]);
        else if (!kMid)
            read_v(0, v[0]);
        u32x4 q3[NQ];
        if (QP < 3 && i % NP == 0)
#pragma unroll
            for (int n = 0; n < NQ; ++n)
                q3[n] = *reinterpret_cast<const u32x4 *>(smem + w.q_at + n * 16 * PaddedTile<HDP>::ROW + i / NP * 64);
        between(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int qp = 0; qp + i % NP < 3; ++qp)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int n = 0; n < NQ; ++n)
                    s[n][t] = mfma(k[i & 1][t], qp < QP ? w.q[n][i / NP][qp < QP ? qp : 0] : q3[n], s[n][t]);
        __builtin_amdgcn_sched_barrier(0);
    }
    if (!full) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const uint32_t bits = seen(n);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][t][i] = bits >> (4 * t + i) & 1 ? s[n][t][i] : -INFINITY;
        }
    }
    // The reference moves only when a score is 2^8 above it (weights stay below 2^8 then): most steps neither
    // reduce over the lanes nor rescale.
    float top[NQ];
    bool move = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        top[n] = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) top[n] = fmaxf(top[n], s[n][t][i]);
        move |= top[n] > w.m[n] + 8.0f;
    }
    if (__any(move)) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const float m = fmaxf(w.m[n], group_max(top[n]));
            const float a = w.m[n] == -INFINITY ? 0.0f : exp2f(w.m[n] - m);
            w.m[n] = m;
            w.l[n] *= a;
#pragma unroll
            for (int d = 0; d < HDP / 16; ++d) w.o[n][d] *= a;
        }
    }
    u32x4 p[NQ][3];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const float ref = w.m[n] == -INFINITY ? 0.0f : w.m[n];
        float e[8];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                e[4 * t + i] = __builtin_amdgcn_exp2f(s[n][t][i] - ref);
                w.l[n] += e[4 * t + i];
            }
        split3(e, p[n], w.pc);
    }
    if constexpr (kMid) {
        mid();
        read_v(0, v[0]);
    }
#pragma unroll
    for (int i = 0; i < VI; ++i) {
        if (i + 1 < VI) read_v(i + 1, v[(i + 1) & 1]);
        between(KI + i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int pp = 0; pp + i % NP < 3; ++pp)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    f32x4 &o = w.o[n][i / NP * 2 + e];
                    o = mfma(v[i & 1][e], p[n][pp], o);
                }
        __builtin_amdgcn_sched_barrier(0);
    }
}

// The rows of a wave: rows row0 .. row0 + 16 NQ - 1 of the request (clamped to its last), q in three parts.
template <int HDP, int NQ, int QP>
__device__ __forceinline__ void wave_init(WaveState<HDP, NQ, QP> &w, const AttnArgs &a, const Request &q, int rows, int kvh,
                                          int row0, int q_off) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, G = (int)a.group.d;
    w.q_at = q_off + c * PaddedTile<HDP>::ROW + 16 * g;
    // Every load before the first answer is used. Past the head's end: its last 8 elements, as 0 (without a branch, which
    // would make each load wait for the one before).
    f32x4 x[NQ][HDP / 32][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int row = min(row0 + 16 * n + c, rows - 1), tok = (int)page_of((uint32_t)row, a.group);
        const float *src = a.q + (size_t)(q.t0 + tok) * a.q_stride + (size_t)(kvh * G + row - tok * G) * a.d.hd;
        w.pos[n] = q.p0 + tok;
#pragma unroll
        for (int st = 0; st < HDP / 32; ++st)
#pragma unroll
            for (int i = 0; i < 2; ++i) x[n][st][i] = ld_f4(src + min(32 * st + 8 * g, a.d.hd - 8) + 4 * i);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        w.m[n] = -INFINITY;
        w.l[n] = 0.0f;
#pragma unroll
        for (int st = 0; st < HDP / 32; ++st) {
            const float scale = 32 * st + 8 * g < a.d.hd ? a.scale2 : 0.0f;
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = x[n][st][i / 4][i % 4] * scale;
            u32x4 part[3];
            split3(y, part, w.pc);
#pragma unroll
            for (int p = 0; p < QP; ++p) w.q[n][st][p] = part[p];
            if (QP < 3)
                *reinterpret_cast<u32x4 *>(smem + w.q_at + n * 16 * PaddedTile<HDP>::ROW + st * 64) = part[2];
        }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int d = 0; d < HDP / 16; ++d) w.o[n][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

// The places (byte offset of the block) of the pages that positions j0 .. j1 - 1 (at most tab_span of them, at least
// one) lie on: ask() for the block numbers, fill() s_tab; 1 for a page outside the cache (whose positions are read
// from offset 0 and not seen): whether there is any. For all threads of the block.
constexpr int kTabBytes = 8 * kTabPages;
__device__ __forceinline__ int tab_span(const AttnArgs &a) {
    return (int)(min((kTabPages - 1) * (long long)a.d.block_size, (long long)kMaxChunk) / 128 * 128);
}
template <int DT>
struct PageTab {
    int b[(kTabPages + 255) / 256], n;
    __device__ __forceinline__ void ask(const AttnArgs &a, int r, int j0, int j1) {
        const int page0 = (int)page_of((uint32_t)j0, a.d.div);
        n = (int)page_of((uint32_t)(j1 - 1), a.d.div) - page0 + 1;
#pragma unroll
        for (int i = 0; i < (kTabPages + 255) / 256; ++i) {
            const int p = (int)threadIdx.x + 256 * i;
            b[i] = p < n ? a.tables[(size_t)r * a.max_blocks + page0 + p] : 0;
        }
    }
    __device__ __forceinline__ bool fill(const AttnArgs &a, uint64_t *s_tab) const {
        bool bad = false;
        __syncthreads();  // the last table has been read
#pragma unroll
        for (int i = 0; i < (kTabPages + 255) / 256; ++i) {
            const int p = (int)threadIdx.x + 256 * i;
            const bool ok = b[i] >= 0 && b[i] < a.d.n_blocks;
            bad |= p < n && !ok;
            if (p < n) s_tab[p] = ok ? (uint64_t)b[i] * a.d.block_stride * (DT == RBT_DT_BF16 ? 2 : 4) : 1;
        }
        return __builtin_amdgcn_readfirstlane(__syncthreads_or(bad)) != 0;
    }
};
// Where a position's row of a head (head_off: the head's bytes in a block) lies in the cache.
template <int DT>
__device__ __forceinline__ uint64_t row_at(const AttnArgs &a, const uint64_t *s_tab, int page0, uint32_t head_off, int pos) {
    const int page = (int)page_of((uint32_t)pos, a.d.div);
    const uint32_t in = (uint32_t)(pos - page * a.d.block_size) * (uint32_t)(a.d.hd * (DT == RBT_DT_BF16 ? 2 : 4));
    return (s_tab[page - page0] & ~(uint64_t)15) + (head_off + in);
}
template <int DT>
__device__ __forceinline__ uint32_t head_offset(const AttnArgs &a, int kvh) {
    return (uint32_t)kvh * (uint32_t)a.d.block_size * (uint32_t)(a.d.hd * (DT == RBT_DT_BF16 ? 2 : 4));
}

// Staging of KEYS positions from j on (those past last repeat it) by THREADS threads: 16-byte chunks of 8 elements
// through registers, so that a tile's loads run during the arithmetic of the one before.
// ONCE: keys and values that one block alone reads stream past the caches.
template <bool ONCE>
__device__ __forceinline__ u32x4 ld_kv(const uint8_t *p) {
    return ONCE ? ld_stream_u4(p) : *reinterpret_cast<const u32x4 *>(p);
}
template <int DT, int HDP, int KEYS, int THREADS, bool ONCE>
struct Stage {
    static constexpr int CH = HDP / 8, ROWS = THREADS / CH, N = KEYS / ROWS;
    static constexpr int LD = DT == RBT_DT_BF16 ? 1 : 2;
    static_assert(N * ROWS == KEYS, "whole passes");
    u32x4 k[N][LD], v[N][LD];
    PartConsts pc;

    template <bool K, bool V>
    __device__ __forceinline__ void load(const AttnArgs &a, const uint64_t *s_tab, int page0, int kvh, int j, int last,
                                         int tid) {
        const int row = tid / CH, chunk = min(tid % CH, a.d.hd / 8 - 1);  // behind the head's end: its last chunk
        const uint32_t head_off = head_offset<DT>(a, kvh);
        constexpr size_t esz = DT == RBT_DT_BF16 ? 2 : 4;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint64_t at = row_at<DT>(a, s_tab, page0, head_off, min(j + row + i * ROWS, last)) + 8 * chunk * esz;
#pragma unroll
            for (int x = 0; x < LD; ++x) {
                if (K) k[i][x] = ld_kv<ONCE>(static_cast<const uint8_t *>(a.kc) + at + 16 * x);
                if (V) v[i][x] = ld_kv<ONCE>(static_cast<const uint8_t *>(a.vc) + at + 16 * x);
            }
        }
    }
    __device__ __forceinline__ void put(const u32x4 (&r)[LD], int off, int part) {
        if constexpr (DT == RBT_DT_BF16) {
            *reinterpret_cast<u32x4 *>(smem + off) = r[0];
        } else {
            float x[8];
            u32x4 p[3];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(r[i / 4][i % 4]);
            split3(x, p, pc);
#pragma unroll
            for (int y = 0; y < 3; ++y) *reinterpret_cast<u32x4 *>(smem + off + y * part) = p[y];
        }
    }
    __device__ __forceinline__ void store(const u32x4 (&r)[N][LD], int to, int part, int tid) {
        const int at = to + tid / CH * PaddedTile<HDP>::ROW + 16 * (tid % CH);
#pragma unroll
        for (int i = 0; i < N; ++i) put(r[i], at + i * ROWS * PaddedTile<HDP>::ROW, part);
    }
};

// The same for a bf16 tile of a block's four waves as direct copies into LDS (SwizzledTile), not waited for. A head dim
// below HDP: the chunks behind it repeat its last (the query's are 0, and the output's are not stored).
template <int HDP, int KEYS>
struct TileCopy {
    using Tile = SwizzledTile<HDP>;
    static constexpr int ROWS = 64 / Tile::CH, N = KEYS / 4 / ROWS;  // rows per copy
    static_assert(N * 4 * ROWS == KEYS, "whole copies");
    uint64_t at[N];
    uint32_t lds0, in[N];
    __device__ __forceinline__ TileCopy() {
        const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)smem + (uint32_t)(wv * N * ROWS * Tile::ROW);
    }
    // The places of the tile from position j on, in two steps: the table is asked, its answers used.
    __device__ __forceinline__ void look(const AttnArgs &a, const uint64_t *s_tab, int page0, uint32_t head_off, int j,
                                         int last) {
        const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = (wv * N + i) * ROWS + lane / Tile::CH, pos = min(j + row, last);
            const int chunk = min((lane % Tile::CH) ^ Tile::key(row), a.d.hd / 8 - 1), page = (int)page_of((uint32_t)pos, a.d.div);
            in[i] = head_off + (uint32_t)(pos - page * a.d.block_size) * (uint32_t)(2 * a.d.hd) + 16u * (uint32_t)chunk;
            at[i] = s_tab[page - page0];
        }
    }
    __device__ __forceinline__ void aim() {
#pragma unroll
        for (int i = 0; i < N; ++i) at[i] = (at[i] & ~(uint64_t)15) + in[i];
    }
    __device__ __forceinline__ void copies(const AttnArgs &a, int buf) const {
#pragma unroll
        for (int i = 0; i < 2 * N; ++i)
            lds_dma16(static_cast<const uint8_t *>(i & 1 ? a.vc : a.kc) + at[i / 2],
                      lds0 + (uint32_t)(buf + ((i & 1) * KEYS + i / 2 * ROWS) * Tile::ROW));
    }
};

// A row's place: its token and head.
struct Place {
    int t, h, pos;
};
__device__ __forceinline__ Place place(const AttnArgs &a, const Request &q, int kvh, int row) {
    const int G = (int)a.group.d, tok = (int)page_of((uint32_t)row, a.group);
    return {q.t0 + tok, kvh * G + row - tok * G, q.p0 + tok};
}

// One of them.
struct Item {
    Request q;
    Cut cut;
    int r, kvh, row0, n_rows, pa, pb, k0, k1;  // rows row0 .. row0 + n_rows - 1 at positions pa .. pb; piece [k0, k1)
    bool split;                                // whether the tile has more than this piece
    float *unit;                               // the piece's partials
};
template <bool THIN, int HDP>
__device__ __forceinline__ Item item_of(const AttnArgs &a, int it, int chunk, const int32_t *s_items,
                                        const int32_t *s_units) {
    constexpr int tr = kTileRows<THIN>;
    Item x;
    // the same for all threads, told to the compiler
    x.r = __builtin_amdgcn_readfirstlane(request_of(s_items, a.n_req, it));
    x.q = request(a, x.r);
    x.cut = cut_of<THIN>(a, x.q, chunk);
    int local = it - __builtin_amdgcn_readfirstlane(s_items[x.r]);
    // With a multiple of eight heads each eighth of the items has its own heads.
    const int hx = a.d.n_kv % 8 == 0 ? a.d.n_kv / 8 : a.d.n_kv;
    const int pieces = (int)pieces_before<THIN>(x.cut, x.cut.nt), group = local / (pieces * hx);
    local -= group * pieces * hx;
    x.kvh = group * hx + local % hx;
    local /= hx;
    const TilePiece tp = tile_piece<THIN>(x.cut, local);
    const int tile = tp.tile, c = tp.piece;
    x.row0 = tile * tr;
    x.n_rows = min(tr, x.cut.rows - x.row0);
    x.pa = place(a, x.q, x.kvh, x.row0).pos;
    x.pb = place(a, x.q, x.kvh, x.row0 + x.n_rows - 1).pos;
    const int lo = a.window > 0 ? max(0, x.pa - a.window + 1) : 0, end = max(x.pb + 1, lo);
    const Pieces pc = pieces_of<THIN>(x.cut, tile);
    x.k0 = (int)min((long long)lo + (long long)c * pc.len, (long long)end);
    x.k1 = x.k0 + min(pc.len, end - x.k0);
    x.split = pc.n > 1;
    x.unit = AttnWs<THIN>::partials(a.ws) +
             ((size_t)__builtin_amdgcn_readfirstlane(s_units[x.r]) +
              ((size_t)x.kvh * pieces + (size_t)pieces_before<THIN>(x.cut, tile) + c) * (tr / 16)) * unit_floats(HDP);
    return x;
}
// An eighth of the items to each XCD (blocks b % 8): with a multiple of eight heads, or an item per block at most, a run
// of them, so that a head's row tiles read its keys and values through one L2; otherwise every eighth item, so that each
// XCD gets large and small ones (prompt of 2048, 8 heads of 256 on 2: 175 us, 255 by runs; 2000 positions, 16 on 4: 77
// and 88; three chunks of 333, 16 heads of 64 on 4: 43.7 and 40.6). A block starts with the item of its own number and, where there are more items than blocks, then takes the next
// one left of its eighth, then of the other eighths: ask() early, its answer used by next() at the item's end.
struct ItemQueue {
    int it, n, xcd, per;  // it < 0: nothing is left
    bool runs, more;
    AttnHeader *hdr;
    __device__ __forceinline__ int start(int x) const { return (int)((long long)n * x / 8); }
    __device__ __forceinline__ int count(int x) const { return runs ? start(x + 1) - start(x) : (n - x + 7) >> 3; }
    __device__ __forceinline__ int item(int x, int k) const { return runs ? start(x) + k : x + 8 * k; }
    __device__ __forceinline__ ItemQueue(int n_items, int n_kv, AttnHeader *header, int block, int blocks)
        : n(n_items), xcd(block & 7), per(blocks >> 3), runs(n_kv % 8 == 0 || n_items <= blocks), more(n_items > blocks), hdr(header) {
        it = (block >> 3) < count(xcd) ? item(xcd, block >> 3) : -1;
    }
    __device__ __forceinline__ int ask() const { return more && threadIdx.x == 0 ? atomicAdd(&hdr->taken[xcd][0], 1) : 0; }
    // for all threads
    __device__ __forceinline__ void next(int ticket, int *s_next) {
        it = -1;
        while (more) {
            if (threadIdx.x < kWave) {  // the answer, or the first other eighth with any left (its counters only grow)
                const int x = threadIdx.x & 7;
                const int k = __builtin_amdgcn_readfirstlane(ticket) + per;
                int got = item(xcd, k);
                if (k >= count(xcd)) {
                    const int t = __hip_atomic_load(&hdr->taken[x][0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    const uint32_t left = (uint32_t)__ballot(per + t < count(x)) & 0xFFu;
                    got = left ? -2 - (__ffs((int)left) - 1) : -1;
                }
                if (threadIdx.x == 0) *s_next = got;
            }
            __syncthreads();
            it = __builtin_amdgcn_readfirstlane(*s_next);
            __syncthreads();
            if (it >= -1) return;
            xcd = -2 - it;
            ticket = ask();
        }
    }
};

// Which of a lane's 16 t + 4 g + i (bit 4 t + i) of 32 positions from j on the query at pos sees.
__device__ __forceinline__ uint32_t seen_bits(const AttnArgs &a, int j, int k1, int pos, const uint64_t *s_tab, int page0,
                                              bool bad) {
    const int g = (threadIdx.x & 63) >> 4;
    const int first = a.window > 0 ? pos - a.window : -1, last = min(k1 - 1, pos);
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int key = j + 16 * (e >> 2) + 4 * g + (e & 3);
        bits |= (uint32_t)((key <= last) & (key > first)) << e;
    }
    if (bad)
        for (int e = 0; e < 8; ++e) {
            const int key = min(j + 16 * (e >> 2) + 4 * g + (e & 3), k1 - 1);
            if (s_tab[(int)page_of((uint32_t)key, a.d.div) - page0] & 1) bits &= ~(1u << e);
        }
    return bits;
}

// The flagged rows of an item again, one by one.
template <int DT, int HDP>
__device__ __forceinline__ void again_rows(const AttnArgs &a, const Item &x, const int *s_flag) {
    for (int row = 0; row < x.n_rows; ++row) {
        if (!s_flag[row]) continue;  // the same for all threads
        const Place pl = place(a, x.q, x.kvh, x.row0 + row);
        const int j0 = a.window > 0 ? max(x.k0, pl.pos - a.window + 1) : x.k0;
        float m, l, o;
        row_any<DT>(a, *reinterpret_cast<RowShared *>(smem), x.r, pl.t, pl.h, j0, min(x.k1, pl.pos + 1), &m, &l, &o);
        if (x.split) {
            float *un = x.unit + (size_t)(row >> 4) * unit_floats(HDP);
            if (threadIdx.x == 0) {
                un[row & 15] = m;
                un[16 + (row & 15)] = l;
            }
            if (threadIdx.x < HDP) un[32 + (row & 15) * HDP + threadIdx.x] = (int)threadIdx.x < a.d.hd ? o : 0.0f;
        } else if ((int)threadIdx.x < a.d.hd) {
            a.out[(size_t)pl.t * a.out_stride + (size_t)pl.h * a.d.hd + threadIdx.x] = l == 0.0f ? 0.0f : o / l;
        }
    }
}

// LDS: [tile | row_any's][pages' places][item and unit prefix sums]
constexpr int kLdsBytes = 156 << 10;  // of 160 KiB: the kernels' fixed shared variables take less than the rest
constexpr int attn_lds(int tile, int n_req) { return tile + kTabBytes + 8 * (n_req + 1); }

// A thin wave on an f32 cache: v_mfma_f32_16x16x4_f32 on f32 operands straight from the cache, 16 positions at a time (a
// decoding row reads every key once: its products wait for memory whichever unit makes them, and nothing has to be
// taken apart). The layout is the bf16 one's with steps of four: S^T leaves lane (c, g) the keys 4 g + i of query c,
// the B operands of four steps of O^T = V^T P^T. K enters 16 bytes per lane (key c, dims 16 s + 4 g + i), V too (key
// 4 g + i, dims 64 h + 4 c + d).
template <int HDP>
struct ThinF32 {
    f32x4 q[HDP / 16], o[HDP / 64][4];  // o[h][d][i]: dim 64 h + 4 (4 g + i) + d
    float m, l;
    int pos;
    f32x4 k[HDP / 16], v[4][HDP / 64];  // the positions at hand; the next ones' are asked for as soon as each is used
    __device__ __forceinline__ void init(const AttnArgs &a, const Item &x) {
        const int c = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
        const Place pl = place(a, x.q, x.kvh, min(x.row0 + c, x.cut.rows - 1));
        const float *src = a.q + (size_t)pl.t * a.q_stride + (size_t)pl.h * a.d.hd;
        pos = pl.pos;
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int s = 0; s < HDP / 16; ++s) {
            const int at = min(16 * s + 4 * g, a.d.hd - 4);
            q[s] = ld_f4(src + at) * (at == 16 * s + 4 * g ? a.scale2 : 0.0f);
        }
#pragma unroll
        for (int h = 0; h < HDP / 64; ++h)
#pragma unroll
            for (int d = 0; d < 4; ++d) o[h][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __device__ __forceinline__ void load_k(const AttnArgs &a, const uint64_t *s_tab, int page0, uint32_t head_off, int j,
                                           int last) {
        const int c = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
        const uint8_t *p = static_cast<const uint8_t *>(a.kc) + row_at<RBT_DT_F32>(a, s_tab, page0, head_off, min(j + c, last));
#pragma unroll
        for (int s = 0; s < HDP / 16; ++s) k[s] = ld_stream_f4(p + 4 * min(16 * s + 4 * g, a.d.hd - 4));
    }
    __device__ __forceinline__ void load_v(const AttnArgs &a, const uint64_t *s_tab, int page0, uint32_t head_off, int j,
                                           int last) {
        const int c = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint8_t *p = static_cast<const uint8_t *>(a.vc) +
                               row_at<RBT_DT_F32>(a, s_tab, page0, head_off, min(j + 4 * g + i, last));
#pragma unroll
            for (int h = 0; h < HDP / 64; ++h) v[i][h] = ld_stream_f4(p + 4 * min(64 * h + 4 * c, a.d.hd - 4));
        }
    }
    // seen(): bit i, whether the lane's query sees key 4 g + i; then_k, then_v: called when the keys, the values
    // have been used
    template <typename Seen, typename ThenK, typename ThenV>
    __device__ __forceinline__ void step(bool full, Seen seen, ThenK then_k, ThenV then_v) {
        f32x4 s2[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int s = 0; s < HDP / 16; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) s2[i & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[s][i], q[s][i], s2[i & 1], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        then_k();
        f32x4 s = s2[0] + s2[1];
        if (!full) {
            const uint32_t bits = seen();
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = bits >> i & 1 ? s[i] : -INFINITY;
        }
        const float top = fmaxf(fmaxf(s.x, s.y), fmaxf(s.z, s.w));
        if (__any(top > m + 8.0f)) {  // as attn_step's
            const float mx = fmaxf(m, group_max(top)), f = m == -INFINITY ? 0.0f : exp2f(m - mx);
            m = mx;
            l *= f;
#pragma unroll
            for (int h = 0; h < HDP / 64; ++h)
#pragma unroll
                for (int d = 0; d < 4; ++d) o[h][d] *= f;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float p = __builtin_amdgcn_exp2f(s[i] - ref);
            l += p;
#pragma unroll
            for (int h = 0; h < HDP / 64; ++h)
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    o[h][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][h][d], p, o[h][d], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        then_v();
    }
};

// Requests of up to 16 rows.
template <int DT, int HDP>
struct ThinShape {
    static constexpr int ROWS = kThinRows * (HDP + 4) * 4;  // a wave's rows, when the waves' states are joined
    static constexpr int WAVE = DT == RBT_DT_BF16 ? 2 * 32 * PaddedTile<HDP>::ROW : ROWS;  // bf16: keys and values before
    static constexpr int TILE = 4 * WAVE;
    static constexpr int PER_CU = HDP <= 128 ? 2 : 1;  // blocks that share a CU
    static_assert(ROWS <= WAVE, "a wave's rows fit its tile");
    static_assert(sizeof(RowShared) <= (size_t)TILE, "row_any's LDS");
};
// Blocks `block` of `blocks`, a multiple of eight.
template <int DT, int HDP>
__device__ __forceinline__ void attn_thin(const AttnArgs &a, int block, int blocks) {
    constexpr int WAVE = ThinShape<DT, HDP>::WAVE;
    __shared__ ScheduleShared s_sched;
    __shared__ float s_m[4][kThinRows], s_l[4][kThinRows];
    __shared__ int s_flag[kThinRows], s_next;
    uint64_t *s_tab = reinterpret_cast<uint64_t *>(smem + ThinShape<DT, HDP>::TILE);
    int32_t *s_items = reinterpret_cast<int32_t *>(s_tab + kTabPages), *s_units = s_items + a.n_req + 1;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const int chunk = __builtin_amdgcn_readfirstlane(schedule<true, HDP>(a, block, blocks, s_items, s_units, s_sched));
    if (chunk == 0) return;
    ItemQueue items(__builtin_amdgcn_readfirstlane(s_items[a.n_req]), a.d.n_kv, AttnWs<true>::header(a.ws), block, blocks);
    const int span = tab_span(a);
    const PaddedTile<HDP> tl;
    while (items.it >= 0) {
        const Item x = item_of<true, HDP>(a, items.it, chunk, s_items, s_units);
        const int ticket = items.ask();
        PageTab<DT> tab;
        if (x.k0 < x.k1) tab.ask(a, x.r, x.k0, x.k0 + min(span, x.k1 - x.k0));
        // fn(w0, w1, page0, bad) over the stretches of the piece that the table holds
        auto stretches = [&](auto fn) {
            for (int w0 = x.k0, w1; w0 < x.k1; w0 = w1) {
                w1 = w0 + min(span, x.k1 - w0);
                if (w0 != x.k0) tab.ask(a, x.r, w0, w1);
                const bool bad = tab.fill(a, s_tab);
                fn(w0, w1, (int)page_of((uint32_t)w0, a.d.div), bad);
            }
        };
        auto whole = [&](int j, int n, int w1, bool bad) {  // whether all rows see all of n positions from j on
            return !bad && j + n <= min(w1, x.pa + 1) && (a.window <= 0 || j > x.pb - a.window);
        };
        const int at = wv * WAVE;
        // each wave's state, and its rows where its tile was
        if constexpr (DT == RBT_DT_BF16) {
            WaveState<HDP, 1> w;
            wave_init(w, a, x.q, x.cut.rows, x.kvh, x.row0, 0);
            const int v_off = at + 32 * PaddedTile<HDP>::ROW;
            stretches([&](int w0, int w1, int page0, bool bad) {
                Stage<DT, HDP, 32, 64, true> st;
                int j = w0 + 32 * wv;
                if (j < w1) st.template load<true, true>(a, s_tab, page0, x.kvh, j, w1 - 1, lane);
                for (; j < w1; j += 128) {
                    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
                    st.store(st.k, at, 0, lane);
                    st.store(st.v, v_off, 0, lane);
                    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
                    if (j + 128 < w1) st.template load<true, true>(a, s_tab, page0, x.kvh, j + 128, w1 - 1, lane);
                    attn_step<HDP, 1, 3, 1, 0>(w, tl, at, v_off, whole(j, 32, w1, bad), [](int) {},
                                               [&](int n) { return seen_bits(a, j, w1, w.pos[n], s_tab, page0, bad); },
                                               NoMid());
                }
            });
            w.l[0] = group_sum(w.l[0]);
            if (g == 0) {
                s_m[wv][c] = w.m[0];
                s_l[wv][c] = w.l[0];
            }
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll
            for (int d = 0; d < HDP / 16; ++d)
                *reinterpret_cast<f32x4 *>(smem + at + (c * (HDP + 4) + 16 * d + 4 * g) * 4) = w.o[0][d];
        } else {
            ThinF32<HDP> w;
            w.init(a, x);
            const uint32_t head_off = head_offset<DT>(a, x.kvh);
            stretches([&](int w0, int w1, int page0, bool bad) {
                int j = w0 + 16 * wv;
                if (j < w1) {
                    w.load_k(a, s_tab, page0, head_off, j, w1 - 1);
                    w.load_v(a, s_tab, page0, head_off, j, w1 - 1);
                }
                for (; j < w1; j += 64)
                    w.step(whole(j, 16, w1, bad), [&]() { return seen_bits(a, j, w1, w.pos, s_tab, page0, bad); },
                           [&]() { if (j + 64 < w1) w.load_k(a, s_tab, page0, head_off, j + 64, w1 - 1); },
                           [&]() { if (j + 64 < w1) w.load_v(a, s_tab, page0, head_off, j + 64, w1 - 1); });
            });
            w.l = group_sum(w.l);
            if (g == 0) {
                s_m[wv][c] = w.m;
                s_l[wv][c] = w.l;
            }
#pragma unroll
            for (int h = 0; h < HDP / 64; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<f32x4 *>(smem + at + (c * (HDP + 4) + 64 * h + 16 * g + 4 * i) * 4) =
                        f32x4{w.o[h][0][i], w.o[h][1][i], w.o[h][2][i], w.o[h][3][i]};
        }
        if (tid < kThinRows) s_flag[tid] = 0;
        __syncthreads();
        const int row = tid >> 4, y = tid & 15;
        float M = -INFINITY, L = 0.0f, wt[4];
#pragma unroll
        for (int z = 0; z < 4; ++z) M = fmaxf(M, s_m[z][row]);
#pragma unroll
        for (int z = 0; z < 4; ++z) {
            wt[z] = state_weight(s_m[z][row], M);
            L += wt[z] * s_l[z][row];
        }
        f32x4 o[HDP / 64];
        float nan = 0.0f * L;
#pragma unroll
        for (int u = 0; u < HDP / 64; ++u) {
            o[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int z = 0; z < 4; ++z)
                o[u] += wt[z] * *reinterpret_cast<const f32x4 *>(smem + z * WAVE + (row * (HDP + 4) + 64 * u + 4 * y) * 4);
            nan += 0.0f * ((o[u].x + o[u].y) + (o[u].z + o[u].w));
        }
        const bool again = ((__ballot(nan != 0.0f) >> (lane & 48)) & 0xFFFFu) != 0;
        if (row < x.n_rows) {
            if (again) {
                if (y == 0) s_flag[row] = 1;
            } else if (x.split) {
                if (y == 0) {
                    x.unit[row] = M;
                    x.unit[16 + row] = L;
                }
#pragma unroll
                for (int u = 0; u < HDP / 64; ++u)
                    *reinterpret_cast<f32x4 *>(x.unit + 32 + row * HDP + 64 * u + 4 * y) = o[u];
            } else {
                const Place pl = place(a, x.q, x.kvh, x.row0 + row);
                float *dst = a.out + (size_t)pl.t * a.out_stride + (size_t)pl.h * a.d.hd;
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
                for (int u = 0; u < HDP / 64; ++u)
                    if (64 * u + 4 * y < a.d.hd) *reinterpret_cast<f32x4 *>(dst + 64 * u + 4 * y) = o[u] * inv;
            }
        }
        if (__syncthreads_or(again && row < x.n_rows)) again_rows<DT, HDP>(a, x, s_flag);
        items.next(ticket, &s_next);
    }
}

// The other requests.
template <int DT, int HDP>
struct WideShape {
    static constexpr int NP = DT == RBT_DT_BF16 ? 1 : 3;
    // bf16: two buffers of keys and values that direct copies fill in turn; f32: one of parts, through registers, of
    // the keys and then of the values, which leaves room for the query rows' third part (prompt of 4096 tokens, 16 heads
    // of 128: 414 us; both at once, the queries in registers, 78 of them spilled: 436; heads of 64: 134 against 130)
    static constexpr bool COPY = DT == RBT_DT_BF16;
    using Tile = std::conditional_t<COPY, SwizzledTile<HDP>, PaddedTile<HDP>>;
    static constexpr int PART = 32 * Tile::ROW, BUF = (COPY ? 2 : 1) * NP * PART;
    // there are registers for two of the query rows' three parts; the third in LDS, where it fits
    static constexpr int QP = HDP == 128 || (!COPY && HDP == 256) ? 2 : 3, Q_AT = COPY ? 2 * BUF : BUF;
    static constexpr int TILE = Q_AT + (QP < 3 ? kWideRows * PaddedTile<HDP>::ROW : 0);
    static constexpr int PER_CU = HDP <= 128 ? 2 : 1;
    static_assert(sizeof(RowShared) <= (size_t)TILE, "row_any's LDS");
};
template <int DT, int HDP>
__device__ __forceinline__ void attn_wide(const AttnArgs &a, int block, int blocks) {
    using Sh = WideShape<DT, HDP>;
    __shared__ ScheduleShared s_sched;
    __shared__ int s_flag[kWideRows], s_next;
    uint64_t *s_tab = reinterpret_cast<uint64_t *>(smem + Sh::TILE);
    int32_t *s_items = reinterpret_cast<int32_t *>(s_tab + kTabPages), *s_units = s_items + a.n_req + 1;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const int chunk = __builtin_amdgcn_readfirstlane(schedule<false, HDP>(a, block, blocks, s_items, s_units, s_sched));
    if (chunk == 0) return;
    ItemQueue items(__builtin_amdgcn_readfirstlane(s_items[a.n_req]), a.d.n_kv, AttnWs<false>::header(a.ws), block, blocks);
    const int span = tab_span(a);
    const typename Sh::Tile tl;
    while (items.it >= 0) {
        const Item x = item_of<false, HDP>(a, items.it, chunk, s_items, s_units);
        const int ticket = items.ask();
        const int wr0 = x.row0 + 32 * wv;
        const bool active = 32 * wv < x.n_rows;
        const int wa = place(a, x.q, x.kvh, min(wr0, x.cut.rows - 1)).pos,
                  wb = place(a, x.q, x.kvh, min(wr0 + 31, x.cut.rows - 1)).pos;
        WaveState<HDP, 2, Sh::QP> w;
        PageTab<DT> tab;
        if (x.k0 < x.k1) tab.ask(a, x.r, x.k0, x.k0 + min(span, x.k1 - x.k0));
        wave_init(w, a, x.q, x.cut.rows, x.kvh, wr0, Sh::Q_AT + 32 * wv * PaddedTile<HDP>::ROW);
        for (int w0 = x.k0, w1; w0 < x.k1; w0 = w1) {
            w1 = w0 + min(span, x.k1 - w0);
            const int page0 = (int)page_of((uint32_t)w0, a.d.div);
            if (w0 != x.k0) tab.ask(a, x.r, w0, w1);
            const bool bad = tab.fill(a, s_tab);
            // the wave's part of 32 staged positions from j on: whether it has any
            auto step = [&](int j, int off, auto between, auto mid) {
                if (!active || j >= w1 || j > wb || (a.window > 0 && j + 31 <= wa - a.window)) return false;
                const bool full = !bad && j + 32 <= min(w1, wa + 1) && (a.window <= 0 || j > wb - a.window);
                attn_step<HDP, 2, Sh::QP, Sh::NP, Sh::PART>(
                    w, tl, off, Sh::COPY ? off + Sh::PART : off, full, between,
                    [&](int n) { return seen_bits(a, j, w1, w.pos[n], s_tab, page0, bad); }, mid);
                return true;
            };
            if constexpr (Sh::COPY) {
                // A tile's copies are made a step ahead, and the places of the tile after it are looked up
                // among the products of that step.
                TileCopy<HDP, 32> cp;
                const uint32_t head_off = head_offset<DT>(a, x.kvh);
                auto look = [&](int j) { cp.look(a, s_tab, page0, head_off, j, w1 - 1); };
                look(w0);
                cp.aim();
                cp.copies(a, 0);
                look(w0 + 32);
                cp.aim();
                int buf = 0;
                for (int j = w0; j < w1; j += 32) {
                    wait_dma<0>();
                    __syncthreads();  // this tile has landed for all, and the last one has been read
                    if (j + 32 < w1) cp.copies(a, buf ^ Sh::BUF);
                    const bool done = step(j, buf, [&](int i) {
                        if (i == 0) look(j + 64);
                        if (i == 2) cp.aim();
                    }, NoMid());
                    if (!done) {
                        look(j + 64);
                        cp.aim();
                    }
                    buf ^= Sh::BUF;
                }
            } else {
                Stage<DT, HDP, 32, 256, false> st;
                st.template load<true, false>(a, s_tab, page0, x.kvh, w0, w1 - 1, tid);
                for (int jt = w0; jt < w1; jt += 32) {
                    __syncthreads();
                    st.store(st.k, 0, Sh::PART, tid);
                    st.template load<false, true>(a, s_tab, page0, x.kvh, jt, w1 - 1, tid);
                    __syncthreads();
                    auto values = [&]() {
                        __syncthreads();  // the keys have been read
                        st.store(st.v, 0, Sh::PART, tid);
                        if (jt + 32 < w1) st.template load<true, false>(a, s_tab, page0, x.kvh, jt + 32, w1 - 1, tid);
                        __syncthreads();
                    };
                    if (!step(jt, 0, [](int) {}, values)) values();
                }
            }
        }
        if (tid < kWideRows) s_flag[tid] = 0;
        __syncthreads();
        bool any = false;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int row = 32 * wv + 16 * n + c;
            const float L = group_sum(w.l[n]);
            float nan = 0.0f * L;
#pragma unroll
            for (int d = 0; d < HDP / 16; ++d)
                nan += 0.0f * ((w.o[n][d].x + w.o[n][d].y) + (w.o[n][d].z + w.o[n][d].w));
            const bool again = ((__ballot(nan != 0.0f) >> c) & 0x0001000100010001ull) != 0;
            if (row >= x.n_rows) continue;
            if (again) {
                s_flag[row] = 1;
                any = true;
            } else if (x.split) {
                float *un = x.unit + (size_t)(row >> 4) * unit_floats(HDP);
                if (g == 0) {
                    un[c] = w.m[n];
                    un[16 + c] = L;
                }
#pragma unroll
                for (int d = 0; d < HDP / 16; ++d)
                    *reinterpret_cast<f32x4 *>(un + 32 + c * HDP + 16 * d + 4 * g) = w.o[n][d];
            } else {
                const Place pl = place(a, x.q, x.kvh, x.row0 + row);
                float *dst = a.out + (size_t)pl.t * a.out_stride + (size_t)pl.h * a.d.hd + 4 * g;
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
                for (int d = 0; d < HDP / 16; ++d)
                    if (16 * d + 4 * g < a.d.hd) *reinterpret_cast<f32x4 *>(dst + 16 * d) = w.o[n][d] * inv;
            }
        }
        if (__syncthreads_or(any)) again_rows<DT, HDP>(a, x, s_flag);
        items.next(ticket, &s_next);
    }
}

// One launch of both: the wide blocks first, which leave at once where no request is theirs; the thin ones fill the
// places that the last wide ones leave (prompts and decoding rows mixed: 29.5 us, 33.6 in two launches; 32 decoding
// sequences: 69.5 and 68.2).
template <int DT, int HDP>
struct AttnShape {
    static constexpr int TILE = std::max(WideShape<DT, HDP>::TILE, ThinShape<DT, HDP>::TILE);
    static constexpr int PER_CU = WideShape<DT, HDP>::PER_CU, BLOCKS = 256 * PER_CU;
    static_assert(PER_CU == ThinShape<DT, HDP>::PER_CU, "one launch bound");
};
template <int DT, int HDP>
__global__ __launch_bounds__(256, (AttnShape<DT, HDP>::PER_CU)) void attn_kernel(AttnArgs a) {
    constexpr int n = AttnShape<DT, HDP>::BLOCKS;
    const int b = (int)blockIdx.x;
    if (b < a.wide * n)
        attn_wide<DT, HDP>(a, b, n);
    else
        attn_thin<DT, HDP>(a, b - a.wide * n, n);
}

// The pieces of cut tiles joined: out = sum_i w_i o_i / sum_i w_i l_i with w_i = 2^(m_i - max m), HDP / 4 lanes to a row.
template <int HDP, bool THIN>
__device__ __forceinline__ void merge_block(const AttnArgs &a, const AttnHeader *hdr, int id, float (*s_state)[4][2],
                                            f32x4 (*s_o)[64]) {
    constexpr int tr = kTileRows<THIN>, tru = tr / 16, LPR = HDP / 4, RPW = 64 / LPR;
    constexpr size_t step = (size_t)tru * unit_floats(HDP);
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, sub = lane % LPR;
    const int r = __builtin_amdgcn_readfirstlane(request_of(hdr->merge, a.n_req, id)), chunk = hdr->chunk;
    const Request q = request(a, r);
    const Cut cut = cut_of<THIN>(a, q, chunk);
    const bool dealt = cut.nc >= kMergeManyPieces;  // the same for the whole block
    const int all = cut.rows * a.d.n_kv, mine = (id - hdr->merge[r]) * merge_rows<HDP>(cut.nc) +
                                                (dealt ? 0 : wv * RPW) + lane / LPR;
    const int at = min(mine, all - 1), kvh = at / cut.rows, row = at - kvh * cut.rows, tile = row / tr;
    const int in = row - tile * tr;
    const int nc = pieces_of<THIN>(cut, tile).n;
    const float *u = AttnWs<THIN>::partials(a.ws) +
                     ((size_t)hdr->units[r] + ((size_t)kvh * (size_t)pieces_before<THIN>(cut, cut.nt) +
                                               (size_t)pieces_before<THIN>(cut, tile)) * tru + (in >> 4)) * unit_floats(HDP) +
                     (in & 15);
    const float *uo = u - (in & 15) + 32 + (in & 15) * HDP + 4 * sub;
    const int i0 = dealt ? wv : 0, by = dealt ? 4 : 1;
    float M = -INFINITY;
    for (int i = i0 + by * sub; i < nc; i += by * LPR) M = fmaxf(M, u[i * step]);
    for (int x = 1; x < LPR; x <<= 1) M = fmaxf(M, __shfl_xor(M, x, 64));
    float L = 0.0f;
    f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int kU = 4;  // pieces in flight
    for (int i = i0; i < nc; i += kU * by) {
        float m[kU], l[kU];
        f32x4 v[kU];
#pragma unroll
        for (int y = 0; y < kU; ++y) {
            const size_t p = (size_t)min(i + y * by, nc - 1) * step;
            m[y] = u[p];
            l[y] = u[p + 16];
            v[y] = ld_f4(uo + p);
        }
#pragma unroll
        for (int y = 0; y < kU; ++y)
            if (i + y * by < nc) {
                const float w = state_weight(m[y], M);
                L += w * l[y];
                o += w * v[y];
            }
    }
    if (dealt) {
        __syncthreads();  // the last states have been read
        if (sub == 0) {
            s_state[wv][lane / LPR][0] = M;
            s_state[wv][lane / LPR][1] = L;
        }
        s_o[wv][lane] = o;
        __syncthreads();
        if (wv != 0) return;
        float Mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) Mx = fmaxf(Mx, s_state[w][lane / LPR][0]);
        L = 0.0f;
        o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float x = state_weight(s_state[w][lane / LPR][0], Mx);
            L += x * s_state[w][lane / LPR][1];
            o += x * s_o[w][lane];
        }
    }
    // a tile of a cut request that is not cut itself was written by its block
    if (mine >= all || nc == 1 || 4 * sub >= a.d.hd) return;
    const Place pl = place(a, q, kvh, row);
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    *reinterpret_cast<f32x4 *>(a.out + (size_t)pl.t * a.out_stride + (size_t)pl.h * a.d.hd + 4 * sub) = o * inv;
}
template <int HDP>
__global__ __launch_bounds__(256) void attn_merge_kernel(AttnArgs a) {
    __shared__ float s_state[4][4][2];
    __shared__ f32x4 s_o[4][64];
    AttnHeader *hw = AttnWs<false>::header(a.ws), *ht = AttnWs<true>::header(a.ws);
    if (blockIdx.x == 0 && threadIdx.x < 8) hw->taken[threadIdx.x][0] = ht->taken[threadIdx.x][0] = 0;
    const int nw = a.wide ? hw->merge_blocks : 0, nt = a.thin ? ht->merge_blocks : 0;
    for (int id = blockIdx.x; id < nw + nt; id += gridDim.x)
        if (id < nt)
            merge_block<HDP, true>(a, ht, id, s_state, s_o);
        else
            merge_block<HDP, false>(a, hw, id - nt, s_state, s_o);
}

__global__ void attn_clear_kernel(uint8_t *ws) {
    if (threadIdx.x < 8)
        AttnWs<false>::header(ws)->taken[threadIdx.x][0] = AttnWs<true>::header(ws)->taken[threadIdx.x][0] = 0;
}

// Rows ids[i] of x in turn: the last new token of each request, for its logits. A block to a row.
__global__ __launch_bounds__(256) void gather_rows_kernel(const float *x, const int32_t *ids, int D, float *out) {
    const float *src = x + (size_t)ids[blockIdx.x] * D;
    for (int i = threadIdx.x; i < D; i += 256) out[(size_t)blockIdx.x * D + i] = src[i];
}

PagedDims dims_of(const rbt_paged_kv &kv) {
    PagedDims d;
    d.n_blocks = kv.n_blocks;
    d.block_size = kv.block_size;
    d.n_kv = kv.n_kv_heads;
    d.hd = kv.head_dim;
    d.block_stride = kv.block_stride ? kv.block_stride
                                     : (uint64_t)kv.n_kv_heads * (uint64_t)kv.block_size * (uint64_t)kv.head_dim;
    d.div = page_div(kv.block_size);
    return d;
}

}  // namespace

namespace {
PlanArgs plan_args(const rbt_paged_plan &p) {
    PlanArgs a;
    a.n_req = p.n_req;
    a.max_blocks = p.max_blocks;
    a.n_blocks = p.n_blocks;
    a.max_tokens = p.max_tokens;
    a.div = page_div(p.block_size);
    a.len = p.len;
    a.new_len = p.new_len;
    a.n_free = p.n_free;
    a.tables = p.tables;
    a.free_list = p.free_list;
    a.kv_len = p.kv_len;
    a.n_free_out = p.n_free_out;
    a.q_start = p.q_start;
    a.slots = p.slots;
    a.positions = p.positions;
    a.status = p.status;
    return a;
}
}  // namespace

hipError_t launch_paged_plan(const Launch &L, const rbt_paged_plan &p) {
    return launch(L, plan_kernel, dim3(1), dim3(kPlanThreads), 0, plan_args(p), (int)(p.max_tokens <= kPlanRowsInOne));
}
hipError_t launch_paged_plan_rows(const Launch &L, const rbt_paged_plan &p) {
    return launch(L, plan_rows_kernel, dim3((unsigned)(((int64_t)p.max_tokens + 255) / 256)), dim3(256), 0, plan_args(p));
}

hipError_t launch_paged_append(const Launch &L, const rbt_paged_kv &kv, const rbt_paged_rows &w) {
    if (w.n_tokens < 1) return hipSuccess;
    AppendArgs a;
    a.d = dims_of(kv);
    const uint64_t qd = (uint64_t)w.n_heads * (uint64_t)kv.head_dim, kvd = (uint64_t)kv.n_kv_heads * (uint64_t)kv.head_dim;
    a.n_heads = w.n_heads;
    a.n_rope = w.n_rope;
    a.q = w.q;
    a.k = w.k;
    a.v = w.v;
    a.q_stride = w.q_stride ? w.q_stride : qd;
    a.k_stride = w.k_stride ? w.k_stride : kvd;
    a.v_stride = w.v_stride ? w.v_stride : kvd;
    a.q_out = w.q_out;
    a.q_norm = w.q_norm;
    a.k_norm = w.k_norm;
    a.eps = w.eps;
    a.rope = reinterpret_cast<const float2 *>(w.rope);
    a.positions = w.positions;
    a.slots = w.slots;
    a.kc = kv.k;
    a.vc = kv.v;
    const dim3 g((unsigned)w.n_tokens);
    const auto a16 = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    if (kv.head_dim % 8 == 0 && qd <= 2048 * kAppendQ && kvd <= 2048 * kAppendK && a16(w.q) && a16(w.k) && a16(w.v) &&
        a16(w.q_out) && a16(w.q_norm) && a16(w.k_norm) && a16(w.rope) && a16(kv.k) && a16(kv.v) && a.q_stride % 4 == 0 &&
        a.k_stride % 4 == 0 && a.v_stride % 4 == 0 && a.d.block_stride % 4 == 0) {
        if (qd <= 2048 && kvd <= 2048)
            return kv.dtype == RBT_DT_BF16 ? launch(L, append_quads_kernel<RBT_DT_BF16, 1, 1>, g, dim3(256), 0, a)
                                           : launch(L, append_quads_kernel<RBT_DT_F32, 1, 1>, g, dim3(256), 0, a);
        return kv.dtype == RBT_DT_BF16 ? launch(L, append_quads_kernel<RBT_DT_BF16, kAppendQ, kAppendK>, g, dim3(256), 0, a)
                                       : launch(L, append_quads_kernel<RBT_DT_F32, kAppendQ, kAppendK>, g, dim3(256), 0, a);
    }
    return kv.dtype == RBT_DT_BF16 ? launch(L, append_kernel<RBT_DT_BF16>, g, dim3(256), 0, a)
                                   : launch(L, append_kernel<RBT_DT_F32>, g, dim3(256), 0, a);
}

namespace {
AttnArgs attn_args(const PagedAttn &p) {
    AttnArgs a;
    a.d = dims_of(p.kv);
    a.n_req = p.batch.n_req;
    a.max_blocks = p.batch.max_blocks;
    a.T = p.T;
    a.n_heads = p.n_heads;
    a.window = p.window;
    a.group = page_div(p.n_heads / p.kv.n_kv_heads);
    a.thin = a.wide = 0;
    a.scale2 = p.scale * 1.44269504088896340736f;
    a.tables = p.batch.tables;
    a.kv_len = p.batch.kv_len;
    a.q_start = p.batch.q_start;
    a.kc = p.kv.k;
    a.vc = p.kv.v;
    a.q = p.q;
    a.out = p.out;
    a.q_stride = p.q_stride;
    a.out_stride = p.out_stride;
    a.ws = static_cast<uint8_t *>(p.ws);
    return a;
}

// LDS past 64 KiB has to be asked for, once per kernel and device.
template <typename F>
hipError_t ask_lds(F kernel, int bytes, std::atomic<uint64_t> &asked) {
    int dev = 0;
    const hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
    if (asked.load(std::memory_order_relaxed) & bit) return hipSuccess;
    const hipError_t f = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (f == hipSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
    return f;
}

// Which blocks a call has, and their LDS. Requests of up to 16 rows have blocks of their own, where their tiles and the
// step's prefix sums fit LDS (a bf16 cache with head dims above 128: up to 2500 requests). Blocks that no request can
// belong to are left out; otherwise each kind finds its requests on the device.
template <int DT, int HDP>
int attn_blocks(AttnArgs &a) {
    using Sh = AttnShape<DT, HDP>;
    const int G = a.n_heads / a.d.n_kv;
    a.thin = G <= kThinRows && attn_lds(Sh::TILE, a.n_req) <= kLdsBytes;
    a.wide = !a.thin || (int64_t)a.T * G > kThinRows;
    static_assert(attn_lds(WideShape<DT, HDP>::TILE, kPagedMaxReq) <= kLdsBytes, "wide blocks take any step");
    return attn_lds(a.thin ? Sh::TILE : WideShape<DT, HDP>::TILE, a.n_req);
}
template <int DT, int HDP>
hipError_t launch_attn(const Launch &L, AttnArgs a, bool merge) {
    using Sh = AttnShape<DT, HDP>;
    const int lds = attn_blocks<DT, HDP>(a);
    if (merge) {  // no more blocks than the rows need, and two rounds of them (prompt of 4096: 208 us against 213 with 1024)
        const int64_t n = (int64_t)a.T * a.n_heads / (256 / HDP) + 1;
        return launch(L, attn_merge_kernel<HDP>, dim3((unsigned)(n < 4096 ? n : 4096)), dim3(256), 0, a);
    }
    static std::atomic<uint64_t> asked{0};
    const hipError_t e = ask_lds(attn_kernel<DT, HDP>, kLdsBytes, asked);
    if (e != hipSuccess) return e;
    return launch(L, attn_kernel<DT, HDP>, dim3((unsigned)(Sh::BLOCKS * (a.wide + a.thin))), dim3(256), (uint32_t)lds, a);
}
hipError_t launch_tiled(const Launch &L, const PagedAttn &p, bool merge) {
    const AttnArgs a = attn_args(p);
    const int hd = a.d.hd;
    if (p.kv.dtype == RBT_DT_BF16)
        return hd <= 64 ? launch_attn<RBT_DT_BF16, 64>(L, a, merge)
                        : hd <= 128 ? launch_attn<RBT_DT_BF16, 128>(L, a, merge) : launch_attn<RBT_DT_BF16, 256>(L, a, merge);
    return hd <= 64 ? launch_attn<RBT_DT_F32, 64>(L, a, merge)
                    : hd <= 128 ? launch_attn<RBT_DT_F32, 128>(L, a, merge) : launch_attn<RBT_DT_F32, 256>(L, a, merge);
}
}  // namespace

// On the matrix cores: 16-byte loads everywhere, offsets within a block in 32 bits.
bool paged_attn_tiled(const PagedAttn &p) {
    const PagedDims d = dims_of(p.kv);
    const auto a16 = [](const void *x) { return (reinterpret_cast<uintptr_t>(x) & 15u) == 0; };
    const uint64_t esz = p.kv.dtype == RBT_DT_BF16 ? 2 : 4;
    return d.hd % 8 == 0 && a16(p.q) && a16(p.out) && a16(p.kv.k) && a16(p.kv.v) && p.q_stride % 4 == 0 &&
           p.out_stride % 4 == 0 && d.block_stride * esz % 16 == 0 &&
           (uint64_t)d.n_kv * (uint64_t)d.block_size * (uint64_t)d.hd * esz <= UINT32_MAX;
}

hipError_t launch_paged_attn(const Launch &L, const PagedAttn &p) {
    if (paged_attn_tiled(p)) return launch_tiled(L, p, false);
    const AttnArgs a = attn_args(p);
    const uint64_t rows = (uint64_t)p.T * (uint64_t)p.n_heads;
    const dim3 g((unsigned)(rows < 65536 ? rows : 65536));
    return p.kv.dtype == RBT_DT_BF16 ? launch(L, attn_any_kernel<RBT_DT_BF16>, g, dim3(256), 0, a)
                                     : launch(L, attn_any_kernel<RBT_DT_F32>, g, dim3(256), 0, a);
}

hipError_t launch_paged_merge(const Launch &L, const PagedAttn &p) { return launch_tiled(L, p, true); }

hipError_t launch_gather_rows(const Launch &L, const float *x, const int32_t *ids, int n, int D, float *out) {
    return launch(L, gather_rows_kernel, dim3((unsigned)n), dim3(256), 0, x, ids, D, out);
}

hipError_t launch_paged_clear(const Launch &L, void *ws) {
    return launch(L, attn_clear_kernel, dim3(1), dim3(64), 0, static_cast<uint8_t *>(ws));
}

}  // namespace rbt
