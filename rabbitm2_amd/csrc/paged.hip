// The paged key/value cache: a step's block tables and slot map from the requests' lengths, the new rows'
// QK-norm + RoPE + write into the pages, and causal attention of the new rows over the pages (include/rbt2_hip.h).
// The engine's State (rabbit2/src/rabbit2.c:427-446) holds one sequence of a fixed context; the arithmetic per
// row is its own (:472-498).
#include <math.h>

#include "paged.h"
#include "rbt2_internal.h"

namespace rbt {
namespace {

typedef __bf16 bf16_t;

// ---------------------------------------------------------------- plan
// One block: three prefix sums over the requests (new rows, blocks needed, blocks given back) in LDS, then the
// blocks pushed and popped and the rows' slots, each by its place in those sums (a binary search), so that one
// long request costs no more than many short ones. All of it is latency; the sums are 64-bit, so that no input
// can wrap them.
constexpr int kPlanThreads = 1024, kPlanPer = kPagedMaxReq / kPlanThreads;

struct PlanArgs {
    int n_req, max_blocks, n_blocks, max_tokens;
    PageDiv div;
    const int32_t *len, *new_len, *n_free;
    int32_t *tables, *free_list, *kv_len, *n_free_out, *q_start, *slots, *positions, *status;
};

// The block's exclusive prefix sums of three values per thread; tot: the sums of all.
__device__ __forceinline__ void block_scan3(long long (&v)[3], long long (&tot)[3], long long (*s_w)[3]) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    long long inc[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) inc[i] = v[i];
    for (int off = 1; off < kWave; off <<= 1)
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const long long up = __shfl_up(inc[i], off, kWave);
            if (lane >= off) inc[i] += up;
        }
    if (lane == kWave - 1)
#pragma unroll
        for (int i = 0; i < 3; ++i) s_w[wv][i] = inc[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        long long before = 0;
        tot[i] = 0;
        for (int w = 0; w < kPlanThreads / kWave; ++w) {
            if (w < wv) before += s_w[w][i];
            tot[i] += s_w[w][i];
        }
        v[i] = before + inc[i] - v[i];
    }
}

// The slot and position of row t of a step whose requests start at `start`.
__device__ __forceinline__ void plan_row(const PlanArgs &a, const int32_t *start, int t, int r, int base) {
    const int pos = base + (t - start[r]), page = (int)page_of((uint32_t)pos, a.div);
    const int b = a.tables[(size_t)r * a.max_blocks + page];
    const bool in = b >= 0 && b < a.n_blocks;
    a.slots[t] = in ? b * (int)a.div.d + (pos - page * (int)a.div.d) : -1;
    a.positions[t] = pos;
}

// rows: whether this launch fills slots and positions too (else plan_rows_kernel does).
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs a, int rows) {
    __shared__ int32_t s_start[kPagedMaxReq + 1], s_need[kPagedMaxReq], s_freed[kPagedMaxReq], s_len[kPagedMaxReq];
    __shared__ long long s_w[kPlanThreads / kWave][3];
    __shared__ int s_bad;
    const int tid = threadIdx.x, bs = (int)a.div.d;
    const long long room = (long long)a.max_blocks * bs;
    const int count = a.n_free[0];
    if (tid == 0) s_bad = count < 0 || count > a.n_blocks;
    int len[kPlanPer], add[kPlanPer], need[kPlanPer], have[kPlanPer];  // requests tid * kPlanPer + i
    bool bad = false, ends[kPlanPer];
    long long v[3] = {0, 0, 0}, tot[3];
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
        const int r = tid * kPlanPer + i;
        const bool live = r < a.n_req;
        len[i] = live ? a.len[r] : 0;
        const int nl = live ? a.new_len[r] : 0;
        ends[i] = nl < 0;
        add[i] = max(nl, 0);
        const bool out = len[i] < 0 || (long long)len[i] + add[i] > room;
        bad |= out;
        const int n0 = out ? 0 : len[i], n1 = out ? 0 : len[i] + add[i];
        have[i] = (int)page_of((uint32_t)n0, a.div) + (n0 % bs != 0);
        need[i] = ends[i] ? 0 : (int)page_of((uint32_t)n1, a.div) + (n1 % bs != 0) - have[i];
        v[0] += add[i];
        v[1] += need[i];
        v[2] += ends[i] ? have[i] : 0;
    }
    __syncthreads();
    if (bad) s_bad = 1;
    block_scan3(v, tot, s_w);
    __syncthreads();
    const long long top = count + tot[2];
    const bool invalid = s_bad || tot[0] > a.max_tokens || top > a.n_blocks;
    const long long lack = invalid ? 0 : tot[1] - top;
    const bool ok = !invalid && lack <= 0;
    if (tid == 0) {
        a.status[0] = invalid ? -1 : lack > 0 ? (int)lack : 0;
        a.n_free_out[0] = ok ? (int)(top - tot[1]) : count;
        a.q_start[a.n_req] = s_start[a.n_req] = ok ? (int)tot[0] : 0;
    }
    const int n_need = ok ? (int)tot[1] : 0, n_freed = ok ? (int)tot[2] : 0;
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
        const int r = tid * kPlanPer + i;
        if (r < a.n_req) {
            s_start[r] = ok ? (int)v[0] : 0;
            s_need[r] = ok ? (int)v[1] : 0;
            s_freed[r] = ok ? (int)v[2] : 0;
            s_len[r] = len[i];
            a.q_start[r] = s_start[r];
            a.kv_len[r] = !ok ? len[i] : ends[i] ? 0 : len[i] + add[i];
        }
        v[0] += add[i];
        v[1] += need[i];
        v[2] += ends[i] ? have[i] : 0;
    }
    __syncthreads();
    for (int i = tid; i < n_freed; i += kPlanThreads) {
        const int r = request_of(s_freed, a.n_req, i);
        a.free_list[count + i] = a.tables[(size_t)r * a.max_blocks + (i - s_freed[r])];
    }
    __syncthreads();
    for (int i = tid; i < n_need; i += kPlanThreads) {
        const int r = request_of(s_need, a.n_req, i), n0 = s_len[r];
        const int first = (int)page_of((uint32_t)n0, a.div) + (n0 % bs != 0);
        a.tables[(size_t)r * a.max_blocks + first + (i - s_need[r])] = a.free_list[(int)top - 1 - i];
    }
    if (!rows) return;
    __syncthreads();
    const int T = s_start[a.n_req];
    for (int t = tid; t < a.max_tokens; t += kPlanThreads) {
        if (t < T) {
            const int r = request_of(s_start, a.n_req, t);
            plan_row(a, s_start, t, r, s_len[r]);
        } else {
            a.slots[t] = a.positions[t] = -1;
        }
    }
}

__global__ __launch_bounds__(256) void plan_rows_kernel(PlanArgs a) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= a.max_tokens) return;
    if (t >= a.q_start[a.n_req]) {
        a.slots[t] = a.positions[t] = -1;
        return;
    }
    const int r = request_of(a.q_start, a.n_req, t);
    plan_row(a, a.q_start, t, r, a.kv_len[r] - (a.q_start[r + 1] - a.q_start[r]));
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

// grid (tokens), 256 threads: prompt_rope_kernel's arithmetic (prompt.hip) with the cache rows in pages.
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

// ---------------------------------------------------------------- attention
struct AttnArgs {
    PagedDims d;
    int n_req, max_blocks, T, n_heads, window;
    float scale;
    const int32_t *tables, *kv_len, *q_start;
    const void *kc, *vc;
    const float *q;
    float *out;
    uint64_t q_stride, out_stride;
};

// Any head dim and alignment: a block per (row, head), rows and heads in turn; 256 positions at a time, a thread
// per position for the scores and a thread per dim for the weighted sum, with a running maximum and sum.
template <int DT>
__global__ __launch_bounds__(256) void attn_any_kernel(AttnArgs a) {
    __shared__ float s_q[kPagedMaxHd], s_p[256], red[8];
    __shared__ uint64_t s_row[256];
    constexpr uint64_t kNone = ~0ull;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, hd = a.d.hd;
    for (uint64_t id = blockIdx.x; id < (uint64_t)a.T * a.n_heads; id += gridDim.x) {
        const int t = (int)(id / a.n_heads), h = (int)(id % a.n_heads);
        if (t < a.q_start[0]) continue;
        const int r = request_of(a.q_start, a.n_req, t), t1 = a.q_start[r + 1];
        if (t >= t1) continue;
        const int kvh = h / (a.n_heads / a.d.n_kv);
        const int n = min(max(a.kv_len[r], 0), a.max_blocks * a.d.block_size), pos = n - t1 + t;
        const int first = a.window > 0 ? max(0, pos - a.window + 1) : 0;
        __syncthreads();  // the previous row's shared values have been read
        if (tid < hd) s_q[tid] = a.q[(size_t)t * a.q_stride + (size_t)h * hd + tid];
        __syncthreads();
        float m = -INFINITY, l = 0.0f, o = 0.0f;
        for (int j0 = first; j0 <= pos; j0 += 256) {
            const int j = j0 + tid;
            float s = -INFINITY;
            uint64_t row = kNone;
            if (j <= pos) {
                const int page = (int)page_of((uint32_t)j, a.d.div);
                const int b = a.tables[(size_t)r * a.max_blocks + page];
                if (b >= 0 && b < a.d.n_blocks) {
                    row = paged_row(a.d, b, kvh, j - page * a.d.block_size);
                    s = 0.0f;
                    for (int i = 0; i < hd; ++i) s += s_q[i] * load_w<DT>(a.kc, row + i);
                    s *= a.scale;
                }
            }
            s_row[tid] = row;
            const float wm = wave_max(s);
            if (lane == 0) red[wv] = wm;
            __syncthreads();
            const float mn = fmaxf(fmaxf(m, fmaxf(red[0], red[1])), fmaxf(red[2], red[3]));
            const float ref = mn == -INFINITY ? 0.0f : mn;  // nothing seen yet: all weights 0
            const float p = row != kNone ? expf(s - ref) : 0.0f;
            s_p[tid] = p;
            const float ps = wave_sum(p);
            if (lane == 0) red[4 + wv] = ps;
            __syncthreads();
            const float alpha = expf(m - ref);
            l = l * alpha + ((red[4] + red[5]) + (red[6] + red[7]));
            o *= alpha;
            if (tid < hd)
                for (int jj = 0; jj < min(256, pos + 1 - j0); ++jj)
                    if (s_row[jj] != kNone) o += s_p[jj] * load_w<DT>(a.vc, s_row[jj] + tid);
            m = mn;
            __syncthreads();  // red, s_p and s_row are rewritten
        }
        if (tid < hd) a.out[(size_t)t * a.out_stride + (size_t)h * hd + tid] = l == 0.0f ? 0.0f : o / l;
    }
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

constexpr int kPlanRowsInOne = 2048;  // rows up to which the plan is one launch

hipError_t launch_paged_plan(const Launch &L, const Launch &Lr, const rbt_paged_plan &p) {
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
    const int rows = p.max_tokens <= kPlanRowsInOne;
    const hipError_t e = launch(L, plan_kernel, dim3(1), dim3(kPlanThreads), 0, a, rows);
    if (e != hipSuccess || rows) return e;
    return launch(Lr, plan_rows_kernel, dim3((unsigned)((p.max_tokens + 255) / 256)), dim3(256), 0, a);
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
    return kv.dtype == RBT_DT_BF16 ? launch(L, append_kernel<RBT_DT_BF16>, g, dim3(256), 0, a)
                                   : launch(L, append_kernel<RBT_DT_F32>, g, dim3(256), 0, a);
}

hipError_t launch_paged_attn(const Launch &L, const rbt_paged_kv &kv, const rbt_paged_batch &b, const float *q,
                             uint64_t q_stride, int T, int n_heads, float scale, int window, float *out,
                             uint64_t out_stride) {
    if (T < 1 || b.n_req < 1) return hipSuccess;
    AttnArgs a;
    a.d = dims_of(kv);
    a.n_req = b.n_req;
    a.max_blocks = b.max_blocks;
    a.T = T;
    a.n_heads = n_heads;
    a.window = window;
    a.scale = scale;
    a.tables = b.tables;
    a.kv_len = b.kv_len;
    a.q_start = b.q_start;
    a.kc = kv.k;
    a.vc = kv.v;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    const uint64_t rows = (uint64_t)T * (uint64_t)n_heads;
    const dim3 g((unsigned)(rows < 65536 ? rows : 65536));
    return kv.dtype == RBT_DT_BF16 ? launch(L, attn_any_kernel<RBT_DT_BF16>, g, dim3(256), 0, a)
                                   : launch(L, attn_any_kernel<RBT_DT_F32>, g, dim3(256), 0, a);
}

}  // namespace rbt
