// Index arithmetic of the paged key/value cache, shared by the kernels (paged.hip) and the host.
#pragma once

#include <stddef.h>
#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define RBT_HD __host__ __device__ __forceinline__
#else
#define RBT_HD inline
#endif

namespace rbt {

constexpr int kPagedMaxReq = 4096;   // requests of a step: their prefix sums sit in LDS
constexpr int kPagedMaxHd = 256;
constexpr int kPagedMaxLen = 0x7FFFFC00;  // positions of a request's table
constexpr int kPlanRowsInOne = 2048;  // rows up to which the plan is one launch
constexpr size_t kPagedWsBytes = 128u << 20;  // the attention's workspace

// n / d for 0 <= n < 2^31 as a product: with s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1,
// n / d = (n + high32(n m)) >> s (the sum stays below 2^32, since the product's high half is at most n).
struct PageDiv {
    uint32_t d, m, s;
};
inline PageDiv page_div(int d) {
    PageDiv p{(uint32_t)d, 1, 0};
    while ((1ull << p.s) < (uint64_t)d) ++p.s;
    p.m = (uint32_t)(((1ull << 32) * ((1ull << p.s) - (uint64_t)d)) / (uint64_t)d + 1);
    return p;
}
RBT_HD uint32_t page_of(uint32_t n, const PageDiv &p) {
    return (n + (uint32_t)(((uint64_t)n * p.m) >> 32)) >> p.s;
}

// What the kernels know of a cache, with the sizes the host has checked.
struct PagedDims {
    int n_blocks, block_size, n_kv, hd;
    uint64_t block_stride;  // elements
    PageDiv div;
};

// Element offset of row `off` of kv head h's rows in block b.
RBT_HD uint64_t paged_row(const PagedDims &d, int b, int h, int off) {
    return (uint64_t)b * d.block_stride + ((uint64_t)h * (uint64_t)d.block_size + (uint64_t)off) * (uint64_t)d.hd;
}

// The last r of [0, n) with start[r] <= t (start[0] <= t): the request of row t where the rows ascend.
RBT_HD int request_of(const int32_t *start, int n, int t) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (start[mid] <= t)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

}  // namespace rbt
