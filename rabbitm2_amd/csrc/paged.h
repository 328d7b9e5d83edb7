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

// ---- how the attention cuts a step (paged.hip)
constexpr int kWideRows = 128, kThinRows = 16;
constexpr int kMaxChunk = kPagedMaxLen;  // positions
static_assert(kMaxChunk % 128 == 0, "whole tiles");
template <bool THIN>
constexpr int kTileRows = THIN ? kThinRows : kWideRows;

RBT_HD int lesser(int a, int b) { return a < b ? a : b; }
RBT_HD int greater(int a, int b) { return a > b ? a : b; }

// A request's rows (tokens times the G query heads of a key/value head, heads fastest; the tokens at positions p0 ..
// n - 1) are cut into nt tiles of tr rows, and each tile's positions into pieces of at most `chunk`. Tile t spans up to
// S(t) = min(p0 + ceil((t + 1) tr / G), limit) positions, which grow with t, so that tiles from T(c) = floor((c chunk -
// p0) G / tr) on have more than c pieces. The first c0 pieces are every tile's, nc is the last tile's number, and
// the tiles before t have pieces_before(t) = c0 t + sum over c >= c0 of max(0, t - T(c)) in all.
struct Cut {
    int rows, nt, nc, c0, p0, limit, chunk, G;
};
template <bool THIN>
RBT_HD Cut cut_rows(int rows, int n, int p0, int G, int window, int chunk) {
    Cut c;
    constexpr int tr = kTileRows<THIN>;
    c.G = G;
    c.rows = rows;
    c.nt = rows / tr + (rows % tr != 0);
    c.p0 = p0;
    // all positions up to a tile's last row, or a window's and what its tokens span
    c.limit = window > 0 && window < n ? lesser(n - window, (tr - 1) / G + 1) + window : n;
    c.chunk = chunk;
    c.nc = greater(1, (int)(((uint32_t)c.limit + (uint32_t)(chunk - 1)) / (uint32_t)chunk));
    c.c0 = p0 > 0 ? lesser(c.nc, p0 / chunk + 1) : 1;
    return c;
}
template <bool THIN>
RBT_HD int64_t first_with(const Cut &c, int piece) {  // T(piece); may be negative below c0
    return ((int64_t)piece * c.chunk - c.p0) * c.G >> (THIN ? 4 : 7);
}
template <bool THIN>
RBT_HD int64_t pieces_before(const Cut &c, int t) {
    int64_t n = (int64_t)c.c0 * t;
    for (int i = c.c0; i < c.nc; ++i) {
        const int64_t d = t - first_with<THIN>(c, i);
        n += d > 0 ? d : 0;
    }
    return n;
}
// Tile t's pieces: n, of len positions each but the last, which may be shorter or, where the tile's positions are fewer
// than S(t), empty. Thin tiles' are equal up to whole tiles of 128 (what they take is memory, shared evenly); wide
// tiles' are whole chunks and a rest.
struct Pieces {
    int n, len;
};
template <bool THIN>
RBT_HD Pieces pieces_of(const Cut &c, int t) {
    const uint32_t last = (uint32_t)(t + 1) * (uint32_t)kTileRows<THIN>, rows = last < (uint32_t)c.rows ? last : (uint32_t)c.rows;
    const uint32_t span = (uint32_t)greater(0, lesser(c.p0 + (int)((rows + (uint32_t)c.G - 1) / (uint32_t)c.G), c.limit));
    const uint32_t m = (span + (uint32_t)(c.chunk - 1)) / (uint32_t)c.chunk, n = m > 0 ? m : 1;
    return {(int)n, THIN ? (int)(((span + n - 1) / n + 127) / 128 * 128) : c.chunk};
}
// Item `local` of a head's pieces_before(nt): its tile and piece, the largest first, so that a queue ends with its
// smallest. Wide tiles' whole chunks, then the rests: a tile t with i + 1 pieces has about t - T(i) rows of positions in
// its rest (times tr / G), so that the rests in descending order are those of the tiles with t - T(i) >= v for falling v.
struct TilePiece {
    int tile, piece;
};
template <bool THIN>
RBT_HD TilePiece tile_piece(const Cut &c, int local) {
    for (int i = c.nc - 1; i >= (THIN ? c.c0 : 1); --i) {
        const int n = c.nt - (i >= c.c0 ? (int)first_with<THIN>(c, i) : 0);
        if (local < n) return {c.nt - 1 - local, THIN ? i : i - 1};
        local -= n;
    }
    if (THIN) return {c.nt - 1 - local % c.nt, c.c0 - 1 - local / c.nt};
    if (c.nc == c.c0) return {c.nt - 1 - local, c.nc - 1};
    // the tiles with i + 1 pieces are [from(i), to(i))
    auto from = [&](int i) { return i >= c.c0 ? first_with<THIN>(c, i) : (int64_t)0; };
    auto to = [&](int i) { return i + 1 < c.nc ? first_with<THIN>(c, i + 1) : (int64_t)c.nt; };
    auto count = [&](int64_t v) {  // tiles with t - T(i) >= v
        int64_t n = 0;
        for (int i = c.c0 - 1; i < c.nc; ++i) {
            const int64_t t = first_with<THIN>(c, i) + v, b = from(i), d = to(i) - (t > b ? t : b);
            n += d > 0 ? d : 0;
        }
        return n;
    };
    const int64_t t0 = first_with<THIN>(c, c.c0 - 1);
    int64_t lo = t0 > 0 ? -t0 : 0, hi = c.nt - t0;  // count(lo) > local >= count(hi)
    while (hi - lo > 1) {
        const int64_t mid = lo + ((hi - lo) >> 1);
        if (count(mid) > local)
            lo = mid;
        else
            hi = mid;
    }
    local -= (int)count(hi);
    for (int i = c.c0 - 1;; ++i) {  // those that have a tile with t - T(i) = lo
        const int64_t t = first_with<THIN>(c, i) + lo;
        if (t >= from(i) && t < to(i) && local-- == 0) return {(int)t, i};
        if (i + 1 >= c.nc) return {c.nt - 1, c.nc - 1};  // not reached
    }
}

}  // namespace rbt
