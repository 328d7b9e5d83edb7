"""The paged cache's entry points on the CPU: their refusals (arguments are checked before the handle, so a NULL
handle shows each message), and the index arithmetic that the kernels share with the host, compiled for
the CPU and run at the borders of its ranges."""
import ctypes as C
import os
import subprocess

import pytest

from rabbitm2_amd import hip

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = C.c_void_p(0x1000)  # never read: every call below ends at a check


def message():
    return hip.lib().rbt_hip_last_error(None).decode()


def kv(**over):
    a = dict(n_blocks=8, block_size=16, n_kv_heads=2, head_dim=64, dtype=hip.DT_BF16, k=P, v=P)
    a.update(over)
    return hip.paged_kv_desc(**a)


def batch(**over):
    a = dict(n_req=2, max_blocks=4, tables=P, kv_len=P, q_start=P)
    a.update(over)
    return hip.paged_batch_desc(**a)


def plan(**over):
    a = dict(n_req=2, max_blocks=4, n_blocks=8, block_size=16, max_tokens=32, len=P, new_len=P, tables=P, free_list=P,
             n_free=P, kv_len=P, n_free_out=P, q_start=P, slots=P, positions=P, status=P)
    a.update(over)
    return hip.paged_plan_desc(**a)


def rows(**over):
    a = dict(n_tokens=4, n_heads=4, q=P, k=P, v=P, q_out=C.c_void_p(0x2000), positions=P, slots=P, rope=P, n_rope=64)
    a.update(over)
    return hip.paged_rows_desc(**a)


def attn(k=None, b=None, q=P, T=4, n_heads=4, out=P, scale=0.0, window=0, q_stride=0, out_stride=0):
    return hip.lib().rbt_hip_paged_attn_dev(None, C.byref(k or kv()), C.byref(b or batch()), q, q_stride, T, n_heads, scale,
                                            window, out, out_stride)


def append(k=None, w=None):
    return hip.lib().rbt_hip_paged_append_dev(None, C.byref(k or kv()), C.byref(w or rows()))


def do_plan(p):
    return hip.lib().rbt_hip_paged_plan_dev(None, C.byref(p))


def test_good_arguments_reach_the_handle_check():
    for ok in (attn(), append(), do_plan(plan())):
        assert ok == 0 and "handle is NULL" in message()
    assert hip.lib().rbt_hip_paged_reserve(None) == 0 and "handle is NULL" in message()
    assert hip.lib().rbt_hip_paged_init(None, 1, 0, 1, 1, 0, 1) == 0 and "handle is NULL" in message()
    assert hip.lib().rbt_hip_forward_paged(None, None, None, None, None) == 0 and "handle is NULL" in message()


BAD_KV = [dict(n_blocks=0), dict(block_size=0), dict(n_kv_heads=0), dict(head_dim=0), dict(head_dim=257),
          dict(n_blocks=1 << 20, block_size=1 << 12), dict(dtype=2), dict(k=None), dict(v=None),
          dict(block_stride=16 * 2 * 64 - 1), dict(block_stride=1 << 62), dict(n_kv_heads=1 << 20)]


@pytest.mark.parametrize("over", BAD_KV, ids=[str(o) for o in BAD_KV])
def test_cache_is_refused(over):
    for name, call in (("paged_attn", attn), ("paged_append", append)):
        assert call(kv(**over)) == 0
        assert message().startswith(name + ": ") and "handle" not in message()


BAD_ATTN = [dict(b=dict(n_req=-1)), dict(b=dict(n_req=4097)), dict(b=dict(max_blocks=0)),
            dict(b=dict(max_blocks=1 << 30)), dict(b=dict(tables=None)), dict(b=dict(kv_len=None)),
            dict(b=dict(q_start=None)), dict(T=-1), dict(n_heads=0), dict(n_heads=3), dict(n_heads=1 << 20), dict(q=None),
            dict(out=None), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(q_stride=255),
            dict(out_stride=255), dict(out_stride=1 << 33), dict(q_stride=300), dict(out_stride=300)]  # out is q


@pytest.mark.parametrize("over", BAD_ATTN, ids=[str(o) for o in BAD_ATTN])
def test_attention_is_refused(over):
    over = dict(over)
    if "b" in over:
        over["b"] = batch(**over["b"])
    assert attn(**over) == 0
    assert message().startswith("paged_attn: ") and "handle" not in message()


BAD_ROWS = [dict(n_tokens=-1), dict(n_heads=0), dict(n_heads=5), dict(k=None), dict(v=None), dict(slots=None),
            dict(q_out=None), dict(positions=None), dict(n_rope=0), dict(q_stride=255), dict(k_stride=127),
            dict(v_stride=127), dict(q_out=P, q_stride=300)]


@pytest.mark.parametrize("over", BAD_ROWS, ids=[str(o) for o in BAD_ROWS])
def test_append_is_refused(over):
    assert append(w=rows(**over)) == 0
    assert message().startswith("paged_append: ") and "handle" not in message()


def test_append_refuses_rope_of_odd_heads():
    assert append(kv(head_dim=65)) == 0 and "rope" in message()


BAD_PLAN = [dict(n_req=-1), dict(n_req=4097), dict(max_blocks=0), dict(n_blocks=0), dict(block_size=0),
            dict(max_tokens=-1), dict(max_blocks=1 << 28), dict(n_blocks=1 << 28)] + [
    {n: None} for n in ("len", "new_len", "tables", "free_list", "n_free", "kv_len", "n_free_out", "q_start", "slots",
                        "positions", "status")]


@pytest.mark.parametrize("over", BAD_PLAN, ids=[str(o) for o in BAD_PLAN])
def test_plan_is_refused(over):
    assert do_plan(plan(**over)) == 0
    assert message().startswith("paged_plan: ") and "handle" not in message()


def test_null_descriptors():
    L = hip.lib()
    assert L.rbt_hip_paged_plan_dev(None, None) == 0 and "NULL" in message()
    assert L.rbt_hip_paged_append_dev(None, None, None) == 0 and "NULL" in message()
    assert L.rbt_hip_paged_append_dev(None, C.byref(kv()), None) == 0 and "NULL" in message()
    assert L.rbt_hip_paged_attn_dev(None, C.byref(kv()), None, P, 0, 1, 4, 0.0, 0, P, 0) == 0 and "NULL" in message()


INDEX_DRIVER = r"""
#include <stdio.h>
#include <initializer_list>
#include <vector>
#include "paged.h"
using namespace rbt;
#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)
template <bool THIN>
int check_cut(int n, int m, int G, int window, int chunk) {
    const int p0 = n - m, tr = kTileRows<THIN>;
    const Cut c = cut_rows<THIN>(m * G, n, p0, G, window, chunk);
    CHECK(c.nt == (m * G + tr - 1) / tr);
    std::vector<std::vector<int>> seen((size_t)c.nt);
    int64_t all = 0;
    for (int t = 0; t < c.nt; ++t) {
        CHECK(pieces_before<THIN>(c, t) == all);
        const Pieces p = pieces_of<THIN>(c, t);
        CHECK(p.n >= 1 && p.len >= 0 && p.len <= chunk && (p.len % 128 == 0 || p.len == chunk));
        // the tile's positions, as its block has them
        const int64_t r1 = (int64_t)(t + 1) * tr < c.rows ? (int64_t)(t + 1) * tr : c.rows;
        const int64_t pa = p0 + (int64_t)t * tr / G, pb = p0 + (r1 - 1) / G;
        const int64_t lo = window > 0 && pa - window + 1 > 0 ? pa - window + 1 : 0, end = pb + 1 > lo ? pb + 1 : lo;
        CHECK((int64_t)p.n * p.len >= end - lo);
        seen[(size_t)t].assign((size_t)p.n, 0);
        all += p.n;
    }
    CHECK(pieces_before<THIN>(c, c.nt) == all);
    for (int64_t i = 0; i < all; ++i) {
        const TilePiece x = tile_piece<THIN>(c, (int)i);
        CHECK(x.tile >= 0 && x.tile < c.nt && x.piece >= 0 && x.piece < (int)seen[(size_t)x.tile].size());
        CHECK(seen[(size_t)x.tile][(size_t)x.piece]++ == 0);
    }
    return 0;
}
int main() {
    // page_of is the quotient, at the borders of every divisor's multiples and of the range
    for (long long d = 1; d <= 2147483647ll; d = d < 70000 ? d + 1 : d * 3 / 2 + 1) {
        const PageDiv p = page_div((int)d);
        for (long long k : {0ll, 1ll, 2ll, 3ll, 1000ll, 2147483647ll / d - 1, 2147483647ll / d})
            for (long long o : {-1ll, 0ll, 1ll}) {
                const long long n = k * d + o;
                if (n < 0 || n > 2147483647ll) continue;
                CHECK((long long)page_of((uint32_t)n, p) == n / d);
            }
    }
    // request_of: the request whose rows hold t, with empty requests before, between and behind
    const int32_t start[] = {0, 0, 3, 3, 3, 4, 9, 9, 9};
    const int of[] = {1, 1, 1, 4, 5, 5, 5, 5, 5};
    for (int t = 0; t < 9; ++t) CHECK(request_of(start, 8, t) == of[t]);
    const int32_t odd[] = {5, 1, 7, -3, 2};  // rows that do not ascend: in bounds all the same
    for (int t = -10; t < 20; ++t) { const int r = request_of(odd, 4, t); CHECK(r >= 0 && r < 4); }
    // the cut of a request: every (tile, piece) is one item, and the pieces cover the tile's positions
    const int ns[] = {0, 1, 5, 100, 128, 129, 700, 1000, 3001}, ms[] = {1, 2, 16, 17, 128, 300, 1500},
              gs[] = {1, 2, 3, 7, 16, 40, 200}, ws[] = {0, 1, 100, 129, 1000, 2147483647}, cs[] = {128, 256, 640, 1408, kMaxChunk};
    for (int n : ns) for (int m : ms) for (int g : gs) for (int w : ws) for (int ch : cs) {
        if ((long long)m * g > 70000) continue;
        if (check_cut<false>(n, m, g, w, ch) || (m * g <= kThinRows && check_cut<true>(n, m, g, w, ch))) {
            printf("n %d m %d G %d window %d chunk %d\n", n, m, g, w, ch);
            return 1;
        }
    }
    // positions and chunks near 2^31
    for (int ch : {1 << 20, 1 << 30, kMaxChunk - 128})
        for (int g : {1, 3, 16, 8192})
            for (int m : {1, 5})
                if (check_cut<false>(kMaxChunk - 3, m, g, 0, ch) || (m * g <= kThinRows && check_cut<true>(kMaxChunk - 3, m, g, 0, ch))) return 1;
    // offsets past 32 bits
    PagedDims d{1 << 20, 128, 8, 128, 8ull * 128 * 128, page_div(128)};
    CHECK(paged_row(d, (1 << 20) - 1, 7, 127) + 128 == (uint64_t)(1 << 20) * 8 * 128 * 128);
    puts("ok");
    return 0;
}
"""


def test_index_arithmetic(tmp_path):
    src, exe = tmp_path / "index.cpp", tmp_path / "index"
    src.write_text(INDEX_DRIVER)
    cmd = ["g++", "-std=c++17", "-O1", "-g", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "rabbitm2_amd", "csrc"),
           str(src), "-o", str(exe)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    assert res.returncode == 0 and res.stdout.strip() == "ok", res.stdout + res.stderr
