"""The paged key/value cache (rbt_hip_paged_plan_dev, _append_dev, _attn_dev) against plain implementations in
64 bits on the host: the plan's whole numbers exactly, floats within bounds that follow from the arithmetic.

Attention: with the engine's formulas in f32, a score q.k * scale of hd products is off by at most about sqrt(hd) *
2^-24 of the sum of their magnitudes A (sums in any order), plus four steps more (the scaled query, the exponent's
difference, the products of parts below 2^-24), and a weight by that much relatively; its power and its products add a
few steps of 2^-24 each (16), sums over n positions sqrt(n). The output, a mean of values under weights that are each
off by a relative w, and whose sum is off by no more, is off by at most 2 w max|v|.

Append: a norm is a sum of n squares (sqrt(n) 2^-24 of it, half of that in the root) and three rounded
products; RoPE adds two products and a sum; a cache of bf16 is off by at most half a step, 2^-8 of the value.
"""
import ctypes as C
import json
import os
import subprocess
import sys

import numpy as np
import pytest

from oracle import pyoracle as po
from rabbitm2_amd import hip

pytestmark = pytest.mark.gpu

F32, BF16 = hip.DT_F32, hip.DT_BF16


class Arrays:
    """Device copies of host arrays, freed together."""

    def __init__(self, dev):
        self.dev, self.bufs = dev, []

    def up(self, a):
        a = np.ascontiguousarray(a)
        b = self.dev.upload_array(a if a.size else np.zeros(1, np.int32))
        self.bufs.append(b)
        return b

    def free(self):
        for b in self.bufs:
            self.dev.free(b)
        self.bufs = []


@pytest.fixture
def up(dev):
    a = Arrays(dev)
    yield a
    a.free()


def to_cache(x, dtype):
    """f32 values as the cache stores them: (stored array, the values it stands for in f64)."""
    if dtype == F32:
        x = x.astype(np.float32)
        return x, x.astype(np.float64)
    raw = po.f32_to_bf16(x.astype(np.float32))
    return raw, po.bf16_to_f32(raw).astype(np.float64)


# ---------------------------------------------------------------- plan
def plan_ref(n, new, tables, free, n_free, bs, n_blocks, max_tokens):
    """The plan in plain Python: a dict of its outputs."""
    R, P = tables.shape
    tables, free = tables.copy(), list(free[:max(n_free, 0)])
    add = [max(int(x), 0) for x in new]
    bad = any(not 0 <= int(n[r]) + add[r] <= P * bs or n[r] < 0 for r in range(R))
    bad = bad or sum(add) > max_tokens or not 0 <= n_free <= n_blocks
    status = -1 if bad else 0
    stack = list(free)
    if not bad:
        for r in range(R):
            if new[r] < 0:
                stack += [int(b) for b in tables[r, :-(-int(n[r]) // bs)]]
        pushed = list(stack)
        if len(stack) > n_blocks:
            status = -1
        need = sum(-(-(int(n[r]) + add[r]) // bs) - -(-int(n[r]) // bs) for r in range(R) if new[r] >= 0)
        if status == 0 and need > len(stack):
            status = need - len(stack)
    if status:
        none = np.full(max_tokens, -1, np.int32)
        return dict(tables=tables, free=free, kv_len=np.asarray(n, np.int32), n_free=n_free,
                    q_start=np.zeros(R + 1, np.int32), slots=none, positions=none, status=status)
    kv, start, slots, pos = [], [0], [], []
    for r in range(R):
        if new[r] < 0:
            kv.append(0)
            start.append(start[-1])
            continue
        kv.append(int(n[r]) + add[r])
        for page in range(-(-int(n[r]) // bs), -(-kv[-1] // bs)):
            tables[r, page] = stack.pop()
        for p in range(int(n[r]), kv[-1]):
            b = int(tables[r, p // bs])
            slots.append(b * bs + p % bs if 0 <= b < n_blocks else -1)
            pos.append(p)
        start.append(start[-1] + add[r])
    pad = [-1] * (max_tokens - len(slots))
    return dict(tables=tables, free=pushed, kv_len=np.array(kv, np.int32), n_free=len(stack),
                q_start=np.array(start, np.int32), slots=np.array(slots + pad, np.int32),
                positions=np.array(pos + pad, np.int32), status=0)


def plan_run(dev, up, n, new, tables, free, n_free, bs, n_blocks, max_tokens, in_place=False):
    R, P = tables.shape
    d_n, d_new, d_t = up.up(np.asarray(n, np.int32)), up.up(np.asarray(new, np.int32)), up.up(tables.astype(np.int32))
    d_f, d_nf = up.up(np.asarray(free, np.int32)), up.up(np.array([n_free], np.int32))
    fill = lambda k: up.up(np.full(max(k, 1), -7, np.int32))  # noqa: E731
    d_kv, d_nfo = (d_n, d_nf) if in_place else (fill(R), fill(1))
    d_qs, d_sl, d_po, d_st = fill(R + 1), fill(max_tokens + 3), fill(max_tokens + 3), fill(1)
    p = hip.paged_plan_desc(R, P, n_blocks, bs, max_tokens, d_n, d_new, d_t, d_f, d_nf, d_kv, d_nfo, d_qs, d_sl, d_po, d_st)
    dev.paged_plan(p)
    g = lambda b, *s: dev.d2h(b, s, np.int32)  # noqa: E731
    sl, po_ = g(d_sl, max_tokens + 3), g(d_po, max_tokens + 3)
    assert (sl[max_tokens:] == -7).all() and (po_[max_tokens:] == -7).all()  # nothing behind the buffers' rows
    return dict(tables=g(d_t, R, P), free=g(d_f, n_blocks), kv_len=g(d_kv, R), n_free=int(g(d_nfo, 1)[0]),
                q_start=g(d_qs, R + 1), slots=sl[:max_tokens], positions=po_[:max_tokens], status=int(g(d_st, 1)[0]))


def plan_check(got, want):
    assert got["status"] == want["status"]
    assert got["n_free"] == want["n_free"]
    for k in ("kv_len", "q_start", "slots", "positions", "tables"):
        assert np.array_equal(got[k], want[k]), k
    top = len(want["free"])
    assert np.array_equal(got["free"][:top], np.array(want["free"], np.int32)[:top])


def plan_state(rng, R, P, bs, max_len, spare):
    """Random requests with their pages, and a free list of `spare` more blocks."""
    n = rng.integers(0, max_len + 1, R)
    have = -(-n // bs)
    n_blocks = int(have.sum()) + spare
    perm = rng.permutation(n_blocks)
    tables = np.full((R, P), -1, np.int32)
    at = 0
    for r in range(R):
        tables[r, :have[r]] = perm[at:at + have[r]]
        at += have[r]
    free = np.full(max(n_blocks, 1), -1, np.int32)
    free[:spare] = perm[at:]
    return n, tables, free, max(n_blocks, 1)


PLANS = [(1, 1, 5, 1), (3, 16, 0, 40), (7, 24, 100, 30), (64, 16, 300, 3), (200, 1, 20, 4), (1025, 8, 90, 5),
         (4096, 32, 500, 2), (5, 128, 3000, 2000), (2, 16, 10, 5000)]  # requests, block, cached up to, new up to


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("shape", PLANS, ids=["R%dbs%dlen%dnew%d" % s for s in PLANS])
def test_plan(dev, up, shape, in_place):
    R, bs, ml, mn = shape
    rng = np.random.default_rng(R * 7 + bs)
    P = -(-(ml + mn) // bs) + 1
    n, tables, free, n_blocks = plan_state(rng, R, P, bs, ml, R * (mn // bs + 2))
    new = rng.integers(0, mn + 1, R)
    if R > 2:
        new[rng.random(R) < 0.1] = -1
    n_free = int((free >= 0).sum())
    M = int(np.maximum(new, 0).sum()) + 5  # and padding behind the last request
    want = plan_ref(n, new, tables, free, n_free, bs, n_blocks, M)
    assert want["status"] == 0
    plan_check(plan_run(dev, up, n, new, tables, free, n_free, bs, n_blocks, M, in_place), want)


def test_plan_uses_blocks_that_just_ended(dev, up):
    """No block is free but those of the requests that end in the same step."""
    tables = np.array([[3, 1, -1], [0, 2, -1], [-1, -1, -1]], np.int32)
    args = ([8, 7, 0], [-1, 1, 9], tables, np.full(4, -1), 0, 4, 4, 16)
    want = plan_ref(*args)
    assert want["status"] == 1  # one block short: 3 needed, 2 come back
    plan_check(plan_run(dev, up, *args), want)
    args = ([8, 7, 0], [-1, 1, 8], tables, np.full(4, -1), 0, 4, 4, 16)
    want = plan_ref(*args)
    assert want["status"] == 0 and want["n_free"] == 0
    plan_check(plan_run(dev, up, *args), want)


T3 = np.array([[0, 1, 2], [3, 4, -1], [-1, -1, -1]], np.int32)
BAD_PLANS = {
    "blocks lacking": ([12, 5, 0], [0, 8, 12], T3, [5, 6, -1, -1, -1, -1, -1], 2, 4, 7, 32),
    "negative length": ([12, -1, 0], [0, 1, 1], T3, [5, 6, -1, -1, -1, -1, -1], 2, 4, 7, 32),
    "length past the table": ([13, 5, 0], [0, 1, 1], T3, [5, 6, -1, -1, -1, -1, -1], 2, 4, 7, 32),
    "new past the table": ([12, 5, 0], [1, 1, 1], T3, [5, 6, -1, -1, -1, -1, -1], 2, 4, 7, 32),
    "huge new": ([12, 5, 0], [0, 2**31 - 1, 2**31 - 1], T3, [5, 6, -1, -1, -1, -1, -1], 2, 4, 7, 32),
    "more rows than the buffers": ([12, 5, 0], [0, 3, 2], T3, [5, 6, -1, -1, -1, -1, -1], 2, 4, 7, 4),
    "free count negative": ([12, 5, 0], [0, 1, 1], T3, [5, 6, -1, -1, -1, -1, -1], -1, 4, 7, 32),
    "free count too large": ([12, 5, 0], [0, 1, 1], T3, [5, 6, -1, -1, -1, -1, -1], 8, 4, 7, 32),
    "more given back than there is room for": ([12, 5, 0], [-1, 1, 1], T3, [5, 6, 5, 6, 5, 6, 5], 5, 4, 7, 32),
}


@pytest.mark.parametrize("name", sorted(BAD_PLANS))
def test_plan_grants_nothing_that_does_not_fit(dev, up, name):
    n, new, tables, free, n_free, bs, n_blocks, M = BAD_PLANS[name]
    want = plan_ref(n, new, tables, np.array(free), n_free, bs, n_blocks, M)
    assert want["status"] != 0
    got = plan_run(dev, up, n, new, tables, free, n_free, bs, n_blocks, M)
    assert np.array_equal(got.pop("free"), free)
    want["free"] = []
    got["free"] = np.zeros(0)
    plan_check(got, want)


def test_plan_of_no_requests_and_no_rows(dev, up):
    got = plan_run(dev, up, [], [], np.zeros((0, 3), np.int32), [2, 1], 2, 16, 2, 4)
    assert got["status"] == 0 and got["n_free"] == 2 and got["q_start"].tolist() == [0]
    assert (got["slots"] == -1).all()
    got = plan_run(dev, up, [3], [0], np.array([[1]], np.int32), [0, -1], 1, 16, 2, 0)
    assert got["status"] == 0 and got["kv_len"].tolist() == [3] and got["q_start"].tolist() == [0, 0]


def test_plan_slots_on_bad_pages_are_none(dev, up):
    """A table entry outside the cache gives its positions no slot."""
    tables = np.array([[9, 1], [-5, 0]], np.int32)
    args = ([2, 1], [3, 4], tables, [3, 2, -1, -1], 2, 4, 4, 16)
    want = plan_ref(*args)
    assert want["slots"].tolist()[:7] == [-1, -1, 8, -1, -1, -1, 12]
    plan_check(plan_run(dev, up, *args), want)


# ---------------------------------------------------------------- append
def append_ref(x, w, cs, heads, hd, eps):
    """QK-norm and RoPE of rows x in 64 bits."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(1, keepdims=True) + eps) * w.astype(np.float64)
    x = x.reshape(len(x), heads, hd)
    if cs is not None:
        c, s = cs[:, None, :, 0].astype(np.float64), cs[:, None, :, 1].astype(np.float64)
        lo, hi = x[..., :hd // 2], x[..., hd // 2:]
        x = np.concatenate((lo * c - hi * s, hi * c + lo * s), -1)
    return x


def rope_table(n, hd):
    a = np.arange(n)[:, None] * 10000.0 ** (-2.0 * np.arange(hd // 2) / hd)
    return np.stack((np.cos(a), np.sin(a)), -1).astype(np.float32)


# tokens, heads, kv heads, head dim, block, dtype, norm, rope, extra floats per row
APPENDS = [(1, 16, 16, 128, 16, BF16, 1, 1, 0), (5, 4, 2, 64, 8, BF16, 1, 1, 0), (33, 6, 2, 80, 24, F32, 0, 1, 0),
           (7, 3, 1, 20, 5, BF16, 1, 1, 3), (9, 5, 5, 7, 3, F32, 1, 0, 1), (130, 8, 1, 256, 32, BF16, 0, 0, 0),
           (300, 16, 16, 128, 16, F32, 1, 1, 256), (21, 32, 32, 128, 16, BF16, 1, 1, 0), (6, 17, 1, 128, 8, F32, 1, 1, 64),
           (3, 65, 5, 128, 4, BF16, 1, 1, 0), (2, 40, 40, 128, 16, F32, 0, 1, 8), (40, 2, 2, 1, 1, BF16, 1, 0, 0), (64, 12, 4, 96, 16, BF16, 1, 1, 4)]


@pytest.mark.parametrize("q_in", ["q", "in place", "no q"])
@pytest.mark.parametrize("shape", APPENDS, ids=["T%dh%dkv%dhd%dbs%ddt%dn%dr%ds%d" % s for s in APPENDS])
def test_append(dev, up, shape, q_in):
    T, H, KV, hd, bs, dt, norm, rope, extra = shape
    rng = np.random.default_rng(T * 31 + hd)
    n_blocks, eps, n_rope = -(-T // bs) + 2, 1e-5, 2 * T + 5
    qd, kd = H * hd, KV * hd
    if q_in == "in place" and extra:
        pytest.skip("q_out may be q only where q is contiguous")
    fused = rng.standard_normal((T, qd + 2 * kd + extra)).astype(np.float32)  # rows as one product leaves them
    row = fused.shape[1]
    d_x = up.up(fused)
    q, k, v = fused[:, :qd], fused[:, qd:qd + kd], fused[:, qd + kd:qd + 2 * kd]
    qs = row
    if q_in == "in place":
        d_q = up.up(q)
        qp, op, qs = C.c_void_p(d_q.ptr), d_q, 0
    else:
        op = up.up(np.full((T, qd), -3.0, np.float32))
        qp = C.c_void_p(d_x.ptr) if q_in == "q" else None
    slots = rng.permutation(n_blocks * bs)[:T].astype(np.int32)
    pos = rng.integers(0, n_rope, T).astype(np.int32)
    dead = rng.random(T) < 0.2  # passed over: a slot or a position out of range
    dead[0] = False
    for i, t in enumerate(np.flatnonzero(dead)):
        if rope and i % 2:
            pos[t] = (-1, n_rope, 2**31 - 1)[i % 3]
        else:
            slots[t] = (-1, n_blocks * bs, -2**31)[i % 3]
    stride = KV * bs * hd + 8  # blocks lie apart
    old = rng.standard_normal((2, n_blocks, stride)).astype(np.float32)
    raw, val = to_cache(old, dt)
    d_k, d_v = up.up(raw[0]), up.up(raw[1])
    qn, kn = (1 + 0.1 * rng.standard_normal(n).astype(np.float32) for n in (qd, kd))
    cs = rope_table(n_rope, hd) if rope else None
    kv = hip.paged_kv_desc(n_blocks, bs, KV, hd, dt, d_k, d_v, stride)
    w = hip.paged_rows_desc(T, H, qp, C.c_void_p(d_x.ptr + 4 * qd), C.c_void_p(d_x.ptr + 4 * (qd + kd)), op, up.up(pos),
                            up.up(slots), q_norm=up.up(qn) if norm else None, k_norm=up.up(kn) if norm else None, eps=eps,
                            rope=up.up(cs) if rope else None, n_rope=n_rope, q_stride=qs, k_stride=row, v_stride=row)
    dev.paged_append(kv, w)
    got_q = dev.d2h(op, (T, qd), np.float32)
    live = np.flatnonzero(~dead)
    c = cs[pos[live]] if rope else None
    # x inv w: the norm's (sqrt(n) + 3) / 2 steps and two products; RoPE: two products and a sum of two such
    tol = lambda n, x: ((n**0.5 + 8) * 2.0**-24 if norm else 2.0**-22) * 2 * np.abs(x).max() + 1e-30  # noqa: E731
    want = append_ref(q[live], qn if norm else None, c, H, hd, eps).reshape(len(live), qd)
    if q_in != "no q":
        assert np.abs(got_q[live] - want).max() <= tol(qd, want)
        assert np.array_equal(got_q[dead], q[dead] if q_in == "in place" else np.full((dead.sum(), qd), -3.0, np.float32))
    else:
        assert (got_q == -3.0).all()
    raw_t = np.float32 if dt == F32 else np.uint16
    for d_c, i, x, wn in ((d_k, 0, k, kn if norm else None), (d_v, 1, v, None)):
        got = dev.d2h(d_c, (n_blocks, stride), raw_t)
        rows = append_ref(x[live], wn, c, KV, hd, eps) if i == 0 else x[live].astype(np.float64).reshape(-1, KV, hd)
        touched = np.zeros((n_blocks, stride), bool)
        t_ = tol(kd, rows) if i == 0 else 0.0
        for j, t in enumerate(live):
            b, off = divmod(int(slots[t]), bs)
            for h in range(KV):
                s = slice((h * bs + off) * hd, (h * bs + off + 1) * hd)
                touched[b, s] = True
                g = got[b, s].astype(np.float64) if dt == F32 else po.bf16_to_f32(got[b, s]).astype(np.float64)
                half = 0.0 if dt == F32 else 2.0**-8 * np.abs(rows[j, h])
                assert (np.abs(g - rows[j, h]) <= t_ * 1.01 + half).all()
        assert np.array_equal(got[~touched], raw[i][~touched])  # everything else as it was


def test_append_keeps_nan_and_infinity(dev, up):
    """bf16 rounding: NaN stays NaN (its low bits all set too), infinities stay, the largest f32 becomes infinity."""
    x = np.array([[np.nan, np.inf, -np.inf, 3.4028234e38, 1.0, -0.0, 1e-45, 65280.0]], np.float32)
    x.view(np.uint32)[0, 0] = 0x7FFFFFFF
    d_x, d_k, d_v = up.up(x), up.up(np.zeros((1, 8), np.uint16)), up.up(np.zeros((1, 8), np.uint16))
    kv = hip.paged_kv_desc(1, 1, 1, 8, BF16, d_k, d_v)
    dev.paged_append(kv, hip.paged_rows_desc(1, 1, None, d_x, d_x, None, None, up.up(np.zeros(1, np.int32))))
    for d in (d_k, d_v):
        g = po.bf16_to_f32(dev.d2h(d, (8,), np.uint16))
        assert np.isnan(g[0]) and g[1] == np.inf and g[2] == -np.inf and g[3] == np.inf
        assert g[4] == 1.0 and g[5] == 0.0 and np.signbit(g[5]) and g[6] == 0.0 and g[7] == 65280.0


# ---------------------------------------------------------------- attention
class Step:
    """Requests with their pages in a random cache, and the reference in 64 bits."""

    def __init__(self, up, lens, heads, kv, hd, bs, dt, seed=1, spare_rows=0, extra_blocks=1, garbage=np.nan, q_scale=1.0,
                 q_extra=0, out_extra=0, stride_extra=0, max_blocks=None):
        rng = np.random.default_rng(seed)
        self.lens = [(int(n), int(m)) for n, m in lens]  # cached, new
        self.H, self.KV, self.hd, self.bs, self.dt = heads, kv, hd, bs, dt
        tot = [n + m for n, m in self.lens]
        pages = [-(-t // bs) for t in tot]
        self.P = max(max(pages, default=0), 1) if max_blocks is None else max_blocks
        self.nb = sum(pages) + extra_blocks
        perm = rng.permutation(self.nb)
        self.tables = np.full((len(tot), self.P), -1, np.int32)
        at = 0
        for r, p in enumerate(pages):
            self.tables[r, :p] = perm[at:at + p]
            at += p
        # everything that is no request's position holds garbage
        self.stride = kv * bs * hd + stride_extra
        dense = np.full((2, self.nb, kv, bs, hd), garbage, np.float32)
        self.k, self.v = [], []
        for r, t in enumerate(tot):
            kr, vr = (to_cache(rng.standard_normal((t, kv, hd)), dt)[1] for _ in range(2))
            self.k.append(kr)
            self.v.append(vr)
            for p in range(t):
                b = self.tables[r, p // bs]
                dense[0, b, :, p % bs], dense[1, b, :, p % bs] = kr[p], vr[p]
        self.dense = dense
        self.T = sum(m for _, m in self.lens)
        self.rows = self.T + spare_rows
        self.qd = heads * hd
        self.q = (q_scale * rng.standard_normal((self.rows, self.qd + q_extra))).astype(np.float32)
        self.out_row = self.qd + out_extra
        self.start = np.concatenate(([0], np.cumsum([m for _, m in self.lens]))).astype(np.int32)
        self.up = up

    def upload(self):
        raw = np.full((2, self.nb, self.stride), 0, np.float32)
        raw[:, :, :self.KV * self.bs * self.hd] = self.dense.reshape(2, self.nb, -1)
        raw = raw if self.dt == F32 else po.f32_to_bf16(raw)
        if self.dt == BF16:
            nan = np.isnan(self.dense.reshape(2, self.nb, -1))
            raw[:, :, :nan.shape[2]][nan] = 0x7FFF
        up = self.up.up
        self.d_k, self.d_v, self.d_q = up(raw[0]), up(raw[1]), up(self.q)
        self.d_t, self.d_n = up(self.tables), up(np.array([n + m for n, m in self.lens], np.int32))
        self.d_s, self.d_o = up(self.start), up(np.full((max(self.rows, 1), self.out_row), -5.0, np.float32))
        self.kv = hip.paged_kv_desc(self.nb, self.bs, self.KV, self.hd, self.dt, self.d_k, self.d_v, self.stride)
        self.batch = hip.paged_batch_desc(len(self.lens), self.P, self.d_t, self.d_n, self.d_s)
        return self

    def call(self, dev, scale=0.0, window=0):
        dev.paged_attn(self.kv, self.batch, self.d_q, self.rows, self.H, self.d_o, scale=scale, window=window,
                       q_stride=self.q.shape[1], out_stride=self.out_row)

    def run(self, dev, scale=0.0, window=0):
        self.call(dev, scale, window)
        return dev.d2h(self.d_o, (self.rows, self.out_row), np.float32)

    def reference(self, scale=0.0, window=0, unseen=None):
        """(outputs [T][qd], tolerance): unseen(r, j) says which positions no row sees."""
        hd, G = self.hd, self.H // self.KV
        sc = scale or 1.0 / np.sqrt(hd)
        out = np.zeros((self.T, self.H, hd))
        A, vmax, nmax = 0.0, 0.0, 1
        for r, (n, m) in enumerate(self.lens):
            if m == 0:
                continue
            tot = n + m
            gone = np.array([bool(unseen and unseen(r, j)) for j in range(tot)])
            q = self.q[self.start[r]:self.start[r + 1], :self.qd].astype(np.float64).reshape(m, self.H, hd)
            pos, j = np.arange(n, tot)[:, None], np.arange(tot)[None]
            seen = (j <= pos) & ~gone[None]
            if window:
                seen &= j > pos - window
            for h in range(self.H):
                k, v = self.k[r][:, h // G], self.v[r][:, h // G]
                with np.errstate(invalid="ignore", over="ignore"):
                    s = np.where(seen, q[:, h] @ np.where(np.isfinite(k), k, 0.0).T * sc, -np.inf)
                    mx = s.max(1, keepdims=True)
                    p = np.exp(s - np.where(np.isfinite(mx), mx, 0.0))
                    l = p.sum(1, keepdims=True)
                    p = p / np.where(l > 0, l, 1.0)
                    fin = np.isfinite(v).all(1)
                    o = p[:, fin] @ v[fin]
                    for jj in np.flatnonzero(~fin):  # 0 times an infinity only where it is seen
                        o = np.where(seen[:, jj:jj + 1], o + p[:, jj:jj + 1] * v[jj], o)
                out[self.start[r]:self.start[r + 1], h] = o
                kf = np.where(np.isfinite(k), k, 0.0)
                A = max(A, float((np.abs(q[:, h]) @ np.abs(kf).T).max() * abs(sc)))
                vmax = max(vmax, float(np.abs(np.where(np.isfinite(v), v, 0.0)).max()))
            nmax = max(nmax, tot)
        w = 2.0**-24 * ((hd**0.5 + 4) * A + nmax**0.5 + 16)
        return out.reshape(self.T, self.qd), 2 * w * vmax

    def check(self, dev, scale=0.0, window=0, unseen=None):
        got = self.run(dev, scale, window)
        want, tol = self.reference(scale, window, unseen)
        err = np.abs(got[:self.T, :self.qd] - want).max() if self.T else 0.0
        print(f"T {self.T}: off by {err:.2e} of {tol:.2e}", flush=True)
        assert err <= tol
        assert (got[:, self.qd:] == -5.0).all() and (got[self.T:] == -5.0).all()  # left as they were
        return got


MIXED = [(0, 1), (0, 37), (5, 0), (100, 1), (63, 1), (64, 3), (31, 33), (0, 0), (17, 130)]
# heads, kv heads, head dim, block, dtype
SHAPES = [(2, 2, 128, 16, F32), (2, 2, 128, 16, BF16), (8, 2, 128, 32, BF16), (8, 2, 64, 16, BF16), (6, 2, 64, 24, F32),
          (5, 1, 80, 7, BF16), (3, 1, 96, 1, F32), (4, 4, 256, 16, BF16), (2, 1, 256, 64, F32), (3, 3, 20, 5, BF16),
          (2, 1, 7, 3, F32), (1, 1, 1, 2, BF16), (40, 1, 128, 128, BF16), (16, 16, 64, 48, BF16), (7, 7, 36, 9, F32),
          (4, 2, 192, 16, BF16)]
IDS = ["h%dkv%dhd%dbs%ddt%d" % s for s in SHAPES]


@pytest.mark.parametrize("window", [0, 1, 40])
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_attention_mixed(dev, up, shape, window):
    """Decoding rows, chunks behind a cache and from its start, requests without rows, rows behind the last."""
    Step(up, MIXED, *shape, spare_rows=3).upload().check(dev, window=window)


@pytest.mark.parametrize("lens", [[(0, 1)], [(0, 300)], [(1000, 1)], [(4000, 2)], [(700, 333)], [(2047, 1)] * 5,
                                  [(n, 1) for n in range(0, 130)], [(0, m) for m in range(1, 70)]],
                         ids=["one", "prompt", "decode", "drafts", "chunk", "same", "each", "chunks"])
@pytest.mark.parametrize("shape", [(2, 2, 128, 16, BF16), (4, 1, 128, 16, F32), (8, 1, 64, 32, BF16)],
                         ids=["bf16", "f32", "grouped"])
def test_attention_lengths(dev, up, shape, lens):
    Step(up, lens, *shape, seed=3).upload().check(dev)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("hd", [128, 40])
def test_attention_long_context(dev, up, dt, hd):
    """Far positions, with and without a window; scores of up to about 30."""
    s = Step(up, [(9000, 1), (20000, 5)], 2, 1, hd, 16, dt, seed=4, q_scale=8.0).upload()
    s.check(dev)
    s.check(dev, window=6000)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("hd", [128, 20])
@pytest.mark.parametrize("scale", [1.0, -0.25, 1e-3, 0.0])
def test_attention_scale(dev, up, dt, hd, scale):
    Step(up, [(50, 1), (3, 40)], 4, 2, hd, 16, dt, seed=5).upload().check(dev, scale=scale)


@pytest.mark.parametrize("shape", [(2, 2, 128, 16, BF16), (6, 2, 64, 16, F32), (3, 1, 20, 5, BF16)], ids=["128", "64", "20"])
@pytest.mark.parametrize("q_extra,out_extra,stride_extra", [(64, 128, 256), (3, 5, 7), (0, 1, 4)])
def test_attention_strides(dev, up, shape, q_extra, out_extra, stride_extra):
    """Rows of q and out among others, blocks apart from each other, aligned and not."""
    Step(up, MIXED, *shape, seed=6, q_extra=q_extra, out_extra=out_extra, stride_extra=stride_extra).upload().check(dev)


@pytest.mark.parametrize("shape", [(2, 2, 128, 16, BF16), (4, 1, 128, 16, F32), (8, 2, 64, 24, BF16), (3, 1, 20, 5, F32)],
                         ids=["bf16", "f32", "64", "20"])
def test_attention_does_not_see_bad_pages(dev, up, shape):
    """Positions on a block outside the cache are not seen; a row that sees none is 0."""
    s = Step(up, [(90, 20), (200, 1), (40, 1), (0, 5)], *shape, seed=7)
    bs = s.bs
    for r, page, b in ((0, 0, -1), (0, 2, s.nb), (1, 1, 2**31 - 1), (1, 3, -2**31), (3, 0, -1)):
        s.tables[r, page] = b
    s.tables[2, :] = s.nb + 5
    bad = lambda r, j: not 0 <= s.tables[r, j // bs] < s.nb  # noqa: E731
    got = s.upload().check(dev, unseen=bad)
    assert (got[s.start[2]:s.start[3], :s.qd] == 0).all()


@pytest.mark.parametrize("shape", [(2, 2, 128, 16, BF16), (4, 1, 128, 16, F32), (3, 1, 20, 5, F32)],
                         ids=["bf16", "f32", "20"])
def test_attention_of_lengths_out_of_range(dev, up, shape):
    """kv_len below the new rows (rows before position 0 see nothing), negative, or past the table: in bounds."""
    s = Step(up, [(30, 8), (10, 3), (20, 2)], *shape, seed=8).upload()
    n = np.array([5, -4, 2**31 - 1], np.int32)
    dev.h2d(s.d_n, n)
    got = s.run(dev)[:, :s.qd]
    assert (got[:3] == 0).all()  # positions -3, -2, -1
    assert (got[8:11] == 0).all()
    want = Step(up, [(0, 5)], *shape, seed=8)
    want.q = s.q[3:8]
    want.k, want.v = [s.k[0][:5]], [s.v[0][:5]]
    ref, tol = want.reference()
    assert np.abs(got[3:8] - ref).max() <= tol


@pytest.mark.parametrize("dt", [F32, BF16])
def test_attention_of_more_rows_than_positions(dev, up, dt):
    """kv_len far below the new rows of a request whose positions are cut: the rows before position 0 are 0, the others
    see what there is."""
    s = Step(up, [(0, 3400), (50, 1)], 2, 2, 64, 16, dt, seed=36).upload()
    n = 3000
    dev.h2d(s.d_n, np.array([n, 51], np.int32))
    got = s.run(dev)[:, :s.qd]
    assert (got[:3400 - n] == 0).all()
    want = Step(up, [(0, n), (50, 1)], 2, 2, 64, 16, dt, seed=36)
    want.q = s.q[3400 - n:]
    want.k, want.v = [s.k[0][:n], s.k[1]], [s.v[0][:n], s.v[1]]
    ref, tol = want.reference()
    assert np.abs(got[3400 - n:] - ref).max() <= tol


@pytest.mark.parametrize("shape", [(200, 1, 64, 16, BF16), (300, 2, 128, 16, F32)], ids=["200", "150"])
def test_attention_of_more_heads_than_a_tile(dev, up, shape):
    Step(up, [(700, 3), (0, 5), (90, 1)], *shape, seed=37).upload().check(dev)


def test_attention_of_rows_out_of_order_stays_in_bounds(dev, up):
    """Row starts that do not ascend or pass the rows: some rows are computed, none outside the buffers."""
    s = Step(up, [(30, 8), (10, 3), (20, 2)], 2, 2, 128, 16, BF16, seed=9, spare_rows=2).upload()
    for start in ([0, 8, 3, 13], [0, 100, 200, 300], [-5, 8, 11, 2**31 - 1], [4, 4, 4, 4], [2**31 - 1, 0, 0, 0]):
        dev.h2d(s.d_s, np.array(start, np.int32))
        got = s.run(dev)
        assert got.shape == (s.rows, s.out_row)


BAD_VALUES = [np.inf, -np.inf, np.nan, -3.3895314e38]


@pytest.mark.parametrize("bad", BAD_VALUES, ids=["inf", "-inf", "nan", "lowest"])
@pytest.mark.parametrize("shape", [(2, 2, 128, 16, BF16), (4, 2, 128, 16, F32), (8, 2, 64, 24, BF16), (3, 1, 20, 5, F32)],
                         ids=["bf16", "f32", "64", "20"])
def test_attention_keeps_later_positions_out(dev, up, shape, bad):
    """Keys and values that are not finite at one position of a chunk: no row before it sees them, whatever tile
    they share; with a window, no row past it either."""
    for at, window in ((20, 0), (64, 0), (95, 0), (20, 16)):
        s = Step(up, [(10, 100), (3, 1)], *shape, seed=10)
        clean = s.upload().run(dev, window=window)
        b, off = s.tables[0, at // s.bs], at % s.bs
        s.dense[:, b, :, off] = bad
        got = s.upload().run(dev, window=window)
        rows = np.arange(10, 110)
        out_of_sight = np.concatenate(((rows < at) | (window > 0) & (rows - window + 1 > at), [True]))
        assert np.isfinite(got[:101][out_of_sight][:, :s.qd]).all()
        _, tol = s.reference(window=window)
        assert np.abs(got[:101][out_of_sight] - clean[:101][out_of_sight])[:, :s.qd].max() <= 2 * tol


@pytest.mark.parametrize("shape", [(2, 2, 128, 16, BF16), (4, 2, 128, 16, F32), (8, 2, 64, 24, BF16), (3, 1, 20, 5, F32)],
                         ids=["bf16", "f32", "64", "20"])
def test_attention_of_seen_infinities(dev, up, shape):
    """A value that is infinite or NaN makes that dim of every row that sees it so, and leaves the others."""
    s = Step(up, [(10, 100), (40, 1), (300, 1)], *shape, seed=11)
    for r, at, d, x in ((0, 30, 3, np.inf), (0, 70, 5, -np.inf), (1, 7, 0, np.nan), (2, 299, 2, np.inf)):
        s.v[r][at, :, d] = x
        s.dense[1, s.tables[r, at // s.bs], :, at % s.bs, d] = x
    got = s.upload().run(dev)[:, :s.qd]
    want, tol = s.reference()
    fin = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fin)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)])
    assert np.abs(got[fin] - want[fin]).max() <= tol


def test_attention_shares_blocks(dev, up):
    """Two requests whose tables name the same blocks (a common prefix) see the same positions."""
    s = Step(up, [(64, 1), (64, 1)], 4, 2, 128, 16, BF16, seed=12)
    s.tables[1, :4] = s.tables[0, :4]
    s.k[1][:64], s.v[1][:64] = s.k[0][:64], s.v[0][:64]
    s.upload().check(dev)


def test_attention_of_many_requests(dev, up):
    rng = np.random.default_rng(13)
    lens = [(int(rng.integers(0, 60)), int(rng.integers(0, 3))) for _ in range(4096)]
    Step(up, lens, 1, 1, 64, 16, BF16, seed=14).upload().check(dev)


# ---------------------------------------------------------------- cut ranges, large caches
# (cached, new) of requests whose positions are cut into pieces that several blocks take
CUT = [(1300, 100), (2500, 1), (700, 0), (900, 2)]
CUT_SHAPES = [(2, 2, 128, 16, BF16), (4, 2, 64, 24, F32), (4, 4, 256, 8, BF16), (3, 1, 72, 1, F32)]
CUT_IDS = ["bf16", "f32", "256", "72"]


@pytest.mark.parametrize("window", [0, 300, 1024])
@pytest.mark.parametrize("shape", CUT_SHAPES, ids=CUT_IDS)
def test_attention_of_cut_ranges(dev, up, shape, window):
    """Pieces, some of whose pages lie outside the cache, a whole piece's among them; values that are not finite are
    seen by some rows of a tile. The same call again gives the same bits."""
    s = Step(up, CUT, *shape, seed=21)
    bs = s.bs
    for r, lo, hi in ((0, 256, 640), (1, 1024, 1300), (3, 0, 130), (1, 2450, 2451)):
        s.tables[r, lo // bs:hi // bs + 1] = -1
    bad = lambda r, j: not 0 <= s.tables[r, j // bs] < s.nb  # noqa: E731
    for r, at, d, x in ((0, 1350, 3, np.inf), (0, 700, 5, np.nan), (1, 2000, 2, -np.inf)):
        s.v[r][at, :, d] = x
        s.dense[1, s.tables[r, at // bs], :, at % bs, d] = x
    got = s.upload().run(dev, window=window)
    want, tol = s.reference(window=window, unseen=bad)
    fin = np.isfinite(want)
    out = got[:, :s.qd]
    assert np.array_equal(np.isfinite(out), fin) and np.array_equal(np.isnan(out), np.isnan(want))
    assert np.abs(out[fin] - want[fin]).max() <= tol
    assert s.run(dev, window=window).tobytes() == got.tobytes()


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("new", [1, 24])
def test_attention_over_more_pages_than_a_table_holds(dev, up, dt, new):
    """Blocks of one position: a piece of a large step lies on more pages than are looked up at a time."""
    lens = [(1500 + 9 * r, new) for r in range(24)]
    s = Step(up, lens, 16, 16, 8, 1, dt, seed=22)
    for r in range(0, 24, 5):
        s.tables[r, 600:603] = (-1, s.nb, 2**31 - 1)
    s.upload().check(dev, unseen=lambda r, j: not 0 <= s.tables[r, j] < s.nb)
    s.check(dev, window=1400, unseen=lambda r, j: not 0 <= s.tables[r, j] < s.nb)


def test_attention_of_many_requests_of_large_heads(dev, up):
    """More requests than leave room in LDS for the tiles of decoding rows: the wide tiles take them."""
    rng = np.random.default_rng(23)
    lens = [(int(rng.integers(0, 40)), int(rng.integers(0, 3))) for _ in range(3000)]
    Step(up, lens, 1, 1, 256, 16, BF16, seed=24).upload().check(dev)


def append_and_attend(dev, up, kv, H, tables, max_blocks, n, seed):
    """n new positions of one request through append and attention: (outputs, what they have to be, tolerance)."""
    KV, hd, bs = kv.n_kv_heads, kv.head_dim, kv.block_size
    x = np.random.default_rng(seed).standard_normal((n, (H + 2 * KV) * hd)).astype(np.float32)
    row, pos = x.shape[1], np.arange(n)
    slots = (tables[pos // bs].astype(np.int64) * bs + pos % bs).astype(np.int32)
    d_x, d_o = up.up(x), up.up(np.full((n, H * hd), -5.0, np.float32))
    dev.paged_append(kv, hip.paged_rows_desc(n, H, None, C.c_void_p(d_x.ptr + 4 * H * hd),
                                             C.c_void_p(d_x.ptr + 4 * (H + KV) * hd), None, None, up.up(slots),
                                             k_stride=row, v_stride=row))
    t = np.full(max_blocks, -1, np.int32)
    t[:len(tables)] = tables
    b = hip.paged_batch_desc(1, max_blocks, up.up(t), up.up(np.array([n], np.int32)), up.up(np.array([0, n], np.int32)))
    dev.paged_attn(kv, b, d_x, n, H, d_o, q_stride=row)
    ref = Step(up, [(0, n)], H, KV, hd, bs if bs < 4096 else 16, kv.dtype)
    ref.q = x[:, :H * hd]
    ref.k, ref.v = ([to_cache(x[:, i * hd:(i + KV) * hd], kv.dtype)[1].reshape(n, KV, hd)] for i in (H, H + KV))
    return dev.d2h(d_o, (n, H * hd), np.float32), *ref.reference()


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("hd", [128, 20])
def test_cache_beyond_32_bits(dev, up, dt, hd):
    """Blocks whose elements lie past 2^32, in the caches' middle and at their end."""
    esz, KV, bs = (4, 2)[dt == BF16], 4, 16
    block = KV * bs * hd
    stride = (1 << 20) + 8 * 128  # elements between blocks
    nb = (1 << 32) // stride + 40
    size = ((nb - 1) * stride + block) * esz
    k, v = dev.malloc(size), dev.malloc(size)
    try:
        kv = hip.paged_kv_desc(nb, bs, KV, hd, dt, k, v, stride)
        tables = np.array([nb - 1, 3, nb - 2, nb // 2, 0, nb - 40], np.int32)
        got, want, tol = append_and_attend(dev, up, kv, 8, tables, 6, 90, 25)
        assert np.abs(got - want).max() <= tol
    finally:
        dev.free(k)
        dev.free(v)


@pytest.mark.parametrize("bs", [1 << 20, (1 << 22) + 1])
def test_blocks_around_4_gib(dev, up, bs):
    """A block just below 4 GiB, whose last head's rows lie past 2^31 bytes, and one beyond."""
    KV, hd = 15, 128
    if bs > 1 << 20:
        KV = 4
    k, v = dev.malloc(2 * KV * bs * hd), dev.malloc(2 * KV * bs * hd)
    try:
        kv = hip.paged_kv_desc(1, bs, KV, hd, BF16, k, v)
        got, want, tol = append_and_attend(dev, up, kv, KV, np.zeros(1, np.int32), 1, 70, 26)
        assert np.abs(got - want).max() <= tol
    finally:
        dev.free(k)
        dev.free(v)


@pytest.mark.parametrize("shape", [(2, 2, 128, 16, BF16), (4, 1, 64, 16, F32), (3, 1, 20, 5, BF16)], ids=["bf16", "f32", "20"])
def test_attention_in_place(dev, up, shape):
    """out may be q: a cut tile's pieces and rows that are computed again read q before it is written."""
    s = Step(up, [(900, 60), (40, 1), (0, 20)], *shape, seed=27)
    s.v[0][930, :, 1] = np.inf
    s.dense[1, s.tables[0, 930 // s.bs], :, 930 % s.bs, 1] = np.inf
    want = s.upload().run(dev)[:, :s.qd]
    dev.paged_attn(s.kv, s.batch, s.d_q, s.rows, s.H, s.d_q)
    assert dev.d2h(s.d_q, (s.rows, s.qd), np.float32).tobytes() == want.tobytes()


# ---------------------------------------------------------------- graphs, handles, failures
class Graph:
    """What fn launches on the handle's stream, captured."""
    L = None

    def __init__(self, dev, fn):
        if Graph.L is None:
            L = Graph.L = C.CDLL("libamdhip64.so")
            L.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
            L.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
            L.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
            L.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
            L.hipGraphExecDestroy.argtypes = L.hipGraphDestroy.argtypes = [C.c_void_p]
        self.dev, self.graph, self.exec = dev, C.c_void_p(), C.c_void_p()
        assert self.L.hipStreamBeginCapture(dev.stream, 2) == 0
        try:
            fn()
        finally:
            assert self.L.hipStreamEndCapture(dev.stream, C.byref(self.graph)) == 0
        assert self.L.hipGraphInstantiate(C.byref(self.exec), self.graph, None, None, 0) == 0

    def replay(self):
        assert self.L.hipGraphLaunch(self.exec, self.dev.stream) == 0

    def free(self):
        self.L.hipGraphExecDestroy(self.exec)
        self.L.hipGraphDestroy(self.graph)


class Pool:
    """The buffers of a serving step (plan, append, attention) on `nb` blocks."""

    def __init__(self, dev, up, R, P, nb, M, H=4, KV=2, hd=64, bs=8, dt=BF16):
        self.dev, self.M, self.nb, self.H, self.hd, self.R = dev, M, nb, H, hd, R
        ints = lambda *s: up.up(np.full(s, -1, np.int32))  # noqa: E731
        self.len, self.t, self.nf = up.up(np.zeros(R, np.int32)), ints(R, P), ints(1)
        self.free, self.new, qs, sl, pos, self.st = ints(nb), ints(R), ints(R + 1), ints(M), ints(M), ints(1)
        esz = np.float32 if dt == F32 else np.uint16
        self.k, self.v = (up.up(np.zeros((nb, KV, bs, hd), esz)) for _ in range(2))
        self.row = (H + 2 * KV) * hd
        self.x, self.q, self.o = (up.up(np.zeros((M, n), np.float32)) for n in (self.row, H * hd, H * hd))
        self.plan = hip.paged_plan_desc(R, P, nb, bs, M, self.len, self.new, self.t, self.free, self.nf, self.len, self.nf,
                                        qs, sl, pos, self.st)
        self.kv = hip.paged_kv_desc(nb, bs, KV, hd, dt, self.k, self.v)
        self.rows = hip.paged_rows_desc(M, H, self.x, C.c_void_p(self.x.ptr + 4 * H * hd),
                                        C.c_void_p(self.x.ptr + 4 * (H + KV) * hd), self.q, pos, sl,
                                        rope=up.up(rope_table(P * bs, hd)), n_rope=P * bs, q_stride=self.row,
                                        k_stride=self.row, v_stride=self.row)
        self.batch = hip.paged_batch_desc(R, P, self.t, self.len, qs)
        self.reset()

    def reset(self):
        self.dev.h2d(self.len, np.zeros(self.R, np.int32))
        self.dev.h2d(self.free, np.arange(self.nb, dtype=np.int32))
        self.dev.h2d(self.nf, np.array([self.nb], np.int32))

    def inputs(self, new, seed):
        self.dev.h2d(self.new, np.array(new, np.int32))
        self.dev.h2d(self.x, np.random.default_rng(seed).standard_normal((self.M, self.row)).astype(np.float32))

    def step(self, dev=None):
        d = dev or self.dev
        d.paged_plan(self.plan)
        d.paged_append(self.kv, self.rows)
        d.paged_attn(self.kv, self.batch, self.q, self.M, self.H, self.o)

    def out(self):
        assert self.dev.d2h(self.st, (1,), np.int32)[0] == 0
        return self.dev.d2h(self.o, (self.M, self.H * self.hd), np.float32)


STEPS = [[600, 0, 17, 1], [1, 40, 20, 1], [1, 1, -1, 1], [70, 1, 60, 1], [-1, 1, 1, 1], [33, 1, 900, 0], [1, 1, 1, 1],
         [0, 0, 0, 0], [1, -1, -1, 1], [9, 80, 2, 5]]


@pytest.mark.parametrize("M", [1000, 2500])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_a_captured_step_replays_for_other_lengths(dev, up, dt, M):
    """One graph of plan, append and attention over steps of other lengths, with eager steps of another pool between
    its replays: each gives the eager step's bits."""
    dev.paged_reserve()
    pool, other = Pool(dev, up, 4, 160, 300, M, dt=dt), Pool(dev, up, 4, 160, 300, M, H=8, KV=1, dt=dt)
    eager = []
    for i, new in enumerate(STEPS):
        pool.inputs(new, 40 + i)
        pool.step()
        eager.append(pool.out().tobytes())
    pool.reset()
    g = Graph(dev, pool.step)
    try:
        dev.memset(pool.o, 0)
        dev.memset(pool.t, 0xFF)
        for i, new in enumerate(STEPS):
            pool.inputs(new, 40 + i)
            other.inputs(STEPS[-1 - i] if min(STEPS[-1 - i]) >= 0 else STEPS[0], i)
            if i % 2:
                other.step()
            g.replay()
            if i % 3:
                other.step()
            dev.synchronize()
            assert pool.out().tobytes() == eager[i], i
            other.reset()
    finally:
        g.free()


def test_two_graphs_of_a_handle_share_its_workspace(dev, up):
    """Replayed in turn, as the handle's stream orders them."""
    dev.paged_reserve()
    steps = [Step(up, CUT, 2, 2, 128, 16, BF16, seed=31).upload(), Step(up, [(2000, 40), (0, 1)], 8, 2, 64, 16, F32, seed=32).upload()]
    want = [s.run(dev).tobytes() for s in steps]
    graphs = [Graph(dev, lambda s=s: s.call(dev)) for s in steps]
    try:
        for i in range(4):
            for s in steps:
                dev.memset(s.d_o, 0)
            for g in graphs[::1 if i % 2 else -1]:
                g.replay()
            dev.synchronize()
            for s, w in zip(steps, want):
                got = dev.d2h(s.d_o, (s.rows, s.out_row), np.float32)
                assert got.tobytes() == w
    finally:
        for g in graphs:
            g.free()


def test_capture_before_the_workspace_is_refused():
    with hip.Device(0) as own:
        a = Arrays(own)
        try:
            s = Step(a, [(30, 8)], 2, 2, 128, 16, BF16, seed=33).upload()
            none = hip.paged_rows_desc(1, 2, None, s.d_q, s.d_q, None, None, a.up(np.array([-1], np.int32)))

            def call():
                with pytest.raises(hip.HipError, match="captured before rbt_hip_paged_reserve"):
                    s.call(own)
                own.paged_append(s.kv, none)
            Graph(own, call).free()
            s.check(own)
        finally:
            a.free()


def test_two_handles_on_one_cache(dev, up):
    """Calls of two handles, each on its own stream and workspace, at once."""
    s = Step(up, CUT + [(300, 300)], 4, 2, 128, 16, BF16, seed=34).upload()
    want = s.run(dev).tobytes()
    with hip.Device(0) as own:
        o = own.upload_array(np.zeros((s.rows, s.out_row), np.float32))
        own.paged_reserve()
        own.synchronize()
        dev.memset(s.d_o, 0)
        dev.synchronize()
        for _ in range(5):
            s.call(dev)
            own.paged_attn(s.kv, s.batch, s.d_q, s.rows, s.H, o, q_stride=s.q.shape[1], out_stride=s.out_row)
        assert own.d2h(o, (s.rows, s.out_row), np.float32).tobytes() == want
        assert dev.d2h(s.d_o, (s.rows, s.out_row), np.float32).tobytes() == want
        own.free(o)


@pytest.mark.parametrize("mode", [1, 2])
def test_profile_names(up, mode):
    with hip.Device(0) as own:
        a = Arrays(own)
        try:
            for M, hd, names in ((1000, 64, {"paged_plan", "paged_append", "paged_attn", "paged_merge"}),
                                 (2500, 20, {"paged_plan", "paged_rows", "paged_append", "paged_attn"})):
                pool = Pool(own, a, 4, 160, 300, M, hd=hd)
                pool.inputs([60, 0, 17, 1], 1)
                own.profile(mode)
                pool.step()
                pool.out()
                after = {n: own.profile_get(n) for n in sorted(names | {"paged_rows", "paged_merge"})}
                own.profile(0)
                for n, (ms, k) in after.items():
                    assert k == (n in names), n
                    assert ms > 0.0 or n not in names
        finally:
            a.free()


CHILD = r"""
import json, sys
sys.path.insert(0, sys.argv[1])
import numpy as np
from rabbitm2_amd import hip
from tests.test_gpu_paged import Arrays, Step, CUT, BF16
res = []
with hip.Device(0) as dev:
    a = Arrays(dev)
    s = Step(a, CUT, 2, 2, 128, 16, BF16, seed=35).upload()
    for _ in range(3):
        dev.memset(s.d_o, 0)
        try:
            got = s.run(dev)
            want, tol = s.reference()
            res.append("ok" if np.abs(got[:s.T] - want).max() <= tol else "wrong")
        except hip.HipError as e:
            res.append(str(e))
    a.free()
print("RESULT " + json.dumps(res), flush=True)
"""


@pytest.mark.parametrize("fault,text", [("malloc:8", "hipMalloc"), ("launch:1", "launch_paged_clear"),
                                        ("launch:2", "launch_paged_attn"), ("launch:3", "launch_paged_merge")])
def test_failures_leave_the_handle_usable(fault, text):
    """The first call fails (the workspace's allocation, one of the launches) and says so; the next ones are right,
    also where the failed one left its items counted and its pieces unjoined. (Seven arrays are allocated before.)"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    print(f"child with RBT_HIP_FAULT={fault}", flush=True)
    r = subprocess.run([sys.executable, "-c", CHILD, root], capture_output=True, text=True, timeout=300, cwd=root,
                       env=dict(os.environ, RBT_HIP_FAULT=fault))
    assert r.returncode == 0, r.stderr[-3000:]
    res = json.loads([ln for ln in r.stdout.splitlines() if ln.startswith("RESULT ")][-1][7:])
    assert text in res[0] and res[1:] == ["ok", "ok"], res


# ---------------------------------------------------------------- a step as it is run
def test_steps_of_a_serving_loop(dev, up):
    """Plan, append and attention over steps in which requests come, read prompts in chunks, decode and end, all
    on one pool of blocks, against the whole history of each request in 64 bits."""
    H, KV, hd, bs, R, P, nb, M = 4, 2, 64, 8, 4, 16, 40, 96
    rng = np.random.default_rng(15)
    cs = rope_table(P * bs, hd)
    qn, kn = (1 + 0.1 * rng.standard_normal(n).astype(np.float32) for n in (H * hd, KV * hd))
    ints = lambda *s: up.up(np.full(s, -1, np.int32))  # noqa: E731
    d_len, d_t, d_free, d_nf = up.up(np.zeros(R, np.int32)), ints(R, P), up.up(np.arange(nb, dtype=np.int32)), \
        up.up(np.array([nb], np.int32))
    d_new, d_qs, d_sl, d_po, d_st = ints(R), ints(R + 1), ints(M), ints(M), ints(1)
    d_k, d_v = (up.up(np.full((nb, KV, bs, hd), 0x7FFF, np.uint16)) for _ in range(2))  # NaN
    d_x, d_q, d_o = (up.up(np.zeros((M, n), np.float32)) for n in ((H + 2 * KV) * hd, H * hd, H * hd))
    row = (H + 2 * KV) * hd
    plan = hip.paged_plan_desc(R, P, nb, bs, M, d_len, d_new, d_t, d_free, d_nf, d_len, d_nf, d_qs, d_sl, d_po, d_st)
    kv = hip.paged_kv_desc(nb, bs, KV, hd, BF16, d_k, d_v)
    w = hip.paged_rows_desc(M, H, d_x, C.c_void_p(d_x.ptr + 4 * H * hd), C.c_void_p(d_x.ptr + 4 * (H + KV) * hd), d_q,
                            d_po, d_sl, q_norm=up.up(qn), k_norm=up.up(kn), eps=1e-5, rope=up.up(cs), n_rope=P * bs,
                            q_stride=row, k_stride=row, v_stride=row)
    batch = hip.paged_batch_desc(R, P, d_t, d_len, d_qs)
    hist = [([], []) for _ in range(R)]
    steps = [[30, 0, 17, 1], [1, 40, 20, 1], [1, 1, -1, 1], [1, 1, 60, 1], [-1, 1, 1, 1], [33, 1, 1, 0], [1, 1, 1, 1],
             [1, -1, -1, 1], [9, 80, 2, 5]]
    for new in steps:
        for r in range(R):
            if new[r] < 0:
                hist[r] = ([], [])
        T = sum(max(n, 0) for n in new)
        x = rng.standard_normal((M, row)).astype(np.float32)
        dev.h2d(d_new, np.array(new, np.int32))
        dev.h2d(d_x, x)
        dev.paged_plan(plan)
        dev.paged_append(kv, w)
        dev.paged_attn(kv, batch, d_q, M, H, d_o)
        assert dev.d2h(d_st, (1,), np.int32)[0] == 0
        got = dev.d2h(d_o, (M, H * hd), np.float32)
        tables = dev.d2h(d_t, (R, P), np.int32)
        cache = [dev.d2h(d, (nb, KV, bs, hd), np.uint16) for d in (d_k, d_v)]
        t = 0
        for r in range(R):
            n = max(new[r], 0)
            if not n:
                continue
            ks, vs = hist[r]
            p0 = len(ks)
            c = cs[p0:p0 + n]
            q = append_ref(x[t:t + n, :H * hd], qn, c, H, hd, 1e-5)
            k = append_ref(x[t:t + n, H * hd:(H + KV) * hd], kn, c, KV, hd, 1e-5)
            ks.extend(list(k))
            vs.extend(list(x[t:t + n, (H + KV) * hd:].astype(np.float64).reshape(n, KV, hd)))
            K, V = np.array(ks), np.array(vs)
            # what the cache holds: each value within half a bf16 step (and the norm's and RoPE's f32 steps)
            slot = np.array([tables[r, p // bs] * bs + p % bs for p in range(len(K))])
            Kc, Vc = (po.bf16_to_f32(c_.transpose(0, 2, 1, 3).reshape(nb * bs, KV, hd)[slot]).astype(np.float64)
                      for c_ in cache)
            assert (np.abs(Kc - K) <= 2.0**-8 * np.abs(K) + 2.0**-18 * np.abs(K).max()).all()
            assert (np.abs(Vc - V) <= 2.0**-8 * np.abs(V)).all()
            for h in range(H):
                s = q[:, h] @ Kc[:, h // 2].T / np.sqrt(hd)
                s[np.arange(len(K))[None] > np.arange(p0, p0 + n)[:, None]] = -np.inf
                p = np.exp(s - s.max(1, keepdims=True))
                o = p / p.sum(1, keepdims=True) @ Vc[:, h // 2]
                # the query rows' f32 steps (16 + 8 of them, test_append) enter the score beside those of the sum
                A = (np.abs(q[:, h]) @ np.abs(Kc[:, h // 2]).T).max() / np.sqrt(hd)
                tol = 2 * (2.0**-17 + 2.0**-24 * ((24 + hd**0.5) * A + 20)) * np.abs(Vc).max()
                assert np.abs(got[t:t + n, h * hd:(h + 1) * hd] - o).max() <= tol
            t += n
        assert t == T
    lens = dev.d2h(d_len, (R,), np.int32)
    assert lens.tolist() == [len(k) for k, _ in hist]
    assert dev.d2h(d_nf, (1,), np.int32)[0] == nb - sum(-(-int(n) // bs) for n in lens)
