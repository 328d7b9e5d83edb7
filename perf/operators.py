"""What is measured: the paged key/value cache of a serving step, as a host program drives it.

A step of many requests runs three operators:

  plan    rbt_hip_paged_plan_dev: from every request's cached length and number of new tokens, the block
          tables (pages taken from and given back to a free list), the slot and position of each new token
          and each request's first row.
  append  rbt_hip_paged_append_dev: QK-norm and RoPE of the new rows, keys and values into their slots.
  attn    rbt_hip_paged_attn_dev: causal attention of the new rows over their request's pages.

The model shape of the benchmark (16 heads of 128 with their own key/value heads, contexts of up to 4096) is one
of the shapes; the grouped heads, other head dims and block sizes are generic. Activations are f32 as everywhere
in the framework, N(0, 1) as a QK-norm leaves them; the cache holds f32 or bf16, the framework's storage types.
"""
import ctypes as C
import math

import numpy as np
import torch

own = False

DEV = "cuda"
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
ESZ = {"f32": 4, "bf16": 2}
EPS, THETA = 1e-5, 10000.0
_handle = []


# ---------------------------------------------------------------- cases
def listed():
    model = {"heads": 16, "kv": 16, "hd": 128}     # the benchmark's model
    grouped = {"heads": 32, "kv": 8, "hd": 128}    # four query heads to a key/value head
    return [
        # one token of one sequence: the step of a single conversation, at the engine's default context
        dict(model, name="attn-decode-1", op="attn", mode="decode", cache="f32", block=16, R=1, q=1, ctx=400, window=0),
        # one step of a batch of sequences of mixed ages
        dict(model, name="attn-decode-32", op="attn", mode="decode", cache="bf16", block=16, R=32, q=1, ctx=2048,
             window=0),
        # the same of many grouped-head sequences with long contexts: the most memory a step reads
        dict(grouped, name="attn-decode-64-long", op="attn", mode="decode", cache="bf16", block=32, R=64, q=1, ctx=8192,
             window=0),
        # one long conversation: a single row per head over 128 Ki positions
        dict(grouped, name="attn-decode-131072", op="attn", mode="chunk", cache="bf16", block=64, R=1, q=1,
             ctx=131071, window=0),
        # a prompt read in at once, the longest that the model's positions allow
        dict(model, name="attn-prompt-4096", op="attn", mode="chunk", cache="bf16", block=16, R=1, q=4096, ctx=0,
             window=0),
        # a chunk of a prompt in the f32 cache that the engine's parity asks for, a ragged length
        dict(model, name="attn-chunk-f32-333", op="attn", mode="chunk", cache="f32", block=16, R=1, q=333, ctx=700,
             window=0),
        # prompt chunks and decoding sequences in one step, small heads, a sliding window, an odd block size
        dict(name="attn-mixed-window", op="attn", mode="mixed", cache="bf16", block=24, R=20, q=200, ctx=1500,
             window=512, heads=12, kv=4, hd=64),
        # one token's keys and values into the cache
        dict(model, name="append-1", op="append", cache="bf16", block=16, T=1, norm=True, rope=True),
        # a long prompt's
        dict(model, name="append-4096", op="append", cache="bf16", block=16, T=4096, norm=True, rope=True),
        # a ragged chunk's into an f32 cache, grouped heads, no QK-norm
        dict(grouped, name="append-f32-777", op="append", cache="f32", block=32, T=777, norm=False, rope=True),
        # a decode step's tables: one token per request, some of them on a new page
        dict(name="plan-32", op="plan", R=32, new=1, ctx=2048, block=16),
        # the tables of a step of many requests with prompt chunks, some requests ending
        dict(name="plan-1024", op="plan", R=1024, new=32, ctx=4096, block=16),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_one(rng):
    op = rng.choices(["attn", "append", "plan"], [6, 2, 2])[0]
    block = rng.choice([8, 16, 16, 24, 32, 64, 128])
    if op == "plan":
        return {"op": op, "R": _log(rng, 1, 1024), "new": _log(rng, 1, 32), "ctx": _log(rng, 64, 4096), "block": block}
    kv = rng.choice([1, 2, 4, 8, 16])
    c = {"op": op, "heads": kv * rng.choice([1, 1, 2, 3, 4, 8]), "kv": kv, "hd": rng.choice([64, 80, 96, 128, 128, 128, 256]),
         "cache": rng.choice(["bf16", "bf16", "f32"]), "block": block}
    if op == "append":
        return dict(c, T=_log(rng, 1, 4096), norm=rng.random() < 0.5, rope=rng.random() < 0.8)
    mode = rng.choice(["decode", "decode", "chunk", "mixed"])
    R = {"decode": _log(rng, 1, 64), "chunk": _log(rng, 1, 4), "mixed": rng.randint(2, 20)}[mode]
    q = 1 if mode == "decode" else _log(rng, 2, 2048 if mode == "chunk" else 200)
    ctx = _log(rng, 16, 8192 if mode == "decode" else 2048)
    return dict(c, mode=mode, R=R, q=q, ctx=ctx, window=rng.choice([0, 0, 0, 64, 500]))


def draw(rng):
    """One more case of the listed ones' ranges; those past the largest one's work, or whose plain form would
    pad too far, are drawn again."""
    while True:
        c = _draw_one(rng)
        w = work(c)
        if max(w["bytes"], w["flops"] / 50) > 1.0e9 or c.get("heads", 1) > 64:
            continue
        if c["op"] == "attn" and (c["R"] * c["heads"] * c["q"] * (c["q"] + c["ctx"]) > 2e8 or
                                  c["R"] * c["kv"] * c["hd"] * (c["q"] + c["ctx"]) > 8e8):
            continue
        return c


def _lengths(c):
    """(cached positions, new tokens) of each request: fixed by the case, so that every seed has the same shapes."""
    r = np.random.RandomState(7919 + 31 * c["R"] + c["ctx"])
    n = c["R"]
    cached = np.maximum(1, (c["ctx"] * r.uniform(0.15, 1.0, n)).astype(np.int64)) if c["ctx"] else np.zeros(n, np.int64)
    cached[0] = c["ctx"]
    new = np.full(n, c["q"], np.int64)
    if c["mode"] == "decode":
        new[:] = 1
    elif c["mode"] == "mixed":  # one request in five reads a prompt chunk of its own length, the others decode
        chunk = np.arange(n) % 5 == 0
        new = np.where(chunk, np.maximum(1, (c["q"] * r.uniform(0.3, 1.0, n)).astype(np.int64)), 1)
        new[0] = c["q"]
    return cached, new


# ---------------------------------------------------------------- inputs
def _normal(seed, stream, shape, dtype=torch.float32):
    g = torch.Generator(device=DEV)
    g.manual_seed((seed * 1000003 + stream) % (1 << 62))
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, 1.0, generator=g)


def _i32(a):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=torch.int32, device=DEV)


def _prepare_attn(c, seed):
    cached, new = _lengths(c)
    R, bs, T = c["R"], c["block"], int(new.sum())
    pages = -(-(cached + new) // bs)
    P, n_blocks = int(pages.max()), int(pages.sum())
    perm = np.random.RandomState(seed % (1 << 31)).permutation(n_blocks)  # pages lie anywhere
    tables = np.full((R, P), -1, np.int64)
    at = np.concatenate(([0], np.cumsum(pages)))
    for r in range(R):
        tables[r, :pages[r]] = perm[at[r]:at[r + 1]]
    shape = (n_blocks, c["kv"], bs, c["hd"])
    return {"c": c, "T": T, "P": P, "Q": int(new.max()), "n_blocks": n_blocks, "k": _normal(seed, 1, shape, DT[c["cache"]]),
            "v": _normal(seed, 2, shape, DT[c["cache"]]), "q": _normal(seed, 3, (T, c["heads"] * c["hd"])),
            "tables": _i32(tables), "kv_len": _i32(cached + new), "q_start": _i32(np.concatenate(([0], np.cumsum(new)))),
            "out": torch.zeros((T, c["heads"] * c["hd"]), device=DEV)}


def _rope_table(n, hd):
    f = THETA ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64) / hd)
    a = torch.arange(n, dtype=torch.float64).unsqueeze(1) * f
    return torch.stack((torch.cos(a), torch.sin(a)), -1)


def _prepare_append(c, seed):
    T, bs = c["T"], c["block"]
    n_blocks = -(-T // bs) + 3
    r = np.random.RandomState(seed % (1 << 31))
    first = int(r.randint(0, 2 * bs))  # tokens already in the request's cache
    perm = r.permutation(n_blocks)
    pos = np.arange(T) + first
    slots = perm[(pos - first + first % bs) // bs] * bs + pos % bs
    qd, kd = c["heads"] * c["hd"], c["kv"] * c["hd"]
    shape = (n_blocks, c["kv"], bs, c["hd"])
    return {"c": c, "n_blocks": n_blocks, "n_rope": T + 2 * bs, "q": _normal(seed, 1, (T, qd)),
            "k": _normal(seed, 2, (T, kd)), "v": _normal(seed, 3, (T, kd)),
            "q_norm": 1.0 + 0.1 * _normal(seed, 4, (qd,)), "k_norm": 1.0 + 0.1 * _normal(seed, 5, (kd,)),
            "rope": _rope_table(T + 2 * bs, c["hd"]).float().to(DEV), "positions": _i32(pos), "slots": _i32(slots),
            "kc": _normal(seed, 6, shape, DT[c["cache"]]), "vc": _normal(seed, 7, shape, DT[c["cache"]]),
            "q_out": torch.zeros((T, qd), device=DEV)}


def _prepare_plan(c, seed):
    R, bs = c["R"], c["block"]
    r = np.random.RandomState(seed % (1 << 31))
    cached = r.randint(0, c["ctx"] + 1, R)
    new = r.randint(0, c["new"] + 1, R) if c["new"] > 1 else np.ones(R, np.int64)
    if R > 8:
        new[r.rand(R) < 0.05] = -1  # requests that ended
    P = -(-(c["ctx"] + c["new"]) // bs)
    have = -(-cached // bs)
    n_blocks = int(R * P)
    perm = r.permutation(n_blocks)
    tables = np.full((R, P), -1, np.int64)
    at = np.concatenate(([0], np.cumsum(have)))
    for i in range(R):
        tables[i, :have[i]] = perm[at[i]:at[i + 1]]
    free = np.full(n_blocks, -1, np.int64)
    n_free = n_blocks - int(at[-1])
    free[:n_free] = perm[at[-1]:]
    M = R * c["new"]  # rows of the step's buffers
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)  # noqa: E731
    return {"c": c, "P": P, "n_blocks": n_blocks, "M": M, "len": _i32(cached), "new": _i32(new), "tables": _i32(tables),
            "free": _i32(free), "n_free": _i32([n_free]), "kv_len": z(R), "n_free_out": z(1), "q_start": z(R + 1),
            "slots": z(M), "positions": z(M), "status": z(1)}


def prepare(case, seed):
    return {"attn": _prepare_attn, "append": _prepare_append, "plan": _prepare_plan}[case["op"]](case, seed)


# ---------------------------------------------------------------- the plain forms, in 32 bits
def _plain_attn(s):
    """All requests padded to the longest: scores, softmax and weighted sum over the gathered pages."""
    c = s["c"]
    R, H, KV, hd, bs = c["R"], c["heads"], c["kv"], c["hd"], c["block"]
    L, Q, G = s["P"] * bs, s["Q"], c["heads"] // c["kv"]
    tables = s["tables"].long().clamp(min=0)
    k = s["k"][tables].float().permute(0, 2, 1, 3, 4).reshape(R, KV, L, hd)
    v = s["v"][tables].float().permute(0, 2, 1, 3, 4).reshape(R, KV, L, hd)
    start, kv_len = s["q_start"].long(), s["kv_len"].long()
    new = start[1:] - start[:-1]
    i, j = torch.arange(Q, device=DEV), torch.arange(L, device=DEV)
    rows = (start[:-1, None] + i).clamp(max=s["T"] - 1)
    q = s["q"].view(-1, H, hd)[rows].permute(0, 2, 1, 3).reshape(R, KV, G * Q, hd)
    pos = (kv_len - new)[:, None] + i                                   # [R][Q]
    seen = j <= pos[:, :, None]
    if c["window"]:
        seen = seen & (j > pos[:, :, None] - c["window"])
    seen = (seen & (i < new[:, None])[:, :, None])[:, None, None]       # [R][1][1][Q][L]
    x = (torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(hd))).view(R, KV, G, Q, L)
    x = x.masked_fill(~seen, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
    n = p.sum(-1, keepdim=True)
    p = p / torch.where(n == 0, torch.ones_like(n), n)
    v = v.masked_fill((j >= kv_len[:, None])[:, None, :, None], 0.0)
    o = torch.matmul(p.view(R, KV, G * Q, L), v).view(R, H, Q, hd)
    t = torch.arange(s["T"], device=DEV)
    r = torch.searchsorted(start, t, right=True) - 1
    return o[r, :, t - start[r]].reshape(s["T"], H * hd)


def _plain_rows(x, w, table, pos, heads, hd):
    if w is not None:
        x = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * w
    x = x.view(-1, heads, hd)
    if table is not None:
        cs = table[pos.long()]
        co, si = cs[:, None, :, 0], cs[:, None, :, 1]
        lo, hi = x[..., :hd // 2], x[..., hd // 2:]
        x = torch.cat((lo * co - hi * si, hi * co + lo * si), -1)
    return x


def _plain_append(s):
    c = s["c"]
    rope, bs = s["rope"] if c["rope"] else None, c["block"]
    q = _plain_rows(s["q"], s["q_norm"] if c["norm"] else None, rope, s["positions"], c["heads"], c["hd"])
    k = _plain_rows(s["k"], s["k_norm"] if c["norm"] else None, rope, s["positions"], c["kv"], c["hd"])
    block, at = s["slots"].long() // bs, s["slots"].long() % bs
    s["kc"][block, :, at] = k.to(s["kc"].dtype)
    s["vc"][block, :, at] = s["v"].view(-1, c["kv"], c["hd"]).to(s["vc"].dtype)
    return q.reshape(s["q"].shape), s["kc"], s["vc"]


def _plain_plan(s):
    c = s["c"]
    bs, P, M = c["block"], s["P"], s["M"]
    n, new, tables, n_free = s["len"].long(), s["new"].long(), s["tables"].long(), s["n_free"].long()
    ends = new < 0
    add = new.clamp(min=0)
    have = (n + bs - 1) // bs
    kv = torch.where(ends, torch.zeros_like(n), n + add)
    freed = torch.where(ends, have, torch.zeros_like(have))
    need = torch.where(ends, torch.zeros_like(have), (kv + bs - 1) // bs - have)
    page = torch.arange(P, device=DEV)
    # freed pages go on top of the free stack in (row, page) order ...
    back = page < freed[:, None]
    put = n_free + (freed.cumsum(0) - freed)[:, None] + page
    free = torch.cat((s["free"].long(), torch.zeros(1, dtype=torch.int64, device=DEV)))
    free = free.scatter(0, torch.where(back, put, torch.full_like(put, s["n_blocks"])).view(-1), tables.view(-1))
    free = free[:-1]
    top = n_free + freed.sum()
    # ... and the needed ones come off its top in the same order
    lack = (need.sum() - top).clamp(min=0)
    ok = lack == 0
    take = (page >= have[:, None]) & (page < (have + need)[:, None]) & ok
    got = top - 1 - ((need.cumsum(0) - need - have)[:, None] + page)
    tables = torch.where(take, free[got.clamp(0, s["n_blocks"] - 1)], tables)
    start = torch.cat((torch.zeros(1, dtype=torch.int64, device=DEV), add.cumsum(0))) * ok
    t = torch.arange(M, device=DEV)
    r = (torch.searchsorted(start, t, right=True) - 1).clamp(max=c["R"] - 1)
    live = t < start[-1]
    pos = n[r] + t - start[r]
    slot = tables[r, (pos // bs).clamp(0, P - 1)] * bs + pos % bs
    none = torch.full_like(t, -1)
    i32 = lambda x: x.to(torch.int32)  # noqa: E731
    return {"tables": i32(tables), "free": i32(torch.where(ok, free, s["free"].long())),
            "kv_len": i32(torch.where(ok, kv, n)), "n_free": i32(torch.where(ok, top - need.sum(), n_free)),
            "q_start": i32(start), "slots": i32(torch.where(live, slot, none)),
            "positions": i32(torch.where(live, pos, none)), "status": i32(lack).view(1)}


# ---------------------------------------------------------------- the framework's calls
def _dev():
    if not _handle:
        from rabbitm2_amd import hip
        _handle.append(hip.Device(0))  # one handle per program, as the engine has
        _handle[0].paged_reserve()
    return _handle[0]


def _ptr(t):
    return C.c_void_p(t.data_ptr())


def _describe(s):
    """The descriptors of a state's buffers, which a program keeps with them."""
    from rabbitm2_amd import hip
    c = s["c"]
    if c["op"] == "plan":
        return {"plan": hip.paged_plan_desc(c["R"], s["P"], s["n_blocks"], c["block"], s["M"], _ptr(s["len"]), _ptr(s["new"]),
                                            _ptr(s["tables"]), _ptr(s["free"]), _ptr(s["n_free"]), _ptr(s["kv_len"]),
                                            _ptr(s["n_free_out"]), _ptr(s["q_start"]), _ptr(s["slots"]),
                                            _ptr(s["positions"]), _ptr(s["status"]))}
    dt = {"f32": hip.DT_F32, "bf16": hip.DT_BF16}[c["cache"]]
    if c["op"] == "append":
        kv = hip.paged_kv_desc(s["n_blocks"], c["block"], c["kv"], c["hd"], dt, _ptr(s["kc"]), _ptr(s["vc"]))
        rows = hip.paged_rows_desc(c["T"], c["heads"], _ptr(s["q"]), _ptr(s["k"]), _ptr(s["v"]), _ptr(s["q_out"]),
                                   _ptr(s["positions"]), _ptr(s["slots"]),
                                   q_norm=_ptr(s["q_norm"]) if c["norm"] else None,
                                   k_norm=_ptr(s["k_norm"]) if c["norm"] else None, eps=EPS,
                                   rope=_ptr(s["rope"]) if c["rope"] else None, n_rope=s["n_rope"])
        return {"kv": kv, "rows": rows}
    kv = hip.paged_kv_desc(s["n_blocks"], c["block"], c["kv"], c["hd"], dt, _ptr(s["k"]), _ptr(s["v"]))
    return {"kv": kv, "batch": hip.paged_batch_desc(c["R"], s["P"], _ptr(s["tables"]), _ptr(s["kv_len"]),
                                                    _ptr(s["q_start"])), "q": _ptr(s["q"]), "out": _ptr(s["out"])}


def _own(s):
    dev, c = _dev(), s["c"]
    if "desc" not in s:
        s["desc"] = _describe(s)
    d = s["desc"]
    if c["op"] == "plan":
        dev.paged_plan(d["plan"])
        return {"tables": s["tables"], "free": s["free"], "kv_len": s["kv_len"], "n_free": s["n_free_out"],
                "q_start": s["q_start"], "slots": s["slots"], "positions": s["positions"], "status": s["status"]}
    if c["op"] == "append":
        dev.paged_append(d["kv"], d["rows"])
        return s["q_out"], s["kc"], s["vc"]
    dev.paged_attn(d["kv"], d["batch"], d["q"], s["T"], c["heads"], d["out"], window=c["window"])
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return {"attn": _plain_attn, "append": _plain_append, "plan": _plain_plan}[state["c"]["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "plan":
        tokens = c["R"] * (c["new"] / 2 if c["new"] > 1 else 1)
        return {"bytes": 16.0 * c["R"] + 8.0 * c["R"] * c["new"] + 8.0 * tokens / c["block"], "flops": 0.0}
    qd, kd, e = c["heads"] * c["hd"], c["kv"] * c["hd"], ESZ[c["cache"]]
    if c["op"] == "append":
        T = c["T"]
        by = T * (8.0 * qd + 2 * kd * (4 + e) + 8 + (4.0 * c["hd"] if c["rope"] else 0)) + (4 * (qd + kd) if c["norm"] else 0)
        return {"bytes": by, "flops": T * (qd + kd) * (4.0 * c["norm"] + 3.0 * c["rope"])}
    cached, new = _lengths(c)
    by, pairs = 0.0, 0
    for n, m in zip(cached.tolist(), new.tolist()):
        pos = np.arange(n, n + m, dtype=np.int64)
        seen = np.minimum(pos + 1, c["window"]) if c["window"] else pos + 1
        pairs += int(seen.sum())
        by += (n + m - (pos[0] + 1 - seen[0])) * 2.0 * kd * e
    return {"bytes": by + 8.0 * qd * int(new.sum()), "flops": 4.0 * c["hd"] * c["heads"] * pairs}


# ---------------------------------------------------------------- the same in 64 bits
def _exact_attn(c, seed):
    s = _prepare_attn(c, seed)
    hd, g, bs = c["hd"], c["heads"] // c["kv"], c["block"]
    lens, start = s["kv_len"].tolist(), s["q_start"].tolist()
    out = torch.zeros((s["T"], c["heads"], hd), dtype=torch.float64, device=DEV)
    for r, n in enumerate(lens):
        m = start[r + 1] - start[r]
        first = max(0, n - m + 1 - c["window"]) if c["window"] else 0  # no row looks further back
        p0, p1 = first // bs, -(-n // bs)
        pages = s["tables"][r, p0:p1].long()
        for h in range(c["kv"]):
            K = s["k"][pages, h].double().reshape(-1, hd)[:n - p0 * bs]
            V = s["v"][pages, h].double().reshape(-1, hd)[:n - p0 * bs]
            at = torch.arange(p0 * bs, n, device=DEV)
            for i0 in range(0, m, 512):
                i1 = min(m, i0 + 512)
                q = s["q"][start[r] + i0:start[r] + i1].double().view(i1 - i0, c["heads"], hd)[:, h * g:(h + 1) * g]
                x = torch.einsum("ihd,jd->ihj", q, K) / math.sqrt(hd)
                pos = torch.arange(n - m + i0, n - m + i1, device=DEV)[:, None]
                bad = at > pos
                if c["window"]:
                    bad |= at <= pos - c["window"]
                x.masked_fill_(bad[:, None], -math.inf)
                out[start[r] + i0:start[r] + i1, h * g:(h + 1) * g] = torch.einsum("ihj,jd->ihd", torch.softmax(x, -1), V)
    return out.view(s["T"], -1)


def _exact_append(c, seed):
    s = _prepare_append(c, seed)
    hd, bs, T = c["hd"], c["block"], c["T"]
    cs = s["rope"].double()[s["positions"].long()]
    turn = torch.complex(cs[..., 0], cs[..., 1])[:, None]

    def rows(x, w, heads):
        x = x.double()
        if c["norm"]:
            x = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / x.shape[1] + EPS) * w.double()
        x = x.reshape(T, heads, hd)
        if c["rope"]:
            z = torch.complex(x[..., :hd // 2].contiguous(), x[..., hd // 2:].contiguous()) * turn
            x = torch.cat((z.real, z.imag), -1)
        return x

    kc, vc = s["kc"].double(), s["vc"].double()
    flat = lambda t: t.permute(0, 2, 1, 3).reshape(-1, c["kv"], hd)  # noqa: E731  a slot is a row
    unflat = lambda t: t.view(s["n_blocks"], bs, c["kv"], hd).permute(0, 2, 1, 3).contiguous()  # noqa: E731
    kc = unflat(flat(kc).index_copy(0, s["slots"].long(), rows(s["k"], s["k_norm"], c["kv"])))
    vc = unflat(flat(vc).index_copy(0, s["slots"].long(), s["v"].double().view(T, c["kv"], hd)))
    return rows(s["q"], s["q_norm"], c["heads"]).reshape(T, -1), kc, vc


def exact(case, seed):
    if case["op"] == "plan":  # whole numbers
        return None
    return (_exact_attn if case["op"] == "attn" else _exact_append)(case, seed)
