"""Whole-model steps on a paged cache (rbt_hip_paged_init / rbt_hip_forward_paged): requests that come, read their
prompts in pieces, decode and end independently. Each request must behave as the engine's forward() on it alone
(rabbit2/src/rabbit2.c:453-548): the oracle runs every request on its own, and each step must match it -- routing
identical for every (layer, token), logits normwise within 1e-3, as for batched decode.
"""
import json
import os
import subprocess
import sys

import numpy as np
import pytest

from oracle import pyoracle as po
from rabbitm2_amd import hip
from tests.common import normwise_err

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MANIFEST = json.load(open(os.path.join(ROOT, "tests", "golden", "manifest.json")))["cases"]
LOGIT_RTOL = 1e-3
F32, BF16 = hip.DT_F32, hip.DT_BF16


def build(case, **over):
    spec = MANIFEST[case]
    cfg = po.Config(**dict(spec["config"], **over))
    g = spec["gen_params"]
    return cfg, po.build_model(cfg, po.GenParams(seed=g["seed"], w_scale=g["w_scale"], fan_in_scale=g["fan_in_scale"],
                                                 emb_scale=g["emb_scale"], norm_jitter=g["norm_jitter"]))


# new tokens of four requests per step; -1: the request ends, and its number starts anew
STEPS = [[7, 0, 3, 1], [1, 5, 1, 1], [1, 1, -1, 1], [4, 1, 6, -1], [1, 1, 1, 0], [-1, 2, 1, 9], [3, 1, -1, 1],
         [0, 0, 0, 0], [1, 1, 2, 1]]


class Requests:
    """Random tokens for a run of steps, and the oracle's answer for each request on its own."""

    def __init__(self, cfg, model, steps, seed):
        rng = np.random.default_rng(seed)
        self.steps, self.cfg = steps, cfg
        self.tokens, self.want = [], []  # per step: tokens [T]; per step and request: (logits, routing rows) or None
        hist, runs = [[] for _ in steps[0]], []
        for new in steps:
            toks, places = [], []
            for r, n in enumerate(new):
                if n < 0:
                    hist[r] = []
                n = max(n, 0)
                t = rng.integers(0, cfg.vocab, n).tolist()
                if n and not hist[r]:
                    runs.append([])
                    hist[r] = runs[-1]
                places.append((hist[r], len(hist[r]), n))
                hist[r].extend(t)
                toks += t
            self.tokens.append(np.array(toks, np.int32))
            self.want.append(places)
        done = {id(r): po.run(model, np.array(r, np.int32), order=po.ORDER_AVX2) for r in runs}
        self.want = [[(done[id(h)][0][p + n - 1], done[id(h)][1][p:p + n]) if n else None for h, p, n in places]
                     for places in self.want]
        self.keep = runs

    def step(self, dev, i):
        c = self.cfg
        return dev.forward_paged(self.steps[i], self.tokens[i], c.vocab, c.n_layers, c.top_k)

    def check(self, got, i):
        logits, routing = got
        t = 0
        for r, w in enumerate(self.want[i]):
            if w is None:
                assert (logits[r] == 0).all()
                continue
            n = len(w[1])
            assert np.array_equal(routing[:, t:t + n].transpose(1, 0, 2), w[1].reshape(n, *routing.shape[::2])), f"step {i} request {r}"
            err = normwise_err(logits[r], w[0])
            assert err <= LOGIT_RTOL, f"step {i} request {r}: logits error {err:.2e}"
            t += n


CASES = ["tiny_olmoe_f32", "ref_odd_shape", "ref_qknorm_norenorm", "tiny_olmoe_bf16", "olmoe_layer_bf16"]


@pytest.mark.parametrize("bs", [1, 4, 16])
@pytest.mark.parametrize("case", CASES)
def test_steps_match_each_request_alone(dev, case, bs):
    cfg, model = build(case)
    dev.upload(model)
    dev.set_router_order(po.ORDER_AVX2)
    q = Requests(cfg, model, STEPS, seed=bs)
    dev.paged_init(4, 16, 4 * -(-16 // bs), bs, F32, 20)
    for i in range(len(STEPS)):
        q.check(q.step(dev, i), i)


def test_more_rows_than_a_wide_tile(dev):
    """Prompts of hundreds of tokens beside decoding requests, at the layer shape of the benchmark's model."""
    cfg, model = build("olmoe_layer_bf16", max_seq=300)
    dev.upload(model)
    dev.set_router_order(po.ORDER_AVX2)
    steps = [[200, 1, 0], [1, 150, 33], [1, 1, 1], [20, -1, 130], [1, 1, 1]]
    q = Requests(cfg, model, steps, seed=5)
    dev.paged_init(3, cfg.max_seq, 40, 24, F32, 250)
    for i in range(len(steps)):
        q.check(q.step(dev, i), i)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_pages_do_not_show_in_the_results(dev, dt):
    """The same steps on other block sizes, and on a pool that other requests have used before: the same bits."""
    cfg, model = build("tiny_olmoe_bf16")
    dev.upload(model)
    dev.set_router_order(po.ORDER_AVX2)
    q = Requests(cfg, model, STEPS, seed=9)
    runs = []
    for bs, used in ((16, False), (4, False), (4, True)):
        dev.paged_init(4, 16, 4 * -(-16 // bs), bs, dt, 20)
        if used:
            for i in (0, 3, 5):
                q.step(dev, i)
            q_end = [-1] * 4
            dev.forward_paged(q_end, np.zeros(0, np.int32), cfg.vocab, cfg.n_layers, cfg.top_k)
        runs.append([q.step(dev, i) for i in range(len(STEPS))])
    for other in runs[1:]:
        for (l0, r0), (l1, r1) in zip(runs[0], other):
            assert l0.tobytes() == l1.tobytes() and r0.tobytes() == r1.tobytes()


def test_refused_steps_change_nothing(dev):
    cfg, model = build("tiny_olmoe_f32")
    dev.upload(model)
    dev.set_router_order(po.ORDER_AVX2)
    q = Requests(cfg, model, STEPS, seed=3)
    dev.paged_init(4, 16, 11, 4, F32, 20)  # the steps need 9 blocks at most
    go = lambda new, toks: dev.forward_paged(new, np.array(toks, np.int32), cfg.vocab, cfg.n_layers, cfg.top_k)  # noqa: E731
    for i in range(len(STEPS)):
        for new, toks, text in (([0, 0, 0, 17], [0] * 17, "positions"), ([0, 1, 0, 0], [cfg.vocab], "out of range"),
                                ([0, 1, 0, 0], [-1], "out of range"), ([9, 9, 2, 1], [0] * 21, "room for 20")):
            if text == "room for 20" and i:
                continue
            with pytest.raises(hip.HipError, match=text):
                go(new, toks)
        q.check(q.step(dev, i), i)
    dev.paged_init(4, 16, 3, 4, F32, 20)
    go([4, 4, 0, 0], [1] * 8)
    with pytest.raises(hip.HipError, match="1 blocks are lacking"):
        go([1, 1, 0, 0], [1, 1])
    go([1, -1, 4, 0], [1] * 5)  # the ended request's block is there for this step
    with pytest.raises(hip.HipError, match="lacking"):
        go([0, 0, 1, 0], [1])


def test_refusals_of_the_state(dev):
    cfg, model = build("tiny_olmoe_f32")
    dev.upload(model)
    with pytest.raises(hip.HipError, match="no paged state"):
        dev.forward_paged([1], [0], cfg.vocab, cfg.n_layers, cfg.top_k)
    good = dict(n_req=2, ctx=8, n_blocks=4, block_size=4, dtype=F32, max_tokens=4)
    for over in (dict(n_req=0), dict(n_req=4097), dict(ctx=-1), dict(n_blocks=0), dict(block_size=0), dict(dtype=2),
                 dict(max_tokens=0), dict(max_tokens=65536), dict(n_blocks=1 << 20, block_size=1 << 12),
                 dict(n_blocks=1, block_size=2**31 - 1)):
        with pytest.raises(hip.HipError, match="paged_init"):
            dev.paged_init(**dict(good, **over))
    dev.paged_init(**good)
    dev.upload(model)  # another model ends the state
    with pytest.raises(hip.HipError, match="no paged state"):
        dev.forward_paged([1, 0], [0], cfg.vocab, cfg.n_layers, cfg.top_k)


def test_other_states_stay(dev):
    """The paged state beside the engine's own: neither disturbs the other."""
    cfg, model = build("tiny_olmoe_bf16")
    dev.upload(model)
    dev.set_router_order(po.ORDER_AVX2)
    q = Requests(cfg, model, STEPS, seed=6)
    toks = np.random.default_rng(7).integers(0, cfg.vocab, len(STEPS)).astype(np.int32)
    want = po.run(model, toks, order=po.ORDER_AVX2)
    dev.state_init(16)
    dev.paged_init(4, 16, 16, 4, F32, 20)
    for i in range(len(STEPS)):
        logits, routing = dev.forward(int(toks[i]), i, cfg.vocab, cfg.n_layers, cfg.top_k)
        assert np.array_equal(routing, want[1][i]) and normwise_err(logits, want[0][i]) <= LOGIT_RTOL
        q.check(q.step(dev, i), i)


CHILD = r"""
import json, sys
sys.path.insert(0, sys.argv[1])
from oracle import pyoracle as po
from rabbitm2_amd import hip
from tests.test_gpu_paged_model import Requests, STEPS, build, F32
res = []
with hip.Device(0) as dev:
    cfg, model = build("tiny_olmoe_bf16")
    dev.upload(model)
    dev.set_router_order(po.ORDER_AVX2)
    q = Requests(cfg, model, STEPS, seed=8)
    dev.paged_init(4, 16, 16, 4, F32, 20)
    for i in range(len(STEPS)):
        for again in range(2):
            try:
                q.check(q.step(dev, i), i)
                break
            except hip.HipError as e:
                res.append([i, str(e)])
print("RESULT " + json.dumps(res), flush=True)
"""


@pytest.mark.parametrize("fault", ["launch:2", "launch:9", "launch:61", "launch:110", "copy:6", "sync:4"])
def test_a_failed_step_can_be_run_again(fault):
    print(f"child with RBT_HIP_FAULT={fault}", flush=True)
    r = subprocess.run([sys.executable, "-c", CHILD, ROOT], capture_output=True, text=True, timeout=300, cwd=ROOT,
                       env=dict(os.environ, RBT_HIP_FAULT=fault))
    assert r.returncode == 0, r.stderr[-3000:]
    res = json.loads([ln for ln in r.stdout.splitlines() if ln.startswith("RESULT ")][-1][7:])
    assert len(res) == 1, res
