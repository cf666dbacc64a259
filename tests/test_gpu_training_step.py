"""The training operators run together, as a step uses them: normalisation, a unary operation whose input is kept in
8 bits, the policy loss, and back through all of them -- eager, recorded and replayed, and next to other work."""
import numpy as np
import pytest

import custos_amd
import operator_refs as refs
from custos_amd import capi

pytestmark = pytest.mark.gpu
CLIP = (0.2, 0.3)


class Step:
    """rows of logits = tanh(group_norm(x)) scaled; loss of chosen tokens; gradients of x, gamma and beta; an SGD step."""

    def __init__(self, dev, n=2, p=70, c=40, groups=4, seed=0):
        self.dev, self.shape, self.groups = dev, (n, p, c), groups
        rng = np.random.default_rng(seed)
        self.rows, self.size = n * p, n * p * c
        self.x = dev.buffer(rng.normal(size=self.size))
        self.gamma, self.beta = dev.buffer(1 + 0.1 * rng.normal(size=c)), dev.buffer(0.1 * rng.normal(size=c))
        self.labels = dev.buffer(rng.integers(0, c, self.rows), "i32")
        self.old = dev.buffer(-np.log(c) + 0.05 * rng.normal(size=self.rows))
        self.ref = dev.buffer(-np.log(c) + 0.05 * rng.normal(size=self.rows))
        self.adv, self.weights = dev.buffer(rng.normal(size=self.rows)), dev.buffer(np.full(self.rows, 1 / self.rows))
        self.h, self.stats = dev.alloc(self.size), dev.alloc(n * groups * 2)
        self.x8, self.h8 = dev.alloc_checkpoint8(self.size), dev.alloc_checkpoint8(self.size)
        self.logits, self.dlogits, self.dh, self.dx = (dev.alloc(self.size) for _ in range(4))
        self.dgamma, self.dbeta = dev.alloc(c), dev.alloc(c)
        self.totals, self.logp = dev.alloc(4), dev.alloc(self.rows)

    def run(self):
        d = self.dev
        d.checkpoint8(self.x, into=self.x8)
        d.group_norm(self.x, self.gamma, self.beta, self.shape, self.groups, "silu", out=self.h, stats=self.stats)
        d.apply_fn_checkpoint8(self.h, lambda v: v.tanh(), out=self.logits, into=self.h8)
        n, p, c = self.shape
        d.policy_loss(self.logits, self.labels, self.old, self.adv, self.weights, (n * p, c), ref_logp=self.ref, clip=CLIP, kl_coef=0.1,
                      logits_grad=self.dlogits, logp=self.logp, totals=self.totals)
        d.clear(self.dh)
        d.add_unary_grad8(self.h8, self.dh, self.dlogits, lambda v: v.tanh().mul(v.tanh()).neg().add(1.0))
        d.add_group_norm_grad(self.x8, self.stats, self.gamma, self.beta, self.dh, self.dx, self.dgamma, self.dbeta, self.shape,
                              self.groups, "silu", overwrite=True)
        d.apply_fn2(self.gamma, self.dgamma, lambda w, g: w.sub(g.mul(0.5)), out=self.gamma)

    def outputs(self):
        return [b.read() for b in (self.logits, self.totals, self.logp, self.dlogits, self.dx, self.dgamma, self.dbeta, self.gamma)]


def same(a, b):
    return all(np.array_equal(x, y) for x, y in zip(a, b))


def test_the_step_against_the_formulas(hip):
    step = Step(hip, seed=3)
    n, p, c = step.shape
    x, gamma, beta = step.x.read().astype(np.float64).reshape(step.shape), step.gamma.read().astype(np.float64), step.beta.read().astype(np.float64)
    step.run()
    logits, totals, logp, dlogits, dx, dgamma, dbeta, new_gamma = step.outputs()
    out, mean, rstd, _ = refs.group_norm(x, gamma, beta, step.groups, "silu", 1e-5)
    want_logits = np.tanh(out)
    # tanh has slopes of at most 1: as far off as its input, and a few steps of its own
    scale = (np.abs(x) + 1) * rstd.max() * np.abs(gamma).max() + 1
    refs.assert_close(logits.reshape(step.shape), want_logits, 2 * refs.STEP * scale, "logits")
    # everything after it is compared on the values that were stored on the way
    z = logits.astype(np.float64).reshape(n * p, c)
    f64 = lambda b: b.read().astype(np.float64)
    t, lp, g, size, t_size = refs.policy_loss(z, step.labels.read(), f64(step.old), f64(step.ref), f64(step.adv), f64(step.weights), 1.0, CLIP, 0.1)
    refs.assert_close(totals, t, refs.U["f32"] * np.abs(t) + refs.STEP * t_size, "totals")
    refs.assert_close(dlogits.reshape(n * p, c), g, refs.U["f32"] * np.abs(g) + 3 * refs.STEP * size * (1 + np.abs(lp))[:, None], "dlogits")
    h = refs.restore8(step.h8.codes.read(), step.h8.scales.read()).astype(np.float64)
    dh = dlogits.astype(np.float64) * (1 - np.tanh(h) ** 2)
    refs.assert_close(f64(step.dh), dh, refs.U["f32"] * np.abs(dh) + 32 * 2.0**-24 * np.abs(dlogits), "dh")
    s = step.stats.read().astype(np.float64).reshape(n, step.groups, 2)
    x8 = refs.restore8(step.x8.codes.read(), step.x8.scales.read()).astype(np.float64).reshape(step.shape)
    (wx, wg, wb), (sx, sg, sb) = refs.group_norm_grad(x8, s[..., 0], s[..., 1], gamma, beta, f64(step.dh).reshape(step.shape), step.groups, "silu")
    refs.assert_close(dx.reshape(step.shape), wx, refs.U["f32"] * np.abs(wx) + refs.STEP * sx, "dx")
    refs.assert_close(dgamma, wg, refs.STEP * sg, "dgamma")
    refs.assert_close(dbeta, wb, refs.STEP * sb, "dbeta")
    assert np.array_equal(new_gamma, gamma.astype(np.float32) - dgamma * np.float32(0.5))


@pytest.mark.parametrize("edges", [capi.GRAPH_EDGES_CHAIN, capi.GRAPH_EDGES_LEVEL_JOINS, capi.GRAPH_EDGES_PER_NODE, capi.GRAPH_EDGES_CHAIN_BY_LEVEL])
@pytest.mark.parametrize("p", [70, 9000])
def test_recorded_and_replayed(edges, p):
    dev = custos_amd.HIP(0)
    try:
        dev.set_graph_edges(edges)
        dev.set_graph_verify(True)
        step, eager = Step(dev, p=p, seed=1), Step(dev, p=p, seed=1)
        dev.capture_begin()
        step.run()
        graph = dev.capture_end()
        names = graph.kernel_names()
        assert any("group_norm" in k for k in names) and any("policy" in k for k in names) and any("save8" in k for k in names)
        other = Step(dev, n=1, p=33, c=24, groups=3, seed=9)
        for replay in range(4):
            # new inputs, the program's own work and waits between the replays
            x = np.random.default_rng(replay).normal(size=step.size)
            step.x.write(x), eager.x.write(x)
            other.run()
            if replay % 2:
                dev.sync()
            graph.launch()
            eager.run()
            assert same(step.outputs(), eager.outputs()), replay
    finally:
        dev.close()


def test_two_graphs_share_the_work_area_and_outlive_its_growth():
    dev = custos_amd.HIP(0)
    try:
        small, large = Step(dev, p=50, seed=1), Step(dev, n=3, p=5000, c=64, groups=8, seed=2)
        check = [Step(dev, p=50, seed=1), Step(dev, n=3, p=5000, c=64, groups=8, seed=2)]
        graphs = []
        for step in (small, large):
            dev.capture_begin()
            step.run()
            graphs.append(dev.capture_end())
        # an operator that needs more than the work area held when the graphs were built
        big = dev.buffer(np.random.default_rng(0).normal(size=300000))
        labels, zeros = dev.buffer(np.zeros(300000), "i32"), dev.buffer(np.zeros(300000))
        for turn in range(3):
            for which, (graph, step, eager) in enumerate(zip(graphs, (small, large), check)):
                dev.policy_loss(big, labels, zeros, zeros, zeros, (300000, 1), logits_grad=False)
                graph.launch()
                eager.run()
                assert same(step.outputs(), eager.outputs()), (turn, which)
    finally:
        dev.close()


def test_a_recording_that_repeats_is_recognised():
    dev = custos_amd.HIP(0)
    try:
        step = Step(dev, seed=4)
        previous = None
        for run in range(4):
            dev.capture_begin()
            step.run()
            graph = dev.capture_end_reuse(previous)
            if previous is not None:
                assert graph is previous
            graph.launch()
            previous = graph
        reused, _, built = dev.capture_stats()
        assert built == 1 and reused == 3
        # one argument that differs makes another graph
        dev.capture_begin()
        step.dev.group_norm(step.x, step.gamma, step.beta, step.shape, step.groups, "relu", out=step.h, stats=step.stats)
        assert dev.capture_end_reuse(previous) is not previous
    finally:
        dev.close()


def test_two_handles_at_once():
    """Each handle has a stream and a work area of its own."""
    a, b = custos_amd.HIP(0), custos_amd.HIP(0)
    try:
        steps = [Step(a, p=3000, seed=5), Step(b, p=3000, seed=6)]
        alone = []
        for step in steps:
            step.run()
            alone.append(step.outputs())
        fresh = [Step(a, p=3000, seed=5), Step(b, p=3000, seed=6)]
        for step in fresh:
            step.run()  # (queued on both streams before either is read)
        assert all(same(step.outputs(), want) for step, want in zip(fresh, alone))
    finally:
        a.close()
        b.close()


def test_a_replayed_graph_of_few_operators_is_issued_directly(hip):
    """A chain of up to four nodes is replayed as plain launches."""
    x = hip.buffer(np.random.default_rng(0).normal(size=2 * 30 * 16))
    out, stats = hip.alloc(x.len), hip.alloc(2 * 4 * 2)
    hip.capture_begin()
    hip.group_norm(x, None, None, (2, 30, 16), 4, out=out, stats=stats)
    saved = hip.checkpoint8(out)
    graph = hip.capture_end()
    assert graph.kernel_nodes <= 4 and graph.edge_count() == 0
    for k in range(3):
        x.write(np.random.default_rng(k).normal(size=x.len))
        graph.launch()
        want, _ = hip.group_norm(x, None, None, (2, 30, 16), 4)
        assert np.array_equal(out.read(), want.read())
        codes, scales = refs.checkpoint8(want.read())
        assert np.array_equal(saved.codes.read(), codes) and np.array_equal(saved.scales.read(), scales)
    graph.destroy()
