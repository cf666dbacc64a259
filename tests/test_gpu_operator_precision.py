"""Where the training operators keep more than a quick sum would: ratios near zero, a KL term that does not count,
temperatures that no f32 holds, a mean far from zero, an outlier among the first values."""
import numpy as np
import pytest

import operator_refs as refs

pytestmark = pytest.mark.gpu
F32 = refs.U["f32"]


def buffers(hip, *arrays):
    return [hip.buffer(np.asarray(a, np.float32).reshape(-1)) for a in arrays]


@pytest.mark.parametrize("vocab", [7, 300, 40000])
def test_the_gradient_of_small_ratios(hip, vocab):
    """exp of the difference itself, relative to its own size, however small."""
    moved = np.array([-3.0, -20.0, -30.0, -34.0, -36.5, -45.0, -60.0])
    rows = len(moved)
    rng = np.random.default_rng(vocab)
    z = rng.normal(size=(rows, vocab)).astype(np.float32)
    labels = rng.integers(0, vocab, rows).astype(np.int32)
    old = (refs.token_logprob(z.astype(np.float64), labels, 1.0)[0] - moved).astype(np.float32)
    advantages, weights = np.linspace(0.5, 2, rows), np.full(rows, 0.25)
    zb, ob, ab, wb = buffers(hip, z, old, advantages, weights)
    _, _, grad = hip.policy_loss(zb, hip.buffer(labels, "i32"), ob, ab, wb, (rows, vocab))
    a32, o64 = advantages.astype(np.float32).astype(np.float64), old.astype(np.float64)
    _, logp, want, size, _ = refs.policy_loss(z.astype(np.float64), labels, o64, None, a32, weights, 1.0, (0.2, 0.2), 0.0)
    assert np.abs(np.exp(logp - o64)[-1]) < 1e-25
    # the f32 sum of the row moves logp, and the gradient by as much relative to itself; p as in the other tests
    refs.assert_close(grad.read().reshape(rows, vocab), want, F32 * np.abs(want) * 1.001 + 3 * refs.STEP * size + 1e-38, "logits_grad")
    # every row by itself: the totals are then its own
    for r in range(rows):
        only = np.zeros(rows)
        only[r] = 0.25
        totals, _, _ = hip.policy_loss(zb, hip.buffer(labels, "i32"), ob, ab, hip.buffer(only.astype(np.float32)), (rows, vocab), logits_grad=False)
        want_ratio = 0.25 * np.exp(logp[r] - o64[r])
        got = totals.read().astype(np.float64)
        assert abs(got[3] - want_ratio) <= refs.STEP * want_ratio, (moved[r], got[3], want_ratio)
        assert abs(got[0] + want_ratio * a32[r]) <= refs.STEP * want_ratio * a32[r], moved[r]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [5, 9000])
def test_a_kl_term_without_weight_moves_nothing(hip, vocab, dtype):
    """ref_logp given to watch the KL term, kl_coef 0: loss and gradient are those of the call without it, also where the KL
    term is beyond its type."""
    rows = 4
    rng = np.random.default_rng(vocab)
    z = rng.normal(size=(rows, vocab))
    labels = rng.integers(0, vocab, rows).astype(np.int32)
    z[1, labels[1]] = -np.inf  # the chosen token is masked: its log-probability is -inf
    logp = refs.token_logprob(z, labels, 1.0)[0]
    ref = np.where(np.isfinite(logp), logp + 0.3, -1.0)
    ref[2] = 800.0             # exp(d) beyond f64
    old, advantages, weights = buffers(hip, np.where(np.isfinite(logp), logp - 0.1, -2.0), np.ones(rows), np.full(rows, 0.25))
    logits, ids = hip.buffer(refs.store(z, dtype).reshape(-1), dtype), hip.buffer(labels, "i32")
    plain = hip.policy_loss(logits, ids, old, advantages, weights, (rows, vocab))
    watched = hip.policy_loss(logits, ids, old, advantages, weights, (rows, vocab), ref_logp=hip.buffer(ref.astype(np.float32)), kl_coef=0.0)
    p, w = plain[0].read(), watched[0].read()
    assert np.isfinite(p).all() and w[0] == p[0] and np.array_equal(w[2:], p[2:])
    g = refs.load(watched[2].read(), dtype)
    assert np.isfinite(g).all() and np.array_equal(g, refs.load(plain[2].read(), dtype))
    # the KL total is still told (rows whose KL term is finite)
    some = hip.buffer(np.array([0.25, 0, 0, 0.25], np.float32))
    kl = hip.policy_loss(logits, ids, old, advantages, some, (rows, vocab), ref_logp=hip.buffer(ref.astype(np.float32)), kl_coef=0.0)[0].read()[1]
    want = 0.5 * (np.expm1(0.3) - 0.3)  # (d is off by f32's rounding of ref, of magnitude log(vocab) + 3, and for bf16 by that of the logits)
    assert abs(kl - want) < (1e-4 if dtype == "f32" else 0.1)


@pytest.mark.parametrize("temperature", [0.7, 1.3, 0.1, 3.0])
def test_temperatures_that_f32_does_not_hold(hip, temperature):
    """Two choices so far apart that the sum is exactly one: logp and lse are quotients, rounded once."""
    rng = np.random.default_rng(4)
    rows = 300
    z = np.zeros((rows, 2), np.float32)
    z[:, 0] = rng.uniform(-2000, 2000, rows)
    z[:, 1] = z[:, 0] - rng.uniform(500, 5000, rows).astype(np.float32)
    labels = np.ones(rows, np.int32)
    lse = hip.alloc(rows)
    got = hip.token_logprob(hip.buffer(z.reshape(-1)), hip.buffer(labels, "i32"), (rows, 2), temperature=temperature, lse=lse).read()
    z64 = z.astype(np.float64)
    refs.assert_close(got, (z64[:, 1] - z64[:, 0]) / temperature, F32 * np.abs(z64[:, 1] - z64[:, 0]) / temperature * (1 + 1e-6), "logp")
    refs.assert_close(lse.read(), z64[:, 0] / temperature, F32 * np.abs(z64[:, 0]) / temperature * (1 + 1e-6), "lse")


@pytest.mark.parametrize("p, c", [(262144, 127), (65536, 127)])
def test_an_outlier_at_the_first_position_does_not_cost_the_deviation(hip, p, c):
    """One value in a group that the others lie up to 3000 deviations away from, where a thread meets it first."""
    rng = np.random.default_rng(p)
    x = rng.normal(size=(1, p, c)).astype(np.float32)
    x[0, 0] = np.geomspace(30, 3000, c)
    out, stats = hip.group_norm(hip.buffer(x.reshape(-1)), None, None, (1, p, c), c)
    x64 = x[0].astype(np.float64)
    mean, var = x64.mean(0), x64.var(0)
    rstd = 1 / np.sqrt(var + 1e-5)
    got = stats.read().astype(np.float64).reshape(c, 2)
    # at most 1024 squares are added one after the other, and 64 operations follow; half of that in the root
    chain = (1024 + 64) * F32
    refs.assert_close(got[:, 0], mean, chain * (np.abs(x64).mean(0)), "mean")
    refs.assert_close(got[:, 1], rstd, (chain / 2 + 2 * F32) * rstd, "rstd")
    z = (x64 - mean) * rstd
    refs.assert_close(out.read().reshape(p, c), z, 4 * chain * (1 + np.abs(z)), "out")


@pytest.mark.parametrize("offset", [300.0, 1000.0, 20011.0])
@pytest.mark.parametrize("p, c", [(4100, 97), (40, 9001), (700, 331), (3, 70000), (20000, 129)])
def test_the_mean_of_one_wide_group_far_from_zero(hip, p, c, offset):
    rng = np.random.default_rng(int(offset) + c)
    x = (rng.normal(size=(1, p, c)) + offset).astype(np.float32)
    _, stats = hip.group_norm(hip.buffer(x.reshape(-1)), None, None, (1, p, c), 1)
    _, mean, rstd, _ = refs.group_norm(x.astype(np.float64), np.ones(c), np.zeros(c), 1, "none", 1e-5)
    got = stats.read().astype(np.float64)
    # the mean of a part and that of the group are each rounded once; everything else is a distance from a value (of size 5 at most)
    assert abs(got[0] - mean[0, 0]) <= 2 * F32 * abs(mean[0, 0]) * 1.001 + refs.STEP * 5, (got[0], mean[0, 0])
    assert abs(got[1] - rstd[0, 0]) <= refs.STEP * rstd[0, 0], (got[1], rstd[0, 0])


@pytest.mark.parametrize("value", [1000.1, -3.3e5, 1e-3])
@pytest.mark.parametrize("p, c", [(4100, 97), (40, 9001), (700, 331), (3, 70000)])
def test_one_wide_group_of_equal_values_has_exactly_their_mean(hip, p, c, value):
    _, stats = hip.group_norm(hip.buffer(np.full(p * c, value)), None, None, (1, p, c), 1)
    assert stats.read()[0] == np.float32(value)
    rstd = 1 / np.sqrt(np.float64(np.float32(1e-5)))
    assert abs(stats.read()[1] - rstd) <= 4 * F32 * rstd  # (a root and a quotient)
