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
