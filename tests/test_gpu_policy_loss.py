"""Token log-probabilities and the clipped policy loss with its gradient, against the 64-bit forms."""
import numpy as np
import pytest

import operator_refs as refs
from custos_amd import capi

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f16", "bf16"]
CLIP = (0.2, 0.3)


class Case:
    def __init__(self, rows, vocab, dtype, pad=0, temperature=1.0, ref=True, masked=True, seed=0):
        rng = np.random.default_rng(seed)
        self.rows, self.vocab, self.dtype, self.pad, self.temperature = rows, vocab, dtype, pad, temperature
        wide = 3 * rng.normal(size=(rows, vocab + pad))
        self.labels = rng.integers(0, vocab, rows).astype(np.int32)
        if masked:
            wide[rng.random(wide.shape) < 0.1] = -np.inf
            wide[np.arange(rows), self.labels] = 2.0
            self.labels[rng.random(rows) < 0.15] = -100
        self.stored = refs.store(wide, dtype)
        self.z = refs.load(self.stored, dtype)[:, :vocab]
        logp, _, _ = refs.token_logprob(self.z, self.labels, temperature)
        # ratios on both sides of the clipping range and inside it, none within rounding of its borders
        ratio = rng.choice([0.5, 0.75, 0.85, 1.0, 1.1, 1.25, 1.35, 2.0], rows) * np.exp(0.02 * (rng.random(rows) - 0.5))
        self.old = (logp - np.log(ratio)).astype(np.float32)
        self.ref = (logp + 0.5 * rng.normal(size=rows)).astype(np.float32) if ref else None
        self.advantages = rng.normal(size=rows).astype(np.float32)
        self.weights = (rng.random(rows) / rows).astype(np.float32)
        self.weights[rng.random(rows) < 0.1] = 0
        self.kl_coef = 0.1 if ref else 0.0


def near(case, got_logp, got_lse, labels=None):
    labels = case.labels if labels is None else labels
    logp, lse, _ = refs.token_logprob(case.z, labels, case.temperature)
    refs.assert_close(got_logp, logp, refs.U["f32"] * np.abs(logp) + refs.STEP * (1 + np.abs(logp)), "logp")
    if got_lse is not None:
        refs.assert_close(got_lse, lse, refs.U["f32"] * np.abs(lse) + refs.STEP * (1 + np.abs(lse)), "lse")


SIZES = [  # rows, vocab, pad
    (1, 1, 0), (3, 2, 1), (5, 7, 0), (4, 8, 3), (9, 9, 0), (130, 33, 5), (3, 2047, 0), (3, 2049, 0), (17, 1000, 24), (3, 8193, 1),
    (2, 32767, 0), (2, 32769, 2), (3, 50021, 0), (2, 65537, 0), (2, 131072, 0), (2, 131075, 1), (1, 200003, 0),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, vocab, pad", SIZES)
def test_logprob(hip, rows, vocab, pad, dtype):
    case = Case(rows, vocab, dtype, pad, temperature=0.7, seed=vocab)
    lse = hip.alloc(rows)
    out = hip.token_logprob(hip.buffer(case.stored.reshape(-1), dtype), hip.buffer(case.labels, "i32"), (rows, vocab), temperature=0.7,
                            pitch=vocab + pad, lse=lse)
    near(case, out.read(), lse.read())


def run(hip, case, **over):
    b = lambda a, d="f32": hip.buffer(np.asarray(a).reshape(-1), d)
    pitch = case.vocab + case.pad
    logits = over.pop("logits", None) or b(case.stored, case.dtype)
    grad = over.pop("logits_grad", None)
    if grad is None:
        grad = b(refs.store(np.full((case.rows, pitch), 3.0), case.dtype), case.dtype)
    return hip.policy_loss(logits, b(case.labels, "i32"), b(case.old), b(case.advantages), b(case.weights), (case.rows, case.vocab),
                           ref_logp=None if case.ref is None else b(case.ref), clip=CLIP, kl_coef=case.kl_coef, temperature=case.temperature,
                           pitch=pitch, logits_grad=grad, grad_pitch=pitch, **over)


def check(case, totals, logp, grad, grad_scale=1.0):
    f64 = lambda a: None if a is None else a.astype(np.float64)
    want, want_logp, want_grad, size, total_size = refs.policy_loss(
        case.z, case.labels, f64(case.old), f64(case.ref), f64(case.advantages), f64(case.weights), case.temperature, CLIP, case.kl_coef, grad_scale)
    refs.assert_close(totals.read(), want, refs.U["f32"] * np.abs(want) + refs.STEP * total_size, "totals")
    refs.assert_close(logp.read(), want_logp, refs.U["f32"] * np.abs(want_logp) + refs.STEP * (1 + np.abs(want_logp)), "logp")
    if grad is None:
        return
    got = refs.load(grad.read(), case.dtype).reshape(case.rows, case.vocab + case.pad)
    # the gradient's factors are off by the errors of logp (twice: ratio and KL term) and of p
    refs.assert_close(got[:, :case.vocab], want_grad,
                      refs.U[case.dtype] * np.abs(want_grad) * 1.001 + 3 * refs.STEP * size * (1 + np.abs(want_logp))[:, None] + refs.TINY[case.dtype],
                      "logits_grad")
    assert np.all(got[:, case.vocab:] == 3)  # between the rows nothing is written


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, vocab, pad", SIZES)
def test_policy_loss(hip, rows, vocab, pad, dtype):
    case = Case(rows, vocab, dtype, pad, temperature=1.3 if vocab % 2 else 1.0, seed=vocab)
    scale = 512.0 * rows if dtype == "f16" else 1.0
    check(case, *run(hip, case, grad_scale=scale), grad_scale=scale)


@pytest.mark.parametrize("rows", [1, 700, 20000, 70000])
def test_totals_of_many_rows(hip, rows):
    case = Case(rows, 5, "f32", seed=rows)
    check(case, *run(hip, case))


def test_without_a_reference_and_without_a_gradient(hip):
    case = Case(40, 500, "bf16", ref=False)
    totals, logp, grad = run(hip, case)
    check(case, totals, logp, grad)
    again, logp2, none = run(hip, case, logits_grad=False)
    assert none is None and np.array_equal(again.read(), totals.read()) and np.array_equal(logp2.read(), logp.read())


@pytest.mark.parametrize("vocab", [7, 100, 40000, 140001])
def test_gradient_in_the_place_of_the_logits(hip, vocab):
    case = Case(6, vocab, "bf16")
    _, _, grad = run(hip, case)
    logits = hip.buffer(case.stored.reshape(-1), "bf16")
    run(hip, case, logits=logits, logits_grad=logits)
    assert np.array_equal(logits.read(), grad.read())


def test_gradient_against_differences(hip):
    """Differences of the 64-bit loss, against the kernel's f32 gradient."""
    case = Case(6, 5, "f32", masked=False, seed=11)
    _, _, grad = run(hip, case)
    got = grad.read().reshape(case.z.shape)
    f64 = lambda a: a.astype(np.float64)

    def loss(z):
        return refs.policy_loss(z, case.labels, f64(case.old), f64(case.ref), f64(case.advantages), f64(case.weights), 1.0, CLIP, case.kl_coef)[0][0]

    h = 1e-5
    for at in np.ndindex(case.z.shape):
        up, down = case.z.copy(), case.z.copy()
        up[at] += h
        down[at] -= h
        assert abs((loss(up) - loss(down)) / (2 * h) - got[at]) < 1e-6, at  # (h^2 times a third derivative; f32 roundings of terms up to 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [5, 700, 9000, 140000])
def test_rows_that_are_masked_or_extreme(hip, vocab, dtype):
    case = Case(9, vocab, dtype, masked=False)
    lowest, largest = {"f32": (-3.4028235e38, 3e38), "f16": (-65504.0, 65504.0), "bf16": (-3.3895314e38, 3.3895314e38)}[dtype]
    z = case.z.copy()
    z[0] = -np.inf                       # nothing can be chosen
    z[1] = lowest                        # all equal, at the end of the range
    z[2] = lowest
    z[2, case.labels[2]] = 1.0           # everything but the label masked with the lowest value
    z[3] = np.nan                        # weight 0: not looked at
    z[4] = -np.inf                       # label -1: not looked at
    z[5] = -np.inf
    z[5, case.labels[5]] = -3.0          # one choice only
    z[6, (case.labels[6] + 1) % vocab] = np.inf
    z[7, case.labels[7]] = -np.inf       # the chosen token is masked
    case.labels[4] = -1
    case.labels[8] = vocab               # behind the vocabulary
    case.weights[:] = 0.25
    case.weights[3] = 0
    case.stored = refs.store(z, dtype)
    b = lambda a, d="f32": hip.buffer(np.asarray(a).reshape(-1), d)
    lse = hip.alloc(9)
    got = hip.token_logprob(b(case.stored, dtype), b(case.labels, "i32"), (9, vocab), temperature=0.5, lse=lse).read()
    assert np.isnan(got[[0, 3, 6, 8]]).all() and got[4] == 0 and got[5] == 0 and got[7] == -np.inf and lse.read()[0] == -np.inf
    bound = refs.STEP * (1 + np.log(vocab))
    assert abs(got[1] + np.log(vocab)) <= bound and got[2] == 0
    case.old = np.zeros(9, np.float32)
    case.ref = None
    case.kl_coef = 0.0
    case.advantages[:] = 1.0
    case.temperature = 1.0
    _, logp, grad = run(hip, case)
    g = refs.load(grad.read(), dtype).reshape(9, vocab)
    assert not g[3].any() and not g[4].any() and logp.read()[3] == 0 and logp.read()[4] == 0
    assert np.isnan(g[0]).all() and np.isnan(g[6]).any() and np.isnan(g[8]).all()
    slope = -0.25 / vocab  # ratio 1 / vocab, inside the clipping range only from below: the gradient passes
    want = np.full(vocab, -slope / vocab)
    want[case.labels[1]] += slope
    refs.assert_close(g[1], want, refs.U[dtype] * np.abs(want) + 4 * refs.STEP * abs(slope) * (1 + np.log(vocab)) + refs.TINY[dtype], "uniform row")
    assert np.abs(g[2]).max() <= refs.TINY[dtype] and np.abs(g[5]).max() <= refs.TINY[dtype] and not g[7].any()


def test_the_same_token_chosen_by_every_row_and_repeated_calls(hip):
    case = Case(300, 64, "f32")
    case.labels[:] = 5
    first = [t.read().view(np.uint8) for t in run(hip, case)]  # (bits: the token is masked in some rows, their terms are not finite)
    again = [t.read().view(np.uint8) for t in run(hip, case)]
    assert all(np.array_equal(a, b) for a, b in zip(first, again))


def test_no_rows(hip):
    one = hip.buffer(np.ones(4))
    labels = hip.buffer(np.zeros(4), "i32")
    totals, _, _ = hip.policy_loss(one, labels, one, one, one, (0, 4), logits_grad=False, logp=hip.alloc(1), totals=hip.buffer(np.ones(4)))
    assert not totals.read().any()
    out = hip.buffer(np.full(1, 7.0))
    hip.token_logprob(one, labels, (0, 4), out=out)
    assert out.read()[0] == 7


def test_python_refusals(hip):
    x = hip.buffer(np.ones(20))
    labels = hip.buffer(np.zeros(4), "i32")
    with pytest.raises(ValueError, match="labels is"):
        hip.token_logprob(x, x, (4, 5))
    with pytest.raises(ValueError, match="logits is"):
        hip.token_logprob(x, labels, (4, 6))
    with pytest.raises(ValueError, match="weights is"):
        hip.policy_loss(x, labels, x, x, hip.alloc(3), (4, 5))
    with pytest.raises(capi.CustosHipError, match="KL term needs"):
        hip.policy_loss(x, labels, hip.alloc(4), hip.alloc(4), hip.alloc(4), (4, 5), kl_coef=0.1)
