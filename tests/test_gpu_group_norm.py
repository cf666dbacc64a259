"""Group norm with an activation, forward and backward, against the 64-bit forms on the same stored inputs."""
import numpy as np
import pytest

import operator_refs as refs
from custos_amd import Checkpoint8, capi

pytestmark = pytest.mark.gpu
EPS = 1e-5


class Case:
    """Stored inputs of one call, and their values in 64 bits."""

    def __init__(self, n, p, c, groups, dtype, params="f32", activation="silu", pad=0, seed=0, offset=0.0):
        rng = np.random.default_rng(seed)
        self.n, self.p, self.c, self.groups, self.dtype, self.params, self.activation = n, p, c, groups, dtype, params, activation
        self.pitch, self.shape = c + pad, (n, p, c)
        wide = (n, p, c + pad)
        self.x_stored = refs.store(rng.normal(size=wide) * rng.uniform(0.5, 2, c + pad) + rng.normal(size=c + pad) + offset, dtype)
        self.gamma_stored = refs.store(1 + 0.3 * rng.normal(size=c), params)
        self.beta_stored = refs.store(0.3 * rng.normal(size=c), params)
        self.x = refs.load(self.x_stored, dtype)[:, :, :c]
        self.gamma, self.beta = refs.load(self.gamma_stored, params), refs.load(self.beta_stored, params)
        self.og = rng.normal(size=wide)
        self.out, self.mean, self.rstd, self.z = refs.group_norm(self.x, self.gamma, self.beta, groups, activation, EPS)
        # (where relu's corner is within the roundings of z, the gradient is not compared: it is sent nothing)
        self.og[:, :, :c][np.abs(self.z) < 1e-3] = 0
        self.og_stored = refs.store(self.og, dtype)
        self.og = refs.load(self.og_stored, dtype)[:, :, :c]

    def out_bound(self):
        per = lambda v: refs._per_channel(v, self.groups, self.c)
        scale = (np.abs(self.x) + np.abs(per(self.mean))) * per(self.rstd) * np.abs(self.gamma) + np.abs(self.beta)
        return refs.U[self.dtype] * np.abs(self.out) * 1.001 + 1.2 * refs.STEP * (scale + np.abs(self.out)) + refs.TINY[self.dtype]

    def stats_stored(self):
        return np.stack((self.mean, self.rstd), -1).astype(np.float32)


def forward(hip, case, **over):
    b = lambda a, d: hip.buffer(a.reshape(-1), d)
    args = dict(x=b(case.x_stored, case.dtype), gamma=b(case.gamma_stored, case.params), beta=b(case.beta_stored, case.params))
    args.update(over)
    return hip.group_norm(args["x"], args["gamma"], args["beta"], case.shape, case.groups, activation=case.activation, eps=EPS,
                          x_pitch=case.pitch, out=over.get("out"), out_pitch=over.get("out_pitch"))


def check_forward(case, out, stats):
    refs.assert_close(refs.load(out.read(), case.dtype).reshape(case.shape), case.out, case.out_bound(), "out")
    s = stats.read().reshape(case.n, case.groups, 2).astype(np.float64)
    size = np.abs(case.x).reshape(case.n, case.p, case.groups, -1).max((1, 3))
    refs.assert_close(s[..., 0], case.mean, refs.STEP * size, "mean")
    # d rstd / d var = -rstd^3 / 2; the variance is off by roundings of its own terms and by those of the values
    # relative to their distance from the mean
    refs.assert_close(s[..., 1], case.rstd, refs.STEP * case.rstd * (1 + size * case.rstd), "rstd")


SIZES = [
    # n, p, c, groups, pad: one value a group of one position; single rows; odd everything
    (1, 1, 8, 8, 0), (1, 1, 64, 1, 0), (2, 1, 33, 3, 5), (1, 2, 5, 1, 0), (1, 17, 1, 1, 0), (3, 7, 6, 6, 1),
    # tiles in registers of every size
    (1, 64, 256, 32, 0), (2, 50, 320, 32, 0), (3, 100, 66, 11, 3), (2, 1024, 40, 2, 0), (1, 3000, 20, 4, 4), (1, 900, 61, 61, 0),
    # streamed: many positions, wide rows, more groups than a tile, one group wider than a workgroup's vectors
    (1, 20000, 24, 3, 0), (2, 5000, 130, 13, 1), (1, 3, 70000, 1, 0), (2, 9, 2600, 1300, 0), (1, 4100, 97, 1, 2), (1, 40, 9001, 1, 0),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n, p, c, groups, pad", SIZES)
def test_forward(hip, n, p, c, groups, pad, dtype):
    case = Case(n, p, c, groups, dtype, pad=pad, seed=p + c)
    check_forward(case, *forward(hip, case))


@pytest.mark.parametrize("activation", ["none", "relu", "gelu"])
@pytest.mark.parametrize("n, p, c, groups", [(2, 50, 48, 4), (1, 9000, 24, 3)])
def test_forward_activations_and_parameter_types(hip, n, p, c, groups, activation):
    case = Case(n, p, c, groups, "bf16", params="bf16", activation=activation)
    check_forward(case, *forward(hip, case))


@pytest.mark.parametrize("p", [40, 30000])
def test_a_large_mean_does_not_cost_the_deviation(hip, p):
    """Values 1000 deviations away from zero, and a first position unlike the rest."""
    case = Case(1, p, 12, 2, "f32", activation="none", offset=1000.0)
    x = case.x_stored.copy()
    x[:, 0] = 0
    case.x_stored, case.x = x, x.astype(np.float64)
    case.out, case.mean, case.rstd, case.z = refs.group_norm(case.x, case.gamma, case.beta, 2, "none", EPS)
    check_forward(case, *forward(hip, case))


def test_without_gamma_and_beta(hip):
    case = Case(2, 30, 16, 4, "f32")
    case.gamma, case.beta = np.ones(16), np.zeros(16)
    case.out, *_ = refs.group_norm(case.x, case.gamma, case.beta, 4, case.activation, EPS)
    check_forward(case, *forward(hip, case, gamma=None, beta=None))


@pytest.mark.parametrize("p", [30, 20000])
def test_a_group_with_nan_or_infinity_is_nan_and_the_others_are_not(hip, p):
    case = Case(2, p, 16, 4, "f32", activation="none")
    x = case.x_stored.copy()
    x[0, 1, 0], x[1, 2, 13] = np.nan, np.inf
    case.x_stored = x
    out, _ = forward(hip, case)
    bad = np.isnan(out.read().reshape(case.shape))
    want = np.zeros(case.shape, bool)
    want[0, :, :4] = want[1, :, 12:] = True
    assert np.array_equal(bad, want)


@pytest.mark.parametrize("p", [30, 9000])
def test_in_place_and_side_by_side(hip, p):
    case = Case(2, p, 17, 1, "f16")
    out, _ = forward(hip, case)
    want = out.read()
    x = hip.buffer(case.x_stored.reshape(-1), "f16")
    forward(hip, case, x=x, out=x)
    assert np.array_equal(x.read(), want)
    # x in the first 17 of 40 columns, out in the next 17: nothing else is written
    wide = np.full((2, p, 40), 7, np.float16)
    wide[:, :, :17] = case.x_stored
    both = hip.buffer(wide.reshape(-1), "f16")
    case.pitch = 40
    forward(hip, case, x=both, out=both.slice(17, both.len), out_pitch=40)
    got = both.read().reshape(2, p, 40)
    assert np.array_equal(got[:, :, :17], case.x_stored) and np.all(got[:, :, 34:] == 7)
    assert np.array_equal(got[:, :, 17:34].reshape(-1), want)


def gradients(hip, case, saved=None, overwrite=True, start=None, **over):
    b = lambda a, d: hip.buffer(a.reshape(-1), d)
    x = saved or b(case.x_stored, case.dtype)
    zeros = [np.zeros(case.n * case.p * case.pitch), np.zeros(case.c), np.zeros(case.c)] if start is None else start
    x_grad = b(refs.store(zeros[0], case.dtype), case.dtype)
    gamma_grad, beta_grad = hip.buffer(zeros[1]), hip.buffer(zeros[2])
    hip.add_group_norm_grad(x, b(case.stats_stored(), "f32"), b(case.gamma_stored, case.params), b(case.beta_stored, case.params),
                            b(case.og_stored, case.dtype), over.get("x_grad", x_grad), over.get("gamma_grad", gamma_grad),
                            over.get("beta_grad", beta_grad), case.shape, case.groups, activation=case.activation, overwrite=overwrite,
                            x_pitch=case.c if saved else case.pitch, out_grad_pitch=case.pitch, x_grad_pitch=case.pitch)
    return refs.load(x_grad.read(), case.dtype).reshape(case.n, case.p, case.pitch), gamma_grad.read(), beta_grad.read()


def check_gradients(case, got, x=None, start=None):
    s = case.stats_stored().astype(np.float64)
    want, scale = refs.group_norm_grad(case.x if x is None else x, s[..., 0], s[..., 1], case.gamma, case.beta, case.og, case.groups,
                                       case.activation)
    start = [np.zeros(case.shape), 0, 0] if start is None else start
    u = refs.U[case.dtype]
    total = want[0] + start[0]
    refs.assert_close(got[0][:, :, :case.c], total, u * np.abs(total) * 1.001 + refs.STEP * (scale[0] + np.abs(total)) + refs.TINY[case.dtype],
                      "x_grad")
    refs.assert_close(got[1], want[1] + start[1], refs.STEP * (scale[1] + np.abs(start[1])), "gamma_grad")
    refs.assert_close(got[2], want[2] + start[2], refs.STEP * (scale[2] + np.abs(start[2])), "beta_grad")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n, p, c, groups, pad", SIZES)
def test_gradients(hip, n, p, c, groups, pad, dtype):
    case = Case(n, p, c, groups, dtype, pad=pad, seed=p + c)
    got = gradients(hip, case)
    check_gradients(case, got)
    assert np.all(got[0][:, :, c:] == 0)  # between the rows nothing is written


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n, p, c, groups, pad", [s for s in SIZES if s[4] == 0])
def test_gradients_from_a_checkpoint(hip, n, p, c, groups, pad, dtype):
    case = Case(n, p, c, groups, dtype, seed=p + c)
    codes, scales = refs.checkpoint8(case.x.astype(np.float32))
    x = refs.restore8(codes, scales).astype(np.float64).reshape(case.shape)
    s = case.stats_stored().astype(np.float64)
    z = (x - refs._per_channel(s[..., 0], groups, c)) * refs._per_channel(s[..., 1], groups, c) * case.gamma + case.beta
    assert case.activation != "relu" and np.all(np.isfinite(z))
    saved = Checkpoint8(hip, hip.buffer(codes, "i8"), hip.buffer(scales), dtype)
    check_gradients(case, gradients(hip, case, saved=saved), x=x)


# more samples than workgroups: of 256 threads, and of 1024
MANY = [(9000, 2, 24, 1), (20000, 1, 10, 5), (2100, 3, 1032, 1)]


@pytest.mark.parametrize("n, p, c, groups", MANY)
def test_many_samples(hip, n, p, c, groups):
    case = Case(n, p, c, groups, "f32", seed=n)
    check_forward(case, *forward(hip, case))
    check_gradients(case, gradients(hip, case))
    start = [np.ones(case.shape)] + [np.full(c, 3, np.float32) for _ in range(2)]
    check_gradients(case, gradients(hip, case, overwrite=False, start=start), start=start)


# few positions, so that a tile takes more channels than it needs to; groups that do not divide by two
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n, p, c, groups", [(600, 5, 90, 9), (300, 64, 80, 10), (1100, 1, 96, 12), (260, 17, 260, 65)])
def test_wide_tiles(hip, n, p, c, groups, dtype):
    case = Case(n, p, c, groups, dtype, seed=n)
    check_forward(case, *forward(hip, case))
    check_gradients(case, gradients(hip, case))


@pytest.mark.parametrize("activation", ["none", "relu", "gelu"])
@pytest.mark.parametrize("n, p, c, groups", [(2, 50, 48, 4), (1, 9000, 24, 3)])
def test_gradients_are_added(hip, n, p, c, groups, activation):
    case = Case(n, p, c, groups, "f32", activation=activation)
    rng = np.random.default_rng(5)
    start = [rng.normal(size=case.shape).astype(np.float32).astype(np.float64)] + [rng.normal(size=c).astype(np.float32) for _ in range(2)]
    check_gradients(case, gradients(hip, case, overwrite=False, start=start), start=start)


@pytest.mark.parametrize("p", [20, 9000])
def test_gradients_that_are_not_wanted(hip, p):
    case = Case(2, p, 24, 3, "f32")
    full = gradients(hip, case)
    only_x = gradients(hip, case, gamma_grad=None, beta_grad=None)
    assert np.array_equal(only_x[0], full[0]) and not only_x[1].any() and not only_x[2].any()
    only_params = gradients(hip, case, x_grad=None)
    assert not only_params[0].any() and np.array_equal(only_params[1], full[1]) and np.array_equal(only_params[2], full[2])


@pytest.mark.parametrize("p", [20, 9000])
def test_gradient_in_the_place_of_what_it_reads(hip, p):
    case = Case(2, p, 19, 1, "bf16")
    want = gradients(hip, case)[0]
    b = lambda a, d: hip.buffer(a.reshape(-1), d)
    for place in ("x", "out_grad"):
        x, og = b(case.x_stored, "bf16"), b(case.og_stored, "bf16")
        target = x if place == "x" else og
        hip.add_group_norm_grad(x, b(case.stats_stored(), "f32"), b(case.gamma_stored, "f32"), b(case.beta_stored, "f32"), og, target, None,
                                None, case.shape, 1, activation="silu", overwrite=True)
        assert np.array_equal(refs.load(target.read(), "bf16").reshape(want.shape), want), place


def test_no_positions(hip):
    g, b = hip.buffer(np.ones(8)), hip.buffer(np.ones(8))
    one = hip.buffer(np.ones(8))
    hip.group_norm(one, None, None, (1, 0, 8), 2, out=one, stats=hip.buffer(np.zeros(4)))
    for overwrite, want in ((False, 1), (True, 0)):
        hip.add_group_norm_grad(one, hip.buffer(np.zeros(4)), None, None, one, hip.buffer(np.zeros(8)), g, b, (1, 0, 8), 2, overwrite=overwrite)
        assert np.all(g.read() == want) and np.all(b.read() == want)


def test_the_same_call_gives_the_same_bits(hip):
    for p in (700, 40000):
        case = Case(2, p, 40, 4, "f32")
        first = gradients(hip, case)
        again = gradients(hip, case)
        assert all(np.array_equal(a, b) for a, b in zip(first, again))


def test_python_refusals(hip):
    x = hip.buffer(np.zeros(100))
    with pytest.raises(ValueError, match="x is 100 x f32"):
        hip.group_norm(x, None, None, (2, 10, 8), 2, out=hip.alloc(160))
    with pytest.raises(ValueError, match="unknown activation"):
        hip.group_norm(x, None, None, (1, 10, 8), 2, activation="swish")
    with pytest.raises(ValueError, match="gamma is 100 x f32"):
        hip.group_norm(x, x, None, (1, 1, 101), 1, out=hip.alloc(101))
    with pytest.raises(capi.CustosHipError, match="divide into the groups"):
        hip.group_norm(x, None, None, (1, 10, 8), 3)
