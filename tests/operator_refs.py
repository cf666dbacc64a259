"""Plain 64-bit forms of the training operators, storage conversions and the bounds the tests compare with.

Bounds.  U[t] is half a step of a storage type relative to the value (the one rounding at the store).  Everything
before it is f32 arithmetic; CHAIN bounds the roundings on any path from the inputs to a value: no kernel adds
more than 200 terms one after the other for the sizes tested here (a thread's rows, then lanes, then wavefronts,
then parts), and fewer than 50 further operations follow.  So a value computed from terms of magnitude `scale`
is off by at most CHAIN * 2^-24 * scale.
"""
import numpy as np

U = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}
CHAIN = 256
STEP = CHAIN * 2.0**-24
TINY = {"f32": 2.0**-149, "f16": 2.0**-24, "bf16": 2.0**-133}  # spacing of the smallest values


def store(a, dtype):
    """`a` rounded to the storage type, as the array a buffer takes."""
    a = np.asarray(a, dtype=np.float32)
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return a.astype(np.float16)
    if dtype == "bf16":
        bits = np.ascontiguousarray(a).view(np.uint32)
        out = ((bits + 0x7FFF + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
        return np.where(np.isnan(a), ((bits >> 16) | 0x40).astype(np.uint16), out)
    return a


def load(a, dtype):
    """The values of a storage array, in 64 bits."""
    if dtype == "bf16":
        return (np.ascontiguousarray(a, dtype=np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return np.asarray(a).astype(np.float64)


def assert_close(got, want, bound, what):
    got, want, bound = np.asarray(got, np.float64), np.asarray(want, np.float64), np.broadcast_to(bound, np.shape(want))
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN in other places"
    infinite = np.isinf(want)
    assert np.array_equal(got[infinite], want[infinite]), f"{what}: infinities"
    ok = np.isnan(want) | infinite | (np.abs(got - np.where(infinite, 0, want)) <= bound)
    if not ok.all():
        at = np.argwhere(~ok)[:5]
        raise AssertionError(f"{what}: {int((~ok).sum())} of {ok.size} beyond the bound, first at {at.tolist()}: "
                             f"{[(got[tuple(i)], want[tuple(i)], bound[tuple(i)]) for i in at]}")


# ---- group norm ----

def _erf(z):
    from scipy.special import erf
    return erf(z)


def act(z, name):
    if name == "relu":
        return np.where(z < 0, 0.0, z)
    if name == "silu":
        with np.errstate(over="ignore"):
            return z / (1 + np.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + _erf(z / np.sqrt(2)))
    return z


def act_grad(z, name):
    if name == "relu":
        return (z > 0).astype(np.float64)
    if name == "silu":
        with np.errstate(over="ignore"):
            s = 1 / (1 + np.exp(-z))
        return s * (1 + z * (1 - s))
    if name == "gelu":
        return 0.5 * (1 + _erf(z / np.sqrt(2))) + z * np.exp(-z * z / 2) / np.sqrt(2 * np.pi)
    return np.ones_like(z)


def _per_channel(v, groups, channels):
    """[n, groups] -> [n, 1, channels]"""
    return np.repeat(v, channels // groups, axis=1)[:, None, :]


def group_norm(x, gamma, beta, groups, activation, eps):
    """(out, mean, rstd, z) of x [n, p, c]."""
    n, p, c = x.shape
    g = x.reshape(n, p, groups, c // groups)
    mean = g.mean(axis=(1, 3))
    var = ((g - mean[:, None, :, None]) ** 2).mean(axis=(1, 3))
    rstd = 1 / np.sqrt(var + eps)
    z = (x - _per_channel(mean, groups, c)) * _per_channel(rstd, groups, c) * gamma + beta
    return act(z, activation), mean, rstd, z


def group_norm_grad(x, mean, rstd, gamma, beta, out_grad, groups, activation):
    """(x_grad, gamma_grad, beta_grad) and, for the bounds, the magnitudes their terms have."""
    n, p, c = x.shape
    m, r = _per_channel(mean, groups, c), _per_channel(rstd, groups, c)
    h = (x - m) * r
    z = h * gamma + beta
    dz = out_grad * act_grad(z, activation)

    def group_mean(v):
        return _per_channel(v.reshape(n, p, groups, c // groups).mean(axis=(1, 3)), groups, c)

    dh = dz * gamma
    x_grad = r * (dh - group_mean(dh) - h * group_mean(dh * h))
    # how far dz can be off: act' has slopes of at most 1.2, and z is off by roundings of its terms
    h_scale = (np.abs(x) + np.abs(m)) * r
    dz_scale = np.abs(out_grad) * (1.2 + 1.2 * (h_scale * np.abs(gamma) + np.abs(beta)))
    dh_scale = dz_scale * np.abs(gamma)
    scale = r * (dh_scale + group_mean(dh_scale) + (1 + h_scale) * group_mean(dh_scale * (1 + h_scale)))
    return ((x_grad, (dz * h).sum((0, 1)), dz.sum((0, 1))),
            (scale, (dz_scale * (1 + h_scale)).sum((0, 1)), dz_scale.sum((0, 1))))


# ---- 8-bit checkpoints ----

def checkpoint8(x):
    """(codes, scales) of a flat f32 array, by the 32-bit steps that define them."""
    x = np.asarray(x, np.float32).reshape(-1)
    n = x.size
    blocks = np.zeros(-(-n // 128) * 128, np.float32)
    blocks[:n] = x
    blocks = blocks.reshape(-1, 128)
    finite = np.isfinite(blocks)
    top = np.where(finite, np.abs(blocks), np.float32(0)).max(1, keepdims=True)
    kept = top >= np.float32(2.0**-100)
    with np.errstate(divide="ignore", invalid="ignore"):
        step = np.where(kept, np.float32(127) / top, np.float32(0)).astype(np.float32)
        codes = np.rint(np.where(finite, blocks, np.float32(0)) * step)
    codes = np.where(finite, codes, -128).astype(np.int8)
    scales = np.where(kept, top * np.float32(1 / 127), np.float32(0)).astype(np.float32)
    return codes.reshape(-1)[:n], scales.reshape(-1)


def restore8(codes, scales):
    """The f32 values codes and scales stand for."""
    v = codes.astype(np.float32) * np.repeat(scales, 128)[:codes.size]
    return np.where(codes == -128, np.float32(np.nan), v).astype(np.float32)


# ---- log-probabilities and the policy loss ----

def token_logprob(z, labels, temperature):
    """(logp, lse, softmax) of rows of logits; a negative label's logp is 0, one behind the vocabulary NaN."""
    z = z / temperature
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        top = z.max(1, keepdims=True)
        e = np.exp(z - np.where(np.isfinite(top), top, 0))
        total = e.sum(1)
        lse = top[:, 0] + np.log(total)
        p = e / total[:, None]
        at = np.clip(labels, 0, z.shape[1] - 1)
        logp = np.where(labels < 0, 0.0, np.where(labels >= z.shape[1], np.nan, z[np.arange(len(labels)), at] - lse))
    return logp, lse, p


def policy_loss(z, labels, old, ref, advantage, weight, temperature, clip, kl_coef, grad_scale=1.0):
    """(totals, logp, gradient) and the magnitude of the gradient's terms at the label and elsewhere."""
    logp, _, p = token_logprob(z, labels, temperature)
    used = (labels >= 0) & (weight != 0)
    logp = np.where(used, logp, 0.0)
    r = np.exp(logp - old)
    bounded = np.clip(r, 1 - clip[0], 1 + clip[1])
    inside = r * advantage <= bounded * advantage
    d = ref - logp if ref is not None else np.zeros_like(logp)
    kl = np.expm1(d) - d
    w = np.where(used, weight, 0.0)
    totals = np.array([(w * (kl_coef * kl - np.minimum(r * advantage, bounded * advantage))).sum(), (w * kl).sum(), (w * ~inside).sum(), (w * r).sum()])
    slope = w * (np.where(inside, -advantage * r, 0.0) - kl_coef * np.expm1(d)) * grad_scale / temperature
    onehot = np.zeros_like(z)
    onehot[np.arange(len(labels)), np.clip(labels, 0, z.shape[1] - 1)] = 1
    grad = np.where(used[:, None], slope[:, None] * (onehot - p), 0.0)
    size = np.abs(w) * (np.abs(advantage) * r + abs(kl_coef) * (np.exp(d) + 1)) * abs(grad_scale) / temperature
    total_size = np.array([(np.abs(w) * (abs(kl_coef) * (kl + np.abs(d) + 1) + np.abs(advantage) * r)).sum(), (np.abs(w) * (kl + np.abs(d) + 1)).sum(),
                           np.abs(w).sum(), (np.abs(w) * r).sum()])
    return totals, logp, grad, np.where(used[:, None], size[:, None] * (onehot + p), 0.0), total_size
