"""The training operators where offsets pass 32 bits: every row or block there gives, bit for bit, what the same
values give in a small buffer."""
import numpy as np
import pytest

import custos_amd
import operator_refs as refs
from custos_amd import Checkpoint8

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev():
    device = custos_amd.HIP(0)  # (of its own: what it allocates goes back when it closes)
    yield device
    device.close()


def spread(dev, values, pitch, dtype):
    """`values` [rows, width] in a buffer whose rows are `pitch` elements apart."""
    rows, width = values.shape
    buf = dev.alloc((rows - 1) * pitch + width, dtype, zeroed=False)
    for r in range(rows):
        buf.slice(r * pitch, r * pitch + width).write(values[r])
    return buf


def gather(buf, rows, width, pitch):
    return np.stack([buf.slice(r * pitch, r * pitch + width).read() for r in range(rows)])


def test_rows_of_logits(dev):
    rows, vocab, pitch = 3, 1000, (1 << 31) + 64
    rng = np.random.default_rng(1)
    z = refs.store(3 * rng.normal(size=(rows, vocab)), "bf16")
    labels = dev.buffer(np.array([0, 999, 500], np.int32), "i32")
    old, adv, weights = (dev.buffer(a.astype(np.float32)) for a in (-rng.random(rows), rng.normal(size=rows), rng.random(rows)))
    small = dev.buffer(z.reshape(-1), "bf16")
    totals, logp, grad = dev.policy_loss(small, labels, old, adv, weights, (rows, vocab))
    far = spread(dev, z, pitch, "bf16")
    far_totals, far_logp, far_grad = dev.policy_loss(far, labels, old, adv, weights, (rows, vocab), pitch=pitch, grad_pitch=pitch)
    assert np.array_equal(far_totals.read(), totals.read()) and np.array_equal(far_logp.read(), logp.read())
    assert np.array_equal(gather(far_grad, rows, vocab, pitch), grad.read().reshape(rows, vocab))
    assert np.array_equal(dev.token_logprob(far, labels, (rows, vocab), pitch=pitch).read(),
                          dev.token_logprob(small, labels, (rows, vocab)).read())


# a tile in registers, and one that is streamed (positions * channels beyond what a lone tile holds)
@pytest.mark.parametrize("n, p, c, groups, pitch", [(3, 5, 96, 4, 1 << 29), (1, 4200, 16, 2, 1 << 20)])
def test_group_norm(dev, n, p, c, groups, pitch):
    rng = np.random.default_rng(2)
    x, og = (refs.store(rng.normal(size=(n * p, c)), "bf16") for _ in range(2))
    gamma, beta = dev.buffer(rng.normal(size=c)), dev.buffer(rng.normal(size=c))
    shape = (n, p, c)

    def run(xb, ogb, row):
        out, stats = dev.group_norm(xb, gamma, beta, shape, groups, activation="silu", x_pitch=row, out_pitch=row)
        out = gather(out, n * p, c, row)
        gg, bg = dev.alloc(c), dev.alloc(c)
        # (x_grad in the place of out_grad)
        dev.add_group_norm_grad(xb, stats, gamma, beta, ogb, ogb, gg, bg, shape, groups, activation="silu", overwrite=True,
                                x_pitch=row, out_grad_pitch=row, x_grad_pitch=row)
        return out, stats.read(), gather(ogb, n * p, c, row), gg.read(), bg.read()

    small = run(dev.buffer(x.reshape(-1), "bf16"), dev.buffer(og.reshape(-1), "bf16"), c)
    far = run(spread(dev, x, pitch, "bf16"), spread(dev, og, pitch, "bf16"), pitch)
    for name, a, b in zip(("out", "stats", "x_grad", "gamma_grad", "beta_grad"), small, far):
        assert np.array_equal(a, b), name


def test_checkpoint(dev):
    first, count = (1 << 32) - 1024, 1024 + 333  # blocks on both sides of 2^32 elements
    n = first + count
    rng = np.random.default_rng(3)
    x, og = (refs.store(rng.normal(size=count), "f16") for _ in range(2))
    f, df = (lambda v: v.sin().mul(2.0)), (lambda v: v.cos().mul(2.0))
    small_out, small_saved = dev.apply_fn_checkpoint8(dev.buffer(x, "f16"), f)
    small_grad = dev.alloc(count, "f16")
    dev.add_unary_grad8(small_saved, small_grad, dev.buffer(og, "f16"), df)
    big = dev.alloc(n, "f16", zeroed=False)
    tail = big.slice(first, n)
    tail.write(x)
    out, saved = dev.apply_fn_checkpoint8(big, f)
    assert isinstance(saved, Checkpoint8)
    codes, scales = saved.codes.slice(first, n), saved.scales.slice(first // 128, saved.scales.len)
    assert np.array_equal(codes.read(), small_saved.codes.read()) and np.array_equal(scales.read(), small_saved.scales.read())
    assert np.array_equal(out.slice(first, n).read(), small_out.read())
    assert np.array_equal(dev.restore8(saved).slice(first, n).read(), dev.restore8(small_saved).read())
    tail.write(og)
    grad = dev.alloc(n, "f16")
    dev.add_unary_grad8(saved, grad, big, df)
    assert np.array_equal(grad.slice(first, n).read(), small_grad.read())
    with pytest.raises(custos_amd.CustosHipError, match="2\\^34"):
        dev._check(dev.lib.custos_hip_checkpoint8_restore(dev.handle, dev.compile(custos_amd.capi.KIND_RESTORE8, "f16", "x", ("x",)),
                                                          saved.codes.ptr, saved.scales.ptr, out.ptr, (1 << 34) + 1))
