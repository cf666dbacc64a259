"""8-bit checkpoints: the codes bit for bit, and what is computed from them."""
import numpy as np
import pytest

import operator_refs as refs
from custos_amd import Checkpoint8, capi

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f16", "bf16"]


def values(n, dtype, seed=0, spread=1.0):
    rng = np.random.default_rng(seed)
    return refs.store(rng.normal(size=n) * spread * np.where(rng.random(n) < 0.01, 30, 1), dtype)


def f32(stored, dtype):
    return refs.load(stored, dtype).astype(np.float32)


def same_checkpoint(saved, codes, scales):
    assert np.array_equal(saved.codes.read(), codes)
    assert np.array_equal(saved.scales.read().view(np.uint32), scales.view(np.uint32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 2, 7, 8, 127, 128, 129, 255, 1023, 4096, 5000, 65539, 300001])
def test_codes_and_scales_bit_for_bit(hip, n, dtype):
    x = values(n, dtype, seed=n)
    saved = hip.checkpoint8(hip.buffer(x, dtype))
    codes, scales = refs.checkpoint8(f32(x, dtype))
    same_checkpoint(saved, codes, scales)
    back = refs.load(hip.restore8(saved).read(), dtype)
    assert np.array_equal(back, refs.load(refs.store(refs.restore8(codes, scales), dtype), dtype))
    # half a scale, the storage type's rounding of the value given back, and the scale's own two roundings
    half = np.repeat(scales, 128)[:n].astype(np.float64) / 2
    refs.assert_close(back, refs.load(x, dtype), half * 1.0001 + refs.U[dtype] * 1.01 * (np.abs(back) + half) + 1e-6 * half * 254, "restored")


@pytest.mark.parametrize("dtype", TYPES)
def test_what_is_not_finite_and_what_is_tiny(hip, dtype):
    n = 128 * 9 + 5
    x = f32(values(n, dtype), dtype)
    x[3], x[130], x[131] = np.nan, np.inf, -np.inf      # among other values
    x[256:384] = np.nan                                 # nothing finite in the block
    x[384:512] = 0.0
    x[512:640] *= np.float32(2.0**-110)                 # below what is kept (f16: zeros already)
    x[640:768] = 0.0
    x[700] = 2.0**-14                                   # one value, kept exactly
    x[768:896] = -0.0
    x[896:1024] = np.inf
    top = {"f32": 3.4028235e38, "f16": 65504.0, "bf16": 3.3895314e38}[dtype]
    x[1024:1152:2], x[1025:1152:2] = top, -top          # the largest values of the type
    stored = refs.store(x, dtype)
    x = f32(stored, dtype)
    saved = hip.checkpoint8(hip.buffer(stored, dtype))
    codes, scales = refs.checkpoint8(x)
    same_checkpoint(saved, codes, scales)
    back = refs.load(hip.restore8(saved).read(), dtype)
    assert np.array_equal(np.isnan(back), ~np.isfinite(x))
    assert np.all(back[384:640] == 0) and back[700] == 2.0**-14
    # a NaN gradient where the input was not finite, whatever the slope
    grad = hip.buffer(refs.store(np.zeros(n), dtype), dtype)
    hip.add_unary_grad8(saved, grad, hip.buffer(refs.store(np.ones(n), dtype), dtype), lambda v: v.mul(2.0), overwrite=True)
    assert np.array_equal(np.isnan(refs.load(grad.read(), dtype)), ~np.isfinite(x) | np.isnan(back * 2))


@pytest.mark.parametrize("dtype", TYPES + ["f16_pernode", "bf16_pernode"])
@pytest.mark.parametrize("n", [1, 130, 70001])
def test_forward_equals_apply_fn_and_saves_the_input(hip, n, dtype):
    storage = dtype.split("_")[0]
    x = values(n, storage, seed=3)
    f = lambda v: v.mul(0.5).tanh().add(v.max(0.25))
    buf = hip.buffer(x, dtype)
    out, saved = hip.apply_fn_checkpoint8(buf, f)
    assert np.array_equal(out.read().view(np.uint8), hip.apply_fn(buf, f).read().view(np.uint8))
    same_checkpoint(saved, *refs.checkpoint8(f32(x, storage)))
    # in place
    again = hip.alloc_checkpoint8(n, dtype)
    hip.apply_fn_checkpoint8(buf, f, out=buf, into=again)
    assert np.array_equal(buf.read().view(np.uint8), out.read().view(np.uint8))
    assert np.array_equal(again.codes.read(), saved.codes.read())


@pytest.mark.parametrize("dtype", TYPES + ["bf16_pernode"])
@pytest.mark.parametrize("n", [1, 131, 70001])
def test_gradient_equals_the_gradient_of_the_restored_input(hip, n, dtype):
    """Exact arithmetic in f' (products and sums of f32 values): the same bits as add_unary_grad over a buffer
    that holds the restored values, in the types where such a buffer holds them exactly."""
    storage = dtype.split("_")[0]
    x, og, g0 = values(n, storage, 4), values(n, storage, 5), values(n, storage, 6)
    saved = hip.checkpoint8(hip.buffer(x, dtype))
    f = lambda v: v.mul(3.0).add(1.0)
    g = hip.buffer(g0, dtype)
    hip.add_unary_grad8(saved, g, hip.buffer(og, dtype), f)
    if dtype in ("f32", "bf16_pernode"):
        want = hip.buffer(g0, dtype)
        hip.add_unary_grad(hip.restore8(saved), want, hip.buffer(og, dtype), f)
        assert np.array_equal(g.read().view(np.uint8), want.read().view(np.uint8))
    v = refs.restore8(saved.codes.read(), saved.scales.read())
    d = v * np.float32(3) + np.float32(1)
    want = refs.load(refs.store(f32(g0, storage) + f32(og, storage) * d, storage), storage)
    if dtype in TYPES:
        assert np.array_equal(refs.load(g.read(), storage), want)
        hip.add_unary_grad8(saved, g, hip.buffer(og, dtype), f, overwrite=True)
        assert np.array_equal(refs.load(g.read(), storage), refs.load(refs.store(f32(og, storage) * d, storage), storage))


@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_of_tanh(hip, dtype):
    n = 20000
    x, og = values(n, dtype, 7), values(n, dtype, 8)
    out, saved = hip.apply_fn_checkpoint8(hip.buffer(x, dtype), lambda v: v.tanh())
    g = hip.alloc(n, dtype)
    hip.add_unary_grad8(saved, g, hip.buffer(og, dtype), lambda v: v.tanh().mul(v.tanh()).neg().add(1.0), overwrite=True)
    v = refs.restore8(saved.codes.read(), saved.scales.read()).astype(np.float64)
    og64 = refs.load(og, dtype)
    want = og64 * (1 - np.tanh(v) ** 2)
    # tanh to a few steps of f32, then the cancelling difference from one
    refs.assert_close(refs.load(g.read(), dtype), want, refs.U[dtype] * np.abs(want) * 1.01 + 16 * 2.0**-24 * np.abs(og64) + refs.TINY[dtype], "tanh")
    # and against differences of the forward operation, at the restored input
    h = 1e-3
    slope = (np.tanh(v + h) - np.tanh(v - h)) / (2 * h)  # off by h^2 / 6 times a third derivative of at most 2
    refs.assert_close(refs.load(g.read(), dtype), og64 * slope, np.abs(og64) * (h * h + 2 * refs.U[dtype]) + refs.TINY[dtype], "differences")


@pytest.mark.parametrize("dtype", TYPES)
def test_slices_at_any_alignment(hip, dtype):
    """Operands that start in the middle of a buffer; what lies around them stays."""
    n, pad = 1000, 64
    x, og = values(n + pad, dtype, 9), values(n + pad, dtype, 10)
    bx, bog = hip.buffer(x, dtype), hip.buffer(og, dtype)
    for start in (1, 3, 8):
        codes = hip.buffer(np.full(n + pad, 77, np.int8), "i8")
        scales = hip.buffer(np.full(20, 5.0))
        out = hip.buffer(refs.store(np.full(n + pad, 9.0), dtype), dtype)
        saved = Checkpoint8(hip, codes.slice(start, start + n), scales.slice(2, 10), dtype)
        hip.apply_fn_checkpoint8(bx.slice(start, start + n), lambda v: v.mul(2.0), out=out.slice(start, start + n), into=saved)
        c, s = refs.checkpoint8(f32(x, dtype)[start:start + n])
        got, got_s = codes.read(), scales.read()
        assert np.array_equal(got[start:start + n], c) and np.all(got[:start] == 77) and np.all(got[start + n:] == 77)
        assert np.array_equal(got_s[2:10], s) and np.all(got_s[:2] == 5) and np.all(got_s[10:] == 5)
        o = refs.load(out.read(), dtype)
        assert np.array_equal(o[start:start + n], 2 * refs.load(x, dtype)[start:start + n])
        assert np.all(o[:start] == 9) and np.all(o[start + n:] == 9)
        hip.add_unary_grad8(saved, out.slice(start, start + n), bog.slice(start, start + n), lambda v: v, overwrite=True)
        o = refs.load(out.read(), dtype)
        want = refs.load(refs.store(f32(og, dtype)[start:start + n] * refs.restore8(c, s), dtype), dtype)
        assert np.array_equal(o[start:start + n], want) and np.all(o[:start] == 9) and np.all(o[start + n:] == 9)


def test_literals_that_change_share_one_kernel(hip):
    n = 300
    x = values(n, "f32")
    saved = hip.checkpoint8(hip.buffer(x))
    v = refs.restore8(saved.codes.read(), saved.scales.read())
    before = hip.cache_stats()[0]
    for k in range(6):
        lr = 0.125 * (k + 1)
        out = hip.restore8(saved, lambda t: t.mul(lr).add(1.0))
        assert np.array_equal(out.read(), v * np.float32(lr) + np.float32(1))
    assert hip.cache_stats()[0] - before <= 2


def test_refusals(hip):
    n = 256
    x, other = hip.buffer(np.ones(n)), hip.buffer(np.ones(n))
    saved = hip.checkpoint8(x)
    lib = hip.lib

    def rc(fn, *args):
        code = fn(hip.handle, *args)
        return code, capi.last_error(hip.handle)

    save = hip.compile(capi.KIND_SAVE8, "f32", "x")
    restore = hip.compile(capi.KIND_RESTORE8, "f32", "x")
    grad = hip.compile(capi.KIND_UNARY_GRAD8, "f32", "x")
    apply = hip.compile(capi.KIND_APPLY, "f32", "x")
    c, s = saved.codes.ptr, saved.scales.ptr
    assert rc(lib.custos_hip_checkpoint8_save, apply, x.ptr, 0, c, s, n)[0] == capi.ERR_KIND_MISMATCH
    assert rc(lib.custos_hip_checkpoint8_restore, save, c, s, other.ptr, n)[0] == capi.ERR_KIND_MISMATCH
    assert rc(lib.custos_hip_add_unary_grad8, restore, c, s, x.ptr, other.ptr, n, 0)[0] == capi.ERR_KIND_MISMATCH
    assert rc(lib.custos_hip_apply_fn, save, x.ptr, other.ptr, n)[0] == capi.ERR_KIND_MISMATCH
    assert rc(lib.custos_hip_add_unary_grad, grad, x.ptr, other.ptr, other.ptr, n)[0] == capi.ERR_KIND_MISMATCH
    assert rc(lib.custos_hip_kernel_prepare_merged, save)[0] == capi.ERR_KIND_MISMATCH
    assert rc(lib.custos_hip_checkpoint8_save, save, x.ptr, 0, c, s, (1 << 40) + 1)[0] == capi.ERR_TOO_LARGE
    assert rc(lib.custos_hip_checkpoint8_save, save, x.ptr, 0, 0, s, n) == (capi.ERR_INVALID_ARGUMENT, "checkpoint save: codes is a null address")
    assert rc(lib.custos_hip_checkpoint8_save, save, x.ptr + 2, 0, c, s, n)[0] == capi.ERR_INVALID_ARGUMENT
    assert rc(lib.custos_hip_checkpoint8_save, save, x.ptr, 0, x.ptr, s, n)[0] == capi.ERR_BAD_OVERLAP
    assert rc(lib.custos_hip_checkpoint8_save, save, x.ptr, x.ptr + 4, c, s, n - 1)[0] == capi.ERR_BAD_OVERLAP
    assert rc(lib.custos_hip_checkpoint8_restore, restore, c, s, c, n // 4)[0] == capi.ERR_BAD_OVERLAP
    assert rc(lib.custos_hip_add_unary_grad8, grad, c, s, other.ptr, other.ptr, n, 0)[0] == capi.ERR_BAD_OVERLAP
    assert rc(lib.custos_hip_add_unary_grad8, grad, c, s, other.ptr, x.ptr, n, 6)[0] == capi.ERR_INVALID_ARGUMENT
    assert rc(lib.custos_hip_checkpoint8_save, save, 0, 0, 0, 0, 0)[0] == 0  # nothing to do
    with pytest.raises(ValueError, match="checkpoint is for 256 x f32"):
        hip.checkpoint8(hip.buffer(np.ones(100)), into=saved)
    with pytest.raises(ValueError, match="differ in length"):
        hip.add_unary_grad8(saved, hip.alloc(100), x, lambda v: v)
    with pytest.raises(ValueError, match="scales is"):
        Checkpoint8(hip, saved.codes, hip.alloc(1), "f32")
    with pytest.raises(capi.CustosHipError, match="f32, f16 and bf16"):
        hip.checkpoint8(hip.buffer(np.ones(4), "f64"))
