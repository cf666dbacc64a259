"""What the training operators refuse, checked on the host before a device is needed: a call without a device
handle that passes every check fails for the missing handle, one that does not names what is wrong."""
import numpy as np
import pytest

from custos_amd import capi

F32, F16, BF16, I32 = (capi.DTYPES[k][0] for k in ("f32", "f16", "bf16", "i32"))
BASE = 1 << 32  # addresses that are never touched


def refused(rc, code, text):
    assert rc == code, (rc, capi.last_error(None))
    assert text in capi.last_error(None), capi.last_error(None)


def gn_desc(**over):
    d = dict(dtype=F32, param_dtype=F32, activation=0, flags=0, samples=2, positions=10, channels=8, groups=2, eps=1e-5)
    return capi.GroupNormDesc(**{**d, **over})


def gn(desc=None, x=BASE, x_pitch=8, gamma=BASE + 0x10000, beta=BASE + 0x20000, out=BASE + 0x30000, out_pitch=8, stats=BASE + 0x40000):
    lib = capi.load_library()
    return lib.custos_hip_group_norm(None, desc, x, x_pitch, gamma, beta, out, out_pitch, stats)


def gn_grad(desc=None, x=BASE, x_pitch=8, codes=0, scales=0, stats=BASE + 0x10000, gamma=0, beta=0, out_grad=BASE + 0x20000, og_pitch=8,
            x_grad=BASE + 0x30000, xg_pitch=8, gamma_grad=BASE + 0x40000, beta_grad=BASE + 0x50000):
    lib = capi.load_library()
    return lib.custos_hip_add_group_norm_grad(None, desc, x, x_pitch, codes, scales, stats, gamma, beta, out_grad, og_pitch, x_grad,
                                              xg_pitch, gamma_grad, beta_grad)


INVALID, OVERLAP, LARGE = capi.ERR_INVALID_ARGUMENT, capi.ERR_BAD_OVERLAP, capi.ERR_TOO_LARGE


def test_calls_that_pass_every_check_need_a_device():
    refused(gn(gn_desc()), INVALID, "device handle is null")
    refused(gn(gn_desc(), gamma=0, beta=0), INVALID, "device handle is null")
    refused(gn(gn_desc(samples=0)), INVALID, "device handle is null")
    refused(gn(gn_desc(), out=BASE), INVALID, "device handle is null")  # in place
    refused(gn(gn_desc(), x_pitch=16, out_pitch=16, out=BASE + 32), INVALID, "device handle is null")  # side by side
    refused(gn_grad(gn_desc()), INVALID, "device handle is null")
    refused(gn_grad(gn_desc(flags=1), x_grad=BASE), INVALID, "device handle is null")
    refused(gn_grad(gn_desc(), x=0, codes=BASE, scales=BASE + 0x8000), INVALID, "device handle is null")
    refused(gn_grad(gn_desc(), x_grad=0, gamma_grad=0, beta_grad=0), INVALID, "device handle is null")


@pytest.mark.parametrize("over, text", [
    (dict(dtype=I32), "f32, f16 or bf16"),
    (dict(dtype=F16, param_dtype=BF16), "f32 or of the element type"),
    (dict(activation=9), "unknown activation"),
    (dict(activation=-1), "unknown activation"),
    (dict(flags=2), "unknown flag"),
    (dict(channels=0), "divide into the groups"),
    (dict(groups=0), "divide into the groups"),
    (dict(groups=3), "divide into the groups"),
    (dict(eps=0.0), "eps is positive"),
    (dict(eps=-1.0), "eps is positive"),
    (dict(eps=float("nan")), "eps is positive"),
    (dict(eps=float("inf")), "eps is positive"),
])
def test_group_norm_descriptions(over, text):
    refused(gn(gn_desc(**over)), INVALID, text)
    refused(gn_grad(gn_desc(**over)), INVALID, text)


def test_group_norm_sizes_beyond_any_memory():
    for over in (dict(channels=1 << 40, groups=1), dict(samples=1 << 40), dict(positions=1 << 60), dict(samples=1 << 30, positions=1 << 39)):
        refused(gn(gn_desc(**over)), LARGE, "beyond any memory")
        refused(gn_grad(gn_desc(**over)), LARGE, "beyond any memory")


@pytest.mark.parametrize("over, code, text", [
    (dict(x=0), INVALID, "x is a null address"),
    (dict(out=0), INVALID, "out is a null address"),
    (dict(stats=0), INVALID, "stats is a null address"),
    (dict(x=BASE + 2), INVALID, "x is not aligned"),
    (dict(gamma=BASE + 0x10001), INVALID, "gamma is not aligned"),
    (dict(x_pitch=7), INVALID, "pitch shorter"),
    (dict(out_pitch=0), INVALID, "pitch shorter"),
    (dict(x=2**64 - 64), INVALID, "wraps around"),
    (dict(x_pitch=1 << 60), LARGE, "larger than any memory"),
    (dict(out=BASE + 32), OVERLAP, "out overlaps x"),
    (dict(out=BASE, out_pitch=16), OVERLAP, "out overlaps x"),
    (dict(out=BASE + 0x10000), OVERLAP, "out overlaps gamma"),
    (dict(stats=BASE + 0x30000), OVERLAP, "out overlaps stats"),
    (dict(stats=BASE), OVERLAP, "stats overlaps x"),
    (dict(x_pitch=12, out_pitch=12, out=BASE + 32), OVERLAP, "out overlaps x"),  # slices of 8 in rows of 12
])
def test_group_norm_operands(over, code, text):
    refused(gn(gn_desc(), **over), code, text)


@pytest.mark.parametrize("over, code, text", [
    (dict(codes=BASE, scales=BASE), INVALID, "either as values or as codes"),
    (dict(x=0), INVALID, "either as values or as codes"),
    (dict(x=0, codes=BASE), INVALID, "either as values or as codes"),
    (dict(stats=0), INVALID, "stats is a null address"),
    (dict(out_grad=0), INVALID, "out_grad is a null address"),
    (dict(gamma_grad=BASE + 0x40002), INVALID, "gamma_grad is not aligned"),
    (dict(x_grad=BASE), OVERLAP, "x_grad overlaps x"),  # it is added to: not in place
    (dict(beta_grad=BASE + 0x40000), OVERLAP, "gamma_grad overlaps beta_grad"),
    (dict(og_pitch=1), INVALID, "pitch shorter"),
])
def test_group_norm_gradient_operands(over, code, text):
    refused(gn_grad(gn_desc(), **over), code, text)


@pytest.mark.parametrize("eps", [1e-300, 1e-40, 1e39])
def test_eps_is_a_normal_number_in_f32(eps):
    refused(gn(gn_desc(eps=eps)), INVALID, "eps is positive")
    refused(gn_grad(gn_desc(eps=eps)), INVALID, "eps is positive")


def test_only_values_may_take_the_place_of_values():
    """What one workgroup writes and another reads is no place for a result, however well the sizes fit."""
    wide = dict(flags=1, channels=8, groups=2)
    for over in (dict(gamma_grad=BASE + 0x60000), dict(beta_grad=BASE + 0x60000)):
        refused(gn_grad(gn_desc(**wide), gamma=BASE + 0x60000, **over), OVERLAP, "overlaps gamma")
    refused(gn_grad(gn_desc(**wide), beta=BASE + 0x60000, beta_grad=BASE + 0x60000), OVERLAP, "overlaps beta")
    refused(gn_grad(gn_desc(**wide), gamma_grad=BASE + 0x10000), OVERLAP, "overlaps stats")
    # one row: x, gamma and the statistics of four groups of two channels have as many bytes
    row = dict(samples=1, positions=1, channels=8, groups=4)
    refused(gn(gn_desc(**row), stats=BASE), OVERLAP, "overlaps x")
    refused(gn(gn_desc(**row), stats=BASE + 0x10000), OVERLAP, "overlaps gamma")
    refused(gn(gn_desc(**row), out=BASE + 0x10000), OVERLAP, "overlaps gamma")
    refused(gn_grad(gn_desc(**row, flags=1), gamma=BASE + 0x30000), OVERLAP, "overlaps gamma")
    refused(gn(gn_desc(**row), out=BASE), INVALID, "device handle is null")


def test_launches_have_fewer_than_2_to_32_threads():
    # (each in less than 2^32 bytes an operand or two)
    refused(gn(gn_desc(samples=1 << 24, positions=1), out=1 << 40, stats=1 << 42), LARGE, "2^32 threads")
    refused(gn_grad(gn_desc(samples=1 << 24, positions=1), x=1 << 46, stats=1 << 44, out_grad=1 << 42, x_grad=1 << 40, gamma_grad=1 << 30, beta_grad=1 << 31), INVALID, "device handle is null")
    refused(logprob(rows=1 << 26, logits=1 << 40, labels=1 << 41, logp=1 << 42), LARGE, "2^32 threads")
    refused(policy(dict(rows=1 << 26), logits=1 << 40, labels=1 << 41, old_logp=1 << 42, advantages=1 << 43, weights=1 << 44,
                   logits_grad=1 << 45, logp=1 << 46, totals=1 << 47), LARGE, "2^32 threads")
    refused(logprob(rows=(1 << 26) - 1, logits=1 << 40, labels=1 << 41, logp=1 << 42), INVALID, "device handle is null")


def test_forward_takes_no_flags():
    refused(gn(gn_desc(flags=1)), INVALID, "no flags")
    refused(gn(None), INVALID, "description is null")


def test_group_norm_formula_against_differences():
    """The gradient formula the kernels are tested with, against differences of the forward formula."""
    import operator_refs as refs
    rng = np.random.default_rng(0)
    n, p, c, groups = 2, 3, 6, 2
    x, og = rng.normal(size=(n, p, c)), rng.normal(size=(n, p, c))
    gamma, beta = rng.normal(size=c), rng.normal(size=c)
    for activation in ("none", "relu", "silu", "gelu"):
        _, mean, rstd, z = refs.group_norm(x, gamma, beta, groups, activation, 1e-3)
        assert np.abs(z).min() > 1e-4  # (no difference steps over relu's corner)
        (xg, gg, bg), _ = refs.group_norm_grad(x, mean, rstd, gamma, beta, og, groups, activation)

        def loss(x_, g_, b_):
            return float((refs.group_norm(x_, g_, b_, groups, activation, 1e-3)[0] * og).sum())

        step = 1e-5
        for which, grad in ((0, xg), (1, gg), (2, bg)):
            args = [x, gamma, beta]
            for at in np.ndindex(args[which].shape):
                moved = []
                for sign in (1, -1):
                    a = [v.copy() for v in args]
                    a[which][at] += sign * step
                    moved.append(loss(*a))
                # (error of a central difference: step^2 times a third derivative, and roundings over the step)
                assert abs((moved[0] - moved[1]) / (2 * step) - grad[at]) < 1e-6, (activation, which, at)


# ---- 8-bit checkpoints ----

@pytest.mark.parametrize("kind", [capi.KIND_SAVE8, capi.KIND_RESTORE8, capi.KIND_UNARY_GRAD8])
def test_checkpoint_kernels_compile_for_the_float_types_and_one_marker(kind):
    for dtype in ("f32", "f16", "bf16", "f16_pernode", "bf16_pernode"):
        assert capi.expr_build_code_object(kind, dtype, "pow((x * 2.0), (x + 1.0))", ["x"]) > 1000
    for dtype in ("f64", "i32", "u8"):
        with pytest.raises(capi.CustosHipError) as e:
            capi.expr_emit(kind, dtype, "x", ["x"])
        assert e.value.code == capi.ERR_EXPR_UNSUPPORTED
    with pytest.raises(capi.CustosHipError) as e:
        capi.expr_emit(kind, "f32", "(x + y)", ["x", "y"])
    assert e.value.code == capi.ERR_ARITY_MISMATCH


def test_unknown_kinds_are_refused():
    for kind in (2, 3, 7, -1):
        with pytest.raises(capi.CustosHipError, match="unknown kernel kind"):
            capi.expr_emit(kind, "f32", "x", ["x"])


def test_checkpoint_entry_points_refuse_a_missing_kernel():
    lib = capi.load_library()
    refused(lib.custos_hip_checkpoint8_save(None, None, BASE, 0, BASE, BASE, 8), INVALID, "null kernel")
    refused(lib.custos_hip_checkpoint8_restore(None, None, BASE, BASE, BASE, 8), INVALID, "null kernel")
    refused(lib.custos_hip_add_unary_grad8(None, None, BASE, BASE, BASE, BASE, 8, 0), INVALID, "null kernel")


def test_checkpoint_formula():
    """Half a scale at most, zeros and the largest magnitude exactly at the ends of the code range."""
    import operator_refs as refs
    rng = np.random.default_rng(1)
    x = rng.normal(size=1000).astype(np.float32)
    codes, scales = refs.checkpoint8(x)
    assert codes.min() >= -127 and np.abs(codes).max() == 127
    assert np.all(np.abs(refs.restore8(codes, scales) - x) <= np.repeat(scales, 128)[:1000] * np.float32(0.50001))


# ---- log-probabilities and the policy loss ----

def logprob(dtype=F32, logits=BASE, pitch=10, labels=BASE + 0x10000, rows=4, vocab=10, temperature=1.0, logp=BASE + 0x20000, lse=0):
    return capi.load_library().custos_hip_token_logprob(None, dtype, logits, pitch, labels, rows, vocab, temperature, logp, lse)


def policy(over=None, **args):
    d = dict(dtype=F32, reserved=0, rows=4, vocab=10, pitch=10, grad_pitch=10, temperature=1.0, clip_low=0.2, clip_high=0.2, kl_coef=0.0, grad_scale=1.0)
    a = dict(logits=BASE, labels=BASE + 0x10000, old_logp=BASE + 0x20000, ref_logp=0, advantages=BASE + 0x30000, weights=BASE + 0x40000,
             logits_grad=BASE + 0x50000, logp=BASE + 0x60000, totals=BASE + 0x70000)
    a.update(args)
    return capi.load_library().custos_hip_policy_loss(None, capi.PolicyDesc(**{**d, **(over or {})}), *a.values())


def test_policy_calls_that_pass_every_check_need_a_device():
    for rc in (logprob(), logprob(lse=BASE + 0x30000), logprob(rows=0), policy(), policy(dict(rows=0)), policy(logits_grad=BASE),
               policy(dict(kl_coef=0.1), ref_logp=BASE + 0x80000), policy(logits_grad=0, logp=0, totals=0),
               policy(dict(pitch=20, grad_pitch=20), logits_grad=BASE + 40)):
        assert rc == INVALID and "device handle is null" in capi.last_error(None)
        refused(rc, INVALID, "device handle is null")


@pytest.mark.parametrize("over, code, text", [
    (dict(dtype=I32), INVALID, "f32, f16 or bf16"),
    (dict(vocab=0), INVALID, "vocabulary is empty"),
    (dict(temperature=0.0), INVALID, "temperature is positive"),
    (dict(temperature=-1.0), INVALID, "temperature is positive"),
    (dict(temperature=float("nan")), INVALID, "temperature is positive"),
    (dict(temperature=float("inf")), INVALID, "temperature is positive"),
    (dict(temperature=1e-320), INVALID, "temperature is positive"),
    (dict(temperature=1e300), INVALID, "temperature is positive"),
    (dict(rows=1 << 31), LARGE, "2^31 rows"),
    (dict(vocab=1 << 30, pitch=1 << 30), LARGE, "2^30 tokens"),
    (dict(pitch=9), INVALID, "pitch shorter"),
])
def test_rows_of_logits(over, code, text):
    refused(logprob(**over), code, text)
    refused(policy(over), code, text)


@pytest.mark.parametrize("over, args, code, text", [
    (dict(reserved=1), {}, INVALID, "reserved"),
    (dict(clip_low=-0.1), {}, INVALID, "clip_low"),
    (dict(clip_low=1.5), {}, INVALID, "clip_low"),
    (dict(clip_high=-0.1), {}, INVALID, "clip_high"),
    (dict(clip_high=float("nan")), {}, INVALID, "clip_high"),
    (dict(kl_coef=float("inf")), {}, INVALID, "finite"),
    (dict(grad_scale=float("nan")), {}, INVALID, "finite"),
    (dict(kl_coef=0.1), {}, INVALID, "needs ref_logp"),
    (dict(grad_pitch=3), {}, INVALID, "pitch shorter"),
    ({}, dict(logits=0), INVALID, "logits is a null"),
    ({}, dict(labels=0), INVALID, "labels is a null"),
    ({}, dict(old_logp=0), INVALID, "old_logp is a null"),
    ({}, dict(advantages=0), INVALID, "advantages is a null"),
    ({}, dict(weights=0), INVALID, "weights is a null"),
    ({}, dict(labels=BASE + 2), INVALID, "labels is not aligned"),
    ({}, dict(logits_grad=BASE + 4), OVERLAP, "overlaps logits"),
    ({}, dict(logp=BASE), OVERLAP, "logp overlaps logits"),
    ({}, dict(logp=BASE + 0x20000), OVERLAP, "overlaps"),
    ({}, dict(totals=BASE + 0x60000), OVERLAP, "overlaps"),
    ({}, dict(totals=BASE + 0x40000), OVERLAP, "overlaps"),
    (dict(vocab=1, pitch=1, grad_pitch=1, rows=1), dict(logits_grad=BASE + 0x20000), OVERLAP, "overlaps old_logp"),
    (dict(vocab=1, pitch=1, grad_pitch=1, rows=1), dict(logp=BASE), OVERLAP, "overlaps logits"),
])
def test_policy_refusals(over, args, code, text):
    refused(policy(over, **args), code, text)


def test_policy_formula_against_differences():
    import operator_refs as refs
    rng = np.random.default_rng(2)
    z, labels = rng.normal(size=(8, 6)), rng.integers(0, 6, 8)
    logp = refs.token_logprob(z, labels, 0.8)[0]
    old, ref = logp - np.log(rng.choice([0.6, 0.9, 1.1, 1.6], 8)), logp + 0.3 * rng.normal(size=8)
    adv, w = rng.normal(size=8), rng.random(8)
    args = (labels, old, ref, adv, w, 0.8, (0.2, 0.3), 0.2)
    grad = refs.policy_loss(z, *args)[2]
    for at in np.ndindex(z.shape):
        up, down = z.copy(), z.copy()
        up[at] += 1e-5
        down[at] -= 1e-5
        assert abs((refs.policy_loss(up, *args)[0][0] - refs.policy_loss(down, *args)[0][0]) / 2e-5 - grad[at]) < 1e-7, at
