"""Group norm where the number of groups has no small divisor (no tile of a few groups is wide enough, and all of them
together are too wide), and its gradients from a checkpoint in every type."""
import numpy as np
import pytest

import operator_refs as refs
from custos_amd import Checkpoint8
from test_gpu_group_norm import SIZES, Case, check_forward, check_gradients, forward, gradients

pytestmark = pytest.mark.gpu

PRIMES = [  # n, p, c, groups, pad, dtype; the last two move more than 64 MiB
    (1, 700, 1025, 41, 0, "f32"), (2, 600, 1032, 43, 3, "f32"), (1, 4096, 1643, 53, 0, "f32"), (1, 900, 1147, 37, 0, "f32"),
    (1, 1000, 2050, 41, 0, "bf16"), (1, 600, 2072, 37, 5, "bf16"), (1, 700, 2120, 53, 0, "f16"), (2, 900, 4066, 38, 0, "f16"),
    (1, 9000, 2159, 17, 0, "bf16"), (1, 9500, 1064, 19, 0, "f32"),
]
KEPT = [s for s in PRIMES if s[4] == 0]


def from_checkpoint(hip, case):
    """Gradients, and the values x stands for."""
    codes, scales = refs.checkpoint8(case.x.astype(np.float32))
    saved = Checkpoint8(hip, hip.buffer(codes, "i8"), hip.buffer(scales), case.dtype)
    return gradients(hip, case, saved=saved), refs.restore8(codes, scales).astype(np.float64).reshape(case.shape)


@pytest.mark.parametrize("n, p, c, groups, pad, dtype", PRIMES)
def test_forward_in_prime_groups(hip, n, p, c, groups, pad, dtype):
    case = Case(n, p, c, groups, dtype, pad=pad, seed=p + c)
    check_forward(case, *forward(hip, case))


@pytest.mark.parametrize("n, p, c, groups, pad, dtype", PRIMES)
def test_gradients_in_prime_groups(hip, n, p, c, groups, pad, dtype):
    case = Case(n, p, c, groups, dtype, pad=pad, seed=p + c)
    check_gradients(case, gradients(hip, case))


@pytest.mark.parametrize("n, p, c, groups, pad, dtype", KEPT)
def test_gradients_in_prime_groups_from_a_checkpoint(hip, n, p, c, groups, pad, dtype):
    case = Case(n, p, c, groups, dtype, seed=p + c)
    got, x = from_checkpoint(hip, case)
    check_gradients(case, got, x=x)


@pytest.mark.parametrize("n, p, c, groups, pad, dtype", KEPT[:5])
def test_gradients_in_prime_groups_are_added(hip, n, p, c, groups, pad, dtype):
    case = Case(n, p, c, groups, dtype, activation="gelu", seed=p + c)
    rng = np.random.default_rng(5)
    start = [refs.load(refs.store(rng.normal(size=case.shape), dtype), dtype)] + [rng.normal(size=c).astype(np.float32) for _ in range(2)]
    check_gradients(case, gradients(hip, case, overwrite=False, start=start), start=start)


@pytest.mark.parametrize("n, p, c, groups, pad, dtype", [KEPT[0], KEPT[3]])
def test_prime_groups_in_place(hip, n, p, c, groups, pad, dtype):
    case = Case(n, p, c, groups, dtype, seed=p + c)
    want = forward(hip, case)[0].read()
    x = hip.buffer(case.x_stored.reshape(-1), dtype)
    forward(hip, case, x=x, out=x)
    assert np.array_equal(x.read(), want)


@pytest.mark.parametrize("n, p, c, groups, pad", [s for s in SIZES if s[4] == 0])
def test_gradients_from_an_f16_checkpoint(hip, n, p, c, groups, pad):
    case = Case(n, p, c, groups, "f16", seed=p + c)
    got, x = from_checkpoint(hip, case)
    check_gradients(case, got, x=x)
