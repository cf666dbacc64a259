"""The training operators around the element-wise path: what is measured, and their plain forms.

A block of a training step is a normalisation with its activation (`group_norm`, channels last), element-wise
operations whose inputs are kept for the backward pass in 8 bits (`apply_fn_checkpoint8`, `add_unary_grad8`,
`restore8`), and at the end the loss that sends the first gradient back (`token_logprob`, `policy_loss`).

`listed()` and `draw()` give cases, `prepare()` the data a program has in hand, `run()` one pass over it -- with
`own` false in elementary torch operations, with `own` true through the framework --, `work()` the bytes and
operations the pass cannot do without, `exact()` its results in 64 bits.
"""
import math

import torch

own = False

BLOCK = 128       # elements that share a scale in an 8-bit checkpoint
TINY = 2.0**-100  # a block whose largest magnitude is below this is kept as zeros
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases ----

def listed():
    return [
        # the norm of the last, smallest map of one sample: a call whose latency counts
        {"name": "norm_small_map", "op": "norm", "n": 1, "positions": 64, "channels": 256, "groups": 32, "pad": 0,
         "dtype": "bf16", "params": "f32", "act": "silu"},
        # the middle maps of a batch
        {"name": "norm_batch", "op": "norm", "n": 8, "positions": 1024, "channels": 640, "groups": 32, "pad": 0,
         "dtype": "bf16", "params": "bf16", "act": "silu"},
        # a map with odd sides and channels that no vector length divides, inside a wider tensor
        {"name": "norm_odd_f32", "op": "norm", "n": 3, "positions": 37 * 53, "channels": 330, "groups": 11, "pad": 7,
         "dtype": "f32", "params": "f32", "act": "gelu"},
        # the full-resolution maps of a large batch: more than the caches hold
        {"name": "norm_large", "op": "norm", "n": 16, "positions": 16384, "channels": 512, "groups": 32, "pad": 0,
         "dtype": "f16", "params": "f32", "act": "silu"},
        # backward of the middle maps
        {"name": "norm_grad_batch", "op": "norm_grad", "n": 4, "positions": 4096, "channels": 320, "groups": 32, "pad": 0,
         "dtype": "bf16", "params": "f32", "act": "silu", "saved": False},
        # backward of large maps whose input was kept in 8 bits
        {"name": "norm_grad_saved_large", "op": "norm_grad", "n": 8, "positions": 16384, "channels": 512, "groups": 32,
         "pad": 0, "dtype": "bf16", "params": "f32", "act": "relu", "saved": True},
        # forward and backward of one unary operation on a small activation of odd length
        {"name": "saved_unary_small", "op": "saved_unary", "len": 65539, "dtype": "f16", "fn": "expmix"},
        # forward and backward of tanh over 2^26 elements, the repository's own unary workload
        {"name": "saved_unary_tanh", "op": "saved_unary", "len": 1 << 26, "dtype": "f32", "fn": "tanh"},
        # an activation put away in 8 bits and taken out again to be computed with
        {"name": "saved_restore_bf16", "op": "saved_restore", "len": 100_000_007, "dtype": "bf16"},
        # log-probabilities of a few tokens, as a sampler or the frozen policy computes them
        {"name": "logprob_few_rows", "op": "logprob", "rows": 8, "vocab": 32768, "pad": 0, "dtype": "f32",
         "temperature": 0.7, "masked": False},
        # the loss over a batch of short answers, odd vocabulary: no two rows start at the same alignment
        {"name": "policy_odd_vocab", "op": "policy", "rows": 1999, "vocab": 50021, "pad": 0, "dtype": "bf16",
         "temperature": 1.0, "ref": True, "masked": True},
        # a large vocabulary and a long batch
        {"name": "policy_large", "op": "policy", "rows": 4096, "vocab": 131072, "pad": 0, "dtype": "bf16",
         "temperature": 1.0, "ref": True, "masked": False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_grad", "norm_grad", "saved_unary", "saved_restore", "logprob", "policy"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op in ("norm", "norm_grad"):
        per_group, groups = _log(rng, 1, 40), rng.choice([1, 2, 5, 8, 11, 16, 32])
        channels = per_group * groups
        positions = max(_log(rng, 1, 20000), -(-16 // per_group))  # (fewer than 16 values have no spread to speak of)
        n = max(1, min(_log(rng, 1, 16), (1 << 26) // (positions * channels)))
        case = {"op": op, "n": n, "positions": positions, "channels": channels, "groups": groups,
                "pad": rng.choice([0, 0, 0, 1, 8, 64]), "dtype": dtype, "params": rng.choice(["f32", dtype]),
                "act": rng.choice(["none", "relu", "silu", "gelu"])}
        if op == "norm_grad":
            case["saved"] = rng.random() < 0.4
            if case["saved"]:
                case["pad"] = 0
        return case
    if op == "saved_unary":
        return {"op": op, "len": _log(rng, 1, 1 << 26), "dtype": dtype, "fn": rng.choice(["tanh", "expmix"])}
    if op == "saved_restore":
        return {"op": op, "len": _log(rng, 1, 100_000_000), "dtype": dtype}
    vocab = _log(rng, 2, 200_000)
    rows = max(1, min(_log(rng, 1, 8192), (1 << 28) // vocab))
    case = {"op": op, "rows": rows, "vocab": vocab, "pad": rng.choice([0, 0, 1, 8, 37]), "dtype": dtype,
            "temperature": rng.choice([1.0, 1.0, 0.7, 1.3]), "masked": rng.random() < 0.3}
    if op == "policy":
        case["ref"] = rng.random() < 0.7
    return case


# ---- data ----

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}
    globals()["_prepare_" + case["op"]](case, g, s)
    if own:  # a program that uses the framework holds its data as the framework's buffers
        import custos_amd

        global _device
        if _device is None:
            _device = custos_amd.HIP(0)
        s["dev"] = _device
        s["b"] = {k: _as_buffer(custos_amd, v) for k, v in s.items() if isinstance(v, torch.Tensor)}
        if "codes" in s:
            kept = case["dtype"]
            s["b"]["saved"] = custos_amd.Checkpoint8(_device, s["b"]["codes"], s["b"]["scales"], kept)
    return s


_device = None
_NAMES = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16", torch.int32: "i32", torch.int8: "i8"}


def _as_buffer(custos_amd, t):
    return custos_amd.Buffer(_device, t.data_ptr(), t.numel(), _NAMES[t.dtype], owned=False)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _maps(case, g):
    """Activations of a convolution: a mean and a spread of its own for every channel."""
    n, p, c, w = case["n"], case["positions"], case["channels"], case["channels"] + case["pad"]
    x = _randn(g, n, p, w)
    return x.mul_(0.5 + torch.rand(w, generator=g, device="cuda")).add_(_randn(g, w)).to(TYPES[case["dtype"]])


def _prepare_norm(case, g, s):
    c, kind = case["channels"], TYPES[case["params"]]
    s["x"] = _maps(case, g)
    s["gamma"] = (1 + 0.2 * _randn(g, c)).to(kind)
    s["beta"] = (0.2 * _randn(g, c)).to(kind)
    if own:
        s["out"] = torch.empty_like(s["x"])
        s["stats"] = torch.empty(case["n"], case["groups"], 2, device="cuda")


def _prepare_norm_grad(case, g, s):
    n, c = case["n"], case["channels"]
    _prepare_norm(case, g, s)
    s["stats"] = _stats(s["x"][:, :, :c], case["groups"], torch.float64).float()
    s["out_grad"] = _randn(g, *s["x"].shape).to(TYPES[case["dtype"]])
    if case["saved"]:
        s["codes"], s["scales"] = _save(s["x"].reshape(-1))
    if own:
        s["x_grad"] = s.pop("out")
        s["gamma_grad"], s["beta_grad"] = (torch.empty(c, device="cuda") for _ in range(2))
    if case["saved"]:
        del s["x"]


def _prepare_saved_unary(case, g, s):
    kind = TYPES[case["dtype"]]
    s["x"] = _randn(g, case["len"]).to(kind)
    s["out_grad"] = (2 * torch.rand(case["len"], generator=g, device="cuda") - 1).to(kind)
    if own:
        _room(case, s)
        s["out"], s["x_grad"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])


def _prepare_saved_restore(case, g, s):
    kind = TYPES[case["dtype"]]
    x = _randn(g, case["len"])
    # a few activations are far larger than the rest, as they are in trained networks
    s["x"] = torch.where(torch.rand(case["len"], generator=g, device="cuda") < 1e-3, x * 30, x).to(kind)
    if own:
        _room(case, s)
        s["out"] = torch.empty_like(s["x"])


def _room(case, s):
    s["codes"] = torch.empty(case["len"], dtype=torch.int8, device="cuda")
    s["scales"] = torch.empty(-(-case["len"] // BLOCK), device="cuda")


def _prepare_logprob(case, g, s):
    r, v, w = case["rows"], case["vocab"], case["vocab"] + case["pad"]
    s["logits"] = (2.5 * _randn(g, r, w)).to(TYPES[case["dtype"]])
    s["labels"] = torch.randint(0, v, (r,), generator=g, device="cuda").int()
    if case["masked"]:  # tokens that may not be sampled, and answers that end before the batch does
        s["logits"].masked_fill_(torch.rand(r, w, generator=g, device="cuda") < 0.1, float("-inf"))
        s["logits"][torch.arange(r, device="cuda"), s["labels"].long()] = 1.0
        s["labels"][torch.rand(r, generator=g, device="cuda") < 0.1] = -1
    if own:
        s["logp"], s["lse"] = torch.empty(r, device="cuda"), torch.empty(r, device="cuda")


def _prepare_policy(case, g, s):
    r = case["rows"]
    _prepare_logprob(case, g, s)
    now = _logprob_rows(s, case)[0]
    # the sampling policy is a few updates old, the reference further away
    s["old_logp"] = (now + 0.15 * _randn(g, r)).float()
    if case["ref"]:
        s["ref_logp"] = (now + 0.3 * _randn(g, r)).float()
    s["advantages"] = _randn(g, r)
    used = torch.rand(r, generator=g, device="cuda") < (0.8 if case["masked"] else 2.0)
    s["weights"] = used.float() / used.sum().clamp(min=1)
    if own:
        s["logits_grad"], s["totals"] = torch.zeros_like(s["logits"]), torch.empty(4, device="cuda")


# ---- one pass ----

CLIP, KL = (0.2, 0.28), 0.05


def _loss_scale(case):
    """16-bit floats without f32's exponents are trained with a scaled loss."""
    return 1024.0 if case["dtype"] == "f16" else 1.0


def run(s):
    return globals()[("_own_" if own else "_plain_") + s["case"]["op"]](s)


_ACTIVATION = {
    "none": lambda z: z,
    "relu": lambda z: z.clamp(min=0),
    "silu": lambda z: z / (1 + torch.exp(-z)),
    "gelu": lambda z: 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5))),
}


def _silu_grad(z):
    sig = 1 / (1 + torch.exp(-z))
    return sig * (1 + z * (1 - sig))


_ACTIVATION_GRAD = {
    "none": lambda z: torch.ones_like(z),
    "relu": lambda z: (z > 0).to(z.dtype),
    "silu": _silu_grad,
    "gelu": lambda z: 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi)),
}
EPS = 1e-5


def _stats(x, groups, kind):
    """Mean and reciprocal deviation of every sample and group: [n, groups, 2]."""
    n, p, c = x.shape
    x = x.to(kind).reshape(n, p, groups, c // groups)
    mean = x.mean((1, 3), keepdim=True)
    var = (x - mean).square().mean((1, 3))
    return torch.stack((mean.reshape(n, groups), torch.rsqrt(var + EPS)), -1)


def _normed(x, stats, groups):
    """x as [n, positions, groups, channels of a group], and the normalised values."""
    n, p, c = x.shape
    x = x.reshape(n, p, groups, c // groups)
    return (x - stats[:, None, :, 0, None]) * stats[:, None, :, 1, None]


def _norm(x, gamma, beta, case):
    stats = _stats(x, case["groups"], x.dtype)
    z = _normed(x, stats, case["groups"]).reshape(x.shape) * gamma + beta
    return _ACTIVATION[case["act"]](z), stats


def _plain_norm(s):
    case = s["case"]
    out, stats = _norm(s["x"][:, :, :case["channels"]].float(), s["gamma"].float(), s["beta"].float(), case)
    return {"out": out.to(s["x"].dtype), "stats": stats}


def _own_norm(s):
    case, b = s["case"], s["b"]
    shape, pitch = (case["n"], case["positions"], case["channels"]), case["channels"] + case["pad"]
    s["dev"].group_norm(b["x"], b["gamma"], b["beta"], shape, case["groups"], activation=case["act"], eps=EPS,
                        out=b["out"], stats=b["stats"], x_pitch=pitch, out_pitch=pitch)
    return {"out": s["out"][:, :, :case["channels"]], "stats": s["stats"]}


def _norm_grad(x, stats, gamma, beta, out_grad, case):
    n, p, c = x.shape
    groups, m = case["groups"], p * (c // case["groups"])
    xhat = _normed(x, stats, groups).reshape(n, p, c)
    dz = out_grad * _ACTIVATION_GRAD[case["act"]](xhat * gamma + beta)
    gamma_grad, beta_grad = (dz * xhat).sum((0, 1)), dz.sum((0, 1))
    dh, xhat = (dz * gamma).reshape(n, p, groups, -1), xhat.reshape(n, p, groups, -1)
    a, b = dh.sum((1, 3), keepdim=True) / m, (dh * xhat).sum((1, 3), keepdim=True) / m
    return ((dh - a - xhat * b) * stats[:, None, :, 1, None]).reshape(n, p, c), gamma_grad, beta_grad


def _plain_norm_grad(s):
    case = s["case"]
    c = case["channels"]
    if case["saved"]:
        x = _restore(s["codes"], s["scales"]).reshape(case["n"], case["positions"], c)
    else:
        x = s["x"][:, :, :c].float()
    dx, dgamma, dbeta = _norm_grad(x, s["stats"], s["gamma"].float(), s["beta"].float(), s["out_grad"][:, :, :c].float(), case)
    return {"x_grad": dx.to(TYPES[case["dtype"]]), "gamma_grad": dgamma, "beta_grad": dbeta}


def _own_norm_grad(s):
    case, b = s["case"], s["b"]
    c, pitch = case["channels"], case["channels"] + case["pad"]
    s["dev"].add_group_norm_grad(b["saved"] if case["saved"] else b["x"], b["stats"], b["gamma"], b["beta"], b["out_grad"],
                                 b["x_grad"], b["gamma_grad"], b["beta_grad"], (case["n"], case["positions"], c),
                                 case["groups"], activation=case["act"], overwrite=True, x_pitch=pitch,
                                 out_grad_pitch=pitch, x_grad_pitch=pitch)
    return {"x_grad": s["x_grad"][:, :, :c], "gamma_grad": s["gamma_grad"], "beta_grad": s["beta_grad"]}


def _save(x):
    """8-bit codes and one scale for every 128 elements; -128 stands for what is not finite."""
    n = x.numel()
    x = torch.nn.functional.pad(x.float(), (0, -n % BLOCK)).reshape(-1, BLOCK)
    finite = torch.isfinite(x)
    largest = torch.where(finite, x, 0).abs().amax(1, keepdim=True)
    kept = largest >= TINY
    step = torch.where(kept, torch.full_like(largest, 127.0) / largest, 0)
    codes = torch.where(finite, torch.round(torch.where(finite, x, 0) * step), -128.0)
    return codes.to(torch.int8).reshape(-1)[:n], torch.where(kept, largest * (1 / 127), 0).reshape(-1)


def _restore(codes, scales):
    n = codes.numel()
    values = torch.nn.functional.pad(codes, (0, -n % BLOCK)).reshape(-1, BLOCK).float() * scales[:, None]
    return values.reshape(-1)[:n].masked_fill_(codes == -128, float("nan"))


_FN = {"tanh": torch.tanh, "expmix": lambda x: torch.exp(0.5 * x) * x + x * x}
_FN_GRAD = {"tanh": lambda x: 1 - torch.tanh(x).square(), "expmix": lambda x: torch.exp(0.5 * x) * (0.5 * x + 1) + 2 * x}
_OWN_FN = {"tanh": lambda x: x.tanh(), "expmix": lambda x: x.mul(0.5).exp().mul(x).add(x.mul(x))}
_OWN_FN_GRAD = {"tanh": lambda x: x.tanh().mul(x.tanh()).neg().add(1.0),
                "expmix": lambda x: x.mul(0.5).exp().mul(x.mul(0.5).add(1.0)).add(x.mul(2.0))}


def _plain_saved_unary(s):
    x, fn = s["x"], s["case"]["fn"]
    out = _FN[fn](x.float()).to(x.dtype)
    grad = s["out_grad"].float() * _FN_GRAD[fn](_restore(*_save(x)))
    return {"out": out, "x_grad": grad.to(x.dtype)}


def _own_saved_unary(s):
    dev, b, fn = s["dev"], s["b"], s["case"]["fn"]
    dev.apply_fn_checkpoint8(b["x"], _OWN_FN[fn], out=b["out"], into=b["saved"])
    dev.add_unary_grad8(b["saved"], b["x_grad"], b["out_grad"], _OWN_FN_GRAD[fn], overwrite=True)
    return {"out": s["out"], "x_grad": s["x_grad"]}


def _plain_saved_restore(s):
    return {"out": _restore(*_save(s["x"])).to(s["x"].dtype)}


def _own_saved_restore(s):
    dev, b = s["dev"], s["b"]
    dev.checkpoint8(b["x"], into=b["saved"])
    dev.restore8(b["saved"], out=b["out"])
    return {"out": s["out"]}


def _softmax_parts(s, case, kind):
    """Per row: exp((z - max) / T), their sum in 64 bits, the scaled logit of the label below the maximum, the maximum."""
    z = s["logits"][:, :case["vocab"]].to(kind)
    top = z.amax(1, keepdim=True)
    d = (z - top) * (1 / case["temperature"])
    chosen = d.gather(1, s["labels"].long().clamp(min=0)[:, None])[:, 0].double()
    return d.exp_(), chosen, top[:, 0].double()


def _logprob_rows(s, case, kind=torch.float32):
    e, chosen, top = _softmax_parts(s, case, kind)
    total = e.sum(1, dtype=torch.float64)
    used = s["labels"] >= 0
    return torch.where(used, chosen - total.log(), 0), top / case["temperature"] + total.log(), e, total


def _plain_logprob(s):
    logp, lse, _, _ = _logprob_rows(s, s["case"])
    return {"logp": logp.float(), "lse": lse.float()}


def _own_logprob(s):
    case, b = s["case"], s["b"]
    s["dev"].token_logprob(b["logits"], b["labels"], (case["rows"], case["vocab"]), temperature=case["temperature"],
                           pitch=case["vocab"] + case["pad"], out=b["logp"], lse=b["lse"])
    return {"logp": s["logp"], "lse": s["lse"]}


def _policy(s, kind):
    """The clipped loss with its KL term and d loss / d logits; the few values per row in 64 bits (a ratio next to the border)."""
    case = s["case"]
    logp, _, e, total = _logprob_rows(s, case, kind)
    used = (s["labels"] >= 0) & (s["weights"] != 0)
    w, adv, old = s["weights"].double(), s["advantages"].double(), s["old_logp"].double()
    ratio = torch.exp(logp - old)
    clipped = ratio.clamp(1 - CLIP[0], 1 + CLIP[1])
    surrogate = torch.minimum(ratio * adv, clipped * adv)
    inside = ratio * adv <= clipped * adv  # the gradient passes where the unclipped term is the smaller one
    behind = s["ref_logp"].double() - logp if case["ref"] else torch.zeros_like(logp)
    kl = torch.expm1(behind) - behind if case["ref"] else torch.zeros_like(logp)
    zero = torch.zeros_like(logp)
    terms = [w * (KL * kl - surrogate), w * kl, w * (~inside), w * ratio]
    totals = torch.stack([torch.where(used, t, zero).sum() for t in terms])
    slope = w * (-adv * ratio * inside + (-KL * torch.expm1(behind) if case["ref"] else 0)) / case["temperature"]
    slope = torch.where(used, slope * _loss_scale(case), zero)
    grad = e.mul_((-slope / total).to(e.dtype)[:, None])
    rows = torch.arange(case["rows"], device=e.device)
    grad[rows, s["labels"].long().clamp(min=0)] += slope.to(e.dtype)
    grad.masked_fill_(~used[:, None], 0)
    return totals, torch.where(used, logp, zero), grad


def _plain_policy(s):
    totals, logp, grad = _policy(s, torch.float32)
    return {"totals": totals.float(), "logp": logp.float(), "logits_grad": grad.to(s["logits"].dtype)}


def _own_policy(s):
    case, b = s["case"], s["b"]
    width = case["vocab"] + case["pad"]
    s["dev"].policy_loss(b["logits"], b["labels"], b["old_logp"], b["advantages"], b["weights"], (case["rows"], case["vocab"]),
                         ref_logp=b.get("ref_logp"), clip=CLIP, kl_coef=KL if case["ref"] else 0.0, temperature=case["temperature"],
                         pitch=width, logits_grad=b["logits_grad"], grad_pitch=width, grad_scale=_loss_scale(case), logp=b["logp"], totals=b["totals"])
    return {"totals": s["totals"], "logp": s["logp"], "logits_grad": s["logits_grad"][:, :case["vocab"]]}


# ---- what a pass cannot do without ----

def work(case):
    size = TYPES[case["dtype"]].itemsize
    if case["op"] in ("norm", "norm_grad"):
        elements = case["n"] * case["positions"] * case["channels"]
        few = case["n"] * case["groups"] * 8 + 2 * case["channels"] * TYPES[case["params"]].itemsize
        if case["op"] == "norm":  # x in, out out; sums of x and of its squares, normalise, scale, shift, activation
            return {"bytes": 2 * size * elements + few, "flops": 12 * elements}
        saved = 1 + 4 / BLOCK if case["saved"] else size
        return {"bytes": (saved + 2 * size) * elements + few + 8 * case["channels"], "flops": 24 * elements}
    if case["op"] == "saved_unary":  # x and out; codes written and read; out_grad and x_grad
        return {"bytes": (4 * size + 2 * (1 + 4 / BLOCK)) * case["len"], "flops": 20 * case["len"]}
    if case["op"] == "saved_restore":
        return {"bytes": (2 * size + 2 * (1 + 4 / BLOCK)) * case["len"], "flops": 6 * case["len"]}
    elements = case["rows"] * case["vocab"]
    if case["op"] == "logprob":
        return {"bytes": size * elements + 12 * case["rows"], "flops": 4 * elements}
    return {"bytes": 2 * size * elements + 24 * case["rows"], "flops": 6 * elements}


# ---- the definitions in 64 bits ----

def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return globals()["_exact_" + case["op"]](case, s)


def _act64(z, name):
    if name == "relu":
        return torch.where(z > 0, z, 0.0), torch.where(z > 0, 1.0, 0.0)
    if name == "silu":
        sig = torch.sigmoid(z)
        return z * sig, sig + z * sig * (1 - sig)
    if name == "gelu":
        phi = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def _exact_norm(case, s):
    n, p, c, g = case["n"], case["positions"], case["channels"], case["groups"]
    gamma, beta = s["gamma"].double().reshape(g, 1, -1), s["beta"].double().reshape(g, 1, -1)
    outs, stats = [], []
    for sample in s["x"]:  # one sample at a time: [groups, positions, channels of a group]
        x = sample[:, :c].double().reshape(p, g, -1).transpose(0, 1)
        var, mean = torch.var_mean(x, (1, 2), correction=0, keepdim=True)
        rstd = 1 / torch.sqrt(var + EPS)
        outs.append(_act64((x - mean) * rstd * gamma + beta, case["act"])[0].transpose(0, 1).reshape(p, c))
        stats.append(torch.stack((mean.reshape(g), rstd.reshape(g)), 1))
    return {"out": torch.stack(outs), "stats": torch.stack(stats)}


def _values64(codes, scales):
    scale = scales.double().repeat_interleave(BLOCK)[:codes.numel()]
    return torch.where(codes == -128, float("nan"), codes.double() * scale)


def _exact_norm_grad(case, s):
    n, p, c, g = case["n"], case["positions"], case["channels"], case["groups"]
    gamma, beta = s["gamma"].double().reshape(g, 1, -1), s["beta"].double().reshape(g, 1, -1)
    source = _values64(s["codes"], s["scales"]).reshape(n, p, c) if case["saved"] else s["x"]
    grads, gammas, betas = [], [], []
    for k in range(n):
        x = source[k, :, :c].double().reshape(p, g, -1).transpose(0, 1)
        dy = s["out_grad"][k, :, :c].double().reshape(p, g, -1).transpose(0, 1)
        mean, rstd = (s["stats"][k, :, i].double().reshape(g, 1, 1) for i in (0, 1))
        h = (x - mean) * rstd
        dz = dy * _act64(gamma * h + beta, case["act"])[1]
        gammas.append((dz * h).sum(1).reshape(c))
        betas.append(dz.sum(1).reshape(c))
        dh = dz * gamma
        grads.append((rstd * (dh - dh.mean((1, 2), keepdim=True) - h * (dh * h).mean((1, 2), keepdim=True))).transpose(0, 1).reshape(p, c))
    return {"x_grad": torch.stack(grads), "gamma_grad": torch.stack(gammas).sum(0), "beta_grad": torch.stack(betas).sum(0)}


def _quantised64(x):
    """What a checkpoint of x stands for; its codes and scales are defined by 32-bit steps."""
    n = x.numel()
    blocks = torch.zeros(-(-n // BLOCK) * BLOCK, device=x.device)
    blocks[:n] = x
    blocks = blocks.reshape(-1, BLOCK)
    top = blocks.abs().max(1, keepdim=True).values
    step = torch.true_divide(torch.full_like(top, 127.0), top)
    values = torch.round(blocks * step).double() * (top * (1 / 127)).double()
    return torch.where(top < TINY, 0.0, values).reshape(-1)[:n]


def _exact_saved_unary(case, s):
    x, v = s["x"].double(), _quantised64(s["x"])
    if case["fn"] == "tanh":
        out, slope = torch.tanh(x), 1 / torch.cosh(v) ** 2
    else:
        out, slope = x * torch.exp(x / 2) + x * x, torch.exp(v / 2) * (1 + v / 2) + 2 * v
    return {"out": out, "x_grad": s["out_grad"].double() * slope}


def _exact_saved_restore(case, s):
    return {"out": _quantised64(s["x"])}


def _exact_rows(case, s):
    """(log-probability of the label, log of the sum) of every row, and the softmax, some rows at a time."""
    step = max(1, (1 << 27) // case["vocab"])
    for at in range(0, case["rows"], step):
        z = s["logits"][at:at + step, :case["vocab"]].double() / case["temperature"]
        lse = torch.logsumexp(z, 1)
        label = s["labels"][at:at + step].long()
        logp = torch.where(label < 0, 0.0, z.gather(1, label.clamp(min=0)[:, None])[:, 0] - lse)
        yield slice(at, at + step), label, logp, lse, z


def _exact_logprob(case, s):
    parts = [(logp, lse) for _, _, logp, lse, _ in _exact_rows(case, s)]
    return {"logp": torch.cat([p[0] for p in parts]), "lse": torch.cat([p[1] for p in parts])}


def _exact_policy(case, s):
    totals, logps = torch.zeros(4, dtype=torch.float64, device="cuda"), []
    grad = torch.empty(case["rows"], case["vocab"], device="cuda")  # (64 bits would not fit three times; 2^-24 is far below its type)
    for rows, label, logp, lse, z in _exact_rows(case, s):
        w, a, old = (s[k][rows].double() for k in ("weights", "advantages", "old_logp"))
        w = torch.where(label < 0, 0.0, w)
        r = torch.exp(logp - old)
        low, high = 1 - CLIP[0], 1 + CLIP[1]
        cut = torch.where(a >= 0, r > high, r < low)
        value = torch.where(cut, torch.where(a >= 0, high, low) * a, r * a)
        kl, kl_slope = torch.zeros_like(r), torch.zeros_like(r)
        if case["ref"]:
            d = s["ref_logp"][rows].double() - logp
            kl, kl_slope = torch.expm1(d) - d, -torch.expm1(d)
        totals += torch.stack([(w * t).sum() for t in (KL * kl - value, kl, cut.double(), r)])
        logps.append(torch.where(w == 0, 0.0, logp))
        slope = w * (KL * kl_slope - torch.where(cut, 0.0, a * r)) * (_loss_scale(case) / case["temperature"])
        p = torch.exp(z - lse[:, None]) * -slope[:, None]
        p[torch.arange(len(label), device="cuda"), label.clamp(min=0)] += slope
        grad[rows] = torch.where(w[:, None] == 0, 0.0, p).float()
    return {"totals": totals, "logp": torch.cat(logps), "logits_grad": grad}
