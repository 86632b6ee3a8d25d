"""The 8-bit row checkpoints and the low-rank adapter products: cases, plain forms and exact results.

Five entry points of `ozaki_jax_b200` are timed here, as four operators:

  rows      restore_rows(checkpoint_rows(X)): an activation matrix held in 8 bits between the forward
            and the backward pass.  Groups of 128 columns of a row share a power of two 2^e; the
            codes are integers in [-127, 127].
  weight    checkpoint_grad(dY, saved) = dY^T X^: the weight gradient of a linear layer from its
            checkpointed input.
  adapters  matmul_adapters(X, W, A, B, ids, scale): Y = X W^T + s_i (X A_i^T) B_i^T, where row m
            of X belongs to adapter i = ids[m] (-1: to none).
  grad      adapters_grad(dY, X or saved, W, A, B, ids, T, scale): dX, dA and dB of the same product.

With `own` false, `run` computes each with elementary torch operations in 32 bits.
"""

import math

import torch

own = False

GROUP = 128  # columns of a row that share one exponent
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FLOOR = {"bf16": -126, "fp16": -24, "fp32": -126}  # smallest exponent of a code's step
CEIL = {"bf16": 121, "fp16": 9, "fp32": 121}       # largest one


def listed():
    return [
        # the round trip of an FP32 matrix of odd size: a small layer's activations
        {"name": "rows_fp32_1000x1001", "op": "rows", "type": "fp32", "m": 1000, "k": 1001},
        # the tall matrix of the gram configuration as one layer's activations
        {"name": "rows_bf16_65536x4096", "op": "rows", "type": "bf16", "m": 65536, "k": 4096},
        # a ragged micro-batch into an FP32 gradient
        {"name": "weight_fp16_1511x1000x777", "op": "weight", "type": "fp16", "out": "fp32",
         "m": 1511, "n": 1000, "k": 777},
        # one training step's tokens through an ordinary square projection
        {"name": "weight_bf16_4096x4096x4096", "op": "weight", "type": "bf16", "out": "bf16",
         "m": 4096, "n": 4096, "k": 4096},
        # the largest: the 8192 x 8192 operand of the headline workload as a weight, 16384 tokens
        {"name": "weight_bf16_16384x8192x8192", "op": "weight", "type": "bf16", "out": "bf16",
         "m": 16384, "n": 8192, "k": 8192},
        # one request decoding: latency
        {"name": "adapters_bf16_1x4096x4096_r16", "op": "adapters", "type": "bf16", "m": 1,
         "n": 4096, "k": 4096, "r": 16, "e": 32, "ids": "tokens"},
        # a decode batch of 64 requests over 64 adapters
        {"name": "adapters_bf16_64x8192x4096_r16", "op": "adapters", "type": "bf16", "m": 64,
         "n": 8192, "k": 4096, "r": 16, "e": 64, "ids": "tokens"},
        # a packed batch of prompts, ragged in every dimension
        {"name": "adapters_fp16_1777x1001x2000_r24", "op": "adapters", "type": "fp16", "m": 1777,
         "n": 1001, "k": 2000, "r": 24, "e": 8, "ids": "runs"},
        # a large prompt or training batch at a high rank
        {"name": "adapters_bf16_8192x8192x4096_r64", "op": "adapters", "type": "bf16", "m": 8192,
         "n": 8192, "k": 4096, "r": 64, "e": 4, "ids": "runs"},
        # backward of a small ragged batch from checkpointed rows
        {"name": "grad_fp16_1023x1000x2048_r8", "op": "grad", "type": "fp16", "m": 1023, "n": 1000,
         "k": 2048, "r": 8, "e": 5, "ids": "runs", "saved": True},
        # backward of an ordinary batch from 16-bit activations
        {"name": "grad_bf16_4096x4096x4096_r16", "op": "grad", "type": "bf16", "m": 4096, "n": 4096,
         "k": 4096, "r": 16, "e": 8, "ids": "runs", "saved": False},
        # backward of a large batch from checkpointed rows
        {"name": "grad_bf16_8192x4096x8192_r32", "op": "grad", "type": "bf16", "m": 8192, "n": 4096,
         "k": 8192, "r": 32, "e": 16, "ids": "runs", "saved": True},
    ]


def _spread(rng, lo, hi):
    """A size spread over the logarithm of its range: a multiple of 64 or of 8, or any number."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    step = rng.choice([64, 64, 8, 1])
    return min(hi, max(lo, int(v) // step * step))


def draw(rng):
    op = rng.choice(["rows", "weight", "weight", "adapters", "adapters", "adapters", "grad", "grad"])
    while True:
        if op == "rows":
            case = {"op": op, "type": rng.choice(["bf16", "fp16", "fp32"]),
                    "m": _spread(rng, 1, 65536), "k": _spread(rng, 1, 16384)}
            if case["m"] * case["k"] <= 65536 * 2048:
                return case
            continue
        kind = rng.choice(["bf16", "fp16"])
        if op == "weight":
            case = {"op": op, "type": kind, "out": rng.choice([kind, "fp32"]),
                    "m": _spread(rng, 1, 16384), "n": _spread(rng, 16, 8192),
                    "k": _spread(rng, 16, 8192)}
        else:
            case = {"op": op, "type": kind, "m": _spread(rng, 1 if op == "adapters" else 64, 8192),
                    "n": _spread(rng, 64, 8192), "k": _spread(rng, 64, 8192),
                    "r": rng.choice([4, 8, 16, 16, 32, 64, 128]), "e": rng.choice([1, 3, 8, 16, 64]),
                    "ids": "runs"}
            if op == "adapters" and case["m"] <= 256:
                case["ids"] = "tokens"
            if op == "grad":
                case["saved"] = rng.random() < 0.5
        if case["m"] * case["n"] * case["k"] <= 8192 * 8192 * 8192:
            return case


# ------------------------------------------------------------------- inputs

def _ids(case, g):
    """Adapter of each row: a row of its own (decoding), or one of a packed batch of requests."""
    m, e = case["m"], case["e"]
    if case["ids"] == "tokens":
        ids = torch.randint(0, e, (m,), generator=g, device="cuda", dtype=torch.int32)
        bare = torch.rand(m, generator=g, device="cuda") < 0.05
        bare[0] = False
        return torch.where(bare, -1, ids).to(torch.int32)
    requests = max(2, min(2 * e, m // 16))
    cuts = torch.randint(0, m + 1, (requests - 1,), generator=g, device="cuda").sort().values
    which = torch.randint(-1, e, (requests,), generator=g, device="cuda", dtype=torch.int32)
    at = torch.searchsorted(cuts, torch.arange(m, device="cuda"), right=True)
    return which[at].contiguous()


def _normal(shape, g, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _activations(m, k, g, dtype):
    """Rows with a few strong columns, as a network's activations have."""
    strong = torch.exp(0.7 * torch.randn(k, generator=g, device="cuda"))
    x = torch.randn(m, k, generator=g, device="cuda")
    return x.mul_(strong).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    t = TYPES[case["type"]]
    m, k = case["m"], case["k"]
    s = {"case": case, "x": _activations(m, k, g, t)}
    if case["op"] == "rows":
        return s
    n = case["n"]
    if case["op"] in ("weight", "grad"):
        s["dy"] = _normal((m, n), g, t, 0.05)
    if case["op"] == "weight" or case.get("saved"):
        # the layer's input is in hand as codes and exponents, kept since the forward pass
        s["codes"], s["exps"] = _codes(s.pop("x"), case["type"])
    if case["op"] != "weight":
        e, r = case["e"], case["r"]
        s["w"] = _normal((n, k), g, t, k ** -0.5)
        s["a"] = _normal((e, r, k), g, t, k ** -0.5)
        s["b"] = _normal((e, n, r), g, t, r ** -0.5)
        s["scale"] = 0.5 + torch.rand(e, generator=g, device="cuda")
        s["ids"] = _ids(case, g)
    if case["op"] == "grad":
        # what the forward pass returned beside Y
        s["t"] = torch.randn(m, case["r"], generator=g, device="cuda")
    return s


# ---------------------------------------------------------- the plain forms

def _two_to(e):
    """2^e in FP32, exactly, for -126 <= e <= 127."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _codes(x, kind):
    """(codes [m, k up to a multiple of 128] int8, exponents [groups, m] int8) of the rows of x."""
    m, k = x.shape
    v = torch.nn.functional.pad(x, (0, -k % GROUP)).view(m, -1, GROUP).float()
    top = v.abs().amax(2)
    whole = torch.isfinite(top)
    e = (torch.frexp(torch.where(whole, top, 1.0)).exponent - 7).clamp(min=FLOOR[kind])
    e = torch.where((top * _two_to(-e)).round() > 127, e + 1, e).clamp(max=CEIL[kind])
    q = (v * _two_to(-e)[:, :, None]).round().clamp(-127, 127)
    q = torch.where(whole[:, :, None], q, 0).to(torch.int8).view(m, -1)
    return q, torch.where(whole, e, -128).to(torch.int8).t().contiguous()


def _values(codes, exps, k):
    """The FP32 values of codes and exponents."""
    m = codes.shape[0]
    e = exps.t().to(torch.int32)
    step = torch.where(e == -128, torch.nan, _two_to(e.clamp(min=-126)))
    return (codes.view(m, -1, GROUP).float() * step[:, :, None]).view(m, -1)[:, :k]


def _own_rows(low, ids, e):
    """[m, e r]: row m's r values in the columns of adapter ids[m], zero elsewhere."""
    mine = ids[:, None] == torch.arange(e, device=ids.device, dtype=ids.dtype)
    return (mine[:, :, None] * low[:, None, :]).view(low.shape[0], -1)


def _pick(all_, ids, scale):
    """[m, r]: of each row's products with every adapter, those of its own one, times its scale."""
    mine = ids[:, None] == torch.arange(all_.shape[1], device=ids.device, dtype=ids.dtype)
    return ((mine * scale)[:, :, None] * all_).sum(1)


def _plain(s):
    case = s["case"]
    t = TYPES[case["type"]]
    m, k = case["m"], case["k"]
    if case["op"] == "rows":
        return _values(*_codes(s["x"], case["type"]), k).to(t)
    x = s["x"].float() if "x" in s else _values(s["codes"], s["exps"], k)
    if case["op"] == "weight":
        return (s["dy"].float().t() @ x).to(TYPES[case["out"]])
    n, e, r = case["n"], case["e"], case["r"]
    w, a, b = s["w"].float(), s["a"].float(), s["b"].float()
    if case["op"] == "adapters":
        low = _pick((x @ a.view(e * r, k).t()).view(m, e, r), s["ids"], s["scale"])
        y = x @ w.t() + _own_rows(low, s["ids"], e) @ b.transpose(1, 2).reshape(e * r, n)
        return y.to(t), low
    dy = s["dy"].float()
    bt = b.transpose(1, 2).reshape(e * r, n)
    up = _own_rows(_pick((dy @ bt.t()).view(m, e, r), s["ids"], s["scale"]), s["ids"], e)
    dx = dy @ w + up @ a.view(e * r, k)
    da = (up.t() @ x).view(e, r, k)
    db = (_own_rows(s["t"], s["ids"], e).t() @ dy).view(e, r, n).transpose(1, 2)
    return dx.to(t), da.to(t), db.to(t).contiguous()


def _calls(s):
    import ozaki_jax_b200 as oz
    case = s["case"]
    if case["op"] == "rows":
        return oz.restore_rows(oz.checkpoint_rows(s["x"]))
    if "codes" in s:
        x = oz.SavedRows(s["codes"], s["exps"], case["k"], TYPES[case["type"]])
    else:
        x = s["x"]
    if case["op"] == "weight":
        return oz.checkpoint_grad(s["dy"], x, dtype=TYPES[case["out"]])
    if case["op"] == "adapters":
        return oz.matmul_adapters(x, s["w"], s["a"], s["b"], s["ids"], s["scale"], return_low=True)
    return oz.adapters_grad(s["dy"], x, s["w"], s["a"], s["b"], s["ids"], s["t"], s["scale"])


def run(state):
    return _calls(state) if own else _plain(state)


# ---------------------------------------------------------------- the bounds

def work(case):
    m, k = case["m"], case["k"]
    size = 4 if case["type"] == "fp32" else 2
    groups = m * -(-k // GROUP)
    held = m * k + groups
    if case["op"] == "rows":
        return {"bytes": 2 * (m * k * size + held), "flops": 4 * m * k}
    n = case["n"]
    if case["op"] == "weight":
        return {"bytes": m * n * 2 + held + n * k * (4 if case["out"] == "fp32" else 2),
                "flops": 2 * m * n * k}
    e, r = case["e"], case["r"]
    requests = m if case["ids"] == "tokens" else max(2, min(2 * e, m // 16))
    used = e * (1 - (1 - 1 / e) ** requests) if e > 1 else 1
    weights = (n * k + used * r * (n + k)) * 2
    if case["op"] == "adapters":
        return {"bytes": int(weights + m * (k + n) * 2 + m * (r + 1) * 4),
                "flops": 2 * m * (n * k + r * (n + k))}
    x = held if case["saved"] else 2 * m * k
    return {"bytes": int(weights + e * r * (n + k) * 2 + m * (n + k) * 2 + x + m * (r + 1) * 4),
            "flops": 2 * m * (n * k + 2 * r * (n + k))}


# ----------------------------------------------- the definitions in 64 bits

def _step(e):
    """2^e in FP64 from its bits: pow(2, e) on the device is not exact."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_rows(x, kind):
    """Value of each element after the round trip, in 64 bits, from the definition: the step 2^e is
    the smallest power of two under which the group's largest value rounds to at most 127."""
    k = x.shape[1]
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for c in range(0, k, GROUP):
        v = x[:, c:c + GROUP].double()
        top = v.abs().max(1, keepdim=True).values
        e = torch.full_like(top, FLOOR[kind])
        # from far below up: floor(log2) may be off by one near a power of two, the loop is not
        e = torch.maximum(e, torch.floor(torch.log2(top.clamp(min=1e-60))) - 8)
        for _ in range(4):
            e = torch.where(torch.round(top / _step(e)) > 127, e + 1, e)
        e = e.clamp(max=CEIL[kind])
        q = torch.round(v / _step(e)).clamp(-127, 127)
        out[:, c:c + GROUP] = q * _step(e)
    return out


def _exact_saved(s, k):
    e = s["exps"].double().repeat_interleave(GROUP, 0).t()
    return (s["codes"].double() * _step(e))[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    m, k = case["m"], case["k"]
    if case["op"] == "rows":
        return _exact_rows(s["x"], case["type"])
    x = s["x"].double() if "x" in s else _exact_saved(s, k)
    if case["op"] == "weight":
        return torch.einsum("mn,mk->nk", s["dy"].double(), x)
    w, ids = s["w"].double(), s["ids"]
    if case["op"] == "adapters":
        y = torch.einsum("mk,nk->mn", x, w)
        low = torch.zeros(m, case["r"], dtype=torch.float64, device=x.device)
        for i in range(case["e"]):
            rows = (ids == i).nonzero()[:, 0]
            t = float(s["scale"][i]) * (x[rows] @ s["a"][i].double().t())
            low[rows] = t
            y[rows] += t @ s["b"][i].double().t()
        return y, low
    dy = s["dy"].double()
    dx = torch.einsum("mn,nk->mk", dy, w)
    da = torch.zeros(s["a"].shape, dtype=torch.float64, device=x.device)
    db = torch.zeros(s["b"].shape, dtype=torch.float64, device=x.device)
    for i in range(case["e"]):
        rows = (ids == i).nonzero()[:, 0]
        u = float(s["scale"][i]) * (dy[rows] @ s["b"][i].double())
        dx[rows] += u @ s["a"][i].double()
        da[i] = u.t() @ x[rows]
        db[i] = dy[rows].t() @ s["t"][rows].double()
    return dx, da, db
