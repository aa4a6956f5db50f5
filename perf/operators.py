"""The query/key path from a projection to attention: its operators, as they are measured.

Four operators, each in a plain form (elementary torch operations in 32 bits) and as calls of this package:

* ``tables``:  cos/sin rows of rotary positions, scaled for long contexts (``rope_tables``)
* ``rope``:    the rotation of queries and keys by those rows (``fused_rope``), with its gradient
* ``qknorm``:  RMSNorm of each query and key head and the rotation in the same pass
               (``fused_qk_norm_rope``), with its gradients
* ``lora``:    low-rank adapters of many requests beside a shared projection (``fused_lora``)

A case is a dict of plain values; ``prepare`` makes its inputs, ``run`` is one pass.
"""

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4}
_EPS = 1e-6
_ORIGINAL = 8192  # positions of the unscaled context that the scalings extend


def _ops():
    """This repository's package (only reached where `own` is true)."""
    if "triton_ops" not in sys.modules:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "triton-fused-ops_b200"))
    import triton_ops

    return triton_ops


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _qk(name, op, batch, seq, hq, hk, dim, rot, layout, dtype, table, pos, train=False):
    return {"name": name, "op": op, "batch": batch, "seq": seq, "hq": hq, "hk": hk, "dim": dim, "rot": rot,
            "layout": layout, "dtype": dtype, "table": table, "pos": pos, "train": train}


def _tables(name, count, rot, scaling, dtype, far):
    return {"name": name, "op": "tables", "count": count, "rot": rot, "scaling": scaling, "dtype": dtype, "far": far}


def _lora(name, tokens, adapters, rank, k, n, dtype, order):
    return {"name": name, "op": "lora", "tokens": tokens, "adapters": adapters, "rank": rank, "k": k, "n": n,
            "dtype": dtype, "order": order}


def listed():
    return [
        # rows for one decode step of 64 requests somewhere in a long context
        _tables("tables decode", 64, 128, "yarn", "f32", 131072),
        # the whole table of a long context, made once when a server starts
        _tables("tables long", 131072, 128, "wavelength", "f32", 131072),
        # one new token of one request: latency is all
        _qk("rope single token", "rope", 1, 1, 32, 8, 128, 128, "half", "bf16", "f32", "given"),
        # a training step of a model whose heads rotate half their width, in pairs
        _qk("rope train partial", "rope", 2, 4096, 32, 8, 128, 64, "pairs", "bf16", "f32", "run", True),
        # one decode step of 64 requests
        _qk("qknorm decode", "qknorm", 64, 1, 32, 8, 128, 128, "half", "bf16", "f32", "given"),
        # a ragged prompt batch, flattened, with a narrow odd head
        _qk("qknorm ragged", "qknorm", 1, 1999, 12, 3, 80, 80, "half", "f16", "f16", "given"),
        # prefill of 8 prompts of 8192 tokens
        _qk("qknorm prefill", "qknorm", 8, 8192, 32, 8, 128, 128, "half", "bf16", "f32", "run"),
        # a training step: both directions, gradients of inputs and weights
        _qk("qknorm train", "qknorm", 2, 4096, 32, 8, 128, 128, "half", "bf16", "f32", "run", True),
        # the same in full precision with head width 64 and as many key heads as query heads
        _qk("qknorm train f32", "qknorm", 2, 1024, 16, 16, 64, 64, "half", "f32", "f32", "run", True),
        # one token of one request beside a 4096 x 4096 projection
        _lora("lora single token", 1, 8, 16, 4096, 4096, "bf16", "mixed"),
        # one decode step: 64 requests over 32 adapters, in any order
        _lora("lora decode", 64, 32, 16, 4096, 4096, "bf16", "mixed"),
        # prefill of 8192 tokens of some tens of requests
        _lora("lora prefill", 8192, 16, 32, 4096, 4096, "bf16", "requests"),
    ]


def _spread(rng, low, high):
    """An integer of [low, high], even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["tables", "rope", "rope", "qknorm", "qknorm", "qknorm", "lora", "lora", "lora"])
    if op == "tables":
        c = _tables("", _spread(rng, 1, 100000), 2 * rng.randint(8, 64), rng.choice(["none", "linear", "ntk", "yarn", "wavelength"]),
                    rng.choice(["f32", "f32", "bf16", "f16"]), rng.choice([8192, 131072, 1000000]))
    elif op == "lora":
        tokens = _spread(rng, 1, 6000)
        c = _lora("", tokens, _spread(rng, 1, 48), rng.choice([4, 8, 8, 16, 16, 24, 32, 64]), _spread(rng, 48, 4096), _spread(rng, 48, 4096),
                  rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice(["mixed", "requests"]))
        if rng.random() < 0.7:  # most projections are a multiple of 64 wide, some are not
            c["k"], c["n"] = -(-c["k"] // 64) * 64, -(-c["n"] // 64) * 64
    else:
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 256])
        rot = rng.choice([dim, dim, dim // 2])
        hk = rng.choice([1, 2, 3, 4, 8])
        hq = hk * rng.choice([1, 2, 4, 5])
        batch = rng.choice([1, 1, 2, 3, 5, 8])
        tokens = _spread(rng, 1, min(30000, 75_000_000 // ((hq + hk) * dim)))
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        c = _qk("", op, batch, max(1, tokens // batch), hq, hk, dim, rot, rng.choice(["half", "half", "pairs"]), dtype,
                rng.choice(["f32", dtype]), rng.choice(["run", "given"]), rng.random() < 0.4)
    c.pop("name")
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    def randint(high, *shape):
        return torch.randint(high, shape, device=dev, generator=g)

    s = dict(case)
    if case["op"] == "tables":
        s["positions"] = randint(case["far"], case["count"])
        return s
    dt = _DTYPES[case["dtype"]]
    if case["op"] == "lora":
        t, m, r = case["tokens"], case["adapters"], case["rank"]
        if case["order"] == "requests":  # each request's tokens lie together
            cuts = torch.rand(t, device=dev, generator=g) < min(1.0, 24.0 / t)
            request = torch.cumsum(cuts, 0)
            ids = (randint(m + 1, t + 1) - 1)[request]  # -1: a request without an adapter
        else:
            ids = torch.where(torch.rand(t, device=dev, generator=g) < 0.1, -1, randint(m, t))
        s["ids"] = ids
        s["x"] = randn(t, case["k"]).to(dt)
        s["base"] = randn(t, case["n"]).to(dt)
        s["a"] = (randn(m, r, case["k"]) / math.sqrt(case["k"])).to(dt)
        s["b"] = (randn(m, case["n"], r) / math.sqrt(r)).to(dt)
        s["scaling"] = 0.5 + 1.5 * torch.rand(m, device=dev, generator=g)
        return s
    b, n, hq, hk, d = (case[k] for k in ("batch", "seq", "hq", "hk", "dim"))
    # queries and keys are the first columns of one fused projection's output
    qkv = randn(b, n, (hq + 2 * hk), d).mul_(0.5 + 1.5 * torch.rand(d, device=dev, generator=g)).to(dt)
    s["q"], s["k"] = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    far = n if case["pos"] == "run" else max(n, 16384)
    freq = 10000.0 ** (-torch.arange(0, case["rot"], 2, device=dev, dtype=torch.float64) / case["rot"])
    angle = torch.arange(far, device=dev, dtype=torch.float64)[:, None] * freq
    angle = torch.cat([angle, angle], dim=-1)
    s["cos"], s["sin"] = angle.cos().to(_DTYPES[case["table"]]), angle.sin().to(_DTYPES[case["table"]])
    s["positions"] = None if case["pos"] == "run" else randint(far, b, n)
    if case["op"] == "qknorm":
        s["wq"], s["wk"] = 1 + 0.1 * randn(d), 1 + 0.1 * randn(d)
    if case["train"]:
        s["gq"], s["gk"] = randn(b, n, hq, d).to(dt), randn(b, n, hk, d).to(dt)
        s["leaves"] = [s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()]
        if case["op"] == "qknorm":
            s["leaves"] += [s["wq"].detach().requires_grad_(), s["wk"].detach().requires_grad_()]
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return {"tables": _run_tables, "rope": _run_rope, "qknorm": _run_qknorm, "lora": _run_lora}[state["op"]](state)


def _run_tables(s):
    dt = _DTYPES[s["dtype"]]
    if own:
        o = _ops()
        scaling = None
        if s["scaling"] != "none":
            scaling = o.RoPEScaling(s["scaling"], factor=8.0, original_max_position=_ORIGINAL)
        return o.rope_tables(s["positions"], s["rot"], 10000.0, scaling, dtype=dt)
    freq, gain = _frequencies(s["rot"], s["scaling"])
    angle = s["positions"].double()[:, None] * torch.tensor(freq, dtype=torch.float64, device=s["positions"].device)
    angle = torch.cat([angle, angle], dim=-1)
    return (angle.cos() * gain).to(dt), (angle.sin() * gain).to(dt)


def _run_rope(s):
    pairs = s["layout"] == "pairs"
    if own:
        o = _ops()
        if not s["train"]:
            return o.fused_rope(s["q"], s["k"], s["cos"], s["sin"], s["positions"], interleaved=pairs)
        q, k = o.fused_rope(*s["leaves"], s["cos"], s["sin"], s["positions"], interleaved=pairs)
        return (q, k, *torch.autograd.grad([q, k], s["leaves"], [s["gq"], s["gk"]]))
    dt = s["q"].dtype
    c, n = _angles(s)
    out = tuple(_rotate(t.float(), c, n, pairs).to(dt) for t in (s["q"], s["k"]))
    if s["train"]:
        out += tuple(_rotate(t.float(), c, -n, pairs).to(dt) for t in (s["gq"], s["gk"]))
    return out


def _run_qknorm(s):
    pairs = s["layout"] == "pairs"
    if own:
        o = _ops()
        if not s["train"]:
            return o.fused_qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], s["positions"], _EPS,
                                        interleaved=pairs)
        q, k = o.fused_qk_norm_rope(*s["leaves"], s["cos"], s["sin"], s["positions"], _EPS, interleaved=pairs)
        return (q, k, *torch.autograd.grad([q, k], s["leaves"], [s["gq"], s["gk"]]))
    dt = s["q"].dtype
    c, n = _angles(s)
    (q, dq, dwq), (k, dk, dwk) = (
        _norm_rope(s[x].float(), s[w], c, n, pairs, s[g].float() if s["train"] else None)
        for x, w, g in (("q", "wq", "gq"), ("k", "wk", "gk")))
    if not s["train"]:
        return q.to(dt), k.to(dt)
    return q.to(dt), k.to(dt), dq.to(dt), dk.to(dt), dwq, dwk


def _run_lora(s):
    if own:
        return _ops().fused_lora(s["x"], s["a"], s["b"], s["ids"], s["scaling"], base=s["base"])
    m, r, k = s["a"].shape
    mine = (s["ids"][:, None] == torch.arange(m, device=s["ids"].device)).float() * s["scaling"]
    low = (s["x"].float() @ s["a"].float().view(m * r, k).t()).view(-1, m, r) * mine[:, :, None]
    delta = low.view(-1, m * r) @ s["b"].float().transpose(1, 2).reshape(m * r, -1)
    return (s["base"].float() + delta).to(s["base"].dtype)


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _frequencies(rot, scaling):
    """Angle per position of each pair of columns, and the factor on cos and sin."""
    factor, gain = 8.0, 1.0
    base = 10000.0 * factor ** (rot / (rot - 2)) if scaling == "ntk" else 10000.0
    freq = [base ** (-2 * i / rot) for i in range(rot // 2)]
    if scaling == "linear":
        freq = [f / factor for f in freq]
    elif scaling == "yarn":
        # pairs that turn more than 32 times over the original context keep their
        # angle, those that turn less than once are slowed down, linear in between
        low, high = (rot * math.log(_ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(10000.0)) for turns in (32.0, 1.0))
        low, high = max(math.floor(low), 0), min(math.ceil(high), rot - 1)
        slow = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(rot // 2)]
        freq = [f * (1 - w) + f / factor * w for f, w in zip(freq, slow)]
        gain = 0.1 * math.log(factor) + 1.0
    elif scaling == "wavelength":
        # kept below a wavelength of original / 4, slowed above original / 1
        keep = [min(1.0, max(0.0, (_ORIGINAL * f / (2 * math.pi) - 1.0) / 3.0)) for f in freq]
        freq = [f * w + f / factor * (1 - w) for f, w in zip(freq, keep)]
    return freq, gain


def _angles(s):
    """cos and sin for each token, [batch, seq, 1, rot / 2], in 32 bits."""
    half = s["rot"] // 2
    at = s["positions"] if s["positions"] is not None else torch.arange(s["seq"], device=s["q"].device)[None]
    return s["cos"][at][..., None, :half].float(), s["sin"][at][..., None, :half].float()


def _rotate(x, c, n, pairs):
    rot = 2 * c.shape[-1]
    first, second = (x[..., 0:rot:2], x[..., 1:rot:2]) if pairs else (x[..., :rot // 2], x[..., rot // 2:rot])
    y = first * c - second * n, first * n + second * c
    y = torch.stack(y, dim=-1).flatten(-2) if pairs else torch.cat(y, dim=-1)
    return torch.cat([y, x[..., rot:]], dim=-1)


def _norm_rope(x, w, c, n, pairs, grad):
    """The normed and rotated heads and, with `grad`, the gradients of x and w."""
    inv = (x.square().mean(-1, keepdim=True) + _EPS).rsqrt()
    unit = x * inv
    out = _rotate(unit * w, c, n, pairs)
    if grad is None:
        return out, None, None
    back = _rotate(grad, c, -n, pairs)  # the inverse rotation
    dunit = back * w
    dx = inv * (dunit - unit * (dunit * unit).mean(-1, keepdim=True))
    return out, dx, (back * unit).double().sum((0, 1, 2)).float()


# ---------------------------------------------------------------------------
# sizes and 64-bit results
# ---------------------------------------------------------------------------
def work(case):
    esize = _BYTES[case["dtype"]]
    if case["op"] == "tables":
        values = case["count"] * case["rot"]
        return {"bytes": 8 * case["count"] + 2 * esize * values, "flops": 2 * values}
    if case["op"] == "lora":
        t, r, both = case["tokens"], case["rank"], case["k"] + case["n"]
        used = min(t, case["adapters"])
        return {"bytes": esize * (t * (both + case["n"]) + used * r * both) + 8 * t, "flops": 2 * t * r * both}
    tokens = case["batch"] * case["seq"]
    values = tokens * (case["hq"] + case["hk"]) * case["dim"]
    rows = case["seq"] if case["pos"] == "run" else tokens
    passes = 4 if case["train"] else 2
    table = rows * case["rot"] * _BYTES[case["table"]] + (8 * tokens if case["pos"] == "given" else 0)
    return {"bytes": passes * esize * values + table, "flops": values * (8 if case["op"] == "qknorm" else 3) * passes / 2}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tables":
        return _exact_tables(case, s["positions"].double())
    if case["op"] == "lora":
        out = s["base"].double()
        for i in range(case["adapters"]):
            at = (s["ids"] == i).nonzero()[:, 0]
            low = torch.einsum("tk,rk->tr", s["x"][at].double(), s["a"][i].double())
            out[at] += torch.einsum("tr,nr->tn", low, s["b"][i].double()) * s["scaling"][i].double()
        return out
    half = case["rot"] // 2
    at = s["positions"] if s["positions"] is not None else torch.arange(case["seq"], device="cuda").expand(case["batch"], -1)
    turn = torch.complex(s["cos"][at][..., :half].double(), s["sin"][at][..., :half].double())[:, :, None]
    leaves = [s[t].double().requires_grad_(case["train"]) for t in ("q", "k", "wq", "wk") if t in s]

    def forward(x, w):
        if w is not None:
            x = x / torch.linalg.vector_norm(torch.cat([x, torch.full_like(x[..., :1], math.sqrt(_EPS * x.shape[-1]))], -1),
                                             dim=-1, keepdim=True) * math.sqrt(x.shape[-1]) * w
        head = x[..., :case["rot"]]
        z = head.unflatten(-1, (half, 2)) if case["layout"] == "pairs" else head.unflatten(-1, (2, half)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
        z = z if case["layout"] == "pairs" else z.transpose(-1, -2)
        return torch.cat([z.flatten(-2), x[..., case["rot"]:]], dim=-1)

    out = [forward(x, leaves[i + 2] if len(leaves) > 2 else None) for i, x in enumerate(leaves[:2])]
    if not case["train"]:
        return tuple(out)
    grads = torch.autograd.grad(out, leaves, [s["gq"].double(), s["gk"].double()])
    return tuple(t.detach() for t in (*out, *grads))


def _exact_tables(case, positions):
    rot, kind = case["rot"], case["scaling"]
    pair = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    exponent, gain = 2 * pair / rot, 1.0
    period = 2 * math.pi * torch.pow(torch.tensor(10000.0, dtype=torch.float64, device="cuda"), exponent)
    if kind == "linear":
        period = period * 8
    elif kind == "ntk":
        period = period * 8.0 ** (2 * pair / (rot - 2))
    elif kind == "yarn":
        def pair_of(turns):  # the (fractional) pair that turns so often over the original context
            return rot / 2 * math.log(_ORIGINAL / (2 * math.pi * turns)) / math.log(10000.0)

        first, last = max(math.floor(pair_of(32.0)), 0), min(math.ceil(pair_of(1.0)), rot - 1)
        slow = ((pair - first) / max(last - first, 0.001)).clamp(0, 1)
        period, gain = period / (1 - slow * 7 / 8), 1.0 + math.log(8.0) / 10
    elif kind == "wavelength":
        keep = ((_ORIGINAL / period - 1) / 3).clamp(0, 1)
        period = period / (keep + (1 - keep) / 8)
    turns = positions[:, None] / period
    turns = (turns - turns.round()) * (2 * math.pi)
    return (gain * torch.cos(turns)).repeat(1, 2), (gain * torch.sin(turns)).repeat(1, 2)
