"""The residual stream of a transformer block and its rotary positions: operators, as they are measured.

Three operators, each in a plain form (elementary torch operations in 32 bits) and as calls of this package:

* ``residual``: a block's branch (normed, dropped out, gated, scaled) added to the residual stream, and the
                norm before the next block, in one pass (``fused_residual_rmsnorm``), with its gradients
* ``dropout``:  dropout from a counter-based generator, alone or with the residual sum (``fused_dropout``),
                with its gradients: the mask is made again, never stored
* ``axes``:     the rotation of queries and keys by positions of several axes (time, height, width):
                ``fused_rope`` and ``fused_qk_norm_rope`` with ``RoPEAxes``, with their gradients

A case is a dict of plain values; ``prepare`` makes its inputs, ``run`` is one pass.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4}
_EPS = 1e-6
_BASE = 10000.0


def _ops():
    """This repository's package (only reached where `own` is true)."""
    if "triton_ops" not in sys.modules:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "triton-fused-ops_b200"))
    import triton_ops

    return triton_ops


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _residual(name, batch, seq, hidden, dtype, stream, norm, gate, mod, p, scale, train=False):
    """`stream`: type of the residual stream; `norm`: the branch is normed; `gate`: none, hidden or sequence (its
    shape); `mod`: the norm's weight is one for all or, with a shift, one for each sequence."""
    return {"name": name, "op": "residual", "batch": batch, "seq": seq, "hidden": hidden, "dtype": dtype, "stream": stream,
            "norm": norm, "gate": gate, "mod": mod, "p": p, "scale": scale, "train": train}


def _dropout(name, rows, cols, dtype, p, add, train=False):
    return {"name": name, "op": "dropout", "rows": rows, "cols": cols, "dtype": dtype, "p": p, "add": add, "train": train}


def _axes(name, batch, seq, hq, hk, dim, sections, order, spectrum, layout, dtype, table, norm, train=False):
    return {"name": name, "op": "axes", "batch": batch, "seq": seq, "hq": hq, "hk": hk, "dim": dim,
            "sections": " ".join(map(str, sections)),
            "order": order, "spectrum": spectrum, "layout": layout, "dtype": dtype, "table": table, "norm": norm, "train": train}


def _sections(case):
    """Pairs of columns that each axis turns."""
    return [int(n) for n in case["sections"].split()]


def listed():
    return [
        # one new token of one request, norms on both sides of the block: latency is all
        _residual("residual single token", 1, 1, 4096, "bf16", "bf16", True, "none", "hidden", 0.0, 1.0),
        # one decode step of 64 requests, the branch scaled
        _residual("residual decode", 64, 1, 4096, "bf16", "bf16", False, "none", "hidden", 0.0, 0.25),
        # prefill of 8 prompts of 8192 tokens
        _residual("residual prefill", 8, 8192, 4096, "bf16", "bf16", True, "none", "hidden", 0.0, 1.0),
        # a training step: norms on both sides, dropout of the branch, both directions
        _residual("residual train", 2, 4096, 4096, "bf16", "bf16", True, "none", "hidden", 0.1, 1.0, True),
        # a training step of an image model: gate, weight and shift made for each sequence from its condition
        _residual("residual train per image", 16, 1025, 1152, "bf16", "bf16", False, "sequence", "sequence", 0.0, 1.0, True),
        # an odd width with a full-precision stream and a gate for each column, flattened prompts
        _residual("residual ragged f32 stream", 1, 1999, 1001, "f16", "f32", False, "hidden", "hidden", 0.0, 1.0),
        # the attention output of a small batch
        _dropout("dropout small", 64, 4096, "bf16", 0.1, False),
        # a training step over a block's output, added to the stream: both directions
        _dropout("dropout train", 8192, 4096, "bf16", 0.1, True, True),
        # an odd number of elements in full precision
        _dropout("dropout odd f32", 1999, 1001, "f32", 0.25, False, True),
        # one decode step of 64 requests about pictures: positions of time, height and width
        _axes("axes decode", 64, 1, 32, 8, 128, (16, 24, 24), "blocks", "shared", "half", "bf16", "f32", True),
        # a training step over pictures and text, the axes taking turns, with the norm of each head
        _axes("axes train", 2, 4096, 32, 8, 128, (24, 20, 20), "cycle", "shared", "half", "bf16", "f32", True, True),
        # one long clip, each axis with its own frequencies, neighbouring columns in pairs, as many key heads
        _axes("axes video", 1, 29999, 24, 24, 128, (8, 28, 28), "blocks", "own", "pairs", "bf16", "f32", False),
    ]


def _spread(rng, low, high):
    """An integer of [low, high], even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["residual", "residual", "residual", "dropout", "dropout", "axes", "axes"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    train = rng.random() < 0.5
    if op == "residual":
        hidden = _spread(rng, 48, 8192)
        if rng.random() < 0.75:  # most models are a multiple of 64 wide, some are not
            hidden = -(-hidden // 64) * 64
        batch = rng.choice([1, 1, 2, 3, 8, 32])
        rows = _spread(rng, 1, min(60000, 50_000_000 // hidden))
        gate = rng.choice(["none", "none", "hidden", "sequence"])
        c = _residual("", batch, max(1, rows // batch), hidden, dtype, rng.choice([dtype, dtype, "f32"]), rng.random() < 0.5, gate,
                      rng.choice(["hidden", "hidden", "sequence"]), rng.choice([0.0, 0.0, 0.1, 0.3]), rng.choice([1.0, 0.25, 0.7]), train)
    elif op == "dropout":
        cols = _spread(rng, 48, 8192)
        if rng.random() < 0.75:
            cols = -(-cols // 64) * 64
        c = _dropout("", _spread(rng, 1, min(60000, 30_000_000 // cols)), cols, dtype, rng.choice([0.05, 0.1, 0.25, 0.5]),
                     rng.random() < 0.5, train)
    else:
        dim, sections = rng.choice([(64, (8, 12, 12)), (64, (12, 10, 10)), (80, (8, 16, 16)), (128, (16, 24, 24)), (128, (24, 20, 20)),
                                    (128, (8, 28, 28)), (128, (16, 16, 16)), (128, (32, 32)), (96, (9, 20, 19)), (256, (44, 42, 42))])
        hk = rng.choice([1, 2, 3, 4, 8])
        hq = hk * rng.choice([1, 2, 4, 5])
        batch = rng.choice([1, 1, 2, 3, 5, 8])
        tokens = _spread(rng, 1, min(30000, 75_000_000 // ((hq + hk) * dim)))
        c = _axes("", batch, max(1, tokens // batch), hq, hk, dim, sections, rng.choice(["blocks", "cycle"]), rng.choice(["shared", "own"]),
                  rng.choice(["half", "half", "pairs"]), dtype, rng.choice(["f32", dtype]), rng.random() < 0.5, train)
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

    s = dict(case)
    dt = _DTYPES[case["dtype"]]
    # the generator's key: on the device, so that a captured step can be replayed with another one
    s["seed"] = torch.randint(2**62, (1,), device=dev, generator=g)
    if case["op"] == "residual":
        b, n, h = case["batch"], case["seq"], case["hidden"]
        wide = _DTYPES[case["stream"]]
        s["x"] = randn(b, n, h).to(dt)
        s["residual"] = (2 * randn(b, n, h)).to(wide)
        s["w1"] = 1 + 0.1 * randn(h) if case["norm"] else None
        s["gate"] = {"none": None, "hidden": 0.5 * randn(h), "sequence": 0.5 * randn(b, h)}[case["gate"]]
        s["w2"] = 1 + 0.1 * (randn(b, h) if case["mod"] == "sequence" else randn(h))
        s["shift"] = 0.2 * randn(b, h) if case["mod"] == "sequence" else None
        if case["train"]:
            s["gh"], s["gy"] = randn(b, n, h).to(wide), randn(b, n, h).to(dt)
        names = ["x", "residual", "w1", "gate", "w2", "shift"]
    elif case["op"] == "dropout":
        s["x"] = randn(case["rows"], case["cols"]).to(dt)
        s["residual"] = randn(case["rows"], case["cols"]).to(dt) if case["add"] else None
        if case["train"]:
            s["g"] = randn(case["rows"], case["cols"]).to(dt)
        names = ["x", "residual"]
    else:
        b, n, hq, hk, d = (case[k] for k in ("batch", "seq", "hq", "hk", "dim"))
        # queries and keys are the first columns of one fused projection's output
        qkv = randn(b, n, hq + 2 * hk, d).mul_(0.5 + 1.5 * torch.rand(d, device=dev, generator=g)).to(dt)
        s["q"], s["k"] = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
        s["w1"] = 1 + 0.1 * randn(d) if case["norm"] else None
        s["w2"] = 1 + 0.1 * randn(d) if case["norm"] else None
        freq = torch.tensor(_frequencies(case), dtype=torch.float64, device=dev)
        angle = torch.arange(max(n, 8192), device=dev, dtype=torch.float64)[:, None] * torch.cat([freq, freq])
        s["cos"], s["sin"] = angle.cos().to(_DTYPES[case["table"]]), angle.sin().to(_DTYPES[case["table"]])
        # frames in order (the first axis), any place in the picture (the others)
        first = torch.sort(torch.randint(max(n, 8192), (b, n), device=dev, generator=g), dim=-1).values
        place = torch.randint(96, (len(_sections(case)) - 1, b, n), device=dev, generator=g)
        s["positions"] = torch.cat([first[None], place])
        if case["train"]:
            s["gq"], s["gk"] = randn(b, n, hq, d).to(dt), randn(b, n, hk, d).to(dt)
        names = ["q", "k", "w1", "w2"]
    if case["train"]:
        s["leaves"] = {k: s[k].detach().requires_grad_() for k in names if s[k] is not None}
    return s


def _axis_of_pairs(case):
    """Which axis turns each pair of columns."""
    sections = _sections(case)
    if case["order"] == "blocks":
        return [a for a, n in enumerate(sections) for _ in range(n)]
    # the axes take turns; one that has all its pairs is passed over
    turns = sorted((k, a) for a, n in enumerate(sections) for k in range(n))
    return [a for _, a in turns]


def _frequencies(case):
    """Angle per position of each pair of columns."""
    axis = _axis_of_pairs(case)
    pairs = len(axis)
    if case["spectrum"] == "shared":
        return [_BASE ** (-i / pairs) for i in range(pairs)]
    # an axis' own frequencies: those of as many columns as it turns
    return [_BASE ** (-axis[:i].count(a) / _sections(case)[a]) for i, a in enumerate(axis)]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return {"residual": _run_residual, "dropout": _run_dropout, "axes": _run_axes}[state["op"]](state)


def _run_residual(s):
    if own:
        o = _ops()
        t = s["leaves"] if s["train"] else s
        out = o.fused_residual_rmsnorm(t["x"], t["residual"], t["w2"], t.get("gate"), branch_norm=s["norm"], branch_weight=t.get("w1"),
                                       shift=t.get("shift"), scale=s["scale"], eps=_EPS, dropout_p=s["p"], seed=s["seed"])
        if not s["train"]:
            return out
        return (*out, *torch.autograd.grad(out, list(t.values()), [s["gh"], s["gy"]]))
    dt, wide = s["x"].dtype, s["residual"].dtype
    x, res = s["x"].float(), s["residual"].float()
    gate, w1 = _per_row(s["gate"], 1.0), _per_row(s["w1"], 1.0)
    w2, shift = _per_row(s["w2"], 1.0), _per_row(s["shift"], 0.0)
    keep = s["scale"] * _keep(x.shape, s["p"], s["seed"]) if s["p"] else s["scale"]
    r1 = (x.square().mean(-1, keepdim=True) + _EPS).rsqrt() if s["norm"] else 1.0
    unit = x * r1
    h = res + unit * w1 * gate * keep
    r2 = (h.square().mean(-1, keepdim=True) + _EPS).rsqrt()
    hat = h * r2
    y = hat * w2 + shift
    if not s["train"]:
        return h.to(wide), y.to(dt)
    gh, gy = s["gh"].float(), s["gy"].float()
    g = gy * w2
    dh = gh + r2 * (g - hat * (g * hat).mean(-1, keepdim=True))
    du = dh * keep
    dunit = du * gate * w1
    dx = r1 * (dunit - unit * (dunit * unit).mean(-1, keepdim=True)) if s["norm"] else dunit
    grads = {"x": dx.to(dt), "residual": dh.to(wide), "w1": _total(du * gate * unit, s["w1"]),
             "gate": _total(du * unit * w1, s["gate"]), "w2": _total(gy * hat, s["w2"]), "shift": _total(gy, s["shift"])}
    return (h.to(wide), y.to(dt), *(grads[k] for k in s["leaves"]))


def _run_dropout(s):
    if own:
        o = _ops()
        t = s["leaves"] if s["train"] else s
        out = o.fused_dropout(t["x"], s["p"], s["seed"], residual=t.get("residual"))
        if not s["train"]:
            return out
        return (out, *torch.autograd.grad([out], list(t.values()), [s["g"]]))
    dt = s["x"].dtype
    keep = _keep(s["x"].shape, s["p"], s["seed"])
    out = s["x"].float() * keep
    out = (out + s["residual"].float() if s["add"] else out).to(dt)
    if not s["train"]:
        return out
    return (out, (s["g"].float() * keep).to(dt), *([s["g"]] if s["add"] else []))


def _run_axes(s):
    pairs = s["layout"] == "pairs"
    if own:
        o = _ops()
        axes = o.RoPEAxes(_sections(s), s["order"], s["spectrum"])
        t = s["leaves"] if s["train"] else s
        if s["norm"]:
            out = o.fused_qk_norm_rope(t["q"], t["k"], t["w1"], t["w2"], s["cos"], s["sin"], s["positions"], _EPS,
                                       interleaved=pairs, axes=axes)
        else:
            out = o.fused_rope(t["q"], t["k"], s["cos"], s["sin"], s["positions"], interleaved=pairs, axes=axes)
        if not s["train"]:
            return out
        return (*out, *torch.autograd.grad(out, list(t.values()), [s["gq"], s["gk"]]))
    dt = s["q"].dtype
    axis = torch.tensor(_axis_of_pairs(s), device=s["q"].device)
    at = s["positions"][axis].movedim(0, -1)  # [batch, seq, pairs]
    column = torch.arange(len(axis), device=at.device)
    c, n = (s[t][at, column][:, :, None].float() for t in ("cos", "sin"))
    (q, dq, dw1), (k, dk, dw2) = (
        _norm_rope(s[x].float(), s[w], c, n, pairs, s[g].float() if s["train"] else None)
        for x, w, g in (("q", "w1", "gq"), ("k", "w2", "gk")))
    if not s["train"]:
        return q.to(dt), k.to(dt)
    return (q.to(dt), k.to(dt), dq.to(dt), dk.to(dt), *([dw1, dw2] if s["norm"] else []))


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _per_row(t, otherwise):
    """A parameter as it multiplies [batch, seq, hidden]: [hidden], or [batch, 1, hidden] of one for each sequence."""
    return otherwise if t is None else t[:, None] if t.dim() == 2 else t


def _total(terms, like):
    """The gradient of a parameter that is shared by the rows."""
    if like is None:
        return None
    return terms.double().sum(1 if like.dim() == 2 else (0, 1)).float()


def _keep(shape, p, seed):
    """0, or 1 / (1 - p), for each element in order.

    Element i is dropped where word i % 4 of the block of counter i // 4 is below p 2^32. Blocks are those of a
    Philox generator of four 32-bit words and ten rounds (Salmon, Moraes, Dror and Shaw, "Parallel random numbers:
    as easy as 1, 2, 3", 2011) with the seed as its key.
    """
    count = math.prod(shape)
    low = 0xFFFFFFFF
    block = torch.arange(-(-count // 4), device=seed.device)
    a, b, c, d = block & low, block >> 32, torch.zeros_like(block), torch.zeros_like(block)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        x, y = a * 0xD2511F53, c * 0xCD9E8D57  # 64 bits that wrap: the words come out of them by shifts and masks
        a, b, c, d = ((y >> 32) & low) ^ b ^ k0, y & low, ((x >> 32) & low) ^ d ^ k1, x & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([a, b, c, d], dim=-1).flatten()[:count].view(shape)
    return (words >= round(p * 2**32)).float() * (1 / (1 - p))


def _rotate(x, c, n, pairs):
    rot = 2 * c.shape[-1]
    first, second = (x[..., 0:rot:2], x[..., 1:rot:2]) if pairs else (x[..., :rot // 2], x[..., rot // 2:rot])
    y = first * c - second * n, first * n + second * c
    y = torch.stack(y, dim=-1).flatten(-2) if pairs else torch.cat(y, dim=-1)
    return torch.cat([y, x[..., rot:]], dim=-1)


def _norm_rope(x, w, c, n, pairs, grad):
    """The heads, normed where there is a weight, rotated and, with `grad`, the gradients of x and w."""
    inv, w = (1.0, 1.0) if w is None else ((x.square().mean(-1, keepdim=True) + _EPS).rsqrt(), w)
    unit = x * inv
    out = _rotate(unit * w, c, n, pairs)
    if grad is None:
        return out, None, None
    back = _rotate(grad, c, -n, pairs)  # the inverse rotation
    if not torch.is_tensor(w):
        return out, back, None
    dunit = back * w
    dx = inv * (dunit - unit * (dunit * unit).mean(-1, keepdim=True))
    return out, dx, (back * unit).double().sum((0, 1, 2)).float()


# ---------------------------------------------------------------------------
# sizes and 64-bit results
# ---------------------------------------------------------------------------
def work(case):
    esize = _BYTES[case["dtype"]]
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        # both directions: x, the stream and its sum, the gradient and x's (the stream's is the gradient itself)
        tensors = (3 if case["add"] else 2) + (2 if case["train"] else 0)
        return {"bytes": esize * n * tensors, "flops": 2 * n * (2 if case["train"] else 1)}
    if case["op"] == "residual":
        n, wide = case["batch"] * case["seq"] * case["hidden"], _BYTES[case["stream"]]
        params = 4 * case["hidden"] * (case["norm"] + {"none": 0, "hidden": 1, "sequence": case["batch"]}[case["gate"]]
                                       + (2 * case["batch"] if case["mod"] == "sequence" else 1))
        # forward: x and the stream, the sum and the normed row; backward: the two again, two gradients in, two out
        return {"bytes": n * 2 * (esize + wide) + params + (n * 3 * (esize + wide) + 2 * params if case["train"] else 0),
                "flops": n * (12 + (24 if case["train"] else 0))}
    tokens = case["batch"] * case["seq"]
    values = tokens * (case["hq"] + case["hk"]) * case["dim"]
    rot, axes = 2 * sum(_sections(case)), len(_sections(case))
    rows = min(tokens, max(case["seq"], 8192))
    moved = 2 if not case["train"] else 5 if case["norm"] else 4
    return {"bytes": moved * esize * values + rows * rot * _BYTES[case["table"]] + 8 * axes * tokens,
            "flops": values * (8 if case["norm"] else 3) * moved / 2}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "dropout":
        keep = _exact_keep(s["x"].shape, case["p"], int(s["seed"]))
        out = s["x"].double() * keep
        out = out + s["residual"].double() if case["add"] else out
        return out if not case["train"] else (out, s["g"].double() * keep, *([s["g"].double()] if case["add"] else []))
    leaves = {k: v.detach().double().requires_grad_() for k, v in s["leaves"].items()} if case["train"] else \
             {k: s[k].double() for k in ("x", "residual", "q", "k", "w1", "gate", "w2", "shift") if s.get(k) is not None}

    def normed(x):
        longer = torch.cat([x, torch.full_like(x[..., :1], math.sqrt(_EPS * x.shape[-1]))], -1)
        return x / torch.linalg.vector_norm(longer, dim=-1, keepdim=True) * math.sqrt(x.shape[-1])

    if case["op"] == "residual":
        wide = (case["batch"], 1, case["hidden"])

        def param(k, otherwise):
            if k not in leaves:
                return otherwise
            return leaves[k].view(wide) if leaves[k].dim() == 2 else leaves[k]

        branch = normed(leaves["x"]) * param("w1", 1.0) if case["norm"] else leaves["x"]
        if case["p"]:
            branch = branch * _exact_keep(branch.shape, case["p"], int(s["seed"]))
        h = leaves["residual"] + case["scale"] * param("gate", 1.0) * branch
        out, given = (h, torch.addcmul(param("shift", torch.zeros((), device=h.device, dtype=h.dtype)), normed(h), param("w2", 1.0))), ("gh", "gy")
    else:
        axis = _axis_of_pairs(case)
        half = len(axis)
        turn = torch.stack([torch.complex(s["cos"][s["positions"][a], i].double(), s["sin"][s["positions"][a], i].double())
                            for i, a in enumerate(axis)], -1)[:, :, None]

        def forward(x, w):
            if case["norm"]:
                x = normed(x) * w
            head = x[..., :2 * half]
            z = head.unflatten(-1, (half, 2)) if case["layout"] == "pairs" else head.unflatten(-1, (2, half)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
            z = z if case["layout"] == "pairs" else z.transpose(-1, -2)
            return torch.cat([z.flatten(-2), x[..., 2 * half:]], dim=-1)

        out, given = (forward(leaves["q"], leaves.get("w1")), forward(leaves["k"], leaves.get("w2"))), ("gq", "gk")
    if not case["train"]:
        return out
    grads = torch.autograd.grad(out, list(leaves.values()), [s[g].double() for g in given])
    return tuple(t.detach() for t in (*out, *grads))


def _exact_keep(shape, p, seed):
    """The plain form's factors from whole numbers of the host."""
    count = math.prod(shape)
    word = np.uint64(0xFFFFFFFF)
    block = np.arange(-(-count // 4), dtype=np.uint64)
    state = [block & word, block >> np.uint64(32), np.zeros_like(block), np.zeros_like(block)]
    key = [seed % 2**32, seed // 2**32]
    for turn in range(10):
        first, third = state[0] * np.uint64(0xD2511F53), state[2] * np.uint64(0xCD9E8D57)
        keys = [np.uint64((key[0] + turn * 0x9E3779B9) % 2**32), np.uint64((key[1] + turn * 0xBB67AE85) % 2**32)]
        state = [third // np.uint64(2**32) ^ state[1] ^ keys[0], third & word,
                 first // np.uint64(2**32) ^ state[3] ^ keys[1], first & word]
    dropped = np.stack(state, axis=1).reshape(-1)[:count] < np.uint64(round(p * 2**32))
    return torch.from_numpy(np.where(dropped, 0.0, 1.0 / (1.0 - p))).to("cuda").view(shape)
