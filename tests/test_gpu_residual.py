"""fused_residual_rmsnorm on the GPU against the formulas in 64 bits.

Error bounds, from the kernels' fp32 arithmetic on the given inputs (one
rounding is u = 2^-24 relative, a result's own rounding eps/2 of its type):

* 1 / sqrt(mean + eps): a row's sum of squares is at most 80 additions of
  positive terms one after the other, halved by the root, rsqrtf within 2 ulp,
  the mean and eps: R = 2^-18
* h: the branch's factors, R + 6 u of it, and the sum's rounding
* y: the error of h times the factors, and of 1/rms: R and the row's mean error of h
* dH, dx: the same errors through their formulas; sums over a row add at most
  K = 100 roundings of the terms' magnitudes
* parameters: the terms' errors, and the roundings of a run of at most 2048 rows
"""

import math

import pytest
import torch

from triton_ops.kernels.dropout import dropout_keep_reference

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-133, torch.float32: 2.0**-149}
U, R, K = 2.0**-24, 2.0**-18, 100
EPS = 1e-5
NAMES = ("x", "residual", "branch_weight", "gate", "weight", "shift")


def check(got, ref, slack, what):
    """|got - ref| <= the result's rounding + slack, NaN and infinity in the same places."""
    assert got.shape == ref.shape, what
    g = got.double()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(g), torch.isnan(ref)), what
    assert torch.equal(g[~fine].nan_to_num(0.5), ref[~fine].nan_to_num(0.5)), what
    bound = (ref.abs() + slack) * (torch.finfo(got.dtype).eps / 2) * 1.01 + TINY[got.dtype] + slack
    over = ((g - ref).abs() - bound)[fine]
    assert over.numel() == 0 or over.max().item() <= 0, f"{what}: {over.max().item():.3e} over the bound"


def formulas(t, branch_norm, scale, keep=None, p=0.0, gh=None, gy=None):
    """{name: (value, slack)} of the outputs and, with gh or gy, the gradients; t: the inputs by name."""
    d = {k: None if v is None else v.double() for k, v in t.items()}
    x, res = d["x"], d["residual"]
    batch = x.shape[0] if x.dim() > 1 else 1

    def rows(v):
        return 1.0 if v is None else v if v.dim() == 1 else v.reshape(batch, *(1,) * (x.dim() - 2), x.shape[-1])

    def mean(v):
        return v.mean(-1, keepdim=True)

    w1, gate, w2 = rows(d["branch_weight"]), rows(d["gate"]), rows(d["weight"])
    shift = 0.0 if d["shift"] is None else rows(d["shift"])
    factor = scale / (1 - p)
    kept = torch.ones_like(x) if keep is None else keep.double()
    r1 = 1 / torch.sqrt(mean(x * x) + EPS) if branch_norm else torch.ones_like(x[..., :1])
    e1 = R if branch_norm else 0.0
    unit, c = x * r1, w1 * gate * factor * torch.ones_like(x)
    u = kept * unit * c
    h = res + u
    eh = u.abs() * (e1 + 6 * U) + U * h.abs()
    r2 = 1 / torch.sqrt(mean(h * h) + EPS)
    e2 = R + mean(eh * eh).sqrt() * r2
    hat = h * r2
    y = hat * w2 + shift
    ehat = r2 * eh + hat.abs() * (e2 + 2 * U)
    wabs = w2.abs() if torch.is_tensor(w2) else w2
    out = {"h": (h, eh), "y": (y, ehat * wabs + 2 * U * (hat * w2).abs() + U * y.abs())}
    if gh is None and gy is None:
        return out
    dh = torch.zeros_like(h) if gh is None else gh.double()
    dy = torch.zeros_like(h) if gy is None else gy.double()
    g = dy * w2
    m = mean(g * hat)
    em = mean(g.abs() * ehat) + K * U * mean((g * hat).abs())
    dH = dh + r2 * (g - hat * m)
    size = dh.abs() + r2 * (g.abs() + (hat * m).abs())
    edH = r2 * (g.abs() * (e2 + 4 * U) + hat.abs() * em + ehat * m.abs() + (hat * m).abs() * (e2 + 6 * U)) + 4 * U * size
    e = kept * dH
    m1 = mean(u * dH)
    em1 = mean(u.abs() * edH) + (e1 + e2 + (K + 10) * U) * mean(u.abs() * size)
    if branch_norm:
        dx = r1 * (c * e - unit * m1)
        edx = r1 * ((c * e).abs() * (e1 + 8 * U) + c.abs() * edH + unit.abs() * em1 + (unit * m1).abs() * (2 * e1 + 8 * U))
    else:
        dx = c * e
        edx = (c * e).abs() * 8 * U + c.abs() * edH
    out["x"], out["residual"] = (dx, edx), (dH, edH)
    per = x.shape[1:-1].numel() if x.dim() > 1 else 1
    run = min(2048, x.numel() // x.shape[-1]) + 20

    def total(name, term, slack):
        v = t[name]
        if v is None:
            return
        own = v.dim() > 1
        shape = (batch, per, x.shape[-1])
        slack = slack + run * U * term.abs()
        term, slack = (torch.broadcast_to(q, x.shape).reshape(shape).sum(1 if own else (0, 1)).view(v.shape) for q in (term, slack))
        out[name] = term, slack

    a, ea = e * unit * factor, (e * unit * factor).abs() * (e1 + 4 * U) + (kept * unit * factor).abs() * edH
    wide = [torch.abs(torch.as_tensor(v, device=x.device)) for v in (w1, gate)]
    total("gate", a * w1, ea * wide[0] + 4 * U * (a * w1).abs())
    total("branch_weight", a * gate, ea * wide[1] + 4 * U * (a * gate).abs())
    total("weight", dy * hat, dy.abs() * ehat + 2 * U * (dy * hat).abs())
    total("shift", dy, torch.zeros_like(dy))
    return out


def randn(shape, dtype, seed, offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = math.prod(shape)
    return torch.randn(n + offset, device="cuda", generator=g).to(DT[dtype])[offset:].view(shape)


def make(shape, dtype, stream, branch_weight=None, gate=None, weight="f32", shift=None, per="", seed=0, offset=0):
    """Inputs by name; parameters by dtype (None: not there), those named in `per` one for each sequence."""
    hidden = shape[-1]

    def param(kind, name, at):
        if kind is None:
            return None
        return (0.5 + randn((shape[0], hidden) if name in per else (hidden,), "f32", seed + at)).to(DT[kind])

    return {"x": randn(shape, dtype, seed + 1, offset), "residual": 2 * randn(shape, stream, seed + 2, offset),
            "branch_weight": param(branch_weight, "branch_weight", 3), "gate": param(gate, "gate", 4),
            "weight": param(weight, "weight", 5), "shift": param(shift, "shift", 6)}


def run(t, branch_norm=False, scale=1.0, p=0.0, seed=7, gh=None, gy=None, offset=0, norm=True):
    """The op's outputs and gradients by name."""
    from triton_ops import fused_residual_rmsnorm

    leaves = {k: v.detach().requires_grad_() for k, v in t.items() if v is not None}
    grads = gh is not None or gy is not None
    given = leaves if grads else t
    h, y = fused_residual_rmsnorm(given["x"], given["residual"], given.get("weight"), given.get("gate"), branch_norm=branch_norm,
                                  branch_weight=given.get("branch_weight"), shift=given.get("shift"), scale=scale, eps=EPS,
                                  dropout_p=p, seed=seed, dropout_offset=offset, norm=norm)
    got = {"h": h, "y": y}
    if grads:
        pairs = [(o, g) for o, g in ((h, gh), (y, gy)) if g is not None]
        got |= dict(zip(leaves, torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [g for _, g in pairs],
                                                    allow_unused=True)))
    return got


def compare(t, got, want, what):
    for name, (ref, slack) in want.items():
        if got.get(name) is None:
            continue
        kind = {"h": t["residual"], "y": t["x"]}.get(name, t.get(name))
        assert got[name].dtype == kind.dtype
        check(got[name], ref, slack, f"{what}: {name}")


# shape, dtype, stream, options of make(), branch_norm, scale, p
CASES = [
    ((1, 1, 4096), "bf16", "bf16", dict(branch_weight="f32"), True, 1.0, 0.0),
    ((64, 1, 4096), "bf16", "bf16", dict(branch_weight="bf16", weight="bf16"), True, 0.25, 0.0),
    ((3, 5, 64), "f16", "f16", dict(gate="f16", weight="f16"), False, 1.0, 0.0),
    ((2, 7, 80), "f16", "f32", dict(branch_weight="f32", gate="f32", shift="f32", per="gate shift"), True, 1.0, 0.1),
    ((4, 9, 1152), "bf16", "bf16", dict(gate="f32", shift="f32", per="gate weight shift"), False, 1.0, 0.0),
    ((4, 300, 136), "bf16", "f32", dict(branch_weight="bf16", gate="bf16", shift="bf16", per="branch_weight weight"), True, 0.7, 0.3),
    ((2, 3, 4104), "bf16", "bf16", dict(branch_weight="f32", gate="f32"), True, 1.0, 0.1),      # two chunks a thread
    ((1, 300, 8192), "bf16", "f32", dict(branch_weight="f32"), True, 1.0, 0.0),
    ((5, 2, 2560), "f32", "f32", dict(branch_weight="f32", gate="f32", shift="f16", per="gate"), True, 1.5, 0.25),
    ((1, 200, 6000), "f32", "f32", dict(gate="f32"), False, 1.0, 0.0),
    ((2, 2, 8200), "f32", "f32", dict(branch_weight="f32"), True, 1.0, 0.5),                     # any width
    ((1, 3, 16384), "f16", "f16", dict(branch_weight="f32", shift="f32"), True, 1.0, 0.1),       # four chunks, any backward
    ((700, 16640), "bf16", "bf16", dict(gate="f32"), True, 1.0, 0.0),                            # any width, both ways
    ((3, 1001), "f16", "f32", dict(gate="f16", shift="bf16"), False, 1.0, 0.1),                  # odd widths
    ((2, 150, 1999), "bf16", "bf16", dict(branch_weight="f32", gate="f32", per="gate"), True, 0.5, 0.2),
    ((2, 3, 2049), "f32", "f32", dict(branch_weight="f32", weight="f16"), True, 1.0, 0.0),
    ((2, 3, 4097), "f16", "f16", dict(branch_weight="f32"), True, 1.0, 0.1),                     # any width, odd
    ((6, 1), "f32", "f32", dict(gate="f32"), False, 1.0, 0.0),
    ((2, 2, 2, 12), "f32", "f32", dict(branch_weight="f32", gate="f32", per="gate"), True, 1.0, 0.0),
    ((5, 33), "bf16", "f32", dict(weight=None), False, 1.0, 0.0),
    ((17,), "f16", "f16", dict(gate="f32", shift="f32"), True, 1.0, 0.0),
    ((3000, 48), "f32", "f32", dict(branch_weight="f32", gate="f32", shift="f32", per="gate"), True, 1.0, 0.1),  # a gate for each row
    ((2, 5000, 256), "bf16", "bf16", dict(branch_weight="f32", gate="f32", shift="f32"), True, 1.0, 0.0),
    ((40, 130, 512), "f16", "f16", dict(gate="f32", shift="f32", per="gate weight shift"), True, 1.0, 0.1),
]


@pytest.mark.parametrize("extension", [True, False])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{'x'.join(map(str, c[0]))}-{c[1]}-{c[2]}")
def test_against_formulas(cuda, monkeypatch, case, extension):
    from triton_ops import _lib

    if not extension:
        monkeypatch.setattr(_lib, "ext", lambda: None)
    shape, dtype, stream, options, branch_norm, scale, p = case
    t = make(shape, dtype, stream, **options)
    keep = dropout_keep_reference(shape, p, 7, 3, "cuda") if p else None
    got = run(t, branch_norm, scale, p, 7, offset=3)
    assert not got["h"].requires_grad and got["h"].is_contiguous() and got["y"].is_contiguous()
    compare(t, got, formulas(t, branch_norm, scale, keep, p), "serving")
    gh, gy = randn(shape, stream, 11), randn(shape, dtype, 12)
    both = run(t, branch_norm, scale, p, torch.tensor([7], device="cuda"), gh, gy, offset=3)
    compare(t, both, formulas(t, branch_norm, scale, keep, p, gh, gy), "training")
    assert torch.equal(both["h"], got["h"]) and torch.equal(both["y"], got["y"])
    again = run(t, branch_norm, scale, p, 7, gh, gy, offset=3)
    assert all(torch.equal(again[k], both[k]) for k in both if both[k] is not None)
    for one in (dict(gh=gh), dict(gy=gy)):  # the gradient of one output alone
        compare(t, run(t, branch_norm, scale, p, 7, offset=3, **one), formulas(t, branch_norm, scale, keep, p, **one), "one output")


def test_without_the_norm(cuda):
    from triton_ops import fused_residual_rmsnorm

    t = make((3, 40, 72), "bf16", "f32", branch_weight="f32", gate="f32", weight=None)
    gh = randn((3, 40, 72), "f32", 11)
    got = run(t, True, 0.5, 0.2, gh=gh, norm=False)
    assert got["y"] is None
    want = formulas(t, True, 0.5, dropout_keep_reference((3, 40, 72), 0.2, 7, 0, "cuda"), 0.2, gh=gh)
    compare(t, got, want, "h alone")
    with torch.no_grad():
        assert fused_residual_rmsnorm(t["x"], t["residual"], norm=False)[1] is None


@pytest.mark.parametrize("extension", [True, False])
def test_strides(cuda, monkeypatch, extension):
    """Columns of wider rows, transposed and expanded tensors, unaligned starts, parts of one conditioning projection."""
    from triton_ops import _lib

    if not extension:
        monkeypatch.setattr(_lib, "ext", lambda: None)
    b, s, h = 3, 20, 64
    wide = randn((b, s, 3 * h), "bf16", 1)
    swapped = randn((s, b, h), "bf16", 2).transpose(0, 1)
    conditions = randn((b, 1, 4 * h), "f32", 3)
    cases = {
        "columns": dict(x=wide[..., h:2 * h], residual=wide[..., 2 * h:]),
        "odd columns": dict(x=wide[..., 1:h + 1], residual=wide[..., 5:h + 5]),
        "transposed": dict(x=swapped, residual=randn((b, s, h), "bf16", 4)),
        "every second": dict(x=wide[..., ::3], residual=wide[..., ::3]),
        "expanded": dict(x=randn((1, 1, h), "bf16", 5).expand(b, s, h), residual=randn((b, 1, h), "bf16", 6).expand(b, s, h)),
        "steps": dict(x=wide[:, ::2, :h], residual=wide[:, 1::2, :h]),
    }
    params = {
        "parts": dict(gate=conditions[..., :h], weight=conditions[..., h:2 * h], shift=conditions[..., 2 * h:3 * h]),
        "odd parts": dict(gate=conditions[:, 0, 1:h + 1], weight=conditions[:, 0, 3:h + 3]),
        "expanded": dict(gate=conditions[:1, 0, :h].expand(b, h), branch_weight=conditions[0, 0, :1].expand(h)),
    }
    for name, t in cases.items():
        for kind, more in params.items():
            full = {k: t.get(k, more.get(k)) for k in NAMES}
            norm = full["branch_weight"] is not None
            shape = full["x"].shape
            gh = randn((shape[-1], *shape[:-1]), "bf16", 7).movedim(0, -1)  # a transposed gradient
            gy = randn((1,), "bf16", 8).expand(shape)
            got = run(full, norm, 1.0, 0.0, 7, gh, gy)
            compare(full, got, formulas(full, norm, 1.0, gh=gh, gy=gy), f"{name}, {kind}")


@pytest.mark.parametrize("shape", [(0, 64), (2, 0, 64), (0, 3, 64)])
@pytest.mark.parametrize("extension", [True, False])
def test_no_rows(cuda, monkeypatch, shape, extension):
    from triton_ops import _lib

    if not extension:
        monkeypatch.setattr(_lib, "ext", lambda: None)
    t = make(shape, "bf16", "f32", branch_weight="f32", gate="f32", shift="f32", per="gate")
    got = run(t, True, 1.0, 0.1, 7, randn(shape, "f32", 1), randn(shape, "bf16", 2))
    assert got["h"].shape == got["y"].shape == shape
    for name in NAMES:
        assert got[name].shape == t[name].shape and (got[name] == 0).all()


def test_some_inputs_want_gradients(cuda):
    """Each input alone, and all but one: the same gradients as together."""
    from triton_ops import fused_residual_rmsnorm

    shape = (2, 30, 96)
    t = make(shape, "f16", "f32", branch_weight="f32", gate="f16", shift="f32", per="gate")
    gh, gy = randn(shape, "f32", 1), randn(shape, "f16", 2)
    every = run(t, True, 0.5, 0.1, 7, gh, gy)
    for chosen in [(n,) for n in NAMES] + [tuple(m for m in NAMES if m != n) for n in NAMES]:
        v = {k: x.detach().requires_grad_(k in chosen) for k, x in t.items()}
        out = fused_residual_rmsnorm(v["x"], v["residual"], v["weight"], v["gate"], branch_norm=True, eps=EPS, scale=0.5,
                                     branch_weight=v["branch_weight"], shift=v["shift"], dropout_p=0.1, seed=7)
        grads = torch.autograd.grad(out, [v[n] for n in chosen], [gh, gy])
        assert all(torch.equal(g, every[n]) for n, g in zip(chosen, grads))


@pytest.mark.parametrize("hidden", [512, 777, 20000])
def test_values_at_the_borders(cuda, hidden):
    """Zero rows, infinities and NaN in rows and at dropped places, rows that cancel."""
    p, seed = 0.5, 5
    t = make((8, hidden), "f32", "f32", branch_weight="f32")
    keep = dropout_keep_reference((8, hidden), p, seed, 0, "cuda")
    x, res = t["x"], t["residual"]
    x[0] = 0
    res[0] = 0
    x[1] = 0
    res[2, 3] = float("inf")
    res[3, 4] = float("nan")
    x[4, 5] = float("inf")
    x[6] *= 1e15
    got = run(t, True, 1.0, p, seed, torch.ones_like(x), torch.ones_like(x))
    fine = [0, 1, 5, 6, 7]
    part = {k: v if v is None or v.dim() == 1 else v[fine] for k, v in t.items()}
    want = formulas(part, True, 1.0, keep[fine], p, torch.ones_like(x[fine]), torch.ones_like(x[fine]))
    for name in ("h", "y", "x", "residual"):
        check(got[name][fine], *want[name], name)
        for row in (0, 1, 5, 6, 7):
            assert torch.isfinite(got[name][row]).all()
    # an infinite element of the stream: h has it, its row's y is 0 beside it and NaN there
    assert got["h"][2, 3] == float("inf") and torch.isfinite(got["h"][2]).sum() == hidden - 1
    assert torch.isnan(got["y"][2, 3]) and (got["y"][2, 4:] == 0).all()
    assert torch.isnan(got["y"][3]).all() and torch.isnan(got["h"][3]).sum() == 1
    # without the branch norm a dropped element is zero whatever it was
    at = (~keep[7]).nonzero()[:2, 0]
    x[7, at[0]], x[7, at[1]] = float("inf"), float("nan")
    t["branch_weight"] = None
    h = run(t, False, 1.0, p, seed)["h"]
    assert torch.equal(h[7, at], res[7, at])
    # x and residual that cancel: h is exactly zero
    both = make((4, hidden), "bf16", "bf16")
    both["residual"] = -both["x"]
    got = run(both, False)
    assert (got["h"] == 0).all() and (got["y"] == 0).all()


@pytest.mark.parametrize("hidden", [200, 512, 777, 4400, 20000])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_dropped_infinities_leave_no_trace(cuda, dtype, hidden):
    """Without the branch norm what lies at dropped places changes nothing, the gate's gradient included."""
    shape, p, seed = (2, 30, hidden), 0.5, 5
    t = make(shape, dtype, dtype, gate="f32", shift="f32")
    dropped = ~dropout_keep_reference(shape, p, seed, 0, "cuda")
    gh, gy = randn(shape, dtype, 11), randn(shape, dtype, 12)
    want = run(t, False, 0.7, p, seed, gh, gy)
    t["x"] = torch.where(dropped, torch.tensor([float("inf"), float("nan")] * (hidden // 2) + [-1.0] * (hidden % 2), device="cuda"),
                         t["x"]).to(DT[dtype])
    got = run(t, False, 0.7, p, seed, gh, gy)
    assert all(torch.equal(got[k], want[k]) for k in want if want[k] is not None)


@pytest.mark.parametrize("dtype,stream,hidden", [
    ("bf16", "bf16", 33), ("f16", "f16", 1001), ("f16", "f32", 1001), ("f32", "f32", 1002), ("bf16", "bf16", 4101),
    ("bf16", "f32", 4101), ("f32", "f32", 4103), ("f16", "f16", 6001), ("bf16", "bf16", 8192), ("f32", "f32", 8000),
])
def test_every_alignment(cuda, dtype, stream, hidden):
    """Rows that start anywhere in a vector, x and the stream at different places of theirs."""
    from triton_ops import fused_residual_rmsnorm

    shape = (2, 9, hidden)
    params = make(shape, dtype, stream, branch_weight="f32", gate="bf16", shift="f32", per="gate")
    keep = dropout_keep_reference(shape, 0.2, 7, 0, "cuda")
    for start in range(8):
        t = {**params, "x": randn(shape, dtype, 1, start), "residual": randn(shape, stream, 2, (3 * start + 1) % 8)}
        gh, gy = randn(shape, stream, 11, (5 * start + 2) % 8), randn(shape, dtype, 12, 7 - start)
        got = run(t, True, 0.7, 0.2, 7, gh, gy)
        compare(t, got, formulas(t, True, 0.7, keep, 0.2, gh, gy), f"start {start}")
        with torch.no_grad():  # a tensor beside the rows is not written
            h, y = fused_residual_rmsnorm(t["x"], t["residual"], t["weight"], t["gate"], branch_norm=True, scale=0.7, eps=EPS,
                                          branch_weight=t["branch_weight"], shift=t["shift"], dropout_p=0.2, seed=7)
        assert torch.equal(h, got["h"]) and torch.equal(y, got["y"])


@pytest.mark.parametrize("dtype,stream,rows,hidden", [
    ("bf16", "bf16", 30000, 4096), ("bf16", "f32", 8000, 4096), ("f32", "f32", 7500, 2560), ("f16", "f16", 3000, 1024),
])
def test_groups_with_many_rows(cuda, dtype, stream, rows, hidden):
    t = make((rows, hidden), dtype, stream, branch_weight="f32")
    at = torch.cat([torch.arange(200), torch.arange(rows // 2, rows // 2 + 200), torch.arange(rows - 900, rows)]).cuda()
    part = {k: v if v is None or v.dim() == 1 else v[at] for k, v in t.items()}
    got = run(t, True)
    compare(part, {k: v[at] for k, v in got.items()}, formulas(part, True, 1.0), "many rows")


def test_captured_beside_an_eager_graph(cuda):
    """A step captured, through leaves of its own, while an eager graph of the same memory waits for its backward pass.

    (torch itself refuses the capture of a backward pass whose leaves an eager graph holds.)
    """
    from triton_ops import fused_dropout, fused_residual_rmsnorm

    x, res = (randn((64, 520), "bf16", i).requires_grad_() for i in (1, 2))
    w = torch.ones(520, device="cuda", requires_grad=True)
    seed = torch.tensor([3], device="cuda")
    eager_leaves = (x, res, w)

    def loss(x, res, w):
        h, y = fused_residual_rmsnorm(x, res, w, branch_norm=True, dropout_p=0.1, seed=seed)
        return fused_dropout(y, 0.2, seed, offset=1, residual=h).float().sum()

    want = torch.autograd.grad(loss(*eager_leaves), eager_leaves)
    eager = loss(*eager_leaves)
    leaves = [t.detach().requires_grad_() for t in eager_leaves]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(loss(*leaves), leaves)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = torch.autograd.grad(loss(*leaves), leaves)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, want))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(eager, eager_leaves), want))


def test_gradients_against_differences(cuda):
    """Central differences of the fp32 op's own formula in 64 bits, along random directions."""
    from triton_ops.kernels.residual import residual_rmsnorm_reference

    shape, p, seed, scale = (3, 4, 24), 0.25, 9, 0.7
    t = make(shape, "f32", "f32", branch_weight="f32", gate="f32", shift="f32", per="gate shift")
    gh, gy = randn(shape, "f32", 1), randn(shape, "f32", 2)
    got = run(t, True, scale, p, seed, gh, gy)
    keep = dropout_keep_reference(shape, p, seed, 0, "cuda")

    def value(v):
        h, y = residual_rmsnorm_reference(v["x"], v["residual"], v["weight"], v["gate"], branch_norm=True, scale=scale, eps=EPS,
                                          branch_weight=v["branch_weight"], shift=v["shift"], keep=keep, dropout_p=p)
        return (h * gh.double()).sum() + (y * gy.double()).sum()

    step = 1e-5
    for name in NAMES:
        wide = {k: v.double() for k, v in t.items()}
        way = randn(t[name].shape, "f32", 3).double()
        up, down = ({**wide, name: wide[name] + s * step * way} for s in (1, -1))
        slope = (value(up) - value(down)) / (2 * step)
        along = (got[name].double() * way).sum()
        # the difference's own error: step^2 and 2^-53 of the sums over the step; the gradient's: fp32
        assert abs(slope - along) <= 1e-5 * (got[name].double() * way).abs().sum(), name


def test_differentiable_once(cuda, monkeypatch):
    from triton_ops import _lib, fused_residual_rmsnorm

    for extension in (True, False):
        if not extension:
            monkeypatch.setattr(_lib, "ext", lambda: None)
        x, res = (randn((2, 3, 16), "f32", i).requires_grad_() for i in (1, 2))
        h, y = fused_residual_rmsnorm(x, res)
        (dx,) = torch.autograd.grad(y.pow(2).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(dx.sum(), x)


def test_changed_inputs_are_noticed(cuda, monkeypatch):
    """autograd's error where a tensor that the backward pass reads was written to, the seed among them."""
    from triton_ops import _lib, fused_residual_rmsnorm

    for extension in (True, False):
        if not extension:
            monkeypatch.setattr(_lib, "ext", lambda: None)
        for which in ("x", "residual", "seed"):
            v = {"x": randn((2, 16), "f32", 1), "residual": randn((2, 16), "f32", 2), "seed": torch.tensor([3], device="cuda")}
            leaf = v["x"].clone().requires_grad_()
            x = leaf * 1
            out = fused_residual_rmsnorm(x, v["residual"], dropout_p=0.5, seed=v["seed"])
            with torch.no_grad():
                (x if which == "x" else v[which]).add_(1)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(out[1].sum(), leaf)


def test_streams_and_graphs(cuda):
    """A side stream, and two captured steps replayed on new inputs and seeds."""
    from triton_ops import fused_residual_rmsnorm

    side = torch.cuda.Stream()
    shape = (2, 40, 264)

    def inputs(seed):
        t = make(shape, "bf16", "bf16", branch_weight="f32", gate="f32", shift="f32", per="gate", seed=100 * seed)
        return [*t.values(), randn(shape, "bf16", 50 + seed), randn(shape, "bf16", 60 + seed), torch.tensor([seed], device="cuda")]

    def leaves(t):
        return [x.clone().requires_grad_(i < 6) for i, x in enumerate(t)]

    def step(x, res, bw, gate, w, shift, gh, gy, seed):
        out = fused_residual_rmsnorm(x, res, w, gate, branch_norm=True, branch_weight=bw, shift=shift, dropout_p=0.1, seed=seed)
        return (*out, *torch.autograd.grad(out, [x, res, bw, gate, w, shift], [gh, gy]))

    plain = {seed: [t.detach() for t in step(*leaves(inputs(seed)))] for seed in (1, 2, 3)}
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = step(*leaves(inputs(1)))
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, plain[1]))
    graphs = []
    for seed in (1, 2):
        static = leaves(inputs(seed))
        with torch.cuda.stream(side):
            step(*static)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(*static)
        graphs.append((graph, static, out))
    for seed in (3, 1, 2):
        new = inputs(seed)
        for _, static, _ in graphs:
            with torch.no_grad():
                for a, b in zip(static, new):
                    a.copy_(b)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for (graph, _, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, plain[seed]))


def test_module(cuda):
    from triton_ops import FusedResidualRMSNorm, fused_residual_rmsnorm

    m = FusedResidualRMSNorm(64, branch_norm=True, layer_scale=0.1, dropout=0.2, dropout_seed=5).cuda()
    x, res = randn((2, 8, 64), "bf16", 1), randn((2, 8, 64), "bf16", 2)
    h, y = m(x, res)
    want = fused_residual_rmsnorm(x, res, m.weight, m.gate, branch_norm=True, branch_weight=m.branch_weight, dropout_p=0.2, seed=5)
    assert torch.equal(h, want[0]) and torch.equal(y, want[1]) and m.seed.item() == 6
    (h.float().sum() + y.float().sum()).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
    assert not torch.equal(m(x, res)[0], h)
    m.eval()
    h, y = m(x, res)
    want = fused_residual_rmsnorm(x, res, m.weight, m.gate, branch_norm=True, branch_weight=m.branch_weight)
    assert torch.equal(h, want[0]) and torch.equal(y, want[1]) and m.seed.item() == 7
    plain = FusedResidualRMSNorm(64).cuda()
    assert torch.equal(plain(x, res, gate=m.gate)[0], fused_residual_rmsnorm(x, res, None, m.gate)[0])


def test_refusals(cuda):
    from torch.autograd import forward_ad

    from triton_ops import fused_residual_rmsnorm
    from triton_ops.exceptions import DeviceError, ShapeMismatchError, UnsupportedDtypeError

    x, res = randn((2, 4, 16), "bf16", 1), randn((2, 4, 16), "bf16", 2)
    w = torch.ones(16, device="cuda")
    for wrong, error in [
        (dict(x=x.double()), UnsupportedDtypeError),
        (dict(residual=res.half()), UnsupportedDtypeError),
        (dict(x=x.float()), UnsupportedDtypeError),  # a 16-bit stream beside an fp32 branch
        (dict(residual=res.cpu()), DeviceError),
        (dict(residual=res[:1]), ShapeMismatchError),
        (dict(weight=w[:8]), ShapeMismatchError),
        (dict(weight=w.expand(3, 16)), ShapeMismatchError),
        (dict(gate=w.expand(1, 16)), ShapeMismatchError),
        (dict(gate=torch.ones(2, 4, 16, device="cuda")), ShapeMismatchError),
        (dict(weight=w.cpu()), DeviceError),
        (dict(weight=w.int()), UnsupportedDtypeError),
        (dict(branch_weight=w), ValueError),
        (dict(norm=False, weight=w), ValueError),
        (dict(dropout_p=1.5, seed=1), ValueError),
        (dict(dropout_p=-0.1, seed=1), ValueError),
        (dict(dropout_p=float("nan"), seed=1), ValueError),
        (dict(dropout_p=0.1), ValueError),
        (dict(dropout_p=0.1, seed=1.5), TypeError),
        (dict(dropout_p=0.1, seed=torch.tensor([1])), DeviceError),
        (dict(dropout_p=0.1, seed=torch.tensor([1, 2], device="cuda")), ShapeMismatchError),
        (dict(dropout_p=0.1, seed=torch.tensor([1], device="cuda", dtype=torch.int32)), UnsupportedDtypeError),
        (dict(dropout_p=0.1, seed=1, dropout_offset=-1), ValueError),
        (dict(x=x.new_ones(()), residual=x.new_ones(())), ShapeMismatchError),
    ]:
        with pytest.raises(error):
            fused_residual_rmsnorm(**{"x": x, "residual": res, **wrong})
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.float(), x.float())
        with pytest.raises((ValueError, NotImplementedError, RuntimeError)):
            fused_residual_rmsnorm(dual, res.float())


def test_many_elements(cuda):
    """More than 2^31 elements: rows at the start, around the border and at the end."""
    hidden = 8192
    rows = 2**31 // hidden + 3
    x = torch.empty(rows, hidden, device="cuda", dtype=torch.bfloat16)
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    res = torch.flip(x, (0,))
    at = torch.tensor([0, 1, rows - 5, rows - 4, rows - 3, rows - 2, rows - 1], device="cuda")
    w = 1 + 0.1 * randn((hidden,), "f32", 2)
    t = {"x": x, "residual": res, "branch_weight": w, "gate": None, "weight": w, "shift": None}
    got = run(t, True)
    part = {k: v if v is None or v.dim() == 1 else v[at] for k, v in t.items()}
    compare(part, {k: v[at] for k, v in got.items()}, formulas(part, True, 1.0), "many")


def test_block_of_operators(cuda):
    """A block's two halves as they follow one another in training: norms, gates and dropout around two projections."""
    from triton_ops import FusedResidualRMSNorm, fused_dropout
    from triton_ops.kernels.residual import residual_rmsnorm_reference

    b, s, h = 2, 33, 128
    g = torch.Generator(device="cuda").manual_seed(3)
    w = [(torch.randn(h, h, device="cuda", generator=g) / math.sqrt(h)).requires_grad_() for _ in range(2)]
    first, second = (FusedResidualRMSNorm(h, branch_norm=True, dropout=0.1, dropout_seed=i).cuda() for i in (20, 30))
    tokens = torch.randn(b, s, h, device="cuda", generator=g).requires_grad_()
    weights = [*w, *first.parameters(), *second.parameters(), tokens]
    stream = fused_dropout(tokens, 0.1, 10)
    h1, y1 = first(stream @ w[0], stream)
    h2, y2 = second(y1 @ w[1], h1)
    got = torch.autograd.grad((h2 * y2).sum(), weights)

    wide = {id(t): t.detach().double().requires_grad_() for t in weights}
    t = [wide[id(v)] for v in weights]
    keep = [dropout_keep_reference((b, s, h), 0.1, seed, 0, "cuda") for seed in (10, 20, 30)]
    at = torch.where(keep[0], t[-1] / 0.9, 0.0)

    def half(m, x, res, kept):
        return residual_rmsnorm_reference(x, res, wide[id(m.weight)], branch_norm=True, eps=m.eps, keep=kept, dropout_p=0.1,
                                          branch_weight=wide[id(m.branch_weight)])

    r1, z1 = half(first, at @ t[0], at, keep[1])
    r2, z2 = half(second, z1 @ t[1], r1, keep[2])
    want = torch.autograd.grad((r2 * z2).sum(), t)
    # fp32 through two matrix products of 128 terms (their own 2^-24 sqrt(128) a term and TF32 off), forward and back
    for a, e in zip(got, want):
        assert (a.double() - e).norm() <= 1e-4 * e.norm()
