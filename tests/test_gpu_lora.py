"""fused_lora and FP8LoRALinear on the GPU against plain formulas in 64 bits.

Error bound of one output, from the kernel's arithmetic (fp32 sums on tensor
instructions, each adding 8 or 16 products with at most two 2^-23 roundings):

* v = A x: (K / 8 + 64) 2^-23 of sum |a| |x| (fp32 operands as two tf32 values
  each, the smallest product left out: 2^-20 more)
* v as two values of the operands' type: 2^-17 (bf16), 2^-22 of the row's
  largest (fp16), 2^-21 (fp32), doubled for the second sum: 2^-16 sum |b| |v|
  and 2^-22 max |v| sum |b| cover all three
* the sum with base: 2^-22 of both magnitudes; the result's own rounding eps/2
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-133, torch.float32: 2.0**-149}


def oracle(x, a, b, ids, scaling, base):
    """(result, bound without the result's rounding) in 64 bits, row by row."""
    t, k = x.shape
    m, r, _ = a.shape
    n = b.shape[1]
    out = base.double().clone() if base is not None else torch.zeros(t, n, device="cuda", dtype=torch.float64)
    slack = 2.0**-22 * out.abs()
    for i in range(m):
        at = (ids == i).nonzero()[:, 0]
        if not len(at):
            continue
        xi, ai, bi = x[at].double(), a[i].double(), b[i].double()
        s = scaling[i].double() if scaling is not None else 1.0
        v, mag = xi @ ai.t(), xi.abs() @ ai.abs().t()
        err = ((k / 8 + 64) * 2.0**-23 + (2.0**-20 if x.dtype == torch.float32 else 0)) * mag
        delta = s * (v @ bi.t())
        out[at] += delta
        slack[at] += s * (err @ bi.abs().t() + 2.0**-16 * (v.abs() @ bi.abs().t())
                          + 2.0**-22 * v.abs().amax(1, keepdim=True) * bi.abs().sum(1)) + 2.0**-22 * delta.abs()
    return out, slack


def check(got, x, a, b, ids, scaling, base, what=""):
    ref, slack = oracle(x, a, b, ids, scaling, base)
    assert got.shape == ref.shape and got.dtype == x.dtype
    bound = slack + ref.abs() * (torch.finfo(x.dtype).eps / 2) * 1.01 + TINY[x.dtype]
    over = ((got.double() - ref).abs() - bound).max().item() if ref.numel() else 0.0
    assert over <= 0, f"{what}: {over:.3e} over the bound"  # NaN fails too


def make(t, m, r, k, n, dtype, seed=0, none=0.1, order="mixed", ids_dtype=torch.int64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DT[dtype]
    x = torch.randn(t, k, device="cuda", generator=g).to(dt)
    a = (torch.randn(m, r, k, device="cuda", generator=g) / k**0.5).to(dt)
    b = (torch.randn(m, n, r, device="cuda", generator=g) / r**0.5).to(dt)
    base = torch.randn(t, n, device="cuda", generator=g).to(dt)
    scaling = 0.5 + torch.rand(m, device="cuda", generator=g)
    ids = torch.randint(m, (t,), device="cuda", generator=g)
    if order == "requests":
        ids = ids.sort().values
    ids = torch.where(torch.rand(t, device="cuda", generator=g) < none, -1, ids).to(ids_dtype)
    return x, a, b, ids, scaling, base


# tokens, adapters, rank, k, n, dtype
CASES = [
    (1, 1, 1, 1, 1, "f32"),
    (1, 8, 16, 4096, 4096, "bf16"),
    (1, 3, 5, 37, 19, "f16"),
    (2, 2, 8, 64, 64, "f32"),
    (17, 1, 16, 128, 96, "bf16"),      # one adapter, a tile and one row
    (33, 4, 4, 200, 72, "f16"),
    (64, 32, 16, 512, 264, "bf16"),
    (100, 300, 24, 96, 40, "bf16"),    # more adapters than rows
    (255, 7, 64, 320, 136, "f16"),
    (256, 5, 33, 130, 257, "f32"),
    (257, 5, 32, 130, 257, "bf16"),    # sorted into tiles from here on
    (500, 1, 8, 256, 512, "f16"),
    (777, 12, 12, 1000, 1500, "f16"),
    (1000, 48, 16, 64, 64, "f32"),
    (1025, 1100, 40, 72, 48, "bf16"),  # more groups than the sort takes at a time
    (2100, 9, 128, 256, 200, "bf16"),
    (300, 3, 256, 512, 72, "f16"),
    (70, 3, 256, 100, 72, "f32"),
    (9000, 20, 8, 64, 64, "bf16"),     # more rows than the sort holds at once
    (20, 16384, 1, 8, 8, "bf16"),      # the most adapters
    (300, 16384, 1, 8, 8, "bf16"),
    (384, 40, 16, 128, 96, "bf16"),    # the most rows of the single launch, and one more
    (385, 40, 16, 128, 96, "bf16"),
    (384, 1, 8, 64, 40, "f32"),
    (500, 3, 256, 512, 72, "f16"),
    (500, 16384, 1, 8, 8, "bf16"),
    (500, 1, 72, 1000, 64, "f16"),
    (500, 2, 200, 128, 64, "f32"),
    (500, 2, 200, 128, 64, "f16"),
    (3000, 16384, 1, 8, 8, "f16"),
    (2049, 5, 4, 16, 8, "f32"),        # a last row alone in its CTA's share of the sort
    (70000, 20, 8, 16, 8, "bf16"),     # more rows than the sort's CTAs hold at once
    (5000, 3, 48, 640, 328, "bf16"),   # full tiles, a last one, columns that end inside a step
    (1500, 40, 128, 512, 264, "f16"),
    (600, 2, 64, 4096, 512, "bf16"),   # a cluster for each tile
    (300, 1, 72, 1000, 64, "f16"),
    (900, 4, 8, 72, 8, "bf16"),
    (7000, 2, 20, 64, 72, "f32"),      # steps of 256 bytes
    (6500, 3, 60, 200, 136, "bf16"),
    (6500, 3, 7, 33, 17, "f16"),
    # each width of the streaming kernels, whole vectors
    (700, 6, 32, 1024, 512, "bf16"),
    (400, 3, 96, 256, 136, "f16"),
    (600, 5, 16, 192, 96, "f32"),
    (320, 2, 64, 128, 200, "f32"),
    (300, 2, 200, 128, 64, "f32"),
    (300, 2, 200, 128, 64, "f16"),
    (90, 3, 100, 256, 96, "bf16"),
    (3, 2, 16, 8192, 2048, "bf16"),    # eight CTAs a tile
]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("order", ["mixed", "requests"])
def test_against_64_bits(cuda, case, order):
    from triton_ops import _lib, fused_lora

    x, a, b, ids, scaling, base = make(*case, seed=sum(case[:5]), order=order)
    keep = base.clone()
    got = fused_lora(x, a, b, ids, scaling, base=base)
    check(got, x, a, b, ids, scaling, base)
    assert _lib.device_error_flags(clear=True) == 0  # no wait ran out
    assert torch.equal(base, keep)
    assert torch.equal(got[ids < 0], base[ids < 0])  # copied bit for bit
    assert torch.equal(got, fused_lora(x, a, b, ids, scaling, base=base))
    delta = fused_lora(x, a, b, ids)
    check(delta, x, a, b, ids, None, None, "no base, no scaling")
    assert not delta[ids < 0].any()
    same = fused_lora(x, a, b, ids.int(), scaling, base=base, out=base)
    assert same is base or same.data_ptr() == base.data_ptr()
    assert torch.equal(base, got)


def test_rows_without_an_adapter_are_left_alone(cuda):
    """In place, their bits stay (NaN payloads and all); out of place they are copied."""
    from triton_ops import fused_lora

    for t in (40, 700):
        x, a, b, ids, scaling, base = make(t, 4, 16, 128, 96, "bf16", seed=3, none=0.5)
        bits = base.view(torch.int16)
        bits[ids < 0] = 0x7FA1  # a NaN with a payload
        before = bits.clone()
        new = fused_lora(x, a, b, ids, scaling, base=base)
        assert torch.equal(new.view(torch.int16)[ids < 0], before[ids < 0])
        fused_lora(x, a, b, ids, scaling, base=base, out=base)
        assert torch.equal(base.view(torch.int16)[ids < 0], before[ids < 0])
        everyone = torch.full_like(ids, -1)
        assert torch.equal(fused_lora(x, a, b, everyone, scaling, base=x[:, :96].contiguous()), x[:, :96])


@pytest.mark.parametrize("t", [9, 600])
def test_nan_and_infinity_stay_in_their_rows(cuda, t):
    from triton_ops import fused_lora

    x, a, b, ids, scaling, base = make(t, 4, 16, 128, 96, "f16", seed=4, none=0)
    ids[:4] = torch.arange(4, device="cuda")
    ref = fused_lora(x, a, b, ids, scaling, base=base)
    x2 = x.clone()
    x2[1, 7], x2[2, 3] = float("nan"), float("inf")
    got = fused_lora(x2, a, b, ids, scaling, base=base)
    assert not torch.isfinite(got[1]).any() and not torch.isfinite(got[2]).any()
    rest = torch.ones(t, dtype=torch.bool, device="cuda")
    rest[1] = rest[2] = False
    assert torch.equal(got[rest], ref[rest])
    # an adapter that no row uses may hold anything
    a2 = torch.cat([a, torch.full_like(a[:1], float("nan"))])
    b2 = torch.cat([b, torch.full_like(b[:1], float("inf"))])
    assert torch.equal(fused_lora(x, a2, b2, ids, torch.cat([scaling, scaling[:1]]), base=base), ref)


def test_large_low_rank_values_in_fp16(cuda):
    """v passes 65504 (fp16's largest) and falls below its smallest while the result stays in range."""
    from triton_ops import fused_lora

    for t in (5, 300, 500):
        x, a, b, ids, _, base = make(t, 2, 16, 256, 64, "f16", seed=5, none=0)
        scaling = torch.tensor([1.0, 2.0**-20], device="cuda")
        x, a = x * 64, a * 1024  # v of order 2^16 and more
        b = b / 256
        b[0] /= 64
        check(fused_lora(x, a, b, ids, scaling, base=base), x, a, b, ids, scaling, base)
        check(fused_lora(x, a, b, ids, scaling), x, a, b, ids, scaling, None)


@pytest.mark.parametrize("t", [3, 300, 500])
@pytest.mark.parametrize("where", ["x", "a"])
def test_infinity_beside_values_past_the_fp16_range(cuda, t, where):
    """Low-rank values 6e7 and 1e6 beside an infinite one, in fp16.

    An infinity in x multiplies the zeros of A too (NaN): all of that row is NaN. One in A makes one low-rank value of
    every row infinite: where B is one for it the row is +inf (the others stay finite, so nothing cancels it), where B
    is zero it is NaN."""
    from triton_ops import fused_lora

    x = torch.zeros(t, 64, device="cuda", dtype=torch.float16)
    x[:, 0], x[:, 1] = 60000.0, 1000.0
    a = torch.zeros(1, 16, 64, device="cuda", dtype=torch.float16)
    a[0, 0, 0], a[0, 1, 1], a[0, 2, 2] = 1000.0, 1000.0, 1.0
    if where == "x":
        x[1, 2] = float("inf")
    else:
        x[:, 2] = 1.0
        a[0, 2, 2] = float("inf")
    b = torch.zeros(1, 32, 16, device="cuda", dtype=torch.float16)
    b[0, :, 0], b[0, :, 1] = 2.0**-14, -(2.0**-14)
    b[0, :8, 2] = 1.0
    got = fused_lora(x, a, b, torch.zeros(t, dtype=torch.int64, device="cuda")).double()
    if where == "a":
        assert (got[:, :8] == float("inf")).all()
        assert torch.isnan(got[:, 8:]).all()
        return
    want = (6e7 - 1e6) * 2.0**-14
    keep = torch.arange(t, device="cuda") != 1
    assert ((got[keep] - want).abs() <= want * 2.0**-10).all()
    assert torch.isnan(got[1]).all()


def test_bad_ids(cuda):
    from triton_ops import _lib, fused_lora

    _lib.device_error_flags(clear=True)
    for t in (20, 400):
        x, a, b, ids, scaling, base = make(t, 4, 16, 128, 96, "bf16", seed=6)
        ref = fused_lora(x, a, b, ids, scaling, base=base)
        assert _lib.device_error_flags(clear=True) == 0
        bad = ids.clone()
        bad[3], bad[11], bad[12] = 4, 2**40, -2**40
        got = fused_lora(x, a, b, bad, scaling, base=base)
        assert _lib.device_error_flags(clear=True) == _lib.ERR_BAD_ADAPTER
        assert torch.isnan(got[3]).all() and torch.isnan(got[11]).all()
        assert torch.equal(got[12], base[12])  # negative: none
        keep = torch.ones(t, dtype=torch.bool, device="cuda")
        keep[[3, 11, 12]] = False
        assert torch.equal(got[keep], ref[keep])


def test_strided_rows_and_shapes(cuda):
    """Views into wider buffers, rows off a 16-byte border, 3-D inputs."""
    from triton_ops import fused_lora

    for t in (30, 600):
        x, a, b, ids, scaling, base = make(t, 4, 16, 128, 96, "bf16", seed=7)
        ref = fused_lora(x, a, b, ids, scaling, base=base)
        for pad, off in ((32, 8), (3, 1)):
            wide_x = torch.zeros(t, 128 + pad, device="cuda", dtype=x.dtype)
            wide_x[:, off:off + 128] = x
            wide = torch.zeros(t, 2 * 96 + pad, device="cuda", dtype=x.dtype)
            wide[:, off:off + 96] = base
            view = wide[:, off:off + 96]
            got = fused_lora(wide_x[:, off:off + 128], a, b, ids, scaling, base=view, out=view)
            check(got, x, a, b, ids, scaling, base)
            assert not wide[:, off + 96:].any() and not wide[:, :off].any()  # the neighbours stay
        flipped = x.t().contiguous().t()  # innermost stride is not 1
        assert torch.equal(fused_lora(flipped, a, b, ids, scaling, base=base), ref)
        shape = (2, t // 2)
        y = fused_lora(x.view(*shape, 128), a, b, ids.view(shape), scaling, base=base.view(*shape, 96))
        assert torch.equal(y.view(t, 96), ref)
        out = torch.empty(*shape, 96, device="cuda", dtype=x.dtype)
        assert fused_lora(x.view(*shape, 128), a, b, ids.view(shape), scaling, base.view(*shape, 96), out) is out
        assert torch.equal(out.view(t, 96), ref)
    broadcast = base[:1].expand(t, 96)  # one bias row for all
    check(fused_lora(x, a, b, ids, scaling, base=broadcast), x, a, b, ids, scaling, broadcast)
    with pytest.raises(ValueError):
        fused_lora(x, a, b, ids, scaling, base=base, out=base[:1].clone().expand(t, 96))


def test_offsets_past_32_bits(cuda):
    """Rows 1.2e9 elements apart, and an adapter past the 2^31st element of lora_b."""
    from triton_ops import fused_lora

    far = 1_200_000_000
    x, a, b, ids, scaling, base = make(3, 2, 8, 64, 64, "bf16", seed=8, none=0)
    big = torch.empty(2 * far + 64, device="cuda", dtype=torch.bfloat16)
    xv = big.as_strided((3, 64), (far, 1))
    xv.copy_(x)
    ref = fused_lora(x, a, b, ids, scaling, base=base)
    assert torch.equal(fused_lora(xv, a, b, ids, scaling, base=base), ref)
    xv.copy_(base)
    assert torch.equal(fused_lora(x, a, b, ids, scaling, base=xv, out=xv), ref)
    del big, xv
    n, m = 1 << 20, 257
    wide = torch.empty(m, n, 8, device="cuda", dtype=torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(1)
    wide[256].copy_(torch.randn(n, 8, device="cuda", generator=g))
    low = torch.zeros(m, 8, 64, device="cuda", dtype=torch.bfloat16)
    low[256] = a[0]
    at = torch.full((1,), 256, device="cuda")
    got = fused_lora(x[:1], low, wide, at)
    check(got, x[:1], low[256:], wide[256:], at - 256, None, None)


def test_empty(cuda):
    from triton_ops import fused_lora

    x, a, b, ids, scaling, base = make(4, 2, 8, 64, 48, "f16")
    assert fused_lora(x[:0], a, b, ids[:0], scaling, base=base[:0]).shape == (0, 48)
    assert fused_lora(x, a, b[:, :0], ids, scaling, base=base[:, :0]).shape == (4, 0)


def test_streams_and_graphs(cuda):
    from triton_ops import fused_lora

    for t in (12, 500):
        data = {seed: make(t, 4, 16, 256, 128, "bf16", seed=seed) for seed in (1, 2, 3)}
        ref = {seed: fused_lora(*d[:5], base=d[5]) for seed, d in data.items()}
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            got = fused_lora(*data[1][:5], base=data[1][5])
        side.synchronize()
        assert torch.equal(got, ref[1])
        graphs = []
        for seed in (1, 2):
            static = [d.clone() for d in data[seed]]
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = fused_lora(*static[:5], base=static[5])
            graphs.append((graph, static, out))
        for first, second in ((3, 1), (2, 3)):
            for (_, static, _), seed in zip(graphs, (first, second)):
                for s, d in zip(static, data[seed]):
                    s.copy_(d)
            torch.cuda.synchronize()
            for graph, _, _ in graphs:  # side by side: their workspaces are their own
                with torch.cuda.stream(torch.cuda.Stream()):
                    graph.replay()
            torch.cuda.synchronize()
            for (_, _, out), seed in zip(graphs, (first, second)):
                assert torch.equal(out, ref[seed])


@pytest.mark.parametrize("extension", [True, False])
def test_threads_on_one_stream(cuda, monkeypatch, extension):
    """Calls of several threads may alternate their launches on the stream: each keeps its own plan."""
    import threading

    from triton_ops import _lib, fused_lora

    if not extension:
        monkeypatch.setattr(_lib, "ext", lambda: None)
    jobs = [make(t, 4, 16, 128, 128, "bf16", seed=t) for t in (300, 700, 40, 1300)]
    ref = [fused_lora(x, a, b, ids, scaling, base=base) for x, a, b, ids, scaling, base in jobs]
    wrong, done, start = [], [], threading.Barrier(len(jobs))

    def work(i):
        x, a, b, ids, scaling, base = jobs[i]
        start.wait(60)
        for _ in range(50):
            if not torch.equal(fused_lora(x, a, b, ids, scaling, base=base), ref[i]):
                wrong.append(i)
        done.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and len(done) == len(threads)


def test_without_the_extension(cuda, monkeypatch):
    from triton_ops import _lib, fused_lora

    for t in (40, 400):
        x, a, b, ids, scaling, base = make(t, 4, 16, 256, 128, "f16", seed=2)
        ref = fused_lora(x, a, b, ids, scaling, base=base)
        with monkeypatch.context() as m:
            m.setattr(_lib, "ext", lambda: None)
            assert torch.equal(fused_lora(x, a, b, ids, scaling, base=base), ref)


def test_module(cuda):
    from triton_ops import FP8LoRALinear
    from triton_ops.exceptions import ShapeMismatchError
    from triton_ops.kernels.lora import lora_reference

    torch.manual_seed(0)
    m = FP8LoRALinear(256, 192, max_adapters=3, rank=16).cuda()
    x = torch.randn(2, 20, 256, device="cuda", dtype=torch.float16)
    ids = torch.randint(-1, 3, (2, 20), device="cuda")
    plain = m(x)
    assert torch.equal(m(x, ids), plain)  # adapters start as zeros
    g = torch.Generator(device="cuda").manual_seed(1)
    for i, r in enumerate((16, 4, 8)):
        m.set_adapter(i, torch.randn(r, 256, device="cuda", generator=g) / 16, torch.randn(192, r, device="cuda", generator=g), 0.5 + i)
    y = m(x, ids)
    flat = (x.view(40, 256), m.lora_a, m.lora_b, ids.view(40), m.scaling, plain.view(40, 192))
    check(y.view(40, 192), *flat)
    # the plain form rounds once more where it adds: within two half steps of it
    ref = lora_reference(*flat)
    assert ((y.view(40, 192).float() - ref.float()).abs() <= 2.0**-10 * ref.float().abs() + 1e-2).all()
    bias = FP8LoRALinear(256, 192, 3, 16, bias=True).cuda()
    assert bias(x, ids).dtype == bias(x).dtype == torch.float32
    assert set(m.state_dict()) >= {"lora_a", "lora_b", "scaling", "weight"}
    with pytest.raises(ShapeMismatchError):
        m.set_adapter(0, torch.zeros(17, 256), torch.zeros(192, 17))
    with pytest.raises(ValueError):
        m.set_adapter(3, torch.zeros(4, 256), torch.zeros(192, 4))


def test_the_path_as_it_is_used(cuda):
    """A decode step: fused projection with adapters, norm and rotation of its heads at given positions."""
    from triton_ops import FP8LoRALinear, FusedQKNormRoPE, RoPEScaling, fused_lora, rope_tables
    from triton_ops.kernels.qk_norm_rope import qk_norm_rope_reference

    hq, hk, d, t, hidden = 8, 2, 64, 24, 512
    torch.manual_seed(1)
    proj = FP8LoRALinear(hidden, (hq + 2 * hk) * d, max_adapters=4, rank=8, adapter_dtype=torch.bfloat16).cuda()
    for i in range(4):
        proj.set_adapter(i, torch.randn(8, hidden) / 8, torch.randn((hq + 2 * hk) * d, 8) / 4)
    norm = FusedQKNormRoPE(d).cuda()
    x = torch.randn(t, hidden, device="cuda", dtype=torch.bfloat16)
    ids = torch.randint(-1, 4, (t,), device="cuda")
    at = torch.randint(100000, (t,), device="cuda")
    with torch.no_grad():
        qkv = proj(x, ids)
        # a second adapter set on the key columns alone, in place
        kv = qkv[:, hq * d:(hq + hk) * d]
        fused_lora(x, proj.lora_a, proj.lora_b[:, hq * d:(hq + hk) * d].contiguous(), ids, proj.scaling, base=kv, out=kv)
        cos, sin = rope_tables(at, d, scaling=RoPEScaling("yarn", 16.0, 8192))
        heads = qkv.view(t, hq + 2 * hk, d)
        v_before = heads[:, hq + hk:].clone()
        q, k = norm(heads[:, :hq], heads[:, hq:hq + hk], cos, sin)
    assert torch.equal(heads[:, hq + hk:], v_before)
    for got, x in ((q, heads[:, :hq]), (k, heads[:, hq:hq + hk])):
        ref = qk_norm_rope_reference(x.double(), torch.ones(d, device="cuda"), cos, sin)
        # heads of unit mean square, rotated: one bf16 rounding of values up to sqrt(2 * 64)
        assert ((got.double() - ref).abs() <= 2.0**-8 * 1.01 * ref.abs() + 2.0**-17 * 12).all()


def test_refusals(cuda):
    from triton_ops import fused_lora
    from triton_ops.exceptions import DeviceError, ShapeMismatchError, UnsupportedDtypeError

    x, a, b, ids, scaling, base = make(8, 3, 16, 64, 48, "f16")
    for bad, error in (
        ((x.cpu(), a, b, ids), DeviceError),
        ((x, a.cpu(), b, ids), DeviceError),
        ((x, a, b, ids.cpu()), DeviceError),
        ((x, a, b, ids, scaling.cpu()), DeviceError),
        ((x.int(), a, b, ids), UnsupportedDtypeError),
        ((x, a.float(), b, ids), UnsupportedDtypeError),
        ((x, a, b.bfloat16(), ids), UnsupportedDtypeError),
        ((x, a, b, ids.float()), UnsupportedDtypeError),
        ((x, a, b, ids, scaling.half()), UnsupportedDtypeError),
        ((x, a, b, ids, scaling, base.float()), UnsupportedDtypeError),
        ((x[:, :32], a, b, ids), ShapeMismatchError),
        ((x, a[0], b, ids), ShapeMismatchError),
        ((x, a, b[:2], ids), ShapeMismatchError),
        ((x, a, b[:, :, :8], ids), ShapeMismatchError),
        ((x, a, b, ids[:7]), ShapeMismatchError),
        ((x, a, b, ids, scaling[:2]), ShapeMismatchError),
        ((x, a, b, ids, scaling, base[:, :40]), ShapeMismatchError),
        ((x, a[:0], b[:0], ids), ShapeMismatchError),
        ((x, a[:, :, ::2], b, ids), ShapeMismatchError),
        ((x, a.transpose(0, 1).contiguous().transpose(0, 1), b, ids), ValueError),
        ((x, a, b.transpose(1, 2).contiguous().transpose(1, 2), ids), ValueError),
        ((x.clone().requires_grad_(), a, b, ids), ValueError),
        ((x, a, b, ids, scaling, base.clone().requires_grad_()), ValueError),
    ):
        with pytest.raises(error):
            fused_lora(*bad)
    with pytest.raises(ShapeMismatchError):
        fused_lora(x, torch.zeros(3, 257, 64, device="cuda").half(), torch.zeros(3, 48, 257, device="cuda").half(), ids)
    with torch.no_grad():
        fused_lora(x.clone().requires_grad_(), a, b, ids)
