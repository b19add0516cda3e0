"""GPU: products with 4-bit weights against the definition in float64, through the public entry points.

Bounds, from the arithmetic: the codes' values enter the products exactly (forward), a product's term passes at most
depth = K / 32 + 2 G + 40 float32 roundings on its way into the sum (32 terms are added inside a matrix instruction, one
sum per 32, one scaled addition per group -- two with a zero point -- and the waves' or splits' sums), each at most 2^-23
of the terms' absolute sum; the result is rounded once: eps / 2 of itself.  In the backward product every weight is first
rounded once, to float16 (11 significant bits, half a step: 2^-11 of it at most), so 2^-11 of the terms' absolute sum.  Results below the type's normal numbers are off by half their step."""
import copy

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

FORMATS = [("int4", 4), ("int4_asym", 4), ("fp4", 4), ("flint4", 4), ("fp4_er_pos", 4), ("fp4_ea_neg", 4), ("fp3", 3), ("int3", 3),
           ("int2_asym", 2)]


@pytest.fixture(scope="module")
def pk():
    from quantization_amd import packed
    return packed


def weight(gen, shape, fmt, bits, g):
    """Codes etc. from the framework's quantizers, packed, and the float64 weight that they stand for."""
    from quantization_amd import packed, quant_weight as qw
    w = (torch.randn(shape, generator=gen, device="cuda") * 0.02).half()
    e = shape[0] if len(shape) == 3 else None
    flat = w.reshape(-1, shape[-1])
    if fmt.startswith("int"):
        deq, q, s, z = qw._int_quant_meta(flat, wq_bits=bits, asym="asym" in fmt, group_size=g)
    else:
        (deq, q, s), z = qw._fp_quant_meta(flat, wq_bits=bits, datatype=fmt, group_size=g), None
    rows, k = flat.shape

    def per(t):
        t = t.double().expand(rows, 1) if t.dim() == 0 else t.double().reshape(rows, -1)
        return t.repeat_interleave(k // t.shape[1], 1)

    v = (q.view(torch.uint8) if "asym" in fmt else q.view(torch.int8) if fmt.startswith("int") else q).double().reshape(rows, k)
    exact = per(s) * (v - per(z) if z is not None else v)
    zmass = per(s) * (v.abs() + (per(z) if z is not None else 0))      # what the sums hold before they cancel
    lead = lambda t: t if e is None or t is None else t.reshape((e, shape[1]) + tuple(t.shape[1:]))
    p = packed.pack_codes(lead(q), lead(s), lead(z), bits, fmt, g)
    return p, exact.reshape(shape), zmass.reshape(shape), deq.reshape(shape)


def depth(k, p):
    groups = k // p.group_size if p.group_size > 0 else 1
    return (k / 32 + 2 * groups + 40) * 2.0 ** -23


def near(got, want, mass, k, p, rounded=False, what=""):
    eps = torch.finfo(got.dtype).eps / 2
    tol = eps * want.abs() + (depth(k, p) + (2.0 ** -11 if rounded else 0)) * (1 + eps) * mass
    tol = tol + torch.finfo(got.dtype).smallest_normal * eps
    off = (got.double() - want).abs()
    bad = off > tol
    assert got.isfinite().all(), (what, "not finite")
    assert not bad.any(), (what, int(bad.sum()), float((off / tol).max()), bad.nonzero()[:4].tolist())


def product(x, w):
    return x.double() @ w.t()


SHAPES = [(16, 128, 32), (48, 96, 32), (1, 64, None), (17, 100, None), (130, 256, 128), (64, 384, 96), (200, 320, 64), (33, 7, None),
          (260, 1024, 256), (96, 640, 160), (2056, 512, 128), (40, 192, -1), (3, 1, None), (66, 4104, None)]


@pytest.mark.parametrize("fmt,bits", FORMATS)
def test_dequantize_has_the_quantizers_bits(pk, fmt, bits):
    gen = torch.Generator(device="cuda").manual_seed(1)
    for n, k, g in SHAPES:
        if g == -1 and not fmt.startswith("int"):
            continue   # (quant_datatype's per-tensor branch is float32 arithmetic)
        p, _, _, deq = weight(gen, (n, k), fmt, bits, g)
        got = p.dequantize()
        assert got.shape == deq.shape
        zero = (got == 0) & (deq == 0)     # (a code has no sign of zero)
        assert torch.equal(torch.where(zero, 0, got.view(torch.int16)), torch.where(zero, 0, deq.view(torch.int16))), (n, k, g)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fmt,bits", FORMATS)
def test_linear_few_rows(pk, fmt, bits, dtype):
    gen = torch.Generator(device="cuda").manual_seed(2)
    for n, k, g in SHAPES:
        p, w, mass, _ = weight(gen, (n, k), fmt, bits, g)
        for m in (1, 2, 5, 16, 17, 32):
            x = torch.randn(m, k, generator=gen, device="cuda").to(dtype)
            near(pk.packed_linear(x, p), product(x, w), product(x.abs(), mass), k, p, what=(n, k, g, m))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fmt,bits", FORMATS)
def test_linear_many_rows_with_bias(pk, fmt, bits, dtype):
    gen = torch.Generator(device="cuda").manual_seed(3)
    for n, k, g in SHAPES:
        p, w, mass, _ = weight(gen, (n, k), fmt, bits, g)
        b = torch.randn(n, generator=gen, device="cuda").to(dtype)
        for m in (33, 64, 65, 128, 130, 301):
            x = torch.randn(m, k, generator=gen, device="cuda").to(dtype)
            near(pk.packed_linear(x, p, b), product(x, w) + b.double(), product(x.abs(), mass) + b.double().abs(), k, p, what=(n, k, g, m))


@pytest.mark.parametrize("g", [32, 64, 128, 256, None])
@pytest.mark.parametrize("fmt", ["int4", "int4_asym"])
def test_every_number_of_blocks(pk, fmt, g):
    """Contractions of one to nine blocks of 128 (windows of zero points in pairs, blocks in two wave sets, cuts) under each
    tile: few rows, one tile to a compute unit, several."""
    gen = torch.Generator(device="cuda").manual_seed(17)
    for blocks in range(1, 10):
        k = blocks * 128
        if g and k % g:
            continue
        p, w, mass, _ = weight(gen, (1100, k), fmt, 4, g)
        for dtype, m in ((torch.float16, 47), (torch.bfloat16, 200), (torch.float16, 1300), (torch.bfloat16, 4200)):
            x = torch.randn(m, k, generator=gen, device="cuda").to(dtype)
            near(pk.packed_linear(x, p), product(x, w), product(x.abs(), mass), k, p, what=(blocks, m))
    # the gradient: the same along the weight's rows
    for blocks in range(1, 10):
        n = blocks * 128 - blocks % 3
        p, w, mass, _ = weight(gen, (n, 1280), fmt, 4, g)
        for dtype, m in ((torch.float16, 47), (torch.bfloat16, 200), (torch.float16, 1300), (torch.bfloat16, 8300)):
            x = torch.zeros(m, 1280, device="cuda", dtype=dtype, requires_grad=True)
            dy = torch.randn(m, n, generator=gen, device="cuda").to(dtype)
            pk.packed_linear(x, p).backward(dy)
            near(x.grad, dy.double() @ w, dy.double().abs() @ mass, n, p, rounded=True, what=("grad", blocks, m))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fmt,bits", FORMATS)
def test_linear_backward(pk, fmt, bits, dtype):
    gen = torch.Generator(device="cuda").manual_seed(4)
    for n, k, g in SHAPES:
        p, w, _, _ = weight(gen, (n, k), fmt, bits, g)
        for m in (1, 17, 64, 130):
            x = torch.randn(m, k, generator=gen, device="cuda").to(dtype).requires_grad_()
            b = torch.randn(n, generator=gen, device="cuda").to(dtype).requires_grad_()
            dy = torch.randn(m, n, generator=gen, device="cuda").to(dtype)
            dx, db = torch.autograd.grad(pk.packed_linear(x, p, b), (x, b), dy)
            near(dx, product(dy, w.t()), product(dy.abs(), w.t().abs()), n, p, rounded=True, what=("dx", n, k, g, m))
            near(db, dy.double().sum(0), dy.double().abs().sum(0) * (m / 16 + 1), n, p, what=("db", n, k, g, m))


def test_bias_gradient_over_many_rows(pk):
    """Runs of rows whose sums a second launch adds; bias alone, without a gradient of x."""
    gen = torch.Generator(device="cuda").manual_seed(17)
    p, *_ = weight(gen, (70, 64), "int4", 4, 32)
    pe, *_ = weight(gen, (3, 70, 64), "int4", 4, 32)
    for m in (512, 513, 1000, 5000):
        x = torch.randn(m, 64, generator=gen, device="cuda").bfloat16()
        dy = torch.randn(m, 70, generator=gen, device="cuda").bfloat16()
        b = torch.zeros(70, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        db, = torch.autograd.grad(pk.packed_linear(x, p, b), b, dy)
        near(db, dy.double().sum(0), dy.double().abs().sum(0) * (m / 16 + 1), 70, p, what=m)
        be = torch.zeros(3, 70, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        c = torch.tensor([m // 2, 0, m - m // 2 - 7])
        db, = torch.autograd.grad(pk.packed_expert_linear(x, pe, c.cuda(), be), be, dy)
        for i, lo, hi in spans(c, m):
            near(db[i], dy[lo:hi].double().sum(0), dy[lo:hi].double().abs().sum(0) * (m / 16 + 1), 70, pe, what=(m, i))


def counts_of(kind, e, rows):
    c = torch.zeros(e, dtype=torch.int64)
    if kind == "even":
        c += rows // e
    elif kind == "one":
        c[e // 2] = rows
    elif kind == "ragged":
        c = torch.multinomial(1 / torch.arange(1., e + 1), rows, replacement=True, generator=torch.Generator().manual_seed(5)).bincount(minlength=e)
        c[0] = max(0, int(c[0]) - 3)       # rows behind the last expert's
    elif kind == "over":
        c += rows                          # more than there are: cut off
    elif kind == "negative":
        c += rows // e
        c[0] = -5
    return c


def spans(counts, rows):
    at = 0
    for e, c in enumerate(counts.tolist()):
        c = min(max(c, 0), rows - at)
        yield e, at, at + c
        at += c


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["even", "one", "ragged", "over", "negative", "none"])
@pytest.mark.parametrize("fmt", ["int4", "int4_asym", "fp4", "flint4"])
def test_experts(pk, fmt, kind, dtype):
    gen = torch.Generator(device="cuda").manual_seed(6)
    for e, n, k, g, rows in [(4, 48, 96, 32, 7), (70, 33, 128, 64, 90), (3, 144, 260, None, 300), (130, 16, 64, 32, 64), (1, 64, 128, 128, 40),
                             (8, 40, 512, 128, 1), (5, 136, 256, 128, 700)]:
        p, w, mass, _ = weight(gen, (e, n, k), fmt, 4, g)
        c = counts_of(kind, e, rows)
        x = torch.randn(rows, k, generator=gen, device="cuda").to(dtype)
        b = torch.randn(e, n, generator=gen, device="cuda").to(dtype)
        dy = torch.randn(rows, n, generator=gen, device="cuda").to(dtype)
        last = [s[2] for s in spans(c, rows)][-1]
        x[last:], dy[last:] = float("nan"), float("nan")      # nobody's rows
        x.requires_grad_(), b.requires_grad_()
        y = pk.packed_expert_linear(x, p, c.to("cuda", torch.int32), b)
        dx, db = torch.autograd.grad(y, (x, b), dy)
        with torch.no_grad():
            assert torch.equal(pk.packed_expert_linear(x, p, c.cuda(), b), y)
            assert not y[last:].any() and not dx[last:].any()
            for i, lo, hi in spans(c, rows):
                xs, ds, what = x[lo:hi], dy[lo:hi], (e, n, k, g, rows, kind, i)
                near(y[lo:hi], product(xs, w[i]) + b[i].double(), product(xs.abs(), mass[i]) + b[i].double().abs(), k, p, what=what)
                near(dx[lo:hi], product(ds, w[i].t()), product(ds.abs(), w[i].t().abs()), n, p, rounded=True, what=("dx",) + what)
                near(db[i], ds.double().sum(0), ds.double().abs().sum(0) * ((hi - lo) / 16 + 1), n, p, what=("db",) + what)


def test_gradient_against_differences(pk):
    """The product is linear in x: <dy, f(x + h) - f(x)> = <dx, h> up to the roundings of its parts."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    p, w, mass, _ = weight(gen, (96, 256), "int4_asym", 4, 64)
    x = torch.randn(40, 256, generator=gen, device="cuda").half().requires_grad_()
    h = torch.randn(40, 256, generator=gen, device="cuda").half()
    dy = torch.randn(40, 96, generator=gen, device="cuda").half()
    dx, = torch.autograd.grad(pk.packed_linear(x, p), x, dy)
    with torch.no_grad():
        up, down = pk.packed_linear(x + h, p).double(), pk.packed_linear(x - h, p).double()
        left, right = (dy.double() * (up - down)).sum() / 2, (dx.double() * h.double()).sum()
        # x +- h are rounded (2^-11 of them through |W|), the three results too
        slack = 2.0 ** -11 * ((dy.double().abs() * ((x.abs() + h.abs()).double() @ mass.t() + up.abs() + down.abs())).sum()
                              + (dx.double().abs() * h.double().abs()).sum() + ((dy.double().abs() @ w.abs()) * h.double().abs()).sum())
    assert abs(left - right) <= slack


def test_layouts_of_the_activations(pk):
    gen = torch.Generator(device="cuda").manual_seed(8)
    for n, k, g in ((48, 256, 64), (32, 100, None)):
        p, w, mass, _ = weight(gen, (n, k), "int4_asym", 4, g)
        wide = torch.randn(200, 2 * k + 9, generator=gen, device="cuda").half()
        views = {"offset": wide[:, 3:3 + k], "every other row": wide[::2, :k], "turned": wide[:k, :150].t() if k <= 200 else wide[:, :k],
                 "one row again": wide[:1, :k].expand(70, k), "three axes": wide[:, :k].reshape(4, 50, k), "one axis": wide[0, 1:1 + k],
                 "overlapping": wide.as_strided((50, k), (k // 2, 1)), "odd rows": wide.reshape(-1)[1:1 + 60 * (k + 1)].view(60, k + 1)[:, :k]}
        for name, x in views.items():
            for rows in (x, x[:3] if x.dim() > 1 else x):
                y = pk.packed_linear(rows, p)
                assert y.shape == rows.shape[:-1] + (n,) and y.is_contiguous(), name
                near(y.reshape(-1, n), product(rows.reshape(-1, k), w), product(rows.abs().reshape(-1, k), mass), k, p, what=name)
        x = wide[:70, :k].clone().requires_grad_()
        y = pk.packed_linear(x, p)
        y.sum().backward()                                        # dy is one value, expanded
        ones = torch.ones(70, n, device="cuda")
        near(x.grad, product(ones, w.t()), product(ones, w.t().abs()), n, p, rounded=True, what="expanded dy")
        shared = wide[:1, :k].clone().requires_grad_()
        pk.packed_linear(shared.expand(70, k), p).sum().backward()    # torch adds the rows of dx in its own order
        assert torch.isfinite(shared.grad).all()


def test_empty_and_refused(pk):
    gen = torch.Generator(device="cuda").manual_seed(9)
    p, *_ = weight(gen, (48, 64), "int4", 4, 32)
    x = torch.empty(0, 64, dtype=torch.float16, device="cuda", requires_grad=True)
    b = torch.zeros(48, dtype=torch.float16, device="cuda", requires_grad=True)
    y = pk.packed_linear(x, p, b)
    dx, db = torch.autograd.grad(y, (x, b), torch.empty_like(y))
    assert y.shape == (0, 48) and dx.shape == (0, 64) and not db.any()
    assert pk.packed_linear(torch.empty(2, 0, 64, dtype=torch.float16, device="cuda"), p).shape == (2, 0, 48)
    pe, *_ = weight(gen, (3, 48, 64), "int4", 4, 32)
    counts = torch.zeros(3, dtype=torch.int32, device="cuda")
    good = torch.zeros(4, 64, dtype=torch.float16, device="cuda")
    assert pk.packed_expert_linear(x, pe, counts).shape == (0, 48)
    for bad in (good.float(), good[:, :63], good[0, 0], good.int()):
        with pytest.raises(ValueError):
            pk.packed_linear(bad, p)
    for bias in (b[:47], b.bfloat16(), b.cpu()):
        with pytest.raises(ValueError):
            pk.packed_linear(good, p, bias)
    with pytest.raises(ValueError):
        pk.packed_linear(good, pe)
    with pytest.raises(ValueError):
        pk.packed_expert_linear(good, p, counts[:1])
    for c in (counts[:2], counts.cpu(), counts.float(), None, counts[None]):
        with pytest.raises(ValueError):
            pk.packed_expert_linear(good, pe, c)
    with pytest.raises(ValueError):
        pk.packed_expert_linear(good[None], pe, counts)
    with pytest.raises(RuntimeError):          # differentiable once
        z = good.clone().requires_grad_()
        g, = torch.autograd.grad(pk.packed_linear(z, p).sum(), z, create_graph=True)
        g.sum().backward()


def test_scales_of_every_size(pk):
    """Scales at both ends of float16, in the same weight: no product of a code and a scale may leave float16's range."""
    gen = torch.Generator(device="cuda").manual_seed(10)
    n, k = 64, 256
    for dtype in (torch.float16, torch.bfloat16):
        for top, lo in ((6.0e4, 3.0e4), (2.0 ** -24, 2.0 ** -24), (1.0e-5, 6.0e-8), (1.0, 2.0 ** -10)):
            s = (torch.rand(n, k // 64, generator=gen, device="cuda") * (top - lo) + lo).half()
            q = torch.randint(-7, 8, (n, k), generator=gen, device="cuda", dtype=torch.int8)
            p = pk.pack_codes(q, s, None, 4, "int4", 64)
            w = q.double() * s.double().repeat_interleave(64, 1)
            for m in (3, 70):
                unit = 1.0 / (top * 64)
                x = torch.randn(m, k, generator=gen, device="cuda").to(dtype)
                if top > 1:
                    x = (x.float() * unit).to(dtype)
                near(pk.packed_linear(x, p), product(x, w), product(x.abs(), w.abs()), k, p, what=(top, m))
                dy = torch.randn(m, n, generator=gen, device="cuda")
                dy = (dy * unit if top > 1 else dy).to(dtype)
                x = x.requires_grad_()
                dx, = torch.autograd.grad(pk.packed_linear(x, p), x, dy)
                near(dx, product(dy, w.t()), product(dy.abs(), w.t().abs()), n, p, rounded=True, what=("dx", top, m))
    # no scale at all
    p = pk.pack_codes(q, torch.zeros_like(s), None, 4, "int4", 64)
    x = torch.randn(5, k, generator=gen, device="cuda").half().requires_grad_()
    y = pk.packed_linear(x, p)
    y.sum().backward()
    assert not y.any() and not x.grad.any()


def test_a_row_that_is_not_finite_stays_its_own(pk):
    gen = torch.Generator(device="cuda").manual_seed(11)
    for fmt in ("int4", "int4_asym"):
        p, w, mass, _ = weight(gen, (48, 256), fmt, 4, 64)
        for m in (5, 100):
            x = torch.randn(m, 256, generator=gen, device="cuda").bfloat16()
            x[2, 7], x[4, 9] = float("nan"), float("inf")
            y = pk.packed_linear(x, p)
            assert y[2].isnan().all() and not y[4].isfinite().any()
            keep = [i for i in range(m) if i not in (2, 4)]
            near(y[keep], product(x[keep], w), product(x[keep].abs(), mass), 256, p, what=(fmt, m))


def test_gradients_of_every_size(pk):
    """Rows of dy of very different size, up to both ends of bfloat16, in one call: each keeps its bits."""
    gen = torch.Generator(device="cuda").manual_seed(19)
    n, k = 200, 128
    p, w, _, _ = weight(gen, (n, k), "int4", 4, 32)
    for m in (30, 200):
        size = torch.logspace(-37, 36, m, device="cuda", dtype=torch.float64)[:, None]
        dy = (torch.randn(m, n, generator=gen, device="cuda").double() * size).bfloat16()
        dy[3], dy[5, 1:] = 0, 0
        x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        dx, = torch.autograd.grad(pk.packed_linear(x, p), x, dy)
        near(dx, product(dy, w.t()), product(dy.abs(), w.t().abs()), n, p, rounded=True, what=m)
        assert not dx[3].any()
        dy[7, 9], dy[8, 9] = float("inf"), float("nan")
        dx, = torch.autograd.grad(pk.packed_linear(x, p), x, dy)
        assert not dx[7:9].isfinite().any()
        keep = [i for i in range(m) if i not in (7, 8)]
        near(dx[keep], product(dy[keep], w.t()), product(dy[keep].abs(), w.t().abs()), n, p, rounded=True, what=m)


def test_streams_and_graphs(pk):
    gen = torch.Generator(device="cuda").manual_seed(12)
    p, w, mass, _ = weight(gen, (96, 512), "int4_asym", 4, 64)
    pe, we, masse, _ = weight(gen, (6, 80, 512), "int4", 4, 128)
    xs = [torch.randn(m, 512, generator=gen, device="cuda").half() for m in (1, 40, 300)]
    want = [pk.packed_linear(x, p) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [pk.packed_linear(x, p) for x in xs]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # two graphs that live side by side, one with a backward pass, replayed with new inputs and counts
    x = torch.zeros(200, 512, dtype=torch.float16, device="cuda", requires_grad=True)
    b = torch.zeros(6, 80, dtype=torch.float16, device="cuda", requires_grad=True)
    dy = torch.zeros(200, 80, dtype=torch.float16, device="cuda")
    counts = torch.full((6,), 30, dtype=torch.int32, device="cuda")
    one = torch.zeros(1, 512, dtype=torch.float16, device="cuda")

    def step():
        y = pk.packed_expert_linear(x, pe, counts, b)
        return (y,) + torch.autograd.grad(y, (x, b), dy)

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), pk.packed_linear(one, p)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        ya, dxa, dba = step()
    with torch.cuda.graph(gb):
        yb = pk.packed_linear(one, p)
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(200, 512, generator=gen, device="cuda"))
            b.copy_(torch.randn(6, 80, generator=gen, device="cuda"))
        dy.copy_(torch.randn(200, 80, generator=gen, device="cuda"))
        one.copy_(torch.randn(1, 512, generator=gen, device="cuda"))
        counts.copy_(torch.tensor([[30] * 6, [200, 0, 0, 0, 0, 0], [0, 1, 0, 2, 0, 3], [50, 0, 100, 7, 0, 43]][i]))
        ga.replay()
        gb.replay()
        got = [t.clone() for t in (ya, dxa, dba, yb)]
        torch.cuda.synchronize()
        for a, e in zip(got, step() + (pk.packed_linear(one, p),)):
            assert torch.equal(a, e), i


def test_offsets_beyond_32_bits(pk):
    """Rows of x, of y and tiles of the weight that lie more than 2^32 bytes from the first."""
    gen = torch.Generator(device="cuda").manual_seed(18)
    n, k = 64, 256
    p, w, mass, _ = weight(gen, (n, k), "int4_asym", 4, 64)
    for stride, rows in ((1 << 23, 300), ((1 << 23) + 8, 300), (1 << 28, 9)):     # read in place, copied first, few rows
        x = torch.empty((rows - 1) * stride + k, dtype=torch.float16, device="cuda").as_strided((rows, k), (stride, 1))
        x.copy_(torch.randn(rows, k, generator=gen, device="cuda"))
        near(pk.packed_linear(x, p), product(x, w), product(x.abs(), mass), k, p, what=stride)
        del x
    n, k, rows = 16400, 32, 140000                                               # y: 4.6 GB, dy too
    p, w, mass, _ = weight(gen, (n, k), "int4", 4, 32)
    x = torch.randn(rows, k, generator=gen, device="cuda").half().requires_grad_()
    y = pk.packed_linear(x, p)
    dx, = torch.autograd.grad(y, x, y.detach())
    with torch.no_grad():
        at = torch.tensor([0, 1, 65535, 131000, 139935, 139999], device="cuda")
        near(y[at], product(x[at], w), product(x[at].abs(), mass), k, p, what="y")
        near(dx[at], product(y[at], w.t()), product(y[at].abs(), w.t().abs()), n, p, rounded=True, what="dx")
    del x, y, dx
    e, n, k = 40, 16384, 16384                                                   # 5.4 GB of codes
    q = torch.randint(-7, 8, (e, n, k), generator=gen, device="cuda", dtype=torch.int8)
    s = (torch.rand(e, n, 1, generator=gen, device="cuda") * 0.01).half()
    p = pk.pack_codes(q, s[..., 0], None, 4, "int4", None)
    counts = torch.zeros(e, dtype=torch.int32, device="cuda")
    counts[-1], counts[0] = 50, 50
    x = torch.randn(100, k, generator=gen, device="cuda").half().requires_grad_()
    y = pk.packed_expert_linear(x, p, counts)
    dx, = torch.autograd.grad(y, x, y.detach())
    with torch.no_grad():
        for i, lo in ((0, 0), (e - 1, 50)):
            w = q[i].double() * s[i].double()
            near(y[lo:lo + 50], product(x[lo:lo + 50], w), product(x[lo:lo + 50].abs(), w.abs()), k, p, what=i)
            near(dx[lo:lo + 50], product(y[lo:lo + 50], w.t()), product(y[lo:lo + 50].abs(), w.t().abs()), n, p, rounded=True, what=i)


def test_repeated_calls_have_the_same_bits(pk):
    gen = torch.Generator(device="cuda").manual_seed(13)
    p, *_ = weight(gen, (256, 2048), "fp4", 4, 64)
    for m in (1, 20, 90, 260):
        x = torch.randn(m, 2048, generator=gen, device="cuda").bfloat16().requires_grad_()
        dy = torch.randn(m, 256, generator=gen, device="cuda").bfloat16()
        runs = []
        for _ in range(3):
            y = pk.packed_linear(x, p)
            runs.append((y, *torch.autograd.grad(y, x, dy)))
        for r in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


@pytest.mark.parametrize("fmt,bits", [("int4", 4), ("int4_asym", 4), ("fp4", 4), ("flint4", 4), ("fp3_er_neg", 3), ("int3_asym", 3)])
@pytest.mark.parametrize("g", [None, 64, -1])
def test_quant_model_packed(pk, fmt, bits, g):
    """quant_model(packed=True): PackedLinear in each Linear's place, the model's output that of the dequantized model."""
    from quantization_amd.quant_weight import quant_model
    torch.manual_seed(14)
    model = nn.Sequential(nn.Linear(128, 192), nn.GELU(), nn.Sequential(nn.Linear(192, 64, bias=False)), nn.Linear(64, 40)).half().cuda()
    names = [n for n, m in model.named_modules() if isinstance(m, nn.Linear)]
    quant_model(model, wq_bits=bits, wq_datatype=fmt, wq_groupsize=g, packed=True)
    mods = dict(model.named_modules())
    assert all(isinstance(mods[n], pk.PackedLinear) for n in names)
    x = torch.randn(50, 128, device="cuda").half()
    for rows in (x, x[:1]):
        h = rows
        for m in (model[0], model[1], model[2][0], model[3]):
            if isinstance(m, pk.PackedLinear):
                w = m.packed.dequantize().float()
                want = F.linear(h.float(), w, None if m.bias is None else m.bias.float())
                mass = h.float().abs() @ w.abs().t() * (16 if "asym" in fmt else 1) + want.abs()
                got = m(h).float()
                # dequantize() rounds each weight to float16 (2^-11), the result once more
                assert ((got - want).abs() <= 2.0 ** -10 * mass + 1e-6).all()
                h = m(h)
            else:
                h = m(h)
        assert torch.equal(model(rows), h)
    # moved, copied, saved and loaded
    again = copy.deepcopy(model)
    assert torch.equal(again.to(torch.device("cuda", 0))(x), model(x))
    state = {k: v.clone() for k, v in model.state_dict().items()}
    with torch.no_grad():
        for t in again.state_dict().values():
            t.zero_()
    again.load_state_dict(state)
    assert torch.equal(again(x), model(x))
    other = copy.deepcopy(model)
    for t in other.state_dict().values():
        t.zero_()
    other.load_state_dict(state, assign=True)
    assert torch.equal(other(x), model(x))
    half = copy.deepcopy(model).bfloat16()     # the packed weight has no floating dtype to change
    assert half(x.bfloat16()).dtype == torch.bfloat16


def test_pack_weight_of_experts_and_host_tensors(pk):
    gen = torch.Generator(device="cuda").manual_seed(15)
    w = (torch.randn(3, 40, 128, generator=gen, device="cuda") * 0.02).half()
    for fmt in ("int4", "int4_asym", "fp4"):
        for g in (64, None, -1):
            if g == -1 and fmt == "fp4":
                continue
            stack = pk.pack_weight(w, 4, fmt, g)
            assert stack.shape == w.shape
            for i in range(3):
                assert torch.equal(stack.dequantize()[i], pk.pack_weight(w[i].cpu(), 4, fmt, g).dequantize()), (fmt, g, i)


def test_a_chain_as_a_model_uses_it(pk):
    """Router, experts' products up and down, and the vocabulary's projection, trained through: against float64."""
    gen = torch.Generator(device="cuda").manual_seed(16)
    e, d, f, v, rows = 6, 128, 192, 300, 150
    up, wu, mu, _ = weight(gen, (e, f, d), "int4", 4, 64)
    down, wd, md, _ = weight(gen, (e, d, f), "int4_asym", 4, 32)
    head, wh, mh, _ = weight(gen, (v, d), "fp4", 4, 128)
    tokens = (torch.randn(rows, d, generator=gen, device="cuda")).bfloat16().requires_grad_()
    expert = torch.randint(0, e, (rows,), generator=gen, device="cuda")
    order = expert.argsort(stable=True)
    counts = torch.bincount(expert, minlength=e)
    h = pk.packed_expert_linear(tokens[order], up, counts)
    o = pk.packed_expert_linear(torch.relu(h), down, counts)
    logits = pk.packed_linear(torch.empty_like(o).index_copy(0, order, o) + tokens, head)
    logits.float().logsumexp(-1).sum().backward()
    t64 = tokens.detach().double().requires_grad_()
    hs = torch.stack([wu[i] @ t64[r] for r, i in enumerate(expert.tolist())])
    os = torch.stack([wd[i] @ torch.relu(hs[r]) for r, i in enumerate(expert.tolist())])
    l64 = (os + t64) @ wh.t()
    l64.logsumexp(-1).sum().backward()
    # three bfloat16 roundings of activations and one of the result on the way forward: 4 * 2^-9 of the norm; the way
    # back rounds each intermediate gradient and each weight: 8 * 2^-9, plus the forward's
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())
    assert rel(logits.detach(), l64.detach()) <= 4 * 2.0 ** -9
    assert rel(tokens.grad, t64.grad) <= 12 * 2.0 ** -9
