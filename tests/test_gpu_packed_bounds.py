"""GPU: how far results of the products with 4-bit weights may be off where the sizes of scales, rows or sums are far apart.
Each bound is derived beside its test from the kernels' arithmetic."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pk():
    from quantization_amd import packed
    return packed


def spread(gen, shape, low, high):
    """Positive float16 numbers, evenly over the binades from 2^low to 2^high."""
    e = torch.rand(shape, generator=gen, device="cuda", dtype=torch.float64) * (high - low) + low
    return (2.0 ** e).half()


def gradient(pk, p, dy):
    x = torch.zeros(dy.shape[0], p.k, dtype=dy.dtype, device="cuda", requires_grad=True)
    return torch.autograd.grad(pk.packed_linear(x, p), x, dy)[0]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fmt", ["int4", "int4_asym", "fp4", "flint4"])
def test_gradient_where_the_scales_are_far_apart(pk, fmt, dtype):
    """dx = dy W with the weights times norm in float16, norm the power of two that brings T = largest |scale| * reach (reach
    16, with zero points 15 + the largest) into [2^14, 2^15).  A scale times norm is exact down to 2^-14 and off by 2^-25 at
    most below; the weight is rounded by 2^-11 of it or, below 2^-14, by 2^-25.  So a weight is off by at most
    2^-11 |W| + 2^-25 (|q - zero| + 1) / norm, and 1 / norm <= T 2^-14.  Rows of bfloat16 are brought to [2^14, 2^15) in their
    turn: an element is off by 2^-25 of that scale, 2^-39 of the row's largest, at most.  The float32 sum passes at most
    n / 16 + 40 additions per term; one rounding of the result."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    n, k, g = 200, 256, 64
    table = {"fp4": [0, 1, 2, 3, 4, 6, 8, 12], "flint4": [0, 1, 2, 3, 4, 6, 8, 16]}.get(fmt)
    for low, high in ((-24, 15), (-24, -1), (-14, 13), (-24, -20)):
        s = spread(gen, (n, k // g), low, high)
        z = None
        if table:
            q = torch.tensor(table, device="cuda").half()[torch.randint(0, 8, (n, k), generator=gen, device="cuda")]
        elif fmt == "int4":
            q = torch.randint(-7, 8, (n, k), generator=gen, device="cuda", dtype=torch.int8)
        else:
            q = torch.randint(0, 16, (n, k), generator=gen, device="cuda", dtype=torch.uint8)
            z = torch.randint(0, 16, (n, k // g), generator=gen, device="cuda").half()
        p = pk.pack_codes(q, s, z, 4, fmt, g)
        wide = lambda t: t.double().repeat_interleave(g, 1)
        d = q.double() - (0 if z is None else wide(z))
        w = d * wide(s)
        top = float(s.double().max()) * (16 if z is None else 15 + float(z.max()))
        off = 2.0 ** -11 * w.abs() + 2.0 ** -25 * (d.abs() + 1) * top * 2.0 ** -14
        # gradients that let the rows of small scales count: dy as large as its scale is small
        balance = (2.0 ** -s.double().log2().mean(1))[None]
        for m in (40, 300):
            dy = torch.randn(m, n, generator=gen, device="cuda", dtype=torch.float64) * balance
            dy = (dy / dy.abs().max() * 2.0 ** 6).to(dtype)
            d64 = dy.double()
            want = d64 @ w
            rows = 2.0 ** -39 * d64.abs().amax(1, keepdim=True) if dtype == torch.bfloat16 else 0.0
            mass = d64.abs() @ w.abs()
            tol = d64.abs() @ off + rows * w.abs().sum(0) * (1 + 2.0 ** -10) + (n / 16 + 40) * 2.0 ** -23 * mass
            eps = torch.finfo(dtype).eps / 2
            tol = tol * (1 + 2 * eps) + eps * want.abs() + torch.finfo(dtype).smallest_normal * eps
            fits = want.abs() + tol < torch.finfo(dtype).max
            got = gradient(pk, p, dy).double()
            bad = ((got - want).abs() > tol) & fits
            assert not bad.any(), (low, high, m, int(bad.sum()), float(((got - want).abs() / tol)[fits].max()))


def runs(rows, experts=1):
    """Into how many runs the rows' sum is cut: up to 512 rows of an expert, on average, in one."""
    per = rows // experts
    return 1 if per <= 512 else min(per // 256, 32)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_bias_gradient_adds_every_row_once(pk, dtype):
    """db = sum of dy over the rows.  A run's rows are added by sixteen waves in turn, the waves' sums and the runs' one after
    the other: a term passes at most rows / (16 runs) + 1 + 15 + runs float32 additions.  Whole numbers whose sums stay below
    2^24 are added without any rounding."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    n, k = 70, 64
    p = pk.pack_weight(torch.randn(n, k, generator=gen, device="cuda").half(), 4, "int4", 32)
    pe = pk.pack_weight(torch.randn(3, n, k, generator=gen, device="cuda").half(), 4, "int4", 32)
    eps = torch.finfo(dtype).eps / 2
    for m in (1, 15, 16, 17, 300, 512, 513, 767, 768, 1000, 1537, 5000, 9000, 20000):
        x = torch.zeros(m, k, device="cuda", dtype=dtype)
        counts = torch.tensor([m // 2, 0, m - m // 2 - m // 7], device="cuda")
        ends = [0, m // 2, m // 2, m - m // 7]
        real = torch.randn(m, n, generator=gen, device="cuda").to(dtype)
        whole = torch.randint(-8, 9, (m, n), generator=gen, device="cuda").to(dtype)
        for dy in (real, whole):
            b = torch.zeros(n, dtype=dtype, device="cuda", requires_grad=True)
            be = torch.zeros(3, n, dtype=dtype, device="cuda", requires_grad=True)
            got, = torch.autograd.grad(pk.packed_linear(x, p, b), b, dy)
            some, = torch.autograd.grad(pk.packed_expert_linear(x, pe, counts, be), be, dy)
            for part, d, r in [(got, dy, runs(m))] + [(some[e], dy[ends[e]:ends[e + 1]], runs(m, 3)) for e in range(3)]:
                want = d.double().sum(0)
                if dy is whole:
                    assert torch.equal(part, want.to(dtype)), m
                    continue
                depth = math.ceil(len(d) / (16 * r)) + 16 + r
                tol = eps * want.abs() + depth * 2.0 ** -24 * (1 + 2 * eps) * d.double().abs().sum(0)
                off = (part.double() - want).abs()
                assert not (off > tol).any(), (m, float((off / tol).max()))


def test_rows_of_large_and_small_activations(pk):
    """Forward, the sums run over code values before the scales come in: a sum of 128 values of up to 16 times an activation
    has to stay in float32, so activations below 2^116 do, and results are right wherever they themselves fit."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    n, k, g = 96, 512, 128
    for fmt in ("int4", "int4_asym", "flint4"):
        p = pk.pack_weight((torch.randn(n, k, generator=gen, device="cuda") * 0.02).half(), 4, fmt, g)
        unit = torch.randn(300, k, generator=gen, device="cuda").clamp_(-4, 4).bfloat16()
        for m in (3, 20, 300):
            want = pk.packed_linear(unit[:m], p)
            for e in (113, 60, -60, -90):
                x = (unit[:m].double() * 2.0 ** e).bfloat16()     # a power of two: every sum is the same times 2^e
                assert torch.equal(pk.packed_linear(x, p).double(), (want.double() * 2.0 ** e)), (fmt, m, e)
