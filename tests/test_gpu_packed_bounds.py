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
