"""GPU: packed weights whose tensors are exchanged, moved, saved or changed under way; calls that are differentiated forwards
or recorded."""
import copy
import io

import pytest
import torch
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad as fa
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pk():
    from quantization_amd import packed
    return packed


def layer(pk, seed=0, n=96, k=256, fmt="int4", bits=4, g=64, bias=True):
    torch.manual_seed(seed)
    return pk.PackedLinear(nn.Linear(k, n, bias=bias).half().cuda(), bits, fmt, g)


def test_a_buffer_with_other_storage(pk):
    """t.data = other: the next call reads the new storage, whatever happens to the old one."""
    x = torch.randn(5, 256, device="cuda").half()
    m = layer(pk)
    want, deq = m(x), m.packed.dequantize()
    for name in ("weight_data", "weight_params", "weight_norm"):
        t = getattr(m, name)
        old = t.detach()
        t.data = t.data.clone()
        old.fill_(-1)
        assert torch.equal(m(x), want) and torch.equal(m.packed.dequantize(), deq), name
    xg = x.clone().requires_grad_()
    dx, = torch.autograd.grad(m(xg), xg, torch.ones_like(want))
    other = layer(pk)
    assert torch.equal(dx, torch.autograd.grad(other(xg), xg, torch.ones_like(want))[0])
    # away from the device under the same tensor object: refused, not read at the old address
    for name in ("weight_data", "weight_params", "weight_norm"):
        t = getattr(m, name)
        t.data = t.data.cpu()
    with pytest.raises(ValueError):
        m(x)


def test_a_layer_that_moves_away_frees_the_device(pk):
    m = layer(pk, n=2048, k=2048, bias=False)
    x = torch.randn(3, 2048, device="cuda").half()
    want = m(x).clone()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    size = sum(b.numel() * b.element_size() for b in m.buffers())
    m.cpu()
    assert torch.cuda.memory_allocated() <= before - size
    with pytest.raises(ValueError):
        m(x)
    assert torch.equal(m.cuda()(x), want)
    back = io.BytesIO()
    torch.save(m, back)
    assert back.tell() < size + (1 << 16)
    assert torch.equal(copy.deepcopy(m)(x), want)


def test_a_state_dict_loaded_between_forward_and_backward(pk):
    m, other = layer(pk), layer(pk, seed=1)
    x = torch.randn(40, 256, device="cuda").half().requires_grad_()
    dy = torch.randn(40, 96, device="cuda").half()
    want, = torch.autograd.grad(m(x), x, dy)
    y = m(x)
    m.load_state_dict(other.state_dict(), assign=True)     # beside the forward's weight
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], want)
    m = layer(pk)
    y = m(x)
    m.load_state_dict({k: v.clone() for k, v in other.state_dict().items()})
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, x, dy)
    assert torch.equal(m(x), other(x))


def test_forward_mode_differentiation(pk):
    """The tangent of a product is the product of the tangents, whether or not gradients are wanted too."""
    w = layer(pk, fmt="int4_asym").packed
    x, t = (torch.randn(5, 256, device="cuda").half() for _ in range(2))
    b, bt = (torch.randn(96, device="cuda").half() for _ in range(2))
    for grad in (False, True):
        with fa.dual_level(), torch.set_grad_enabled(grad):
            y, yt = fa.unpack_dual(pk.packed_linear(fa.make_dual(x, t), w, fa.make_dual(b, bt)))
            assert torch.equal(y, pk.packed_linear(x, w, b)) and torch.equal(yt, pk.packed_linear(t, w, bt))
            y, yt = fa.unpack_dual(pk.packed_linear(fa.make_dual(x, t), w, b))
            assert torch.equal(yt, pk.packed_linear(t, w))
            _, yt = fa.unpack_dual(pk.packed_linear(x, w, fa.make_dual(b, bt)))
            assert torch.equal(yt, bt.expand(5, 96))
            assert fa.unpack_dual(pk.packed_linear(x, w, b)).tangent is None
    e = pk.pack_weight(torch.randn(3, 96, 256, device="cuda").half(), 4, "int4", 64)
    c, be, bet = torch.tensor([2, 0, 2], device="cuda"), torch.randn(3, 96, device="cuda").half(), torch.randn(3, 96, device="cuda").half()
    with fa.dual_level():
        y, yt = fa.unpack_dual(pk.packed_expert_linear(fa.make_dual(x, t), e, c, fa.make_dual(be, bet)))
    assert torch.equal(y, pk.packed_expert_linear(x, e, c, be)) and torch.equal(yt, pk.packed_expert_linear(t, e, c, bet))
    with pytest.raises(RuntimeError):      # transforms that wrap tensors
        torch.func.jvp(lambda v: pk.packed_linear(v, w), (x,), (t,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda v: pk.packed_linear(v, w))(x[:, None])


class Counting(TorchDispatchMode):
    """Notes the operators that run inside."""

    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func.__name__)
        return func(*args, **(kwargs or {}))


class Named(torch.Tensor):
    pass


def test_recorded_products_replay_what_was_recorded(pk):
    """Traced, captured, exported and compiled programs multiply; they do not return memory that nobody has written."""
    m = layer(pk, fmt="int4_asym")
    stack = pk.pack_weight(torch.randn(3, 96, 256, device="cuda").half(), 4, "fp4", 64)
    counts = torch.tensor([2, 1, 2], device="cuda")
    x, x2 = (torch.randn(5, 256, device="cuda").half() for _ in range(2))
    w, b = m.packed, m.bias.detach()
    both = lambda x: (pk.packed_linear(x, w, b), pk.packed_expert_linear(x, stack, counts), stack.dequantize())
    with torch.no_grad():
        want = [t.clone() for t in both(x2)]
        traced = torch.jit.trace(both, x)
        file = io.BytesIO()
        layer_traced = torch.jit.trace(m, x)
        torch.jit.save(layer_traced, file)
        file.seek(0)
        programs = {"traced": traced, "make_fx": make_fx(both)(x),
                    "compiled": torch.compile(both, backend="aot_eager", fullgraph=True)}
        for name, f in programs.items():
            torch.full((1 << 16,), float("nan"), device="cuda")       # (what the allocator hands out next)
            assert all(torch.equal(a, b) for a, b in zip(f(x2), want)), name
        for f in (layer_traced, torch.jit.load(file), torch.export.export(m, (x,), strict=False).module()):
            assert torch.equal(f(x2), want[0])
    # with gradients: each program's own backward pass
    xg = x2.clone().requires_grad_()
    dy = torch.randn(5, 96, device="cuda").half()
    want = torch.autograd.grad(m(xg), (xg, m.bias), dy)
    for f in (torch.jit.trace(m, x), torch.compile(m, backend="aot_eager", fullgraph=True)):
        y = f(xg)
        assert torch.equal(y, m(xg))
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (xg, m.bias), dy), want))

    def gradients(x, dy):
        x = x.detach().requires_grad_()
        return torch.autograd.grad(pk.packed_linear(x, m.packed), x, dy)[0]

    assert torch.equal(make_fx(gradients)(x, dy)(x2, dy), want[0])
    # others that look on: the operator has a name, the results are the same
    with Counting() as seen:
        y = m(xg)
        got = torch.autograd.grad(y, (xg, m.bias), dy)
    assert "packed_product.default" in seen.names and "packed_product_grad.default" in seen.names
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    y = m(xg)
    with Counting() as seen:                                          # the backward pass alone
        got = torch.autograd.grad(y, (xg, m.bias), dy)
    assert "packed_product_grad.default" in seen.names and all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        assert torch.equal(torch.Tensor(m(x2.as_subclass(Named))), m(x2))
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        assert m(mode.from_tensor(x)).shape == (5, 96)
    assert torch.equal(m(xg), y)


def test_the_operators_refuse_what_does_not_fit(pk):
    w = layer(pk).packed
    tensors, form = w._operands()
    x, dy = torch.zeros(3, 256, device="cuda").half(), torch.zeros(3, 96, device="cuda").half()
    f, g = torch.ops.quantization_amd.packed_product, torch.ops.quantization_amd.packed_product_grad
    c = torch.zeros(1, dtype=torch.int32, device="cuda")
    for bad in (lambda: f(x[:, :255], *tensors, None, None, *form), lambda: f(x[0], *tensors, None, None, *form),
                lambda: f(x, *tensors, dy[0, :95], None, *form), lambda: f(x, *tensors, None, c, *form),
                lambda: f(x, *tensors, None, None, 2, *form[1:]), lambda: f(x, tensors[0][:4], *tensors[1:], None, None, *form),
                lambda: g(x, *tensors, None, *form, True, True), lambda: g(dy.float(), *tensors, None, *form, True, True),
                lambda: g(dy, *tensors, c, *form, True, True)):
        with pytest.raises(ValueError):
            bad()
    dx, db = g(dy, *tensors, None, *form, False, False)
    assert not dx.numel() and not db.numel()


def test_a_state_dict_of_another_format_is_refused(pk):
    x = torch.randn(5, 256, device="cuda").half()
    m, other = layer(pk), layer(pk, fmt="fp4")
    want = m(x)
    for assign in (False, True):
        with pytest.raises(RuntimeError):
            m.load_state_dict(other.state_dict(), assign=assign)
        assert torch.equal(m(x), want)
    again = layer(pk, seed=1)
    again.load_state_dict({k: v.cpu() for k, v in m.state_dict().items()})
    assert torch.equal(again(x), want)


def test_packing_refuses_codes_that_it_would_change(pk):
    s = torch.ones(8, 2, dtype=torch.float16, device="cuda")
    q = torch.randint(-7, 8, (8, 64), dtype=torch.int8, device="cuda")
    assert torch.equal(pk.pack_codes(q, s, group_size=32).dequantize(), q.half())
    for v in (-8, 8):
        q[3, 5] = v
        with pytest.raises(ValueError):
            pk.pack_codes(q, s, group_size=32)
    u = torch.randint(0, 16, (8, 64), dtype=torch.uint8, device="cuda")
    assert torch.equal(pk.pack_codes(u, s, s, datatype="int4_asym", group_size=32).dequantize(), u.half() - 1)
    u[0, 0] = 16
    with pytest.raises(ValueError):
        pk.pack_codes(u, s, s, datatype="int4_asym", group_size=32)
    t = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12], device="cuda").half().repeat(8, 8)
    assert torch.equal(pk.pack_codes(t, s, datatype="fp4", group_size=32).dequantize(), t)
    for v in (5, float("nan"), 16, float("-inf"), 0.5):
        u = t.clone()
        u[7, 63] = v
        with pytest.raises(ValueError):
            pk.pack_codes(u, s, datatype="fp4", group_size=32)
    from quantization_amd.fused import TABLE_LISTS
    for fmt, bits in (("flint4", 4), ("fp4_ea_pos", 4), ("fp4_er_neg", 4), ("fp3", 3), ("fp3_ea_neg", 3)):
        values = torch.tensor(sorted(set(TABLE_LISTS[fmt])), device="cuda").half()
        rows = values[torch.randint(0, len(values), (2, 33, 71), device="cuda")]
        rows[0, 0, :len(values)], rows[0, 0, 40] = values, -0.0
        one = torch.ones(2, 33, dtype=torch.float16, device="cuda")
        assert torch.equal(pk.pack_codes(rows, one, None, bits, fmt).dequantize(), rows)
        for v in (-16 if fmt == "fp4_ea_pos" else 7, float("nan"), 9, 1.5):
            bad = rows.clone()
            bad[1, 32, 70] = v
            with pytest.raises(ValueError):
                pk.pack_codes(bad, one, None, bits, fmt)


@pytest.mark.parametrize("fmt,bits", [("fp4", 4), ("flint4", 4), ("fp4_er_pos", 4), ("fp4_ea_neg", 4), ("fp3", 3), ("int4", 4),
                                      ("int4_asym", 4)])
def test_dequantize_with_one_scale_per_tensor(pk, fmt, bits):
    """The bits of the quantizers' dequantized weight (for tables not quant_datatype's, which are float32 arithmetic's)."""
    from quantization_amd import quant_weight as qw
    torch.manual_seed(3)
    w = (torch.randn(200, 320, device="cuda") * 0.02).half()
    got = pk.pack_weight(w, bits, fmt, -1).dequantize()
    if fmt.startswith("int"):
        want, again = qw._int_quant_meta(w, bits, "asym" in fmt, -1)[0], qw.quant_int_asym if "asym" in fmt else qw.quant_int
        again = again(w, bits, -1)
    else:
        want, again = qw._fp_quant_meta(w, bits, fmt, -1)[0], None
    bits_of = lambda t: torch.where(t == 0, 0, t.view(torch.int16))
    assert torch.equal(bits_of(got), bits_of(want))
    assert again is None or torch.equal(bits_of(got), bits_of(again))


def test_second_derivatives_forward_over_reverse(pk):
    """A Hessian times a vector: of f(x) = sum(y^2) / 2, y = x W^T + b, it is (v W^T) W."""
    w = layer(pk).packed
    b = torch.randn(96, device="cuda").half()
    x = (torch.randn(40, 256, device="cuda") * 0.1).half().requires_grad_()
    v = (torch.randn(40, 256, device="cuda") * 0.1).half()
    with fa.dual_level():
        y = pk.packed_linear(fa.make_dual(x, v), w, b)
        at, moves = fa.unpack_dual(y)
        dx, = torch.autograd.grad(y, x, fa.make_dual(at.detach(), moves.detach()))     # (detach alone would drop the tangent)
        primal, tangent = fa.unpack_dual(dx)
    with torch.no_grad():
        yv = pk.packed_linear(v, w)
    z = torch.zeros_like(x, requires_grad=True)
    assert torch.equal(primal, torch.autograd.grad(pk.packed_linear(z, w), z, pk.packed_linear(x, w, b).detach())[0])
    assert torch.equal(tangent, torch.autograd.grad(pk.packed_linear(z, w), z, yv)[0])


def test_the_operators_keep_torchs_rules(pk):
    """Schema, shapes and types without data, gradients and their recording, as torch checks its own operators."""
    tests = ("test_schema", "test_autograd_registration", "test_faketensor", "test_aot_dispatch_dynamic")
    for bias in (False, True):
        tensors, form = layer(pk, fmt="int4_asym").packed._operands()
        x = torch.randn(5, 256, device="cuda").half().requires_grad_()
        b = torch.randn(96, device="cuda").half().requires_grad_() if bias else None
        torch.library.opcheck(pk._product_op, (x, *tensors, b, None, *form), test_utils=tests)
        torch.library.opcheck(pk._gradient_op, (torch.randn(5, 96, device="cuda").half(), *tensors, None, *form, True, bias),
                              test_utils=tests)
    stack = pk.pack_weight(torch.randn(3, 96, 256, device="cuda").half(), 4, "fp4", 64)
    tensors, form = stack._operands()
    c = torch.tensor([2, 0, 2], device="cuda", dtype=torch.int32)
    be = torch.randn(3, 96, device="cuda").half().requires_grad_()
    torch.library.opcheck(pk._product_op, (x, *tensors, be, c, *form), test_utils=tests)
    torch.library.opcheck(pk._gradient_op, (torch.randn(5, 96, device="cuda").half(), *tensors, c, *form, True, True),
                          test_utils=tests)
    torch.library.opcheck(pk._dequantize_op, (*tensors, *form), test_utils=tests)
