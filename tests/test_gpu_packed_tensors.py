"""GPU: packed weights whose tensors are exchanged, moved, saved or changed under way; calls that are differentiated forwards
or recorded."""
import copy
import io

import pytest
import torch
import torch.nn as nn
from torch.autograd import forward_ad as fa

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
