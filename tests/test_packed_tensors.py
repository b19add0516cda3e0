"""CPU: which tensors, addresses and formats a packed weight hands on, with a stand-in for the launches."""
import copy
import ctypes
import io
import pickle
import weakref

import pytest
import torch
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad as fa
from torch.fx.experimental.proxy_tensor import make_fx

from quantization_amd import packed
from quantization_amd.quant_weight import quant_model


class StandIn:
    """libmq.so with launches that only note the addresses of the weight and the rows; sizes come from the library itself."""

    def __init__(self, real):
        self.real, self.seen, self.rows, self.bias = real, [], [], []

    def __getattr__(self, name):
        return getattr(self.real, name)

    def _note(self, ref, x):
        self.rows.append(x)
        c = ctypes.cast(ref, ctypes.POINTER(packed._W4)).contents
        self.seen.append((c.data, c.params, c.norm))
        return 0

    def mq_linear4(self, ref, x, dtype, rows, ld, bias, *args):
        self.bias.append(bias)
        return self._note(ref, x)

    def mq_linear4_grad(self, ref, dy, *args):
        return self._note(ref, dy)


@pytest.fixture
def launches(monkeypatch):
    s = StandIn(packed._bind())
    monkeypatch.setattr(packed, "_bound", s)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    monkeypatch.setattr(packed, "_on_device", lambda call, t, *args: call(t, *args, 0))
    return s


def host_weight(n=32, k=128, group=64, bits=4, fmt="int4", fill=0):
    """A weight whose tensors lie on the host."""
    c = packed._W4(experts=1, n=n, k=k, group=max(group, 0), kind=packed._kind_of(bits, fmt)[0])
    L = packed._bind()
    data = torch.full((L.mq_w4_data_bytes(1, n, k) // 4,), fill, dtype=torch.int32)
    params = torch.full((L.mq_w4_params_bytes(ctypes.byref(c)) // 2,), fill, dtype=torch.int16)
    return packed.PackedWeight(data, params, torch.ones(1, dtype=torch.int32), None, n, k, group, bits, fmt)


def addresses(w):
    return w.data.data_ptr(), w.params.data_ptr(), w.norm.data_ptr()


def rows(m=3, k=128):
    return torch.zeros(m, k, dtype=torch.float16)


def run(x, w, bias=None, counts=None):
    return packed._on_device(packed._forward, x, w, bias, counts)


def test_a_tensor_with_other_storage_is_taken_up(launches):
    """t.data = other keeps the tensor object and frees its memory."""
    w = host_weight()
    run(rows(), w)
    assert launches.seen[-1] == addresses(w)
    keep = []   # (the old memory must not be given out again at the same address)
    for name in ("data", "params", "norm"):
        t = getattr(w, name)
        keep.append(t.detach())
        t.data = t.data.clone()
        run(rows(), w)
        assert launches.seen[-1] == addresses(w), name
    w.data.data = w.data.data[:-4].clone()
    with pytest.raises(ValueError):
        run(rows(), w)


@pytest.fixture
def host_linear(monkeypatch):
    """PackedLinear on the host."""
    monkeypatch.setattr(packed, "pack_weight",
                        lambda w, bits, fmt, g: host_weight(w.shape[0], w.shape[1], g or 0, bits, fmt))
    return lambda n=32, k=128, group=64, bits=4, fmt="int4": packed.PackedLinear(nn.Linear(k, n).half(), bits, fmt, group)


BUFFERS = ("weight_data", "weight_params", "weight_norm")


@pytest.mark.parametrize("way", ["applied", "assigned", "loaded"])
def test_exchanged_buffers_are_let_go_at_once(host_linear, way):
    """The weight that a module no longer holds takes no memory: moving it away frees the device's."""
    m = host_linear()
    assert m.packed.data is m.weight_data
    old = [weakref.ref(getattr(m, b)) for b in BUFFERS]
    if way == "applied":
        m._apply(lambda t: t.clone())
    elif way == "assigned":
        for b in BUFFERS:
            setattr(m, b, getattr(m, b).clone())
    else:
        m.load_state_dict({k: v.clone() for k, v in m.state_dict().items()}, assign=True)
    assert [r() for r in old] == [None] * 3
    assert m.packed.data is m.weight_data and m.packed.params is m.weight_params and m.packed.norm is m.weight_norm


def test_a_saved_module_holds_its_weight_once(host_linear):
    m = host_linear(256, 1024)
    m.packed
    once = sum(getattr(m, b).numel() * getattr(m, b).element_size() for b in BUFFERS)
    for again in (pickle.loads(pickle.dumps(m)), copy.deepcopy(m)):
        assert again.packed.data is again.weight_data and again.packed.shape == m.packed.shape
        assert repr(again) == repr(m)
    m._buffers["weight_data"] = m.weight_data.clone()   # past the module's own ways
    file = io.BytesIO()
    torch.save(m, file)
    assert once < file.tell() < once + (1 << 16)
    assert m.packed.data is m.weight_data
    state = dict(m.__dict__, _packed=m.packed)          # as modules were saved that kept no description of their own
    del state["_form"]
    old = packed.PackedLinear.__new__(packed.PackedLinear)
    old.__setstate__(state)
    assert repr(old) == repr(m)


def test_a_weight_changed_between_forward_and_backward(launches, host_linear):
    """As torch does for the weights of its own products: the gradient is that of the forward's weight, or an error."""
    def forward(w):
        x = rows().requires_grad_()
        b = torch.zeros(w.n, dtype=torch.float16, requires_grad=True)
        return x, b, packed._PackedProduct.apply(x, b, w, None)

    for name in ("data", "params", "norm"):
        w = host_weight()
        x, b, y = forward(w)
        getattr(w, name).add_(1)
        with pytest.raises(RuntimeError, match="forward"):
            torch.autograd.grad(y, x, torch.ones_like(y))
        b = torch.zeros(w.n, dtype=torch.float16, requires_grad=True)
        y = packed._PackedProduct.apply(rows(), b, w, None)
        getattr(w, name).add_(1)
        torch.autograd.grad(y, b, torch.ones_like(y))      # a bias's gradient alone does not read the weight
        x, b, y = forward(w)
        torch.autograd.grad(y, x, torch.ones_like(y))
    # a state dict loaded under way: copied into the buffers, or (assign) beside the forward's
    m = host_linear()
    state = {k: v.clone() for k, v in m.state_dict().items()}
    x, b, y = forward(m.packed)
    m.load_state_dict(state)
    with pytest.raises(RuntimeError, match="forward"):
        torch.autograd.grad(y, x, torch.ones_like(y))
    x, b, y = forward(m.packed)
    was = addresses(m.packed)
    m.load_state_dict(state, assign=True)
    torch.autograd.grad(y, x, torch.ones_like(y))
    assert launches.seen[-1] == was != addresses(m.packed)
    with torch.inference_mode():                    # tensors without versions
        w = host_weight()
    x, b, y = forward(w)
    torch.autograd.grad(y, x, torch.ones_like(y))


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_differentiation_has_a_tangent(launches, grad):
    """The product is linear in x and in the bias: the tangent is one more product."""
    w = host_weight()
    bias = torch.zeros(w.n, dtype=torch.float16)
    for with_x, with_bias in ((True, True), (True, False), (False, True)):
        with fa.dual_level(), torch.set_grad_enabled(grad):
            x = fa.make_dual(rows(), rows()) if with_x else rows()
            b = fa.make_dual(bias, torch.ones_like(bias)) if with_bias else bias
            before = len(launches.seen)
            y = packed._run(x, w, b, None)
            assert fa.unpack_dual(y).tangent is not None
            assert fa.unpack_dual(y).tangent.shape == y.shape
            assert len(launches.seen) == before + 2
    with fa.dual_level():     # a tangent without memory
        y = packed._run(fa.make_dual(rows(), torch._efficientzerotensor((3, 128), dtype=torch.float16)), w, None, None)
        assert fa.unpack_dual(y).tangent is not None and launches.rows[-1]
    with fa.dual_level():     # nothing to differentiate
        y = packed._run(rows(), w, bias, None)
        assert fa.unpack_dual(y).tangent is None


def fakes(mode, w):
    with mode:
        at = lambda t: torch.empty(t.shape, dtype=t.dtype, device="cuda")
        return packed.PackedWeight(at(w.data), at(w.params), at(w.norm), w.experts, w.n, w.k, w.group_size, w.wq_bits, w.datatype)


def test_a_recorded_product_is_an_operator_of_the_graph():
    """Not the allocation of its result alone, which a replay would return unwritten."""
    mode = FakeTensorMode()
    w = fakes(mode, host_weight())
    with mode:
        x, b = (torch.empty(s, dtype=torch.float16, device="cuda") for s in ((4, 3, 128), (32,)))
        c = torch.empty(1, dtype=torch.int64, device="cuda")
    e = packed.PackedWeight(w.data, w.params, w.norm, 1, w.n, w.k, w.group_size, w.wq_bits, w.datatype)
    names = lambda g: [n.target.__name__ for n in g.graph.nodes if n.op == "call_function"]
    g = make_fx(lambda x, b: packed.packed_linear(x, w, b))(x, b)
    assert "packed_product.default" in names(g)
    g = make_fx(lambda x, c, b: packed.packed_expert_linear(x, e, c, b))(x[0], c, b[None])
    assert "packed_product.default" in names(g)
    assert "packed_dequantize.default" in names(make_fx(lambda x: w.dequantize() + x)(x[0, 0]))
    with mode:      # shapes and types alone
        assert packed.packed_linear(x, w, b).shape == (4, 3, 32) and w.dequantize().shape == (32, 128)
        tensors, form = w._operands()
        dx, db = torch.ops.quantization_amd.packed_product_grad(x[0, :, :32], *tensors, None, *form, True, False)
        assert dx.shape == (3, 128) and db.shape == (0,) and dx.dtype == torch.float16


def test_what_cannot_be_recorded_raises(launches):
    w = host_weight()
    with pytest.raises(NotImplementedError):        # (the operator has no host form)
        torch.jit.trace(lambda x: packed._run(x, w, None, None), rows())
    with pytest.raises(NotImplementedError):
        make_fx(lambda x: packed._run(x, w, None, None))(rows())
    assert not launches.seen
    q, s = torch.zeros(32, 128, dtype=torch.int8), torch.ones(32, 2, dtype=torch.float16)
    for record in (torch.jit.trace, lambda f, a: make_fx(f)(*a)):
        with pytest.raises(RuntimeError, match="recorded"):
            record(lambda q, s: packed.pack_codes(q, s, group_size=64).data, (q, s))
    x, b = rows(), torch.zeros(32, dtype=torch.float16)
    for f in (lambda: torch.ops.quantization_amd.packed_product(x, w.data, w.params, w.norm, b, None, 0, 32, 128, 64, 4, "int4"),
              lambda: torch.ops.quantization_amd.packed_dequantize(w.data, w.params, w.norm, 0, 32, 128, 64, 4, "int4")):
        with pytest.raises(NotImplementedError):
            f()


def test_a_state_dict_says_its_format(host_linear):
    """int4 and fp4 have buffers of the same sizes: the one's codes are not the other's."""
    forms = [dict(), dict(fmt="fp4"), dict(fmt="flint4"), dict(fmt="fp4_er_pos"), dict(fmt="fp3", bits=3)]
    for a in forms:
        state = host_linear(**a).state_dict()
        for b in forms:
            m = host_linear(**b)
            for assign in (False, True):
                for strict in (False, True):
                    if a == b:
                        m.load_state_dict(state, strict=strict, assign=assign)
                        continue
                    kept = {k: v.clone() for k, v in m.state_dict().items()}
                    state["weight_data"].fill_(7)
                    with pytest.raises(RuntimeError, match="format"):
                        m.load_state_dict(state, strict=strict, assign=assign)
                    assert all(torch.equal(v, kept[k]) for k, v in m.state_dict().items())
    # names and groupings that are decoded alike
    host_linear(bits=3, fmt="int3").load_state_dict(host_linear().state_dict())
    host_linear(group=None).load_state_dict(host_linear(group=-1).state_dict())
    host_linear(group=128).load_state_dict(host_linear(group=None).state_dict())
    # in a model, through a file, and from one that says nothing
    model = nn.Sequential(host_linear(), host_linear())
    file = io.BytesIO()
    torch.save(model.state_dict(), file)
    file.seek(0)
    state = torch.load(file, weights_only=True)
    model.load_state_dict(state)
    assert set(state) == {f"{i}.{b}" for i in (0, 1) for b in BUFFERS + ("bias", "weight_format")}
    with pytest.raises(RuntimeError, match="format"):
        nn.Sequential(host_linear(), host_linear(fmt="fp4")).load_state_dict(state)
    bare = {k: v for k, v in state.items() if not k.endswith("format")}
    with pytest.warns(UserWarning, match="format"):
        model.load_state_dict(bare)
    with pytest.raises(RuntimeError, match="spare"):     # strictness is as it was
        model.load_state_dict(dict(state, **{"0.spare": torch.zeros(1)}))
    assert "weight_format" not in dict(model.named_buffers())


def test_codes_that_the_format_does_not_hold_are_refused():
    """The kernel would keep them within its four bits, which is another weight."""
    check = packed._check_integers
    for dtype in (torch.int8, torch.uint8):      # bytes, read as the kind's integers
        check(torch.arange(16).to(dtype), packed.INT_ASYM)
        check(torch.arange(-7, 8).to(torch.int8).view(dtype), packed.INT_SYM)
        for v, kind in ((16, packed.INT_ASYM), (-1, packed.INT_ASYM), (-128, packed.INT_ASYM), (8, packed.INT_SYM),
                        (-8, packed.INT_SYM), (127, packed.INT_SYM), (-128, packed.INT_SYM)):
            with pytest.raises(ValueError, match="codes"):
                check(torch.tensor([3, v, 1], dtype=torch.int8).view(dtype), kind)


def test_quant_model_packs_a_shared_layer_in_all_its_places(host_linear):
    class Twice(nn.Module):
        def __init__(self):
            super().__init__()
            self.down = nn.Linear(128, 128)
            self.again = self.down
            self.blocks = nn.ModuleList([nn.Sequential(nn.Linear(128, 32), self.down)])
            self.blocks.append(self.blocks[0])

    m = Twice()
    quant_model(m, wq_bits=4, wq_datatype="int4", wq_groupsize=64, packed=True)
    assert isinstance(m.down, packed.PackedLinear) and isinstance(m.blocks[0][0], packed.PackedLinear)
    assert m.down is m.again is m.blocks[0][1] and m.blocks[0] is m.blocks[1]
    assert not [x for x in m.modules() if isinstance(x, nn.Linear)]
    # nothing holds a Linear that is the model itself: it cannot be swapped
    root = nn.Linear(128, 32)
    with pytest.raises(ValueError, match="PackedLinear"):
        quant_model(root, wq_bits=4, wq_datatype="int4", wq_groupsize=64, packed=True)
    assert list(root.named_children()) == []


def test_rows_of_another_shape_never_reach_the_library(launches):
    w = host_weight()
    for shape in ((128,), (2, 3, 128)):
        with pytest.raises(ValueError):
            run(torch.zeros(shape, dtype=torch.float16), w)
    assert not launches.seen


def test_forward_mode_over_a_backward_pass(launches):
    """dx and db are linear in dy: where dy has a tangent they have one, and operators called by name refuse one."""
    w = host_weight()
    x = rows().requires_grad_()
    b = torch.zeros(w.n, dtype=torch.float16, requires_grad=True)
    y = packed._run(x, w, b, None)
    with fa.dual_level():
        before = len(launches.seen)
        dx, db = torch.autograd.grad(y, (x, b), fa.make_dual(torch.ones_like(y), torch.ones_like(y)))
        assert fa.unpack_dual(dx).tangent is not None and fa.unpack_dual(db).tangent is not None
        assert len(launches.seen) == before + 2
    with fa.dual_level():      # the bias's tangent is read as it lies in memory: whole rows of it
        dual = fa.make_dual(torch.zeros(w.n, dtype=torch.float16), torch.ones(1, dtype=torch.float16).expand(w.n))
        packed._run(rows(), w, dual, None)
        assert launches.bias[-1] and launches.bias[-1] != launches.bias[-2]
    tensors, form = w._operands()
    forward, backward = packed._product_op._init_fn, packed._gradient_op._init_fn
    with fa.dual_level():
        with pytest.raises(NotImplementedError):
            forward(fa.make_dual(rows(), rows()), *tensors, None, None, *form)
        with pytest.raises(NotImplementedError):
            backward(fa.make_dual(rows(k=32), rows(k=32)), *tensors, None, *form, True, True)


def test_formats_in_other_clothes(host_linear):
    """A text of another integer type is read; one without contents (meta tensors) says nothing."""
    m = host_linear()
    state = dict(m.state_dict())
    state["weight_format"] = state["weight_format"].long()
    m.load_state_dict(state)
    meta = {k: v.to("meta") for k, v in state.items()}
    m.load_state_dict(meta, assign=True)
    assert m.weight_data.is_meta


def test_tensors_without_memory_are_not_taken_for_none(launches):
    """A wrapper's address is 0, which the library reads as "no bias" and "no counts"."""
    w = host_weight()
    e = packed.PackedWeight(w.data, w.params, w.norm, 1, w.n, w.k, w.group_size, w.wq_bits, w.datatype)
    b, c, y = torch.zeros(w.n, dtype=torch.float16), torch.ones(1, dtype=torch.int32), rows(k=w.n)
    calls = [(lambda b: run(rows(), w, b), b), (lambda c: run(rows(), e, None, c), c),
             (lambda c: packed._on_device(packed._backward, y, e, c, True, True), c)]
    for call, t in calls:
        call(t)
        before = len(launches.seen)
        with pytest.raises(RuntimeError):
            torch.func.functionalize(call)(t)
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(t[None])
        assert len(launches.seen) == before
