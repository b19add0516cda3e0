"""CPU: what the 4-bit products refuse and decide before any GPU call."""
import ctypes

import pytest
import torch
import torch.nn as nn

from quantization_amd import _lib, packed
from quantization_amd.fused import TABLE_LISTS, lut_values


def _c(experts=1, n=64, k=256, group=128, kind=packed.INT_SYM, ptr=4096):
    return packed._W4(data=ptr, params=ptr, norm=ptr, experts=experts, n=n, k=k, group=group, kind=kind)


def test_table_order_holds_every_list():
    for name in ("fp3", "fp3_er_pos", "fp3_er_neg", "fp3_ea_pos", "fp3_ea_neg", "flint4", "fp4_er_pos", "fp4_er_neg", "fp4_ea_pos",
                 "fp4_ea_neg"):
        t = packed.table_order(TABLE_LISTS[name])
        assert len(t) == 16 and t[0] == 0.0 and set(t) == set(TABLE_LISTS[name]), name
    assert packed.table_order(lut_values("fp4")) == [0, 1, 2, 3, 4, 6, 8, 12, 0, -1, -2, -3, -4, -6, -8, -12]
    with pytest.raises(ValueError):
        packed.table_order(range(-8, 9))


@pytest.mark.parametrize("bits,name", [(8, "int8"), (5, "int5"), (1, "int4"), (4, "fp5"), (8, "fp8_e4m3"), (4, "mx_fp4"),
                                       (4, "mixed_bitmod"), (4, ""), (4, None), (3, "fp4")])
def test_formats_that_are_refused(bits, name):
    with pytest.raises(ValueError):
        packed._kind_of(bits, name)


def test_library_refuses_before_any_launch():
    L = packed._bind()
    ref = ctypes.byref
    big = 1 << 40
    assert L.mq_w4_data_bytes(1, 17, 129) == 2 * 2 * 1024
    assert L.mq_w4_data_bytes(0, 1, 1) == 0 and L.mq_w4_data_bytes(1, 1 << 23, 1) == 0 and L.mq_w4_data_bytes(1, 1, 1 << 21) == 0
    assert L.mq_w4_params_bytes(ref(_c(n=17, k=96, group=32))) == 2 * 4 * 16 * 2    # groups of the padded 128 columns
    assert L.mq_w4_params_bytes(ref(_c(n=17, k=96, group=0, kind=packed.INT_ASYM))) == 2 * 16 * 4
    assert L.mq_w4_params_bytes(ref(_c(k=250))) == 0
    call = lambda c, rows=4, dt=_lib.F16, x=4096, ld=256, y=4096, counts=None, ws=None, size=0: L.mq_linear4(
        ref(c), x, dt, rows, ld, None, counts, y, ws, size, None)
    assert call(_c(), rows=0) == _lib.OK
    assert call(_c(), rows=-1) == _lib.ERR_ARG
    assert call(_c(), rows=big) == _lib.ERR_TOO_LARGE
    assert call(_c(), dt=_lib.F32) == _lib.ERR_UNSUPPORTED
    assert call(_c(group=100)) == _lib.ERR_GROUP
    assert call(_c(k=240, group=48)) == _lib.ERR_UNSUPPORTED
    assert call(_c(group=-1)) == _lib.ERR_ARG
    assert call(_c(kind=4)) == _lib.ERR_ARG
    assert call(_c(experts=2)) == _lib.ERR_ARG                  # experts without counts
    assert call(_c(), ld=255) == _lib.ERR_ARG                   # rows that overlap
    assert call(_c(), x=None) == _lib.ERR_ARG
    assert call(_c(), x=4097) == _lib.ERR_ALIGN
    assert call(_c(), y=4104) == _lib.ERR_ALIGN
    assert call(_c(ptr=4098)) == _lib.ERR_ALIGN
    assert call(_c(), counts=4098) == _lib.ERR_ALIGN
    bad = _c(kind=packed.TABLE)
    bad.values[1] = 17.5                                        # not an e4m3 number
    assert call(bad) == _lib.ERR_UNSUPPORTED
    bad.values[0], bad.values[1] = 1.0, 1.0
    assert call(bad) == _lib.ERR_UNSUPPORTED                    # entry 0 is what padding decodes to
    assert call(_c(n=1 << 22, k=1 << 20, group=0), rows=1 << 27, ld=1 << 20) in (_lib.ERR_TOO_LARGE, _lib.ERR_WORKSPACE)
    need = L.mq_linear4_workspace_bytes(ref(_c()), _lib.F16, 4, 1, 0, 1)     # the gradient's turned operand
    assert need >= 16 * 1024
    back = lambda dx, db, ws, size, c=_c(), dt=_lib.F16: L.mq_linear4_grad(ref(c), 4096, dt, 4, 64, None, dx, db, ws, size, None)
    assert back(4096, None, None, 0) == _lib.ERR_WORKSPACE
    assert back(4096, None, 4096, need - 1) == _lib.ERR_WORKSPACE
    assert back(None, None, 4096, big) == _lib.ERR_ARG
    assert back(None, 4097, 4096, big) == _lib.ERR_ALIGN
    assert back(None, 4096, 4096, big, dt=_lib.F32) == _lib.ERR_UNSUPPORTED
    assert back(None, 4096, 4096, big, c=_c(experts=3)) == _lib.ERR_ARG
    assert L.mq_linear4_workspace_bytes(ref(_c()), _lib.F16, 4, 1, 0, 2) == 0
    assert L.mq_linear4_workspace_bytes(ref(_c()), _lib.F16, 4096, 1, 0, 2) > 0      # runs of rows, added by a second launch
    assert L.mq_w4_pack(ref(_c()), None, 4096, None, None) == _lib.ERR_ARG
    assert L.mq_w4_pack(ref(_c()), 4096, 4096, 4096, None) == _lib.ERR_ARG         # a zero point with symmetric codes
    assert L.mq_w4_unpack(ref(_c()), None, None) == _lib.ERR_ARG


def test_pack_codes_refuses_what_does_not_belong_together():
    q, s = torch.zeros(8, 64, dtype=torch.int8), torch.ones(8, 2, dtype=torch.float16)
    bad = [dict(q=q.float(), scale=s, group_size=32), dict(q=q, scale=s.float(), group_size=32), dict(q=q, scale=s[:4], group_size=32),
           dict(q=q, scale=s, zp=s, group_size=32), dict(q=q, scale=s, datatype="int4_asym", group_size=32),
           dict(q=q, scale=s, datatype="fp4", group_size=32), dict(q=q[:0], scale=s[:0], group_size=32),
           dict(q=q, scale=s, group_size=None), dict(q=q, scale=torch.ones(8, 4, dtype=torch.float16), group_size=16),
           dict(q=q[None], scale=s, group_size=32)]
    for kw in bad:
        with pytest.raises(ValueError):
            packed.pack_codes(**kw)
    with pytest.raises(RuntimeError):   # as the reference's reshape
        packed.pack_codes(q, s, group_size=48)


def test_products_refuse_host_tensors_and_quant_model_refuses_other_formats():
    w = object.__new__(packed.PackedWeight)
    w.n, w.k, w.experts = 8, 64, None
    with pytest.raises(RuntimeError):
        packed.packed_linear(torch.zeros(1, 64, dtype=torch.float16), w)
    with pytest.raises(TypeError):
        packed.packed_linear(torch.zeros(1, 64, dtype=torch.float16), torch.zeros(8, 64))
    from quantization_amd.quant_weight import quant_model
    model = nn.Sequential(nn.Linear(32, 32))
    for bits, name in ((4, "mx_fp4"), (4, "mixed_bitmod"), (8, "int8"), (8, "fp8_e4m3")):
        with pytest.raises(ValueError):
            quant_model(model, wq_bits=bits, wq_datatype=name, wq_groupsize=None, packed=True)
    assert isinstance(model[0], nn.Linear)
