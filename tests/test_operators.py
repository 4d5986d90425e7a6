"""The operators on device buffers without a GPU: their sizes, and the calls that they refuse before they touch a device
(the pointers here are never followed)."""
import ctypes as C
import os
import re

import numpy as np
import pytest

from tests import ops_ref as ref
from tests.harness import moe
from c0ven_amd import _lib

P = 1 << 20  # a well aligned address


def refused(call, *words):
    with pytest.raises(moe.MoeError) as e:
        call()
    assert e.value.status == _lib.MOE_BAD_ARGUMENT
    for w in words:
        assert w in str(e.value)


def test_struct_layouts():
    rows = {name: (off, size) for name, off, size in moe.abi_layout()}
    for sname, cls in (("moe_route_config", _lib.MoeRouteConfig), ("moe_mx4_matrix", _lib.Mx4Matrix),
                       ("moe_mx4_experts", _lib.MoeMx4Experts)):
        assert rows[sname] == (0, C.sizeof(cls))
        for f, _ in cls._fields_:
            d = getattr(cls, f)
            assert rows["%s.%s" % (sname, f)] == (d.offset, d.size)


def test_sizes():
    for rows, cols in ((1, 1), (3, 128), (7, 129), (5, 2560), (1 << 20, 1 << 14)):
        c = ref.pad128(cols)
        assert moe.mx4_code_bytes(rows, cols) == rows * c // 2
        assert moe.mx4_scale_bytes(rows, cols) == rows * c // 32


GOOD = dict(n_expert=64, n_used=4)


@pytest.mark.parametrize("bad", [dict(n_expert=0), dict(n_expert=513), dict(n_used=0), dict(n_used=17), dict(n_expert=3),
                                 dict(score=2), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
                                 dict(type=moe.QT_Q8_0), dict(n_group=5, top_group=1), dict(n_group=8, top_group=0),
                                 dict(n_group=8, top_group=9), dict(n_group=8, top_group=2, group_top=3),
                                 dict(n_group=8, top_group=2, group_top=0), dict(n_group=32, top_group=1),
                                 dict(n_expert=128, n_group=128, top_group=4)])
def test_route_refusals(bad):
    r = moe.Router(**{**GOOD, **bad})
    refused(lambda: r.route_async(P, 1, P, P))


@pytest.mark.parametrize("args", [dict(logits=None), dict(logits=P + 2), dict(ids=None), dict(w=None), dict(ids=P + 1),
                                  dict(load=P + 2), dict(bias=P + 1), dict(stride=63), dict(ntok=(1 << 24) + 1)])
def test_route_refuses_buffers(args):
    a = {**dict(logits=P, ntok=1, ids=P, w=P), **args}
    refused(lambda: moe.Router(**GOOD).route_async(**a))


def mat(rows=64, cols=256, codes=P, scales=P):
    return moe.Mx4Matrix(codes, scales, rows, cols)


@pytest.mark.parametrize("m", [mat(cols=0), mat(codes=None), mat(scales=None), mat(codes=P + 8), mat(scales=P + 4),
                               mat(cols=(1 << 20) + 1), mat(rows=(1 << 27) + 1)])
def test_mx4_refuses_matrices(m):
    big = 1 << 40
    refused(lambda: moe.mx4_quantize_async(moe.QT_F32, P, m, stride=big))
    refused(lambda: moe.mx4_dequantize_async(m, moe.QT_F32, P, stride=big))
    refused(lambda: moe.mx4_matmul_async(m, mat(), moe.QT_F32, P, P, big))
    refused(lambda: moe.mx4_matmul_async(mat(), m, moe.QT_F32, P, P, big, y_stride=big))
    refused(lambda: moe.mx4_linear_async(moe.QT_F32, P, 1, m, moe.QT_F32, P, P, big, x_stride=big, y_stride=big))


def test_mx4_refuses_buffers():
    m, big = mat(), 1 << 40
    for t, p, stride in ((moe.QT_Q8_0, P, 256), (moe.QT_F32, None, 256), (moe.QT_F32, P + 2, 256), (moe.QT_F16, P + 1, 256),
                         (moe.QT_F32, P, 255), (moe.QT_F32, P, big + 1)):
        refused(lambda: moe.mx4_quantize_async(t, p, m, stride=stride))
        refused(lambda: moe.mx4_dequantize_async(m, t, p, stride=stride))
        refused(lambda: moe.mx4_matmul_async(m, mat(256), t, p, P, big, y_stride=stride))
        refused(lambda: moe.mx4_linear_async(moe.QT_F32, P, 4, mat(256), t, p, P, big, y_stride=stride))
        refused(lambda: moe.mx4_linear_async(t, p, 4, m, moe.QT_F32, P, P, big, x_stride=stride))
    refused(lambda: moe.mx4_linear_async(moe.QT_F32, P, (1 << 27) + 1, m, moe.QT_F32, P, P, big), "tokens")
    refused(lambda: moe.mx4_matmul_async(mat(1 << 27), mat((1 << 11) + 1), moe.QT_F32, P, P, big), "2^38")
    refused(lambda: moe.mx4_matmul_async(m, mat(cols=257), moe.QT_F32, P, P, big), "same cols")
    need = moe.mx4_linear_work_bytes(m, 40)
    assert need > 0
    for work, n in ((P, need - 1), (None, need), (P + 8, need)):
        refused(lambda: moe.mx4_linear_async(moe.QT_F32, P, 40, m, moe.QT_F32, P, work, n), "work")
    with pytest.raises(moe.MoeError):
        _lib._op(_lib.lib.moe_mx4_quantize_async(0, moe.QT_F32, P, 256, None, None))


@pytest.mark.parametrize("cols", [0, (1 << 20) + 1, 0xFFFFFF00, 0xFFFFFF81, 0xFFFFFFFF])
@pytest.mark.parametrize("rows,ntok", [(64, 40), (64, 4000), ((1 << 27) + 1, 40), (64, 1)])
def test_work_of_refused_sizes(rows, ntok, cols):
    """Sizes that the calls refuse ask for no work, where 32 bits hold no row's length rounded up among them."""
    m = mat(rows, cols)
    assert moe.mx4_matmul_work_bytes(m, ntok) == 0 and moe.mx4_linear_work_bytes(m, ntok) == 0


def test_work_of_sizes():
    m = mat(64, 1 << 20, None, None)
    assert moe.mx4_matmul_work_bytes(m, 40) > 0 and moe.mx4_linear_work_bytes(m, 40) > 0
    for rows, ntok in (((1 << 27) + 1, 40), (64, (1 << 27) + 1)):
        m = mat(rows, 256)
        assert moe.mx4_matmul_work_bytes(m, ntok) == 0 and moe.mx4_linear_work_bytes(m, ntok) == 0


def experts(E=8, H=256, F=96, K=2, gate=None, up=None, down=None, **kw):
    return moe.Mx4Experts(H, F, E, K, gate or mat(F, H), up or mat(F, H), down or mat(H, F), **kw)


@pytest.mark.parametrize("bad", [dict(E=0), dict(E=513), dict(K=0), dict(K=17), dict(H=0), dict(F=0), dict(H=16385),
                                 dict(F=16385), dict(gate=mat(95, 256)), dict(up=mat(96, 255)), dict(down=mat(96, 256)),
                                 dict(gate=mat(96, 256, codes=None)), dict(up=mat(96, 256, scales=P + 1)),
                                 dict(x_type=moe.QT_Q4_K), dict(y_type=8), dict(swiglu_limit=-1.0),
                                 dict(swiglu_limit=float("nan"))])
def test_experts_refusals(bad):
    e = experts(**bad)
    assert e.work_bytes(4) == 0
    refused(lambda: e.forward_async(P, 4, P, P, P, P, 1 << 40))


def test_experts_refuses_buffers():
    e = experts()
    n = e.work_bytes(4)
    assert n > 0 and e.work_bytes(16385) == 0
    good = dict(x=P, ntok=4, ids=P, w=P, y=P, work=P, work_bytes=n)
    for bad in (dict(x=None), dict(x=P + 1), dict(y=None), dict(y=P + 1), dict(ids=None), dict(ids=P + 2), dict(w=None),
                dict(w=P + 2), dict(work=None), dict(work=P + 4), dict(work_bytes=n - 1), dict(ntok=16385),
                dict(x_stride=255), dict(y_stride=255)):
        refused(lambda: e.forward_async(**{**good, **bad}))


@pytest.mark.parametrize("E", [8, 512])
def test_experts_of_no_tokens(E):
    """No work, nothing to do, no device touched."""
    e = experts(E=E)
    assert e.work_bytes(0) == 0
    e.forward_async(P, 0, P, P, P, None, 0)
    refused(lambda: e.forward_async(P, 0, P, P, P, None, 0, x_stride=255))


def test_empty_batches():
    """Buffers of no tokens may be null, as an empty tensor's are; those that do hold something may not."""
    w, none = mat(), moe.Mx4Matrix(None, None, 0, 256)
    moe.Router(**GOOD).route_async(None, 0, None, None)
    moe.mx4_quantize_async(moe.QT_F16, None, none)
    moe.mx4_dequantize_async(none, moe.QT_F16, None)
    moe.mx4_matmul_async(none, w, moe.QT_F32, None)
    moe.mx4_linear_async(moe.QT_F32, None, 0, w, moe.QT_F32, None, None, 0)
    moe.mx4_linear_async(moe.QT_F32, P, 4, none, moe.QT_F32, None, None, 0)
    experts().forward_async(None, 0, None, None, None, None, 0)
    refused(lambda: moe.mx4_matmul_async(none, mat(codes=None), moe.QT_F32, None))
    refused(lambda: moe.mx4_linear_async(moe.QT_F32, None, 4, none, moe.QT_F32, None, None, 0))
    refused(lambda: experts(gate=mat(96, 256, None)).forward_async(None, 0, None, None, None, None, 0))
    refused(lambda: moe.Router(**GOOD).route_async(None, 0, P + 1, None))


def test_null_descriptions():
    assert _lib.lib.moe_route_async(None, P, 8, None, 1, P, P, None, None) == _lib.MOE_BAD_ARGUMENT
    assert _lib.lib.moe_mx4_experts_async(None, P, 8, 1, P, P, P, 8, P, 8, None) == _lib.MOE_BAD_ARGUMENT
    assert _lib.lib.moe_mx4_experts_work_bytes(None, 1) == 0
    assert _lib.lib.moe_mx4_linear_work_bytes(None, 1) == 0 and _lib.lib.moe_mx4_matmul_work_bytes(None, 1) == 0


def test_reference_quantisation():
    """The plain implementation against the format's own table: every value of it is kept, halves go to the even code."""
    x = np.concatenate([ref.VALUES, -ref.VALUES, ref.BORDERS, [6.0]])[None]
    got = ref.mx4(x)[0]
    assert np.array_equal(got[:16], x[0, :16])
    assert np.array_equal(got[16:23], [0, 1, 1, 2, 2, 4, 4])
    assert np.array_equal(ref.mx4(np.array([[7.9, 5.1, 0.2]])), [[6, 6, 0]])


def test_kernels_do_not_spill():
    """Every kernel of the operators holds what it needs in registers; the experts' tiles of 64 run three waves a SIMD."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "c0ven_amd", "_build", "kernel_resources.txt")
    if not os.path.exists(path):
        pytest.skip("no build in this tree (run __graft_entry__.build())")
    rows = {}
    for line in open(path):
        name, *kv = line.split()
        if re.match(r"_ZN5c0ven\d+(mx4_|moe_route|route_)", name):
            rows[name] = {k: int(v) if v.isdigit() else v for k, v in (x.split("=") for x in kv)}
    assert len(rows) >= 60
    for n, r in rows.items():
        assert r["scratch"] == 0, (n, r)
        if re.search(r"mx4_(gate_up|down)_tilesILi1ELi2E", n):
            assert r["occupancy"] >= 3, (n, r)
