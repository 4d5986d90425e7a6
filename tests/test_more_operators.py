"""The dispatch of routed tokens and the 8-bit integer operators without a GPU: their sizes, and the calls that they refuse before
they touch a device (the pointers here are never followed)."""
import ctypes as C
import os
import random
import re

import numpy as np
import pytest

from tests import more_ref as ref
from tests.harness import moe
from tests.test_operators import refused
from c0ven_amd import _lib

P = 1 << 20  # a well aligned address
BIG = 1 << 40


def test_struct_layouts():
    rows = {name: (off, size) for name, off, size in moe.abi_layout()}
    for sname, cls in (("moe_dispatch_config", _lib.MoeDispatchConfig), ("moe_i8_matrix", _lib.I8Matrix),
                       ("moe_i8_experts", _lib.MoeI8Experts)):
        assert rows[sname] == (0, C.sizeof(cls))
        for f, _ in cls._fields_:
            d = getattr(cls, f)
            assert rows["%s.%s" % (sname, f)] == (d.offset, d.size)


# ---- dispatch

GOOD = dict(n_expert=64, n_used=4, n_embd=256, type=moe.QT_F32)


def calls(d, **args):
    """Every call of d, with some of its arguments replaced."""
    a = {**dict(x=P, ntok=8, ids=P, xs=P, order=P, places=P, offsets=P, work=P, work_bytes=BIG, y=P, dw=P, w=P, stride=256), **args}
    return {
        "dispatch": lambda: d.dispatch_async(a["x"], a["ntok"], a["ids"], a["xs"], a["order"], a["places"], a["offsets"], a["work"],
                                             a["work_bytes"], x_stride=a["stride"], xs_stride=a["stride"]),
        "combine": lambda: d.combine_async(a["x"], a["ntok"], a["places"], a["y"], a["w"], o_stride=a["stride"]),
        "combine to": lambda: d.combine_async(P, a["ntok"], a["places"], a["y"], a["w"], y_stride=a["stride"]),
        "dispatch_backward": lambda: d.dispatch_backward_async(a["x"], a["ntok"], a["places"], a["y"], dxs_stride=a["stride"]),
        "combine_backward": lambda: d.combine_backward_async(a["x"], a["ntok"], a["places"], P, a["y"], a["dw"], a["w"],
                                                             dy_stride=a["stride"]),
        "combine_backward of": lambda: d.combine_backward_async(P, a["ntok"], a["places"], a["x"], a["y"], a["dw"], a["w"],
                                                                o_stride=a["stride"]),
        "combine_backward to": lambda: d.combine_backward_async(P, a["ntok"], a["places"], P, a["y"], a["dw"], a["w"],
                                                                dout_stride=a["stride"]),
    }


@pytest.mark.parametrize("bad", [dict(n_expert=0), dict(n_expert=513), dict(n_used=0), dict(n_used=17), dict(n_embd=0),
                                 dict(n_embd=(1 << 20) + 1), dict(type=moe.QT_Q8_0), dict(type=99)])
def test_dispatch_refusals(bad):
    d = moe.Dispatch(**{**GOOD, **bad})
    assert d.work_bytes(1 << 18) == 0
    for call in calls(d).values():
        refused(call)


@pytest.mark.parametrize("args,which", [
    (dict(ntok=(1 << 20) + 1), "dispatch combine dispatch_backward combine_backward"), (dict(stride=255), "all"), (dict(stride=BIG + 1), "all"),
    (dict(places=None), "all"), (dict(places=P + 2), "all"), (dict(x=None), "dispatch combine dispatch_backward combine_backward"),
    (dict(x=P + 2), "dispatch combine dispatch_backward combine_backward"), (dict(ids=None), "dispatch"), (dict(ids=P + 1), "dispatch"),
    (dict(xs=P + 2), "dispatch"), (dict(order=None), "dispatch"), (dict(order=P + 2), "dispatch"), (dict(offsets=None), "dispatch"),
    (dict(offsets=P + 2), "dispatch"), (dict(y=None), "combine dispatch_backward"), (dict(y=P + 2), "combine dispatch_backward combine_backward"),
    (dict(w=P + 2), "combine combine_backward"), (dict(dw=P + 2), "combine_backward")])
def test_dispatch_refuses_buffers(args, which):
    for name, call in calls(moe.Dispatch(**GOOD), **args).items():
        if which == "all" or name in which.split():
            refused(call)


def test_dispatch_work():
    d = moe.Dispatch(512, 16, 256)
    assert d.work_bytes(1) == d.work_bytes(0) == 0 and d.work_bytes((1 << 20) + 1) == 0
    need = d.work_bytes(1 << 20)
    assert 0 < need <= 256 * 512 * 4
    for work, n in ((P, need - 1), (None, need), (P + 8, need)):
        refused(lambda: d.dispatch_async(P, 1 << 20, P, P, P, P, P, work, n), "work")


def test_dispatch_of_no_tokens():
    """The ways back do nothing; rows may be null, strides are checked all the same."""
    d = moe.Dispatch(**GOOD)
    d.combine_async(None, 0, None, None)
    d.dispatch_backward_async(None, 0, None, None)
    d.combine_backward_async(None, 0, None, None, None, P)
    d.combine_backward_async(P, 8, P)  # (neither gradient asked for)
    refused(lambda: d.combine_async(None, 0, None, None, o_stride=255))
    refused(lambda: d.dispatch_async(None, 0, None, None, None, None, None))  # (offsets are written)


# ---- 8-bit integers


def mat(rows=64, cols=256, codes=P, scales=P):
    return moe.I8Matrix(codes, scales, rows, cols)


def test_sizes():
    for rows, cols in ((1, 1), (3, 128), (7, 129), (5, 2560), (1 << 27, 1 << 16)):
        assert moe.i8_code_bytes(rows, cols) == rows * ref.pad128(cols)


@pytest.mark.parametrize("m", [mat(cols=0), mat(codes=None), mat(scales=None), mat(codes=P + 8), mat(scales=P + 2),
                               mat(cols=(1 << 16) + 1), mat(rows=(1 << 27) + 1)])
def test_i8_refuses_matrices(m):
    refused(lambda: moe.i8_quantize_async(moe.QT_F32, P, m, stride=BIG))
    refused(lambda: moe.i8_dequantize_async(m, moe.QT_F32, P, stride=BIG))
    refused(lambda: moe.i8_matmul_async(m, mat(), moe.QT_F32, P, P, BIG))
    refused(lambda: moe.i8_matmul_async(mat(), m, moe.QT_F32, P, P, BIG, y_stride=BIG))
    refused(lambda: moe.i8_linear_async(moe.QT_F32, P, 1, m, moe.QT_F32, P, P, BIG, x_stride=BIG, y_stride=BIG))


def test_i8_refuses_buffers():
    m = mat()
    for t, p, stride in ((moe.QT_Q8_0, P, 256), (moe.QT_F32, None, 256), (moe.QT_F32, P + 2, 256), (moe.QT_F16, P + 1, 256),
                         (moe.QT_F32, P, 255), (moe.QT_F32, P, BIG + 1)):
        refused(lambda: moe.i8_quantize_async(t, p, m, stride=stride))
        refused(lambda: moe.i8_dequantize_async(m, t, p, stride=stride))
        refused(lambda: moe.i8_matmul_async(m, mat(256), t, p, P, BIG, y_stride=stride))
        refused(lambda: moe.i8_linear_async(moe.QT_F32, P, 4, mat(256), t, p, P, BIG, y_stride=stride))
        refused(lambda: moe.i8_linear_async(t, p, 4, m, moe.QT_F32, P, P, BIG, x_stride=stride))
    refused(lambda: moe.i8_linear_async(moe.QT_F32, P, (1 << 27) + 1, m, moe.QT_F32, P, P, BIG), "tokens")
    refused(lambda: moe.i8_matmul_async(mat(1 << 27), mat((1 << 11) + 1), moe.QT_F32, P, P, BIG), "2^38")
    refused(lambda: moe.i8_matmul_async(m, mat(cols=257), moe.QT_F32, P, P, BIG), "same cols")
    need = moe.i8_linear_work_bytes(m, 40)
    assert need > 0
    for work, n in ((P, need - 1), (None, need), (P + 8, need)):
        refused(lambda: moe.i8_linear_async(moe.QT_F32, P, 40, m, moe.QT_F32, P, work, n), "work")
    with pytest.raises(moe.MoeError):
        _lib._op(_lib.lib.moe_i8_quantize_async(0, moe.QT_F32, P, 256, None, None))


@pytest.mark.parametrize("cols", [0, (1 << 16) + 1, 0xFFFFFF00, 0xFFFFFF81, 0xFFFFFFFF])
@pytest.mark.parametrize("rows,ntok", [(64, 40), (64, 4000), ((1 << 27) + 1, 40), (64, 1)])
def test_work_of_refused_sizes(rows, ntok, cols):
    m = mat(rows, cols)
    assert moe.i8_matmul_work_bytes(m, ntok) == 0 and moe.i8_linear_work_bytes(m, ntok) == 0


def test_work_of_sizes():
    m = mat(64, 1 << 16, None, None)
    assert moe.i8_matmul_work_bytes(m, 40) > 0 and moe.i8_linear_work_bytes(m, 40) > 0
    assert moe.i8_linear_work_bytes(m, 0) == 0 and moe.i8_matmul_work_bytes(m, 0) == 0
    for rows, ntok in (((1 << 27) + 1, 40), (64, (1 << 27) + 1)):
        m = mat(rows, 256)
        assert moe.i8_matmul_work_bytes(m, ntok) == 0 and moe.i8_linear_work_bytes(m, ntok) == 0


def experts(E=8, H=256, F=96, K=2, gate=None, up=None, down=None, **kw):
    return moe.I8Experts(H, F, E, K, gate or mat(F, H), up or mat(F, H), down or mat(H, F), **kw)


@pytest.mark.parametrize("bad", [dict(E=0), dict(E=513), dict(K=0), dict(K=17), dict(H=0), dict(F=0), dict(H=16385),
                                 dict(F=16385), dict(gate=mat(95, 256)), dict(up=mat(96, 255)), dict(down=mat(96, 256)),
                                 dict(gate=mat(96, 256, codes=None)), dict(up=mat(96, 256, scales=P + 1)),
                                 dict(x_type=moe.QT_Q4_K), dict(y_type=8), dict(swiglu_limit=-1.0),
                                 dict(swiglu_limit=float("nan")), dict(swiglu_limit=float("inf"))])
def test_experts_refusals(bad):
    e = experts(**bad)
    assert e.work_bytes(4) == 0
    refused(lambda: e.forward_async(P, 4, P, P, P, P, BIG))


def test_experts_refuses_buffers():
    e = experts()
    n = e.work_bytes(4)
    assert n > 0 and e.work_bytes(16385) == 0
    good = dict(x=P, ntok=4, ids=P, w=P, y=P, work=P, work_bytes=n)
    for bad in (dict(x=None), dict(x=P + 1), dict(y=None), dict(y=P + 1), dict(ids=None), dict(ids=P + 2), dict(w=None),
                dict(w=P + 2), dict(work=None), dict(work=P + 4), dict(work_bytes=n - 1), dict(ntok=16385),
                dict(x_stride=255), dict(y_stride=255)):
        refused(lambda: e.forward_async(**{**good, **bad}))


def test_empty_batches():
    w, none = mat(), moe.I8Matrix(None, None, 0, 256)
    moe.i8_quantize_async(moe.QT_F16, None, none)
    moe.i8_dequantize_async(none, moe.QT_F16, None)
    moe.i8_matmul_async(none, w, moe.QT_F32, None)
    moe.i8_linear_async(moe.QT_F32, None, 0, w, moe.QT_F32, None, None, 0)
    moe.i8_linear_async(moe.QT_F32, P, 4, none, moe.QT_F32, None, P, moe.i8_linear_work_bytes(none, 4))
    for E, H in ((8, 256), (512, 256), (8, 5)):
        assert experts(E=E, H=H).work_bytes(0) == 0
        experts(E=E).forward_async(None, 0, None, None, None, None, 0)
    refused(lambda: moe.i8_matmul_async(none, mat(codes=None), moe.QT_F32, None))
    refused(lambda: moe.i8_linear_async(moe.QT_F32, None, 4, none, moe.QT_F32, None, None, 0))
    refused(lambda: experts(gate=mat(96, 256, None)).forward_async(None, 0, None, None, None, None, 0))


def test_null_descriptions():
    lib, bad = _lib.lib, _lib.MOE_BAD_ARGUMENT
    assert lib.moe_dispatch_async(None, P, 8, 1, P, P, 8, P, P, P, P, 8, None) == bad
    assert lib.moe_combine_async(None, P, 8, 1, P, P, P, 8, None) == bad
    assert lib.moe_dispatch_backward_async(None, P, 8, 1, P, P, 8, None) == bad
    assert lib.moe_combine_backward_async(None, P, 8, 1, P, P, 8, P, P, 8, P, None) == bad
    assert lib.moe_i8_experts_async(None, P, 8, 1, P, P, P, 8, P, 8, None) == bad
    for size in (lib.moe_dispatch_work_bytes, lib.moe_i8_experts_work_bytes, lib.moe_i8_linear_work_bytes, lib.moe_i8_matmul_work_bytes):
        assert size(None, 1) == 0


# ---- the plain implementations


def test_reference_quantisation():
    """Halves go to the even code, every multiple of the scale is kept, the largest is 127; tiny, empty and infinite rows."""
    codes, s = ref.i8_quantize([[127, 0.5, 1.5, -2.5, 126.5, -127], [2.0 ** -149, 0, 0, 0, 0, 0], [0] * 6, [1, np.inf, 0, 0, 0, 0]])
    assert codes.tolist() == [[127, 0, 2, -2, 126, -127], [0] * 6, [0] * 6, [0] * 6]
    assert s[0] == 1 and s[1] == s[2] == 2.0 ** -100 and np.isnan(s[3])


def test_reference_dispatch():
    order, places, offsets = ref.dispatch(np.array([[2, 0], [0, -1], [5, 2]]), 3)
    assert order.tolist() == [1, 2, 0, 5, -1, -1] and offsets.tolist() == [0, 2, 2, 4]
    assert places.tolist() == [[2, 0], [1, -1], [-1, 3]]


@pytest.mark.parametrize("seed", range(4))
def test_code_by_sign(seed):
    """The kernels' rule for a code (floor of x / s by an approximate reciprocal, then the sign of x - (k + 1/2) s) gives the nearest
    integer of the exact quotient, next to borders and on them too."""
    r = random.Random(seed)
    from fractions import Fraction

    for _ in range(2000):
        s = np.float32(r.uniform(1, 2) * 2.0 ** r.randint(-100, 100))
        k = r.randint(-127, 126)
        x = np.float32((k + 0.5) * float(s)) if r.random() < 0.7 else np.float32(r.uniform(-127, 127) * float(s))
        for _ in range(r.randint(0, 2)):
            x = np.nextafter(x, np.float32(r.choice([-np.inf, np.inf])))
        inv = np.float32(np.float32(1) / s)
        inv = np.nextafter(inv, np.float32(r.choice([0, np.inf])))  # (a reciprocal off by a unit)
        f = int(np.floor(np.float32(x * inv)))
        d = Fraction(float(x)) - (f + Fraction(1, 2)) * Fraction(float(s))
        code = f + (1 if d > 0 else 0 if d < 0 else f & 1)
        exact = Fraction(float(x)) / Fraction(float(s))
        assert code == round(exact)


def test_kernels_do_not_spill():
    """Every kernel of these operators holds what it needs in registers; the experts' tiles of 64 run three waves a SIMD."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "c0ven_amd", "_build", "kernel_resources.txt")
    if not os.path.exists(path):
        pytest.skip("no build in this tree (run __graft_entry__.build())")
    rows = {}
    for line in open(path):
        name, *kv = line.split()
        if re.match(r"_ZN5c0ven\d+(i8_|sort_|dispatch_|combine_)", name):
            rows[name] = {k: int(v) if v.isdigit() else v for k, v in (x.split("=") for x in kv)}
    assert len(rows) >= 60
    for n, r in rows.items():
        assert r["scratch"] == 0, (n, r)
        if re.search(r"i8_(gate_up|down)_tilesILi1ELi2E", n):
            assert r["occupancy"] >= 3, (n, r)
