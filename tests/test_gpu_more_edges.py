"""The dispatch and the 8-bit integer operators on the GPU with every buffer at its least alignment, and with scales that are no
numbers among the experts: the bits of a call on aligned buffers, and nothing beside the buffers written."""
import numpy as np
import pytest

from tests import more_ref as ref
from tests.harness import moe
from tests.ops_dev import TYPES, encode, hip
from tests.test_gpu_dispatch import draw_ids, say
from tests.test_gpu_i8 import operand
from tests.test_gpu_i8_experts import Model, run, tokens

pytestmark = pytest.mark.gpu


class Room:
    """Buffers of bytes, each `by` bytes past an aligned address, between guards."""

    def __init__(self, far):
        self.far, self.all = far, []

    def put(self, a, by):
        """a's copy at its least alignment (`by` bytes), or aligned; its pointer."""
        a = np.ascontiguousarray(a)
        at = 256 + (by if self.far else 0)
        raw = np.full(at + a.nbytes + 256, 0xA5, np.uint8)
        raw[at:at + a.nbytes] = a.reshape(-1).view(np.uint8)
        b = hip.put(raw)
        self.all.append((b, at, a))
        return b.ptr + at

    def get(self, i):
        b, at, a = self.all[i]
        raw = b.get()
        assert (raw[:at] == 0xA5).all() and (raw[at + a.nbytes:] == 0xA5).all()
        return raw[at:at + a.nbytes].view(a.dtype).reshape(a.shape)


def alike(call):
    """call(room) returns which of the room's buffers are results: the same bytes at the least alignment."""
    got = []
    for far in (False, True):
        room = Room(far)
        got.append([room.get(i) for i in call(room)])
        for i in range(len(room.all)):
            room.get(i)  # (guards)
    for a, b in zip(*got):
        assert np.array_equal(a, b)
    return got[0]


def bytes_of(n):
    return np.full(max(n, 16), 0xA5, np.uint8)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("T,K,H", [(1, 10, 2048), (30, 3, 5), (700, 4, 130), (999, 4, 2561)])
def test_dispatch(T, K, H, type):
    say("aligned dispatch", T, K, H, type)
    E, size = 60, 4 if type == "f32" else 2
    r = np.random.default_rng(T)
    ids = draw_ids(T, K, E, T)
    x = encode(r.normal(size=(T, H)), type)
    zero = np.zeros_like(encode(np.zeros((T * K, H)), type))
    o, dy, w = encode(r.normal(size=(T * K, H)), type), encode(r.normal(size=(T, H)), type), r.normal(size=(T, K)).astype(np.float32)
    d = moe.Dispatch(E, K, H, TYPES[type])

    def call(room):
        p = [room.put(a, by) for a, by in ((x, size), (ids, 4), (zero, size), (np.zeros(T * K, np.int32), 4), (np.zeros((T, K), np.int32), 4),
                                           (np.zeros(E + 1, np.int32), 4), (bytes_of(d.work_bytes(T)), 16), (o, size), (w, 4),
                                           (np.zeros_like(x), size), (dy, size), (zero, size), (np.zeros((T, K), np.float32), 4),
                                           (np.zeros_like(x), size))]
        d.dispatch_async(p[0], T, p[1], p[2], p[3], p[4], p[5], p[6], d.work_bytes(T))
        d.combine_async(p[7], T, p[4], p[9], p[8])
        d.combine_backward_async(p[10], T, p[4], p[7], p[11], p[12], p[8])
        d.dispatch_backward_async(p[7], T, p[4], p[13])
        return 2, 3, 4, 5, 9, 11, 12, 13

    got = alike(call)
    order, places, offsets = ref.dispatch(ids, E)
    assert np.array_equal(got[1], order) and np.array_equal(got[2], places) and np.array_equal(got[3], offsets)


@pytest.mark.parametrize("type", ["f32", "f16"])
@pytest.mark.parametrize("M,N,K", [(1, 100, 2048), (5, 77, 5), (16, 40, 3000), (17, 100, 3000), (300, 300, 130), (1500, 1500, 130),
                                   (600, 8200, 200), (3500, 3500, 200)])
def test_products(M, N, K, type):
    say("aligned products", M, N, K, type)
    size = 4 if type == "f32" else 2
    w, s = operand(N, K, 3)
    codes, scales = ref.i8_padded(w), s.astype(np.float32)
    x = encode(np.random.default_rng(M).normal(size=(M, K)), type)

    def call(room):
        p = [room.put(a, by) for a, by in ((x, size), (codes, 16), (scales, 4), (np.zeros((M, ref.pad128(K)), np.int8), 16),
                                           (np.zeros(M, np.float32), 4), (encode(np.zeros((M, N)), type), size), (encode(np.zeros((M, N)), type), size),
                                           (np.zeros_like(x), size))]
        wm, xm = moe.I8Matrix(p[1], p[2], N, K), moe.I8Matrix(p[3], p[4], M, K)
        n, n2 = moe.i8_matmul_work_bytes(wm, M), moe.i8_linear_work_bytes(wm, M)
        work, work2 = room.put(bytes_of(n), 16), room.put(bytes_of(n2), 16)
        moe.i8_quantize_async(TYPES[type], p[0], xm)
        moe.i8_matmul_async(xm, wm, TYPES[type], p[5], work, n)
        moe.i8_linear_async(TYPES[type], p[0], M, wm, TYPES[type], p[6], work2, n2)
        moe.i8_dequantize_async(xm, TYPES[type], p[7])
        return 3, 4, 5, 6, 7

    got = alike(call)
    assert np.array_equal(got[2], got[3])


@pytest.mark.parametrize("T,H,F,E,K", [(1, 300, 129, 20, 10), (8, 512, 96, 12, 4), (16, 256, 600, 12, 10), (60, 2100, 200, 8, 3), (900, 256, 100, 12, 4)])
def test_experts(T, H, F, E, K):
    say("aligned experts", T, H, F, E, K)
    x, ids, w = tokens(T, H, E, K, T, 0.1)
    x, ids, w = encode(x, "bf16"), ids.astype(np.int32), w.astype(np.float32)
    r, mats = np.random.default_rng(H), []
    for rows, cols in ((F, H), (F, H), (H, F)):
        c, s = ref.i8_quantize((r.normal(size=(E * rows, cols)) * 0.05).astype(np.float32))
        mats.append((ref.i8_padded(c), s.astype(np.float32), rows, cols))

    def call(room):
        p = [room.put(a, by) for a, by in ((x, 2), (ids, 4), (w, 4), (np.zeros_like(x), 2))]
        m = [moe.I8Matrix(room.put(c, 16), room.put(s, 4), rows, cols) for c, s, rows, cols in mats]
        op = moe.I8Experts(H, F, E, K, *m)
        n = op.work_bytes(T)
        op.forward_async(p[0], T, p[1], p[2], p[3], room.put(bytes_of(n), 16), n)
        return (3,)

    assert alike(call)[0].any()


@pytest.mark.parametrize("T", [2, 16, 60, 900])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_scales_that_are_no_numbers(T, which):
    """NaN in the scales of one expert's matrix: its tokens' results are NaN (down: in that row's column), the others have the bits
    that they have without."""
    say("nan scales", T, which)
    E, H, F, K, bad = 8, 256, 96, 2, 3
    model = Model(E, H, F, 4)
    x, ids, w = tokens(T, H, E, K, 3, 0.1)
    ids[0, 0], ids[1] = bad, [1, 2]
    clean, _ = run(model, x, ids, w)
    values, buf = model.hold[2 * which + 1]
    rows = model.m[which].rows
    poisoned = values.copy()
    at = bad * rows + rows - 1  # (the matrix's last row: the next expert's follow)
    poisoned[at] = np.nan
    buf.put(poisoned)
    got, _ = run(model, x, ids, w)
    hit = (ids == bad).any(-1)
    if which == 2:
        assert np.isnan(got[hit, H - 1]).all()
        assert np.array_equal(got[:, :H - 1], clean[:, :H - 1])
    else:
        assert np.isnan(got[hit]).all()
    assert np.array_equal(got[~hit], clean[~hit]) and not hit[1]


def replayed(inputs, results, call):
    """call(results, stream) captured and replayed on new inputs, between eager calls on other results: the same bytes. inputs: (buffer,
    maker of its contents); results: twice the same buffers."""
    s1, s2 = hip.stream(), hip.stream()
    launch = hip.capture(s1, lambda: call(results[0], s1))
    for i in range(3):
        for b, make in inputs:
            b.put(make(i))
        launch()
        call(results[1], s2)
        for a, b in zip(*results):  # (work, where it is among them, too)
            assert np.array_equal(a.get(), b.get())


def test_graph_of_many_tokens():
    """The dispatch of several slices of ids and the ways back, captured."""
    say("graph of many tokens")
    T, K, E, H = 1500, 8, 60, 300
    d = moe.Dispatch(E, K, H)
    x, ids, w = hip.full((T, H), 0, np.uint16), hip.full((T, K), 0, np.int32), hip.full((T, K), 0)
    n = d.work_bytes(T)
    assert n > 0

    def results():
        return [hip.full((T * K, H), 0, np.uint16), hip.full(T * K, 0, np.int32), hip.full((T, K), 0, np.int32), hip.full(E + 1, 0, np.int32),
                hip.full((T, H), 0, np.uint16), hip.full((T * K, H), 0, np.uint16), hip.full((T, K), 0), hip.full((T, H), 0, np.uint16),
                hip.full(n, 0xA5, np.uint8)]

    def call(b, s):
        d.dispatch_async(x.ptr, T, ids.ptr, b[0].ptr, b[1].ptr, b[2].ptr, b[3].ptr, b[8].ptr, n, stream=s)
        d.combine_async(b[0].ptr, T, b[2].ptr, b[4].ptr, w.ptr, stream=s)
        d.combine_backward_async(x.ptr, T, b[2].ptr, b[0].ptr, b[5].ptr, b[6].ptr, w.ptr, stream=s)
        d.dispatch_backward_async(b[5].ptr, T, b[2].ptr, b[7].ptr, stream=s)

    replayed([(x, lambda i: encode(np.random.default_rng(i).normal(size=(T, H)), "bf16")), (ids, lambda i: draw_ids(T, K, E, i, 0.0)),
              (w, lambda i: np.random.default_rng(i).normal(size=(T, K)).astype(np.float32))], [results(), results()], call)


@pytest.mark.parametrize("M,N,K", [(17, 100, 3000), (1500, 1500, 130), (700, 8192, 200), (3500, 3500, 200)])
def test_graph_of_products(M, N, K):
    """Parts of k and each size of tiles, captured."""
    say("graph of products", M, N, K)
    w, s = operand(N, K, 3)
    codes, scales = hip.put(ref.i8_padded(w)), hip.put(s.astype(np.float32))
    wm, x = moe.I8Matrix(codes.ptr, scales.ptr, N, K), hip.full((M, K), 0)
    n = moe.i8_linear_work_bytes(wm, M)
    results = [[hip.full((M, N), 0), hip.full(n, v, np.uint8)] for v in (0, 0xA5)]

    def call(b, s):
        moe.i8_linear_async(moe.QT_F32, x.ptr, M, wm, moe.QT_F32, b[0].ptr, b[1].ptr, n, stream=s)

    replayed([(x, lambda i: np.random.default_rng(i).normal(size=(M, K)).astype(np.float32))], [r[:1] for r in results],
             lambda b, s: call(results[0] if b[0] is results[0][0] else results[1], s))


@pytest.mark.parametrize("T,H,F,E,K", [(1100, 256, 100, 12, 4), (4200, 2300, 8, 400, 8)])
def test_graph_of_experts(T, H, F, E, K):
    """Several slices of ids; values in several turns; captured."""
    say("graph of experts", T, H, F, E, K)
    model = Model(E, H, F, 6)
    op = model.op(K)
    n = op.work_bytes(T)
    x, ids, w = hip.full((T, H), 0), hip.full((T, K), 0, np.int32), hip.full((T, K), 0)
    results = [[hip.full((T, H), 0)] for _ in range(2)]
    work = [hip.full(n, v, np.uint8) for v in (0, 0xA5)]

    def call(b, s):
        op.forward_async(x.ptr, T, ids.ptr, w.ptr, b[0].ptr, work[0 if b is results[0] else 1].ptr, n, stream=s)

    made = {}

    def make(i, j):
        if i not in made:
            a = tokens(T, H, E, K, i, 0.1, True)
            made[i] = (a[0], a[1].astype(np.int32), a[2].astype(np.float32))
        return made[i][j]

    replayed([(b, lambda i, j=j: make(i, j)) for j, b in enumerate((x, ids, w))], results, call)
