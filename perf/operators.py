"""Routing to experts and the microscaled 4-bit products, as measurable cases.

A serving program whose experts are kept in microscaled 4-bit floats calls, a layer: the routing of its router's
logits (moe_route_async), the experts on the routed tokens (moe_mx4_experts_async) and, for its dense matrices, the
product with float rows (moe_mx4_linear_async) or with rows that are quantised already (moe_mx4_matmul_async); it
quantises weights and activations with moe_mx4_quantize_async. Everything is on the device and in the program's
buffers.

The format: 32 values along a row share a power of two (a biased exponent in a byte, 2^(s - 127)); a value is a sign,
two bits of exponent and one of mantissa (0, 0.5, 1, 1.5, 2, 3, 4, 6), two in a byte, the earlier one low. Rows are
padded with zeros to 128 values.
"""
import math

import torch

own = False  # the framework's kernels instead of the plain forms

FLOATS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIGMA = 0.02  # of the weights


def _route(name, T, E, K, score="softmax", bias=False, groups=0, kept=0, best=1, renorm=True, scale=1.0, type="f32",
           masked=0.0, empty=0):
    return {"name": name, "kind": "route", "T": T, "E": E, "K": K, "score": score, "bias": bias, "groups": groups,
            "kept": kept, "best": best, "renorm": renorm, "scale": scale, "type": type, "masked": masked, "empty": empty}


def _quantize(name, rows, cols, type):
    return {"name": name, "kind": "quantize", "rows": rows, "cols": cols, "type": type}


def _product(name, kind, M, N, K, type, out):
    return {"name": name, "kind": kind, "M": M, "N": N, "K": K, "type": type, "out": out}


def _experts(name, T, H, F, E, K, zipf=0.0, type="bf16", limit=0.0, dropped=0.0):
    return {"name": name, "kind": "experts", "T": T, "H": H, "F": F, "E": E, "K": K, "zipf": zipf, "type": type,
            "limit": limit, "dropped": dropped}


def listed():
    return [
        # One generated token's routing: the smallest call, launch and latency.
        _route("route_1", 1, 512, 10),
        # A prompt's routing with everything that is in use: sigmoid scores, a bias that balances the experts, the best
        # 4 of 8 groups, weights that are renormalised and scaled, some experts masked, padded rows at the end.
        _route("route_groups_999", 999, 256, 8, "sigmoid", True, 8, 4, 2, True, 2.5, "bf16", 0.05, 7),
        # The largest chunk the block takes.
        _route("route_16384", 16384, 512, 10),
        # A few tokens' activations.
        _quantize("quantize_8x2560", 8, 2560, "f32"),
        # A weight matrix, or a long chunk's activations.
        _quantize("quantize_16384x8192", 16384, 8192, "bf16"),
        # One generated token through a dense matrix.
        _product("linear_1", "linear", 1, 8192, 2048, "bf16", "bf16"),
        # A short prompt's quantised rows, sizes that no tile divides, 32-bit results.
        _product("matmul_301", "matmul", 301, 2565, 1000, "f32", "f32"),
        # A whole chunk through a large dense matrix: bound by the matrix cores.
        _product("linear_4096", "linear", 4096, 8192, 8192, "bf16", "bf16"),
        # One generated token through its experts.
        _experts("experts_1", 1, 2048, 512, 512, 10),
        # A verify step of 8 tokens with the skewed expert use of real routing.
        _experts("experts_8", 8, 2048, 512, 512, 10, 1.1),
        # An ordinary prompt on the model file's shape, ranks without an expert among them.
        _experts("experts_301", 301, 2560, 640, 512, 10, 1.1, "f16", 7.0, 0.05),
        # A large prefill chunk.
        _experts("experts_4096", 4096, 2048, 512, 512, 10, 1.1),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    """A case of the same ranges, its sizes spread over their logarithms."""
    kind = rng.choice(["route", "quantize", "linear", "matmul", "experts"])
    type = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind == "route":
        E = rng.choice([8, 60, 64, 96, 128, 160, 256, 384, 511, 512])
        groups = rng.choice([0, 0, 4, 8]) if E % 8 == 0 and E >= 32 else 0
        kept = rng.randint(2, groups) if groups else 0
        T = _log(rng, 1, 16384)
        c = _route("", T, E, rng.randint(1, min(16, E // groups * kept if groups else E)), rng.choice(["softmax", "sigmoid"]),
                   rng.random() < 0.5, groups, kept, rng.choice([1, 2]) if groups else 1, rng.random() < 0.7,
                   rng.choice([1.0, 2.5]), type, rng.choice([0.0, 0.1, 0.5]), rng.choice([0, T // 10]))
    elif kind == "quantize":
        cols = _log(rng, 1, 16384)
        c = _quantize("", min(_log(rng, 1, 65536), 16384 * 8192 // cols), cols, type)
    elif kind == "experts":
        H, F = rng.choice([(2048, 512), (2560, 640), (1024, 704), (1000, 200), (512, 1536)])
        E = rng.choice([8, 40, 128, 512])
        T = _log(rng, 1, 4096 * 2048 * 512 // max(H * F, 2048 * 512))
        c = _experts("", T, H, F, E, rng.randint(1, min(10, E)), rng.choice([0.0, 1.1]), rng.choice(["f16", "bf16"]),
                     rng.choice([0.0, 7.0]), rng.choice([0.0, 0.1]))
    else:
        c = _product("", kind, _log(rng, 1, 4096), _log(rng, 1, 8192), _log(rng, 1, 8192), type,
                     rng.choice(["f32", "f16", "bf16"]))
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------------------------
# The plain forms


def _pad(n):
    return -(-n // 128) * 128


def _to_mx4(x):
    """Rows of floats to codes and scales. A block that holds an infinity or a NaN has the scale 255 and codes 0."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.float(), (0, _pad(cols) - cols)).view(rows, -1, 32)
    most = v.abs().amax(-1, keepdim=True)
    fine = most < math.inf
    e = (torch.frexp(torch.where(fine & (most > 0), most, torch.full_like(most, 2.0 ** -126)))[1] - 3).clamp(min=-127)
    e = torch.where(most > 0, e, torch.full_like(e, -127))
    a = torch.where(fine, torch.ldexp(v, -e), torch.zeros_like(v))
    m = a.abs()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    q = (torch.round(m / step) * step).clamp(max=6)  # torch.round takes halves to even, the format's rule
    code = torch.where(q <= 2, 2 * q, torch.where(q <= 4, q + 2, torch.full_like(q, 7))).to(torch.uint8)
    code = (code | (torch.signbit(a).to(torch.uint8) << 3)).view(rows, -1)
    scale = torch.where(fine, e + 127, torch.full_like(e, 255)).to(torch.uint8).view(rows, -1)
    return code[:, 0::2] | (code[:, 1::2] << 4), scale


def _from_mx4(codes, scales, cols):
    """Codes (.., n / 2) and scales (.., n / 32) to 32-bit values."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    table = torch.cat([table, -table])
    v = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], -1).view(*codes.shape[:-1], -1, 32)
    s = torch.where(scales == 255, math.nan, torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127))
    return (v * s.unsqueeze(-1)).flatten(-2)[..., :cols]


def _plain_route(c, logits, bias):
    T, E, K = c["T"], c["E"], c["K"]
    x = logits.double()  # the order of the scores is decided in 64 bits
    known = x > -math.inf  # neither minus infinity nor NaN
    x = torch.where(known, x, torch.full_like(x, -math.inf))
    if c["score"] == "softmax":
        top = x.amax(-1, keepdim=True)
        p = torch.where(x == top, 1.0, torch.exp(x - top)) * known
        s = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    else:
        s = torch.where(known, 1 / (1 + torch.exp(-x)), 0.0)
    if bias is not None:
        key = torch.where(known & (bias > -math.inf), s + bias.double(), -math.inf)
    else:
        key = torch.where(known, s, -math.inf) if c["groups"] and c["best"] > 1 else x
    if c["groups"]:
        g = key.view(T, c["groups"], -1)
        best = g.sort(dim=-1, descending=True).values[..., :c["best"]]
        total = torch.where(best > -math.inf, best, 0.0).sum(-1)
        total = torch.where(best[..., 0] > -math.inf, total, -math.inf)
        keep = total.sort(dim=-1, descending=True, stable=True).indices[:, :c["kept"]]
        stays = torch.zeros_like(total, dtype=torch.bool).scatter_(1, keep, True)
        key = torch.where(stays.unsqueeze(-1), g, -math.inf).view(T, E)
    order = key.sort(dim=-1, descending=True, stable=True)
    ids, there = order.indices[:, :K], order.values[:, :K] > -math.inf
    w = torch.where(there, s.gather(1, ids), 0.0)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-20)
    ids = torch.where(there, ids, -1).int()
    load = torch.bincount(ids.flatten() + 1, minlength=E + 1)[1:].int()
    return {"ids": ids, "w": (w * c["scale"]).float(), "load": load}


def _plain_experts(c, s):
    T, H, F, K = c["T"], c["H"], c["F"], c["K"]
    # The assignments by expert, each of the used experts' padded to the most that one has.
    flat = s.ids.flatten().long()
    taken = (flat >= 0).nonzero().flatten()
    used, at = torch.unique(flat[taken], return_inverse=True)
    order = at.argsort(stable=True)
    counts = torch.bincount(at, minlength=len(used))
    y = torch.zeros(T, K, H, device=s.x.device)
    if len(used):
        expert = at[order]
        place = torch.arange(len(order), device=at.device) - (counts.cumsum(0) - counts)[expert]
        cap = int(counts.max())
        xs = _from_mx4(*_to_mx4(s.x), H)[taken[order] // K]
        rows = torch.zeros(len(used), cap, H, device=xs.device)
        rows[expert, place] = xs
        rows = rows.transpose(1, 2).contiguous()
        g, u = (torch.bmm(_from_mx4(*(m[used] for m in w), H), rows) for w in (s.gate, s.up))
        g, u = (v.transpose(1, 2)[expert, place].double() for v in (g, u))  # values next to a border of the codes
        if c["limit"]:
            g, u = g.clamp(max=c["limit"]), u.clamp(-c["limit"], c["limit"])
        h = (g / (1 + torch.exp(-g)) * u).float()
        rows = torch.zeros(len(used), cap, F, device=xs.device)
        rows[expert, place] = _from_mx4(*_to_mx4(h), F)
        o = torch.bmm(_from_mx4(*(m[used] for m in s.down), F), rows.transpose(1, 2).contiguous())
        y.view(T * K, H)[taken[order]] = o.transpose(1, 2)[expert, place]
    w = torch.where(s.ids >= 0, s.w, 0.0)
    return (y * w.unsqueeze(-1)).sum(1).to(FLOATS[c["type"]])


# ---------------------------------------------------------------------------------------------------------------------
# The framework's calls


def _start(s):
    """What a program keeps beside its buffers: the framework's descriptions of them, and the calls' workspaces."""
    import c0ven_amd as moe

    c, dev = s.case, s.device
    ptr = torch.Tensor.data_ptr
    types = {"f32": moe.QT_F32, "f16": moe.QT_F16, "bf16": moe.QT_BF16}

    def room(n):
        return torch.empty(n, dtype=torch.uint8, device=dev)

    def mx4(pair, cols):
        return moe.Mx4Matrix(ptr(pair[0]), ptr(pair[1]), pair[0].shape[-2], cols)

    if c["kind"] == "route":
        router = moe.Router(c["E"], c["K"], {"softmax": moe.MOE_SCORE_SOFTMAX, "sigmoid": moe.MOE_SCORE_SIGMOID}[c["score"]],
                            c["groups"], c["kept"], c["best"], c["renorm"], c["scale"], types[c["type"]])
        ids = torch.empty(c["T"], c["K"], dtype=torch.int32, device=dev)
        w = torch.empty(c["T"], c["K"], device=dev)
        load = torch.empty(c["E"], dtype=torch.int32, device=dev)
        a = (ptr(s.logits), c["T"], ptr(ids), ptr(w), ptr(load), None if s.bias is None else ptr(s.bias))
        out = {"ids": ids, "w": w, "load": load}
        return lambda: (router.route_async(*a, stream=s.stream), out)[1]
    if c["kind"] == "quantize":
        rows, cols = c["rows"], c["cols"]
        codes, scales = room((rows, _pad(cols) // 2)), room((rows, _pad(cols) // 32))
        out = torch.empty(rows, cols, dtype=FLOATS[c["type"]], device=dev)
        m, t = mx4((codes, scales), cols), types[c["type"]]

        def both():
            moe.mx4_quantize_async(t, ptr(s.x), m, stream=s.stream)
            moe.mx4_dequantize_async(m, t, ptr(out), stream=s.stream)
            return {"values": out}

        return both
    if c["kind"] == "experts":
        experts = moe.Mx4Experts(c["H"], c["F"], c["E"], c["K"], *(mx4(m, n) for m, n in ((s.gate, c["H"]), (s.up, c["H"]),
                                 (s.down, c["F"]))), x_type=types[c["type"]], y_type=types[c["type"]], swiglu_limit=c["limit"])
        y = torch.empty(c["T"], c["H"], dtype=FLOATS[c["type"]], device=dev)
        s.work = work = room(experts.work_bytes(c["T"]))
        a = (ptr(s.x), c["T"], ptr(s.ids), ptr(s.w), ptr(y), ptr(work), work.numel())
        return lambda: (experts.forward_async(*a, stream=s.stream), {"y": y})[1]
    y = torch.empty(c["M"], c["N"], dtype=FLOATS[c["out"]], device=dev)
    w = mx4(s.w, c["K"])
    if c["kind"] == "matmul":
        x = mx4(s.x, c["K"])
        s.work = work = room(moe.mx4_matmul_work_bytes(w, c["M"]))
        a = (x, w, types[c["out"]], ptr(y), ptr(work), work.numel())
        return lambda: (moe.mx4_matmul_async(*a, stream=s.stream), {"y": y})[1]
    s.work = work = room(moe.mx4_linear_work_bytes(w, c["M"]))
    a = (types[c["type"]], ptr(s.x), c["M"], w, types[c["out"]], ptr(y), ptr(work), work.numel())
    return lambda: (moe.mx4_linear_async(*a, stream=s.stream), {"y": y})[1]


# ---------------------------------------------------------------------------------------------------------------------


class State:
    call = None


def _rng(seed, device):
    return torch.Generator(device=device).manual_seed(seed)


def _weights(rows, cols, g, n=0):
    """A matrix of N(0, 0.02) values (or n of them) in the format."""
    made = [_to_mx4(torch.randn(rows, cols, generator=g, device=g.device) * SIGMA) for _ in range(max(1, n))]
    return tuple(torch.stack([m[i] for m in made]) if n else made[0][i] for i in (0, 1))


def _activations(rows, cols, type, g):
    """What a norm gives: N(0, 1), with the few channels of large values that models have."""
    x = torch.randn(rows, cols, generator=g, device=g.device)
    return (x * torch.where(torch.rand(cols, generator=g, device=g.device) < 0.01, 8.0, 1.0)).to(FLOATS[type])


def _zipf(E, s, g):
    """A bias of the logits under which the experts' use falls off as rank^-s."""
    return -s * torch.log1p(torch.randperm(E, generator=g, device=g.device).float())


def prepare(case, seed):
    s = State()
    s.case, s.device = case, torch.device("cuda")
    s.stream = torch.cuda.current_stream().cuda_stream
    g = _rng(seed, s.device)
    c = case
    if c["kind"] == "route":
        x = torch.randn(c["T"], c["E"], generator=g, device=s.device) * 1.5
        x = torch.where(torch.rand(c["T"], c["E"], generator=g, device=s.device) < c["masked"], -math.inf, x)
        x[c["T"] - c["empty"]:] = -math.inf
        s.logits = x.to(FLOATS[c["type"]])
        s.bias = torch.randn(c["E"], generator=g, device=s.device) * 0.1 if c["bias"] else None
    elif c["kind"] == "quantize":
        s.x = _activations(c["rows"], c["cols"], c["type"], g)
    elif c["kind"] == "experts":
        T, H, F, E, K = c["T"], c["H"], c["F"], c["E"], c["K"]
        # Matrices of 16 experts at a time: each expert has values of its own.
        n = math.gcd(E, 16)
        s.gate, s.up, s.down = (tuple(m.view(E, a, -1) for m in _weights(n * a, b, g, E // n))
                                for a, b in ((F, H), (F, H), (H, F)))
        s.x = _activations(T, H, c["type"], g)
        logits = torch.randn(T, E, generator=g, device=s.device) + (_zipf(E, c["zipf"], g) if c["zipf"] else 0.0)
        top = logits.topk(K, -1)
        s.w = top.values.softmax(-1)
        s.ids = torch.where(torch.rand(T, K, generator=g, device=s.device) < c["dropped"], -1, top.indices).int()
    else:
        s.w = _weights(c["N"], c["K"], g)
        x = _activations(c["M"], c["K"], c["type"], g)
        s.x = _to_mx4(x) if c["kind"] == "matmul" else x
    return s


def run(s):
    if own:
        if s.call is None:
            s.call = _start(s)
        return s.call()
    c = s.case
    if c["kind"] == "route":
        return _plain_route(c, s.logits, s.bias)
    if c["kind"] == "quantize":
        return {"values": _from_mx4(*_to_mx4(s.x), c["cols"]).to(FLOATS[c["type"]])}
    if c["kind"] == "experts":
        return {"y": _plain_experts(c, s)}
    x = _from_mx4(*(s.x if c["kind"] == "matmul" else _to_mx4(s.x)), c["K"])
    return {"y": (x @ _from_mx4(*s.w, c["K"]).T).to(FLOATS[c["out"]])}


def _used(c):
    """How many experts the case's tokens use, on logits of its distribution."""
    g = _rng(7, "cpu")
    logits = torch.randn(c["T"], c["E"], generator=g) + (_zipf(c["E"], c["zipf"], g) if c["zipf"] else 0.0)
    ids = logits.topk(c["K"], -1).indices
    return len(torch.unique(ids[torch.rand(c["T"], c["K"], generator=g) >= c["dropped"]]))


def work(case):
    c = case
    if "type" in c:
        size = FLOATS[c["type"]].itemsize

    def mx4(rows, cols):
        return rows * cols * (0.5 + 1 / 32)

    if c["kind"] == "route":  # the scores: an exponential, a division and the comparisons that a value takes
        return {"bytes": c["T"] * (c["E"] * size + 8 * c["K"]) + 4 * c["E"] * (2 if c["bias"] else 1), "flops": 24.0 * c["T"] * c["E"]}
    if c["kind"] == "quantize":  # values read, the format written, read again for the values it stands for, those written
        n = c["rows"] * c["cols"]
        return {"bytes": 2 * n * size + 2 * mx4(c["rows"], c["cols"]), "flops": 8.0 * n}
    if c["kind"] == "experts":
        T, H, F, K = c["T"], c["H"], c["F"], c["K"]
        return {"bytes": _used(c) * mx4(3 * H, F) + 2 * T * H * size + 8 * T * K, "flops": 6.0 * T * K * (1 - c["dropped"]) * F * H}
    M, N, K = c["M"], c["N"], c["K"]
    return {"bytes": mx4(N, K) + (mx4(M, K) if c["kind"] == "matmul" else M * K * size) + M * N * FLOATS[c["out"]].itemsize,
            "flops": 2.0 * M * N * K}


# ---------------------------------------------------------------------------------------------------------------------
# The same in 64 bits, from the definitions


def _exact_values(codes, scales, cols):
    """sign * m * 2^(s - 127) of each code, m from its exponent and mantissa bits."""
    c = torch.stack([codes % 16, codes // 16], -1).flatten(-2)[..., :cols].to(torch.int16)
    s = scales.repeat_interleave(32, -1)[..., :cols]
    e, m = (c // 2) % 4, (c % 2).double()
    v = torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2((e - 1).double())) * (1 - 2 * (c // 8)).double()
    return torch.where(s == 255, math.nan, v * torch.exp2(s.double() - 127))


def _exact_rounded(x):
    """Each value as the nearest of the format's under its block's scale: 2^(floor(log2 of the block's largest) - 2)."""
    rows, cols = x.shape
    v = torch.zeros(rows, -(-cols // 32) * 32, dtype=torch.float64, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, -1, 32)
    most = v.abs().max(-1, keepdim=True).values
    e = torch.floor(torch.log2(most.clamp(min=2.0 ** -1074)))
    e = e + (torch.exp2(e + 1) <= most) - (torch.exp2(e) > most).double()  # the logarithm may round to a power of two
    unit = torch.exp2((e - 2).clamp(min=-127))
    m = v.abs() / unit
    # The borders between neighbours; one that lies halfway goes to the value with the even mantissa.
    r = torch.zeros_like(m)
    for border, value, up in ((0.25, 0.5, False), (0.75, 1, True), (1.25, 1.5, False), (1.75, 2, True), (2.5, 3, False), (3.5, 4, True), (5, 6, False)):
        r = torch.where((m >= border) if up else (m > border), value, r)
    return torch.where(most < math.inf, r * unit * v.sign(), math.nan).view(rows, -1)[:, :cols]


def _exact_route(c, s):
    x = s.logits.double()
    there = torch.isfinite(x) | (x == math.inf)
    if c["score"] == "softmax":
        most = torch.where(there, x, -math.inf).max(-1, keepdim=True).values
        score = torch.where(there, torch.exp(torch.where(there, x - most, 0.0)), 0.0)
        score = torch.where(there.any(-1, keepdim=True), score / score.sum(-1, keepdim=True), 0.0)
    else:
        score = torch.where(there, torch.sigmoid(x), 0.0)
    order = score + (s.bias.double() if c["bias"] else 0.0)
    order = torch.where(there, order, -math.inf)
    if c["groups"]:
        n = c["E"] // c["groups"]
        worth = [torch.topk(order[:, i * n:(i + 1) * n], c["best"], -1).values for i in range(c["groups"])]
        worth = torch.stack([torch.where(v[:, 0] == -math.inf, -math.inf, torch.nan_to_num(v, neginf=0.0).sum(-1)) for v in worth], -1)
        place = (-worth).argsort(dim=-1, stable=True).argsort(dim=-1)  # equal groups: the first ones
        order = torch.where((place < c["kept"]).repeat_interleave(n, -1), order, -math.inf)
    top = torch.topk(order, c["K"], -1)
    w = torch.where(top.values > -math.inf, score.gather(-1, top.indices), 0.0)
    if c["renorm"]:
        w = w / torch.clamp(w.sum(-1, keepdim=True), min=1e-20)
    return {"ids": None, "w": w * c["scale"], "load": None}


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "route":
        return _exact_route(c, s)
    if c["kind"] == "quantize":
        return {"values": _exact_rounded(s.x.double())}
    if c["kind"] != "experts":
        x = _exact_values(*s.x, c["K"]) if c["kind"] == "matmul" else _exact_rounded(s.x.double())
        return {"y": x @ _exact_values(*s.w, c["K"]).T}
    x = _exact_rounded(s.x.double())
    y = torch.zeros(c["T"], c["H"], dtype=torch.float64, device=s.device)
    for e in torch.unique(s.ids).tolist():
        if e < 0:
            continue
        t, k = (s.ids == e).nonzero(as_tuple=True)
        g, u = (x[t] @ _exact_values(m[0][e], m[1][e], c["H"]).T for m in (s.gate, s.up))
        if c["limit"]:
            g, u = g.clamp(max=c["limit"]), u.clamp(-c["limit"], c["limit"])
        h = _exact_rounded(g * torch.sigmoid(g) * u)
        y.index_put_((t,), s.w[t, k].double().unsqueeze(-1) * (h @ _exact_values(s.down[0][e], s.down[1][e], c["F"]).T), accumulate=True)
    return {"y": y}
