"""Cases that measure the framework's operators for attention blocks: rotary positions over several axes
(forward and backward), Newton-Schulz orthogonalisation of updates, and products in 8-bit integers with a
scale for each token and output channel.

Where ``own`` is false, ``run`` computes an operator in elementary torch operations (32 bits, angles and the
matrices' norms in 64); where it is true, it calls the framework's kernels.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}

# coefficients of the quintic Newton-Schulz step and the norm's guard
_NS = (3.4445, -4.7750, 2.0315)
_NS_STEPS = 5
_NS_EPS = 1e-7
_SLOPE = 0.01


def listed():
    return [
        # one token of a batch of two streams at a far position, 3-axis sections: a decoding step, latency counts
        {"name": "rotary token", "op": "rotary", "type": "bf16", "b": 2, "h": 1, "w": 1, "heads": 10, "dim": 128,
         "tail": 0, "sections": "16,24,24", "layout": "half", "ladder": "shared", "list": True, "train": False},
        # q | k of a window-attention block's qkv map (8 + 8 heads of 24 on a 64 x 64 map, batch 32), rows and columns
        {"name": "rotary image", "op": "rotary", "type": "f16", "b": 32, "h": 64, "w": 64, "heads": 16, "dim": 24,
         "tail": 0, "sections": "6,6", "layout": "half", "ladder": "axis", "list": False, "train": False},
        # a training step's positions on the whole qkv map (v passes through), gradient included
        {"name": "rotary train", "op": "rotary", "type": "bf16", "b": 8, "h": 64, "w": 64, "heads": 16, "dim": 24,
         "tail": 192, "sections": "6,6", "layout": "pairs", "ladder": "axis", "list": False, "train": True},
        # a long video sequence with listed positions and a head that is rotated in part only
        {"name": "rotary video", "op": "rotary", "type": "bf16", "b": 1, "h": 1, "w": 61440, "heads": 20, "dim": 128,
         "tail": 0, "sections": "16,16,16", "layout": "half", "ladder": "axis", "list": True, "train": False},
        # one small convolution's update (128 <- 64 channels, 3 x 3): latency of the chain of products
        {"name": "orthogonalize one", "op": "ortho", "type": "f32", "shapes": "128x576"},
        # one training step's worth of a codec's convolutions and Linears, sizes as in this repository's models
        {"name": "orthogonalize codec", "op": "ortho", "type": "f32",
         "shapes": "12*192x1728,2*192x4800,4*256x2304,6*192x192,4*576x192,5*96x864,4*64x576,3*16x144,1*512x2304,"
                   "1*352x768"},
        # a wide transformer's square projection
        {"name": "orthogonalize square", "op": "ortho", "type": "f32", "shapes": "2048x2048"},
        # a tall feed-forward weight, gradients kept in 16 bits
        {"name": "orthogonalize tall", "op": "ortho", "type": "bf16", "shapes": "4096x1024"},
        # one token through a 4096 -> 4096 projection: bound by the weights' bytes
        {"name": "int8 token", "op": "int8", "type": "bf16", "m": 1, "k": 4096, "n": 4096, "act": "none", "res": False},
        # a window-attention block's qkv Linear on a 64 x 64 map, batch 32: bound by the activations' bytes
        {"name": "int8 qkv", "op": "int8", "type": "f16", "m": 131072, "k": 192, "n": 576, "act": "none", "res": False},
        # odd sizes on every side, 32-bit activations, activation and shortcut
        {"name": "int8 odd", "op": "int8", "type": "f32", "m": 1037, "k": 333, "n": 517, "act": "lrelu", "res": True},
        # a prompt through a wide projection: bound by the products
        {"name": "int8 wide", "op": "int8", "type": "bf16", "m": 8192, "k": 4096, "n": 8192, "act": "none", "res": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rotary", "ortho", "int8"))
    if op == "rotary":
        dim = rng.choice((16, 24, 32, 40, 48, 64, 72, 80, 96, 128))
        naxes = rng.choice((1, 2, 3))
        pairs = rng.randint(naxes, dim // 2)
        cuts = sorted(rng.sample(range(1, pairs), naxes - 1)) if naxes > 1 else []
        sections = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
        heads = rng.randint(1, 24)
        tokens = _log_int(rng, 1, max(2, 60000 * 20 * 128 // (heads * dim * 3)))
        b = rng.choice((1, 2, 3))
        h = max(1, min(64, int(math.sqrt(tokens / b)))) if rng.random() < 0.5 else 1
        return {"op": "rotary", "type": rng.choice(("f32", "f16", "bf16")), "b": b, "h": h,
                "w": max(1, min(60000, tokens // (b * h))), "heads": heads, "dim": dim,
                "tail": rng.choice((0, 0, dim, 2 * dim + 2)), "sections": ",".join(map(str, sections)),
                "layout": rng.choice(("half", "pairs")), "ladder": rng.choice(("axis", "shared")),
                "list": rng.random() < 0.5, "train": rng.random() < 0.4}
    if op == "ortho":
        count = rng.choice((1, 1, 2, 5, 9))
        shapes = []
        for _ in range(count):
            m = _log_int(rng, 8, 1500 if count == 1 else 400)
            n = _log_int(rng, m, 4 * m + 700)
            shapes.append("%dx%d" % ((m, n) if rng.random() < 0.7 else (n, m)))
        return {"op": "ortho", "type": rng.choice(("f32", "f32", "bf16", "f16")), "shapes": ",".join(shapes)}
    m, k, n = _log_int(rng, 1, 8192), _log_int(rng, 16, 4096), _log_int(rng, 16, 8192)
    return {"op": "int8", "type": rng.choice(("f32", "f16", "bf16")), "m": m, "k": k, "n": n,
            "act": rng.choice(("none", "relu", "lrelu")), "res": rng.random() < 0.4}


def _shapes(case):
    out = []
    for part in case["shapes"].split(","):
        count, _, size = part.rpartition("*")
        m, n = size.split("x")
        out += [(int(m), int(n))] * int(count or 1)
    return out


def _sections(case):
    return [int(s) for s in case["sections"].split(",")]


def work(case):
    e = _BYTES[case["type"]]
    if case["op"] == "rotary":
        tokens, c = case["b"] * case["h"] * case["w"], case["heads"] * case["dim"] + case["tail"]
        passes = 2 if case["train"] else 1
        listed_bytes = 4 * len(_sections(case)) * tokens if case["list"] else 0
        return {"bytes": passes * (2 * tokens * c * e + listed_bytes),
                "flops": passes * 6 * tokens * case["heads"] * sum(_sections(case))}
    if case["op"] == "ortho":
        nbytes = flops = 0
        for m, n in _shapes(case):
            m, n = min(m, n), max(m, n)
            nbytes += 2 * m * n * e
            # X X^T and A A are symmetric: half of their products; the update needs all of its own
            flops += _NS_STEPS * (m * m * n + m * m * m + 2 * m * m * n)
        return {"bytes": nbytes, "flops": flops}
    m, k, n = case["m"], case["k"], case["n"]
    return {"bytes": m * k * e + n * k + m * n * e * (2 if case["res"] else 1) + 8 * n, "flops": 2 * m * k * n}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _frequencies(case):
    """(axis of each pair, angle of each pair at position 1) in 64 bits."""
    sections = _sections(case)
    axis, freq = [], []
    for a, count in enumerate(sections):
        for i in range(count):
            p = len(axis)
            axis.append(a)
            freq.append(10000.0 ** (-(p / sum(sections) if case["ladder"] == "shared" else i / count)))
    return (torch.tensor(axis, device="cuda"), torch.tensor(freq, dtype=torch.float64, device="cuda"))


def _quantize_rows(x):
    """8-bit codes (as 32-bit floats) and the scale of each row: rint(127 x / max|x|), max|x| / 127.  16-bit
    values divide in 32 bits without meeting a border that is not theirs; 32-bit ones need 64."""
    x = x.double() if x.dtype == torch.float32 else x.float()
    top = x.abs().amax(dim=1, keepdim=True)
    codes = torch.where(top > 0, torch.round(x * 127.0 / top), torch.zeros_like(x))
    return codes.float(), (top / 127.0).float()


def prepare(case, seed):
    g = _generator(seed)
    t = _TYPES[case["type"]]
    s = {"case": case}

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["op"] == "rotary":
        b, h, w = case["b"], case["h"], case["w"]
        c = case["heads"] * case["dim"] + case["tail"]
        s["x"] = normal(b, h, w, c).to(t)
        s["axis"], s["freq"] = _frequencies(case)
        if case["list"]:
            # frames / rows / columns of a token list, anywhere in a long context
            n = len(_sections(case))
            start = torch.randint(0, 1 << 20, (n, b, 1, 1), device="cuda", generator=g)
            s["pos"] = (start + torch.randint(0, 4096, (n, b, h, w), device="cuda", generator=g)).to(torch.int32)
        else:
            s["pos"] = None
        if case["train"]:
            s["dy"] = normal(b, h, w, c).to(t)
            s["x"].requires_grad_(True)
        if own:
            from lic_amd import functional as Fn
            s["plan"] = Fn.RotaryPlan(case["dim"], _sections(case), base=10000.0, layout=case["layout"],
                                      shared_ladder=case["ladder"] == "shared", device="cuda")
    elif case["op"] == "ortho":
        mats = []
        for m, n in _shapes(case):
            # a gradient: a decaying low-rank part and noise
            r = max(1, min(m, n) // 4)
            decay = torch.logspace(0, -2, r, device="cuda")
            low = (normal(m, r) * decay) @ normal(r, n) / math.sqrt(r)
            mats.append((1e-3 * (low + 0.02 * normal(m, n))).to(t))
        s["mats"] = mats
    else:
        m, k, n = case["m"], case["k"], case["n"]
        # activations with a few loud channels, weights of a trained layer's spread
        s["x"] = (normal(m, k) * torch.exp(0.7 * normal(1, k))).to(t)
        weight, s["bias"] = normal(n, k) / math.sqrt(k), 0.1 * normal(n)
        codes, scale = _quantize_rows(weight)
        s["codes"], s["scale"] = codes.to(torch.int8), scale.reshape(n)
        s["res"] = normal(m, n).to(t) if case["res"] else None
        if own:
            from lic_amd import functional as Fn
            s["pack"] = Fn.pack_linear_int8(weight, s["bias"])
    return s


def _angles(case, s):
    """[b, h, w, 1, pairs] angles in 64 bits; without a list, the positions are those of the grid."""
    b, h, w = case["b"], case["h"], case["w"]
    if s["pos"] is not None:
        pos = s["pos"]
    else:
        n = len(_sections(case))
        at = torch.arange(b * h * w, device="cuda").reshape(b, h, w)
        frame, row, col = at // (h * w), at // w % h, at % w
        pos = torch.stack({1: [at % (h * w)], 2: [row, col], 3: [frame, row, col]}[n])
    return (pos.double()[s["axis"]].movedim(0, -1) * s["freq"]).unsqueeze(-2)


def _rotate(case, x, cos, sin):
    """One rotation of the heads' pairs in x's working precision; what is not rotated passes through."""
    b, h, w, _ = x.shape
    wide = case["heads"] * case["dim"]
    pairs = cos.shape[-1]
    v = x[..., :wide].reshape(b, h, w, case["heads"], case["dim"])
    u, rest = v[..., :2 * pairs], v[..., 2 * pairs:]
    if case["layout"] == "half":
        p, q = u[..., :pairs], u[..., pairs:]
        u = torch.cat((p * cos - q * sin, p * sin + q * cos), dim=-1)
    else:
        p, q = u[..., 0::2], u[..., 1::2]
        u = torch.stack((p * cos - q * sin, p * sin + q * cos), dim=-1).flatten(-2)
    return torch.cat((torch.cat((u, rest), dim=-1).reshape(b, h, w, wide), x[..., wide:]), dim=-1)


def _newton_schulz(mats):
    """Matrices of one shape together, as a batch."""
    g = torch.stack(mats)
    tall = g.shape[1] > g.shape[2]
    x = g.float().transpose(1, 2).contiguous() if tall else g.float()
    x = (x / (x.double().square().sum(dim=(1, 2), keepdim=True).sqrt() + _NS_EPS)).float()
    a, b, c = _NS
    for _ in range(_NS_STEPS):
        gram = torch.matmul(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return list((x.transpose(1, 2) if tall else x).to(g.dtype).unbind())


def _activate(y, act):
    return torch.where(y > 0, y, torch.zeros_like(y) if act == "relu" else _SLOPE * y) if act != "none" else y


def run(s):
    case = s["case"]
    if own:
        from lic_amd import _ffi, autograd as A, functional as Fn
        if case["op"] == "rotary":
            if case["train"]:
                y = A.rotary(s["x"], s["plan"], case["heads"], s["pos"])
                dx, = torch.autograd.grad(y, s["x"], s["dy"])
                return {"y": y, "dx": dx}
            return {"y": Fn.rotary(Fn.Act(s["x"]), s["plan"], case["heads"], s["pos"]).t}
        if case["op"] == "ortho":
            return Fn.orthogonalize(s["mats"], steps=_NS_STEPS, coeffs=_NS, eps=_NS_EPS)
        act = {"none": _ffi.ACT_NONE, "relu": _ffi.ACT_RELU, "lrelu": _ffi.ACT_LRELU}[case["act"]]
        m, k, n = case["m"], case["k"], case["n"]
        res = Fn.Act(s["res"].view(1, 1, m, n)) if case["res"] else None
        return {"y": Fn.linear_int8(Fn.Act(s["x"].view(1, 1, m, k)), s["pack"], act=act, slope=_SLOPE,
                                    r1=res).t.view(m, n)}
    if case["op"] == "rotary":
        angles = _angles(case, s)
        cos, sin = torch.cos(angles).float(), torch.sin(angles).float()
        x = s["x"].detach()
        y = {"y": _rotate(case, x.float(), cos, sin).to(x.dtype)}
        if case["train"]:
            y["dx"] = _rotate(case, s["dy"].float(), cos, -sin).to(x.dtype)
        return y
    if case["op"] == "ortho":
        outs, alike = [None] * len(s["mats"]), {}
        for i, g in enumerate(s["mats"]):
            alike.setdefault(tuple(g.shape), []).append(i)
        for where in alike.values():
            for i, x in zip(where, _newton_schulz([s["mats"][i] for i in where])):
                outs[i] = x
        return outs
    x = s["x"]
    codes, scale = _quantize_rows(x)
    y = _activate((codes @ s["codes"].float().t()) * scale * s["scale"] + s["bias"], case["act"])
    return {"y": (y + s["res"].float() if case["res"] else y).to(x.dtype)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        # each pair as a complex number, turned by exp(i t)
        angles = _angles(case, s)
        turn = torch.polar(torch.ones_like(angles), angles)

        def turned(x, turn):
            b, h, w, c = x.shape
            wide, pairs, dim = case["heads"] * case["dim"], turn.shape[-1], case["dim"]
            order = torch.arange(2 * pairs, device="cuda")
            order = order.reshape(2, pairs).t() if case["layout"] == "half" else order.reshape(pairs, 2)
            y = x.detach().double()
            heads = y[..., :wide].reshape(b, h, w, case["heads"], dim).clone()
            z = torch.complex(heads[..., order[:, 0]], heads[..., order[:, 1]]) * turn
            heads[..., order[:, 0]], heads[..., order[:, 1]] = z.real, z.imag
            return torch.cat((heads.reshape(b, h, w, wide), y[..., wide:]), dim=-1)

        y = {"y": turned(s["x"], turn)}
        if case["train"]:
            y["dx"] = turned(s["dy"], turn.conj())
        return y
    if case["op"] == "ortho":
        # on the shorter side: X <- X p(X^T X) or p(X X^T) X are the same odd polynomial of G
        a, b, c = _NS
        outs = []
        for g in s["mats"]:
            x = g.double()
            x = x / (torch.linalg.matrix_norm(x) + _NS_EPS)
            left = x.shape[0] <= x.shape[1]
            one = torch.eye(min(x.shape), dtype=torch.float64, device="cuda")
            for _ in range(_NS_STEPS):
                gram = torch.mm(x, x.t().contiguous()) if left else torch.mm(x.t().contiguous(), x)
                p = a * one + torch.mm(b * one + c * gram, gram)
                x = torch.mm(p, x) if left else torch.mm(x, p)
            outs.append(x)
        return outs
    x = s["x"].double()
    top = x.abs().amax(dim=1)
    safe = torch.where(top > 0, top, torch.ones_like(top))
    y = torch.mm(torch.round(x * 127.0 / safe[:, None]), s["codes"].double().t().contiguous())
    y = y * (top / 127.0)[:, None] * s["scale"].double() + s["bias"].double()
    if case["act"] == "relu":
        y = y.clamp(min=0)
    elif case["act"] == "lrelu":
        y = torch.maximum(y, _SLOPE * y)
    return {"y": y + s["res"].double() if case["res"] else y}
