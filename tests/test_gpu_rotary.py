"""Rotary positions (lic_rotary) against a rotation in 64 bits.

Tolerance: the kernel's cos / sin are off by at most 2.5e-7 (the angle's reduction and scaling: two fp32 roundings of a
value up to pi/4; the series: three roundings and 2e-9 of terms left out), its two products and their sum round three
times: |error| <= 5e-7 (|a| + |b|), and the result is rounded to its type, eps / 2 relative (fp16: or half of 2^-24)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _grid(B, H, W, naxes):
    at = torch.arange(B * H * W).view(B, H, W)
    full = [at // (H * W), at // W % H, at % W]
    return torch.stack([at % (H * W)] if naxes == 1 else full[3 - naxes:])


def _oracle(x, plan, heads, pos, inverse=False):
    """([B, H, W, C] rotated in 64 bits, the same with |a| + |b| in the place of each rotated element)."""
    B, H, W, C = x.shape
    d, P = plan.head_dim, plan.pairs
    ang = pos.double()[torch.tensor(plan.axes)].movedim(0, -1) * torch.tensor(plan.freqs, dtype=torch.float64)
    c, s = torch.cos(ang)[..., None, :], torch.sin(ang)[..., None, :]
    if inverse:
        s = -s
    y, size = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    v, z = y[..., :heads * d].view(B, H, W, heads, d), size[..., :heads * d].view(B, H, W, heads, d)
    i0 = torch.arange(P) if plan.layout == "half" else 2 * torch.arange(P)
    i1 = i0 + (P if plan.layout == "half" else 1)
    a, b = v[..., i0].clone(), v[..., i1].clone()
    v[..., i0], v[..., i1] = a * c - b * s, a * s + b * c
    z[..., i0] = z[..., i1] = a.abs() + b.abs()
    y[..., :heads * d], size[..., :heads * d] = v.reshape(B, H, W, -1), z.reshape(B, H, W, -1)
    return y, size


def _check(got, want, size):
    dt = got.dtype
    tol = 5e-7 * size + (want.abs() + 5e-7 * size) * torch.finfo(dt).eps / 2 + (2.0 ** -25 if dt == torch.float16 else 0)
    rotated = size > 0
    err = (got.cpu().double() - want).abs()
    assert (err <= tol)[rotated].all(), (err - tol)[rotated].max()
    assert torch.equal(got.cpu().double()[~rotated], want[~rotated])   # copied, or 0 turned to 0


CASES = [
    # B, H, W, heads, head_dim, tail channels, sections, layout, ladder, positions
    (1, 1, 1, 1, 2, 0, (1,), "half", False, "grid"),
    (1, 1, 1, 10, 128, 0, (16, 24, 24), "half", True, "image"),
    (2, 8, 8, 16, 24, 192, (6, 6), "half", False, "grid"),
    (2, 8, 8, 16, 24, 192, (6, 6), "pairs", False, "grid"),
    (3, 5, 7, 3, 40, 1, (3, 8), "pairs", False, "grid"),
    (3, 5, 7, 3, 40, 13, (2, 3, 4), "half", True, "grid"),
    (1, 1, 515, 5, 80, 0, (40,), "half", False, "shared"),
    (2, 1, 129, 7, 36, 5, (1, 2, 3, 5), "pairs", False, "image"),
    (1, 3, 1000, 2, 72, 0, (7, 8), "half", False, "shared"),
    (2, 2, 33, 4, 64, 8, (32,), "pairs", True, "image"),
    (1, 1, 2100, 20, 128, 0, (16, 16, 16), "half", False, "image"),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,H,W,heads,d,tail,sections,layout,shared,kind", CASES)
def test_rotary_matches_64_bits(dtype, B, H, W, heads, d, tail, sections, layout, shared, kind):
    import lic_amd.functional as Fn
    g = torch.Generator().manual_seed(B * 100 + W + d)
    plan = Fn.RotaryPlan(d, sections, layout=layout, shared_ladder=shared, device=DEV)
    x = torch.randn(B, H, W, heads * d + tail, generator=g).to(dtype)
    pos = None
    if kind != "grid":
        shape = (len(sections), H, W) if kind == "shared" else (len(sections), B, H, W)
        pos = torch.randint(-(1 << 22), 1 << 22, shape, generator=g, dtype=torch.int32)
    full = _grid(B, H, W, len(sections)) if pos is None else pos if pos.dim() == 4 else pos[:, None].expand(-1, B, -1, -1)
    for inverse in (False, True):
        got = Fn.rotary(Fn.Act(x.to(DEV)), plan, heads, pos.to(DEV) if pos is not None else None, inverse=inverse).t
        _check(got, *_oracle(x, plan, heads, full, inverse))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "pairs"])
@pytest.mark.parametrize("total,c0,c", [(96, 0, 64), (96, 24, 64), (67, 3, 48), (65, 1, 49)])
def test_rotary_channel_windows_in_place(dtype, layout, total, c0, c):
    """A channel window at any offset, into another window, and in place: the same bits as on a packed copy, nothing
    outside the rotated heads touched."""
    import lic_amd.functional as Fn
    g = torch.Generator().manual_seed(total + c0)
    plan = Fn.RotaryPlan(16, (3, 4), base=50.0, layout=layout, device=DEV)
    x = torch.randn(2, 3, 5, total, generator=g).to(dtype).to(DEV)
    packed = Fn.rotary(Fn.Act(x[..., c0:c0 + c].contiguous()), plan, c // 16).t
    before = x.clone()
    view = Fn.Act(x, c0, c)
    y = torch.full((2, 3, 5, total + 8), 7.0, dtype=dtype, device=DEV)
    Fn.rotary(view, plan, c // 16, out=Fn.Act(y, 5, c))
    assert torch.equal(y[..., 5:5 + c], packed)
    y[..., 5:5 + c] = 7.0
    assert (y == 7.0).all() and torch.equal(x, before)
    Fn.rotary(view, plan, c // 16, out=view)
    assert torch.equal(x[..., c0:c0 + c], packed)
    x[..., c0:c0 + c] = before[..., c0:c0 + c]
    assert torch.equal(x, before)


def test_rotary_odd_alignment_matches_packed():
    """A tensor that starts off the 16-byte grid takes narrower accesses and gives the same bits."""
    import lic_amd.functional as Fn
    plan = Fn.RotaryPlan(32, (8, 8), device=DEV)
    for dtype in TYPES:
        flat = torch.randn(1 + 4 * 6 * 64, device=DEV).to(dtype)
        x = flat[1:].view(1, 4, 6, 64)
        want = Fn.rotary(Fn.Act(x.clone()), plan, 2).t
        assert torch.equal(Fn.rotary(Fn.Act(x), plan, 2).t, want)


def test_rotary_far_positions_and_inverse():
    """The largest positions: angles stay those of 64-bit arithmetic (position * freq there is exact to 2^-22 turns at
    2^31), and turning back restores x."""
    import lic_amd.functional as Fn
    plan = Fn.RotaryPlan(64, (32,), device=DEV)
    x = torch.randn(1, 1, 4, 128)
    pos = torch.tensor([2 ** 31 - 1, -2 ** 31, 2 ** 30 + 12345, -1], dtype=torch.int32).view(1, 1, 4)
    y = Fn.rotary(Fn.Act(x.to(DEV)), plan, 2, pos.to(DEV))
    want, size = _oracle(x, plan, 2, pos[:, None])
    # the oracle's own angle: 2^31 * 2^-53 = 2.4e-7
    assert ((y.t.cpu().double() - want).abs() <= 1e-6 * size + 2 ** -24 * want.abs()).all()
    back = Fn.rotary(y, plan, 2, pos.to(DEV), inverse=True).t.cpu()
    assert ((back - x).abs() <= 2.5e-6 * (size.float() + 1e-6)).all()


def test_rotary_infinities_stay_in_their_pair():
    import lic_amd.functional as Fn
    plan = Fn.RotaryPlan(8, (4,), layout="pairs", device=DEV)
    x = torch.randn(1, 1, 3, 8, device=DEV)
    x[0, 0, 1, 2] = float("inf")
    x[0, 0, 2, 5] = float("nan")
    y = Fn.rotary(Fn.Act(x), plan, 1).t
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[0, 0, 1, 2:4] = True
    want[0, 0, 2, 4:6] = True
    assert torch.equal(bad, want)


def test_rotary_empty_and_refusals():
    import lic_amd.functional as Fn
    plan = Fn.RotaryPlan(16, (4, 4), device=DEV)
    assert Fn.rotary(Fn.Act(torch.empty(0, 4, 4, 32, device=DEV)), plan, 2).t.shape == (0, 4, 4, 32)
    x = Fn.Act(torch.zeros(2, 4, 4, 64, device=DEV))
    with pytest.raises(ValueError, match="overlaps"):
        Fn.rotary(x.ch(0, 32), plan, 2, out=x.ch(16, 48))
    with pytest.raises(ValueError, match="another size"):
        Fn.rotary(x, plan, 2, out=x.ch(0, 32))
    with pytest.raises(ValueError, match="int32"):
        Fn.rotary(x, plan, 2, torch.zeros(2, 4, 4, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError, match="int32"):
        Fn.rotary(x, plan, 2, torch.zeros(1, 4, 4, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="explicit positions"):
        Fn.rotary(x, Fn.RotaryPlan(16, (1, 1, 1, 1), device=DEV), 2)
    with pytest.raises(ValueError, match="not on the GPU"):
        Fn.rotary(x, plan, 2, torch.zeros(2, 4, 4, dtype=torch.int32))
    # strided positions are read by value
    pos = torch.arange(64, dtype=torch.int32, device=DEV).view(4, 4, 4)[::2]
    y = Fn.rotary(x, plan, 2, pos)
    assert torch.equal(y.t, Fn.rotary(x, plan, 2, pos.contiguous()).t)


@pytest.mark.parametrize("layout", ["half", "pairs"])
def test_rotary_gradient(layout):
    """Against the formula (the rotation back, in 64 bits) and against differences: the map is linear, so a difference
    quotient at any step is the directional derivative up to rounding."""
    import lic_amd.functional as Fn
    from lic_amd import autograd as AG
    g = torch.Generator().manual_seed(4)
    plan = Fn.RotaryPlan(20, (4, 5), layout=layout, device=DEV)
    x = torch.randn(2, 3, 4, 3 * 20 + 11, generator=g)
    dy = torch.randn(x.shape, generator=g)
    leaf = x.to(DEV).requires_grad_(True)
    y = AG.rotary(leaf, plan, 3)
    dx, = torch.autograd.grad(y, leaf, dy.to(DEV), create_graph=True)
    want, size = _oracle(dy, plan, 3, _grid(2, 3, 4, 2), inverse=True)
    _check(dx.detach(), want, size)
    step = torch.randn(x.shape, generator=g)
    up, down = (Fn.rotary(Fn.Act((x + h * step).to(DEV)), plan, 3).t.double().cpu() for h in (1.0, -1.0))
    slope = ((up - down) / 2 * dy.double()).sum()
    terms = ((up.abs() + down.abs()) * dy.abs()).sum() + (step.abs() * dx.detach().cpu().abs()).sum()
    assert abs(slope - (step.double() * dx.detach().cpu().double()).sum()) <= 2e-6 * terms
    # the gradient's gradient is the forward rotation again
    v = torch.randn(x.shape, generator=g).to(DEV)
    probe = dy.to(DEV).requires_grad_(True)
    y2 = AG.rotary(leaf, plan, 3)
    dx2, = torch.autograd.grad(y2, leaf, probe, create_graph=True)
    ddy, = torch.autograd.grad(dx2, probe, v)
    assert torch.equal(ddy, Fn.rotary(Fn.Act(v), plan, 3).t)


def test_rotary_other_stream_and_graph():
    """On a side stream, and captured (out of place, in place, backward) and replayed with new data between replays."""
    import lic_amd.functional as Fn
    from lic_amd import autograd as AG
    plan = Fn.RotaryPlan(24, (6, 6), device=DEV)
    x = torch.randn(2, 8, 8, 16 * 24, device=DEV)
    want = Fn.rotary(Fn.Act(x), plan, 16).t.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = Fn.rotary(Fn.Act(x), plan, 16).t
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    sx, sg = x.clone().requires_grad_(True), torch.randn_like(x)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = AG.rotary(sx, plan, 16)
        dx, = torch.autograd.grad(y, sx, sg)
        z = Fn.Act(y.detach().clone())
        Fn.rotary(z, plan, 16, out=z, inverse=True)
    for k in range(3):
        with torch.no_grad():
            sx.copy_(torch.randn_like(x))
            sg.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, Fn.rotary(Fn.Act(sx.detach()), plan, 16).t)
        assert torch.equal(dx, Fn.rotary(Fn.Act(sg), plan, 16, inverse=True).t)
        assert torch.equal(z.t, Fn.rotary(Fn.Act(y.detach()), plan, 16, inverse=True).t)


def test_rotary_more_workgroups_than_a_grid_dimension():
    """From 2^24 workgroups of 256 threads on (here one token each: rows of 1025 elements are read one by one) a launch
    takes a second dimension: tokens on both sides of its rows, zeros everywhere else (34 GB each way)."""
    import lic_amd.functional as Fn
    H = W = 4100
    assert H * W > 1 << 24
    plan = Fn.RotaryPlan(1025, (200, 312), device=DEV)
    at = torch.tensor([0, 1, (1 << 22) - 1, 1 << 22, (1 << 22) + 1, (1 << 24) - 1, 1 << 24, H * W - 1])
    x = torch.zeros(1, H, W, 1025, dtype=torch.bfloat16, device=DEV)
    rows = torch.randn(at.numel(), 1025, generator=torch.Generator().manual_seed(2)).bfloat16()
    x.view(H * W, 1025)[at.to(DEV)] = rows.to(DEV)
    y = Fn.rotary(Fn.Act(x), plan, 1).t.view(H * W, 1025)
    got = y[at.to(DEV)].clone()
    y[at.to(DEV)] = 0
    assert all(int(torch.count_nonzero(part)) == 0 for part in y.split(1 << 20))
    del x, y
    torch.cuda.empty_cache()
    pos = torch.stack([at // W, at % W])[:, None, None]
    _check(got.view(1, 1, -1, 1025), *_oracle(rows.view(1, 1, -1, 1025), plan, 1, pos))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "pairs"])
@pytest.mark.parametrize("listed", [False, True])
def test_rotary_gradient_16_bit(dtype, layout, listed):
    """The training path's types: forward and gradient of a map with channels that pass through, a gradient that arrives
    strided, positions of the grid and listed, against 64 bits."""
    import lic_amd.functional as Fn
    from lic_amd import autograd as AG
    g = torch.Generator().manual_seed(6)
    plan = Fn.RotaryPlan(24, (6, 6), layout=layout, device=DEV)
    x, dy = (torch.randn(2, 8, 12, 72, generator=g).to(dtype) for _ in range(2))
    pos = torch.randint(-5000, 5000, (2, 2, 8, 12), generator=g, dtype=torch.int32) if listed else None
    full = pos if listed else _grid(2, 8, 12, 2)
    leaf = x.to(DEV).requires_grad_(True)
    y = AG.rotary(leaf, plan, 2, pos.to(DEV) if listed else None)
    strided = dy.to(DEV).permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)
    dx, = torch.autograd.grad(y, leaf, strided)
    _check(y.detach(), *_oracle(x, plan, 2, full))
    _check(dx, *_oracle(dy, plan, 2, full, inverse=True))
