"""Newton-Schulz orthogonalisation (lic_orthogonalize) and the Muon optimiser against 64 bits.

Tolerance: the kernel's products take operands of 22 bits (two fp16 parts) with fp32 sums, the same iteration in fp32
takes 24: its error against 64 bits is at most 2^-22 / 2^-24 = 4 times that of fp32 products (2-norm, plus 1e-7 for the
scaling by the norm), and a 16-bit result adds its own rounding, eps / 2 of each value."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
C = (3.4445, -4.7750, 2.0315)


def _newton_schulz(g, steps, coeffs, eps, dt):
    a, b, c = coeffs
    g = g.to(dt) if dt == torch.float64 else g.float()
    tall = g.shape[0] > g.shape[1]
    x = (g.t() if tall else g).contiguous()
    x = (x.double() / (torch.linalg.vector_norm(x.double()) + eps)).to(dt)
    for _ in range(steps):
        gram = x @ x.t().contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.t().contiguous() if tall else x


def _gradient(m, n, g, dt, size=1e-3):
    r = max(1, min(m, n) // 4)
    low = (torch.randn(m, r, generator=g) * torch.logspace(0, -2, r)) @ torch.randn(r, n, generator=g) / math.sqrt(r)
    return (size * (low + 0.02 * torch.randn(m, n, generator=g))).to(dt)


def _check(got, g, steps=5, coeffs=C, eps=1e-7):
    want = _newton_schulz(g.cpu(), steps, coeffs, eps, torch.float64)
    plain = _newton_schulz(g.cpu(), steps, coeffs, eps, torch.float32).double()
    dt = got.dtype
    norm = want.norm()
    tol = 4 * (plain - want).norm() + 1e-7 * norm
    if dt != torch.float32:
        tol = tol + torch.finfo(dt).eps / 2 * norm + 2.0 ** -25 * math.sqrt(want.numel())
    err = (got.cpu().double() - want).norm()
    assert got.is_contiguous() and err <= tol, (tuple(g.shape), float(err / norm), float(tol / norm))


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 3), (8, 8), (16, 144), (31, 33), (33, 31), (64, 64), (65, 300), (300, 65), (127, 129),
          (128, 576), (192, 192), (200, 1000), (257, 256), (384, 128), (50, 5000)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_orthogonalize_list(dtype):
    """All sizes in one call, and each alone: the same bits, near 64 bits."""
    import lic_amd.functional as Fn
    g = torch.Generator().manual_seed(1)
    mats = [_gradient(m, n, g, dtype).to(DEV) for m, n in SHAPES]
    outs = Fn.orthogonalize(mats)
    for a, o in zip(mats, outs):
        _check(o, a)
        assert torch.equal(Fn.orthogonalize([a])[0], o)


@pytest.mark.parametrize("m,n", [(700, 900), (1030, 520), (640, 640), (70000, 24), (24, 70000)])
def test_orthogonalize_larger(m, n):
    import lic_amd.functional as Fn
    a = _gradient(m, n, torch.Generator().manual_seed(m), torch.float32).to(DEV)
    _check(Fn.orthogonalize([a])[0], a)


@pytest.mark.parametrize("steps", [1, 2, 3, 10])
@pytest.mark.parametrize("coeffs", [C, (2.0, -1.5, 0.5), (1.875, -1.25, 0.375)])
def test_orthogonalize_steps_and_coefficients(steps, coeffs):
    import lic_amd.functional as Fn
    g = torch.Generator().manual_seed(steps)
    for m, n in ((40, 70), (96, 96), (90, 20)):
        a = torch.randn(m, n, generator=g).to(DEV)
        _check(Fn.orthogonalize([a], steps=steps, coeffs=coeffs)[0], a, steps, coeffs)


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e-8, 1e-6, 1.0, 1e6, 1e30])
def test_orthogonalize_scales(size):
    """Gradients of any size: far below eps they stay small (divided by eps), far above fp16's and fp32's squares they
    are normalised."""
    import lic_amd.functional as Fn
    a = _gradient(48, 80, torch.Generator().manual_seed(2), torch.float32, size).to(DEV)
    _check(Fn.orthogonalize([a])[0], a)


def test_orthogonalize_zero_nan_and_views():
    import lic_amd.functional as Fn
    g = torch.Generator().manual_seed(5)
    good = torch.randn(60, 90, generator=g).to(DEV)
    nan = good.clone()
    nan[3, 4] = float("nan")
    inf = good.clone()
    inf[5, 6] = float("inf")
    wide = torch.randn(64, 400, generator=g).to(DEV)
    views = [wide[:, 3:203:2], wide.t(), wide[::3], wide.view(64, 20, 20)[:, 1], wide[2:3].expand(8, 400)]
    want = [Fn.orthogonalize([v.contiguous()])[0] for v in views]
    outs = Fn.orthogonalize([good, torch.zeros(30, 40, device=DEV), nan, torch.empty(0, 5, device=DEV), inf] + views)
    assert torch.equal(outs[0], Fn.orthogonalize([good])[0])      # a neighbour's NaN stays with it
    assert (outs[1] == 0).all() and not torch.isfinite(outs[2]).any() and outs[3].shape == (0, 5)
    assert not torch.isfinite(outs[4]).all()
    assert all(torch.equal(a, b) for a, b in zip(outs[5:], want))


def test_orthogonalize_many_and_eps():
    """More matrices than one launch carries, and eps = 0."""
    import lic_amd.functional as Fn
    g = torch.Generator().manual_seed(6)
    mats = [torch.randn(8 + i % 13, 8 + i % 17, generator=g).to(DEV) for i in range(150)]
    for a, o in zip(mats, Fn.orthogonalize(mats, eps=0.0)):
        _check(o, a, eps=0.0)


def test_orthogonalize_result_does_not_depend_on_the_list():
    """Long lists, whose many tiles take kernels of another shape, give every matrix the bits that it has alone."""
    import lic_amd.functional as Fn
    g = torch.Generator().manual_seed(8)
    shapes = [(192, 1728)] * 12 + [(256, 2304)] * 4 + [(300, 300), (40, 5000), (128, 576), (700, 800), (2048, 2048)]
    mats = [_gradient(m, n, g, torch.float32).to(DEV) for m, n in shapes]
    outs = Fn.orthogonalize(mats)
    for a, o in zip(mats, outs):
        assert torch.equal(Fn.orthogonalize([a])[0], o), tuple(a.shape)
    for a, o in zip(mats[:1] + mats[-3:], outs[:1] + outs[-3:]):
        _check(o, a)


def test_orthogonalize_streams_and_graph():
    import lic_amd.functional as Fn
    lists = [[torch.randn(96, 160, device=DEV), torch.randn(200, 64, device=DEV)], [torch.randn(128, 128, device=DEV)]]
    want = [[o.clone() for o in Fn.orthogonalize(l)] for l in lists]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in lists], [None, None]
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            got[i] = Fn.orthogonalize(lists[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
    graphs, outs = [torch.cuda.CUDAGraph() for _ in lists], [None, None]
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph):
            outs[i] = Fn.orthogonalize(lists[i])
    for k in range(3):
        for l in lists:
            for a in l:
                a.copy_(torch.randn_like(a))
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):       # both at once: their workspaces are their own
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for l, o in zip(lists, outs):
            assert all(torch.equal(a, b) for a, b in zip(Fn.orthogonalize(l), o))


@pytest.mark.parametrize("nesterov,adjust,wd", [(True, "rms", 0.0), (False, "shape", 0.1)])
def test_muon_step(nesterov, adjust, wd):
    """Two steps against the optimiser's definition in 64 bits.  The update is lr * scale * NS(u) with every factor
    within fp32 rounding: 1e-5 of the step's norm covers the products (4 * 2.5e-6) and the scaling."""
    from lic_amd.optim import Muon
    g = torch.Generator().manual_seed(7)
    shapes = [(24, 16, 3, 3), (64, 32), (16, 40, 1, 1)]
    params = [torch.nn.Parameter(torch.randn(s, generator=g).to(DEV)) for s in shapes]
    opt = Muon(params, lr=0.02, momentum=0.9, nesterov=nesterov, adjust=adjust, weight_decay=wd)
    ref, mom = [p.detach().cpu().double() for p in params], [torch.zeros(s, dtype=torch.float64) for s in shapes]
    for _ in range(2):
        for i, p in enumerate(params):
            grad = torch.randn(p.shape, generator=g)
            p.grad = grad.to(DEV)
            before = ref[i].clone()
            mom[i] = 0.9 * mom[i] + 0.1 * grad.double()
            u = 0.9 * mom[i] + 0.1 * grad.double() if nesterov else mom[i]
            o = _newton_schulz(u.reshape(u.shape[0], -1), 5, C, 1e-7, torch.float64).view(u.shape)
            rows, cols = u.shape[0], u[0].numel()
            scale = 0.2 * math.sqrt(max(rows, cols)) if adjust == "rms" else math.sqrt(max(1, rows / cols))
            ref[i] = before * (1 - 0.02 * wd) - 0.02 * scale * o
        opt.step()
    for p, r, s in zip(params, ref, shapes):
        assert ((p.detach().cpu().double() - r).norm() <= 2e-5 * 0.02 * 10 * math.sqrt(min(s[0], r[0].numel())) +
                2 ** -23 * r.norm())
        assert opt.state[p]["momentum"].dtype == torch.float32
    opt.load_state_dict(opt.state_dict())
    opt.step()


def test_muon_captured_step_matches_eager():
    from lic_amd.optim import Muon
    torch.manual_seed(0)
    init = [torch.randn(48, 32, 3, 3, device=DEV), torch.randn(64, 64, device=DEV)]
    grads = [[torch.randn_like(p) for p in init] for _ in range(4)]

    def params():
        ps = [torch.nn.Parameter(p.clone()) for p in init]
        for p in ps:
            p.grad = torch.zeros_like(p)
        return ps
    eager, cap = params(), params()
    oe, oc = (Muon(ps, lr=torch.tensor(0.01, device=DEV), weight_decay=0.01) for ps in (eager, cap))
    for p, q, g in zip(eager, cap, grads[0]):
        p.grad.copy_(g)
        q.grad.copy_(g)
    oe.step()
    oc.step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        oc.step()
    for k in (1, 2, 3):
        for p, q, g in zip(eager, cap, grads[k]):
            p.grad.copy_(g)
            q.grad.copy_(g)
        if k == 3:   # a schedule's change reaches the captured step
            for o in (oe, oc):
                o.param_groups[0]["lr"].fill_(0.005)
        oe.step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(eager, cap))


def test_muon_16_bit_weights():
    """bf16 weights move by the fp32 update and are rounded once; empty ones are left alone."""
    from lic_amd.optim import Muon
    g = torch.Generator().manual_seed(9)
    w, grad = torch.randn(40, 64, generator=g).bfloat16(), torch.randn(40, 64, generator=g).bfloat16()
    p, none = torch.nn.Parameter(w.to(DEV)), torch.nn.Parameter(torch.zeros(0, 8, device=DEV))
    p.grad, none.grad = grad.to(DEV), torch.zeros(0, 8, device=DEV)
    Muon([p, none], lr=0.1, momentum=0.0, adjust="shape").step()
    want = w.double() - 0.1 * _newton_schulz(grad.double(), 5, C, 1e-7, torch.float64)
    # the update's own error, 4 * 2.5e-6 of its norm, is below a value's rounding here
    tol = torch.finfo(torch.bfloat16).eps / 2 * want.abs() + 0.1 * 1e-5 * math.sqrt(40)
    assert ((p.detach().cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("mode", ["--eager", "--graph"])
def test_train_cli_with_muon(mode, monkeypatch, capsys):
    """train_net_unet.py --optimizer muon (at its 256 x 256 crops, which the net's windows need): eager and captured steps
    run and print a finite epoch summary."""
    import re
    import sys
    import train_net_unet
    monkeypatch.setattr(sys, "argv", ["train_net_unet.py", "--optimizer", "muon", mode, "--batch_size", "1",
                                      "--steps_per_epoch", "2", "--warmup", "2", "--lr", "1e-4"])
    train_net_unet.main()
    out = capsys.readouterr().out
    loss = float(re.search(r"\[Epoch 0000 TRAIN\] Loss: (\S+)", out).group(1))
    assert math.isfinite(loss) and loss > 0


@pytest.mark.parametrize("wd", [0.05, 2.0])
def test_muon_16_bit_decay(wd):
    """bf16 weights, decay and update are rounded together, once: also a decay (lr wd = 5e-4 of the weight) that a bf16
    multiply would lose (half a step is 2^-8).  Tolerance: half a step of the result, and the update's own error, 1e-5 of
    its norm at most (4 * 2.5e-6)."""
    from lic_amd.optim import Muon
    g = torch.Generator().manual_seed(10)
    w, grad = torch.randn(40, 64, generator=g).bfloat16(), torch.randn(40, 64, generator=g).bfloat16()
    x = _newton_schulz(grad.double(), 5, C, 1e-7, torch.float64)
    for lr in (0.01, torch.tensor(0.01, device=DEV)):
        p = torch.nn.Parameter(w.to(DEV))
        p.grad = grad.to(DEV)
        Muon([p], lr=lr, momentum=0.0, adjust="shape", weight_decay=wd).step()
        want = w.double() * (1 - 0.01 * wd) - 0.01 * x
        tol = torch.finfo(torch.bfloat16).eps / 2 * want.abs() + 0.01 * 1e-5 * math.sqrt(40)
        assert ((p.detach().cpu().double() - want).abs() <= tol).all()
        lost = (w.double() - 0.01 * x).bfloat16()
        assert not torch.equal(p.detach().cpu(), lost)


def test_muon_captured_without_a_step_before_is_refused():
    """A graph that created the momentum would set it to zero at every replay."""
    from lic_amd.optim import Muon
    p = torch.nn.Parameter(torch.randn(16, 16, device=DEV))
    p.grad = torch.randn_like(p)
    opt, before, graph = Muon([p], lr=torch.tensor(0.01, device=DEV)), p.detach().clone(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="eager step"):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    assert torch.equal(p, before) and not opt.state[p]
    opt.step()
    assert not torch.equal(p, before) and "momentum" in opt.state[p]


# error against that of fp32 products, and the bound: midway between the recorded ratio and the one without what the shape
# is there for (16 x 144, 64 x 64: the third part of X, 1.20 and 1.25 without; 128 x 576, 2048 x 2048: short chains of the
# matrix instructions' own additions, 1.32 and 0.71 with chains of 16 steps)
@pytest.mark.parametrize("m,n,bound", [(16, 144, (0.81 + 1.20) / 2), (64, 64, (1.02 + 1.25) / 2),
                                       (128, 576, (1.09 + 1.32) / 2), (2048, 2048, (0.54 + 0.71) / 2)])
def test_orthogonalize_error_against_fp32_products(m, n, bound):
    """Frobenius norms, averaged over four seeds; fp32 products by the library's plain fp32 matrix product."""
    import lic_amd.functional as Fn

    def products(g, dt):
        a, b, c = C
        x = g.double()
        x = (x / (torch.linalg.vector_norm(x) + 1e-7)).to(dt)
        for _ in range(5):
            gram = torch.mm(x, x.t().contiguous())
            x = a * x + torch.mm(b * gram + c * torch.mm(gram, gram), x)
        return x.double()
    kernel = plain = 0.0
    for seed in range(4):
        g = _gradient(m, n, torch.Generator().manual_seed(20 + seed), torch.float32).to(DEV)
        want = products(g, torch.float64)
        kernel += float((Fn.orthogonalize([g])[0].double() - want).norm())
        plain += float((products(g, torch.float32) - want).norm())
    assert kernel <= bound * plain, (kernel / plain, bound)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_orthogonalize_infinity_leaves_nothing_finite(dtype):
    import lic_amd.functional as Fn
    g = torch.Generator().manual_seed(11)
    mats = [torch.randn(s, generator=g).to(dtype).to(DEV) for s in ((1, 1), (1, 9), (5, 1), (60, 90), (300, 70), (64, 64))]
    for m in mats:
        m[m.shape[0] // 2, m.shape[1] // 3] = float("-inf")
    assert not any(torch.isfinite(o).any() for o in Fn.orthogonalize(mats))
