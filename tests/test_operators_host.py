"""Rotary plans and the refusals of the rotary, 8-bit and orthogonalisation operators (no GPU: every call here is
refused before anything is launched, or never reaches the device)."""
import ctypes
import math

import pytest
import torch

import lic_amd
import lic_amd.functional as Fn
from lic_amd import _ffi
from lic_amd.functional import Act


def _plan(*a, **k):
    return Fn.RotaryPlan(*a, device="cpu", **k)


def test_rotary_plan_frequencies():
    p = _plan(32, (4, 6), base=100.0, scale=(1.0, 0.5))
    assert p.pairs == 10 and p.naxes == 2 and p.axes == [0] * 4 + [1] * 6
    want = [100.0 ** (-i / 4) for i in range(4)] + [0.5 * 100.0 ** (-i / 6) for i in range(6)]
    assert p.freqs == pytest.approx(want, rel=1e-15)
    shared = _plan(32, (4, 6), base=100.0, shared_ladder=True)
    assert shared.freqs == pytest.approx([100.0 ** (-i / 10) for i in range(10)], rel=1e-15)


@pytest.mark.parametrize("pos", [0, 1, -1, 12345, 2 ** 31 - 1, -2 ** 31])
def test_rotary_table_angles(pos):
    """The fixed-point turns times any int32 position, modulo 2^64, is the angle modulo one turn: off by at most
    |pos| / 2 steps of 2^-64 turns (the table's rounding: |pos| pi 2^-64 rad), the 64-bit reference's own rounding of
    pos * freq (2^-53 relative) and its 2 pi (2.5e-16 off, once a turn: under pos * freq * 2^-54)."""
    p = _plan(64, (16,), base=10000.0)
    for turns, freq in zip(p.table[:, 0].tolist(), p.freqs):
        got = (turns * pos) % 2 ** 64 / 2 ** 64 * 2 * math.pi
        want = pos * freq
        tol = abs(pos) * math.pi * 2 ** -64 + abs(pos) * freq * 2 ** -51 + 1e-12
        assert abs(math.remainder(got - want, 2 * math.pi)) <= tol


@pytest.mark.parametrize("args,kw", [((16, ()), {}), ((16, (4, 5)), {}), ((16, (4, 0)), {}), ((64, (1,) * 5), {}),
                                     ((16, (4,)), {"layout": "thirds"}), ((16, (4,)), {"base": 0.0}),
                                     ((16, (4, 4)), {"scale": (1.0,)}), ((16, (4,)), {"scale": float("inf")})])
def test_rotary_plan_refusals(args, kw):
    with pytest.raises(ValueError, match="RotaryPlan"):
        _plan(*args, **kw)


def test_host_tensors_are_refused():
    x = Act(torch.zeros(1, 2, 2, 32))
    with pytest.raises(ValueError, match="not on the GPU"):
        Fn.rotary(x, _plan(16, (4,)), 2)
    with pytest.raises(ValueError, match="not on the GPU"):
        Fn.quantize_tokens(x)
    with pytest.raises(ValueError, match="not on the GPU"):
        Fn.pack_linear_int8(torch.zeros(4, 32))
    with pytest.raises(ValueError, match="not on the GPU"):
        Fn.linear_int8(x, Fn.Int8Pack(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4), None, 32))
    with pytest.raises(ValueError, match="not on the GPU"):
        Fn.orthogonalize([torch.zeros(4, 4)])


def test_size_refusals():
    x = Act(torch.zeros(1, 2, 2, 32))
    with pytest.raises(ValueError, match="do not fit"):
        Fn.rotary(x, _plan(16, (4,)), 3)
    with pytest.raises(ValueError, match="do not fit"):
        Fn.rotary(x, _plan(16, (4,)), 0)
    with pytest.raises(ValueError, match="channels"):
        Fn.linear_int8(x, Fn.Int8Pack(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4), None, 31))
    with pytest.raises(ValueError, match="weight must be"):
        Fn.pack_linear_int8(torch.zeros(4, 4, 1))
    with pytest.raises(ValueError, match="bias"):
        Fn.pack_linear_int8(torch.zeros(4, 4), torch.zeros(5))
    with pytest.raises(ValueError, match="one dtype"):
        Fn.orthogonalize([torch.zeros(4, 4), torch.zeros(4, 4, dtype=torch.float16)])
    with pytest.raises(ValueError, match="one dtype"):
        Fn.orthogonalize([torch.zeros(4)])
    assert Fn.orthogonalize([]) == []


def test_overlap_rule():
    t = torch.zeros(1, 2, 2, 32)
    a = Act(t, 0, 16)
    assert Fn._overlaps(a, Act(t, 8, 16)) and Fn._overlaps(a, a)
    assert not Fn._overlaps(a, Act(t, 16, 16)) and not Fn._overlaps(a, Act(torch.zeros(1, 2, 2, 32)))
    assert not Fn._overlaps(Act(t[:, :1].clone()), Act(t)) and Fn._overlaps(Act(t[:, 1:]), Act(t))
    assert not Fn._overlaps(Act(t[:, :1]), Act(t[:, 1:])) and not Fn._overlaps(Act(t[:0]), Act(t[:0]))
    assert Fn._overlaps(Act(t.view(1, 1, 4, 32), 0, 16), Act(t, 16, 16))   # other shapes: refused on byte ranges


def _refused(status, text):
    assert status != 0 and text in _ffi._lib.lic_last_error().decode(), _ffi._lib.lic_last_error()


def test_c_entry_refusals():
    """Arguments the C ABI refuses; the fake pointers are never read."""
    lib = lic_amd.load_library()
    f = 4096   # a non-null, aligned address that nothing dereferences

    def rot(dtype=0, x=f, ldx=64, n=1, h=2, w=2, c=64, heads=2, dim=32, pairs=8, layout=0, table=f, naxes=2, pos=None,
            y=f, ldy=64):
        return lib.lic_rotary(dtype, x, ldx, n, h, w, c, heads, dim, pairs, layout, table, naxes, pos, 0, 0, y, ldy,
                              None)
    _refused(rot(dtype=7), "dtype")
    _refused(rot(heads=3), "fit the view")
    _refused(rot(heads=2 ** 30, dim=2 ** 30), "fit the view")
    _refused(rot(pairs=17), "fit the view")
    _refused(rot(pairs=0), "fit the view")
    _refused(rot(ldx=63), "fit the view")
    _refused(rot(layout=2), "layout")
    _refused(rot(naxes=0), "naxes")
    _refused(rot(naxes=4), "naxes")
    _refused(rot(naxes=5, pos=f), "naxes")
    _refused(rot(n=-1), "negative")
    _refused(rot(table=None), "null")
    _refused(rot(y=f, ldy=80), "in place")
    assert rot(n=0) == 0

    def quant(dtype=0, x=f, ldx=100, m=4, k=100, codes=f, kpad=128, scale=f):
        return lib.lic_quantize_int8(dtype, x, ldx, m, k, codes, kpad, scale, None)
    _refused(quant(dtype=3), "dtype")
    _refused(quant(kpad=96), "out of range")
    _refused(quant(kpad=100), "out of range")
    _refused(quant(k=0), "out of range")
    _refused(quant(k=200000, kpad=200000), "out of range")
    _refused(quant(m=-1), "out of range")
    _refused(quant(ldx=99), "stride")
    _refused(quant(codes=f + 8), "aligned")
    assert quant(m=0) == 0

    def lin(dtype=0, x=f, ldx=100, xc=None, xs=None, m=4, k=100, w=f, kpad=128, ws=f, n=8, act=0, r1=None, ldr1=0, y=f,
            ldy=8, work=f, nbytes=1 << 20):
        return lib.lic_linear_int8(dtype, x, ldx, xc, xs, m, k, w, kpad, ws, None, n, act, 0.0, r1, ldr1, y, ldy, work,
                                   nbytes, None)
    _refused(lin(dtype=-1), "dtype")
    _refused(lin(n=0), "n out of range")
    _refused(lin(act=4), "act")
    _refused(lin(ldy=7), "stride below n")
    _refused(lin(r1=f, ldr1=7), "stride below n")
    _refused(lin(x=None), "x or xcodes")
    _refused(lin(xc=f, xs=f), "x or xcodes")
    _refused(lin(x=None, xc=f), "x or xcodes")
    _refused(lin(w=f + 4), "aligned")
    _refused(lin(ldx=99), "stride below k")
    big = dict(m=5, k=400, ldx=400, kpad=448)
    _refused(lin(work=None, **big), "workspace")
    _refused(lin(work=f + 8, **big), "workspace")
    _refused(lin(nbytes=16, **big), "workspace")
    assert lin(m=0) == 0
    assert lib.lic_linear_int8_workspace(5, 448, 8) >= 5 * 448 + 20
    assert lib.lic_linear_int8_workspace(-1, 128, 8) == -1 and lib.lic_linear_int8_workspace(1, 128, 0) == -1
    for m in (1, 4, 5, 64, 65, 1037, 16384, 16385, 131072):
        for kpad in (64, 384, 448, 4096, 4160):
            for n in (1, 64, 65, 517, 16384):
                assert lib.lic_linear_int8_workspace(m, kpad, n) == Fn._int8_workspace(m, kpad, n)

    def ortho(rows=8, cols=8, g=f, out=f, steps=5, eps=1e-7, dtype=0, count=1, ws=f, nbytes=1 << 30, coeffs=True):
        m = (_ffi.OrthoMat * 1)()
        m[0].g, m[0].rs, m[0].cs, m[0].out, m[0].rows, m[0].cols = g, max(cols, 1), 1, out, rows, cols
        co = (ctypes.c_float * 3)(*Fn.NEWTON_SCHULZ) if coeffs else None
        return lib.lic_orthogonalize(dtype, count, m, steps, co, eps, ws, nbytes, None)
    _refused(ortho(rows=0), "out of range")
    _refused(ortho(rows=65537, cols=65537), "out of range")
    _refused(ortho(rows=(1 << 24) + 1), "out of range")
    _refused(ortho(cols=(1 << 24) + 1), "out of range")
    _refused(ortho(g=None), "null")
    _refused(ortho(out=None), "null")
    _refused(ortho(steps=0), "steps")
    _refused(ortho(eps=-1.0), "eps")
    _refused(ortho(eps=float("nan")), "eps")
    _refused(ortho(dtype=9), "dtype")
    _refused(ortho(count=-1), "null")
    _refused(ortho(coeffs=False), "null")
    _refused(ortho(ws=None), "workspace")
    _refused(ortho(ws=f + 8), "workspace")
    _refused(ortho(nbytes=64), "workspace")
    assert ortho(count=0) == 0
    m = (_ffi.OrthoMat * 1)()
    m[0].g, m[0].rs, m[0].cs, m[0].out, m[0].rows, m[0].cols = f, 8, 1, f, 8, 8
    wild = (ctypes.c_float * 3)(10.0, 10.0, 10.0)
    _refused(lib.lic_orthogonalize(0, 1, m, 9, wild, 1e-7, f, 1 << 30, None), "run away")
    assert lib.lic_orthogonalize_workspace(0, 1, m) > 0 and lib.lic_orthogonalize_workspace(0, -1, m) == -1


def test_ortho_struct_matches_c_compiler(tmp_path):
    import shutil
    import subprocess
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    from tests.test_capi import ROOT
    py = _ffi.OrthoMat
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "lic.h"\nint main(void) {\n'
                   'printf("%zu", sizeof(lic_ortho_mat));\n' +
                   "".join(f'printf(" %zu", offsetof(lic_ortho_mat, {n[0]}));\n' for n in py._fields_) + "return 0; }")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(py)] + [getattr(py, n[0]).offset for n in py._fields_]
    assert lic_amd.load_library().lic_args_size(8) == ctypes.sizeof(py)


def test_muon_refusals_and_split():
    from lic_amd.layers import Conv2d, ConvTranspose2d, Linear
    from lic_amd.optim import Muon, split_muon_params
    net = torch.nn.Sequential(Conv2d(16, 32, 3), Conv2d(16, 16, 3, groups=16), ConvTranspose2d(32, 16, 5), Linear(16, 4),
                              torch.nn.LayerNorm(16))
    mats, others = split_muon_params(net, net.parameters())
    assert [tuple(p.shape) for p in mats] == [(32, 16, 3, 3), (32, 16, 5, 5)]
    assert len(mats) + len(others) == len(list(net.parameters()))
    with pytest.raises(ValueError, match="matrices"):
        Muon([torch.nn.Parameter(torch.zeros(4))])
    with pytest.raises(ValueError, match="adjust"):
        Muon(mats, adjust="none")
    with pytest.raises(ValueError, match="momentum"):
        Muon(mats, momentum=1.0)
    with pytest.raises(ValueError, match="lr"):
        Muon(mats, lr=-1.0)


def test_together_steps_all_or_none():
    """One scheduler reaches every group, a state comes back whole, and a GradScaler that meets a NaN in one optimiser's
    gradients leaves the other's weights alone too."""
    from lic_amd.optim import Muon, Together
    with pytest.raises(ValueError, match="at least one"):
        Together()
    p, q = (torch.nn.Parameter(torch.ones(3)) for _ in range(2))
    opt = Together(torch.optim.Adam([p], lr=0.5), torch.optim.SGD([q], lr=0.25))
    sch = torch.optim.lr_scheduler.MultiStepLR(opt, [1], 0.5)
    p.grad, q.grad = torch.ones(3), torch.ones(3)
    opt.step()
    sch.step()
    assert torch.allclose(p, torch.full((3,), 0.5)) and torch.equal(q, torch.full((3,), 0.75))
    assert [o.param_groups[0]["lr"] for o in opt.optimizers] == [0.25, 0.125]
    other = Together(torch.optim.Adam([p], lr=0.5), torch.optim.SGD([q], lr=0.25))
    other.load_state_dict(opt.state_dict())
    assert [g["lr"] for g in other.param_groups] == [0.25, 0.125] and other.optimizers[0].state[p]["step"] == 1
    scaler = torch.amp.GradScaler("cpu", init_scale=4.0)
    scaler.scale(torch.ones(()))
    before = [p.detach().clone(), q.detach().clone()]
    p.grad, q.grad = torch.tensor([1.0, float("nan"), 1.0]), torch.ones(3)
    scaler.unscale_(opt)
    scaler.step(opt)
    scaler.update()
    assert torch.equal(p, before[0]) and torch.equal(q, before[1])
    opt.zero_grad(set_to_none=True)
    assert p.grad is None and q.grad is None
    m = Muon([torch.nn.Parameter(torch.zeros(4, 4))])
    with pytest.raises(ValueError, match="matrices"):
        m.add_param_group({"params": [torch.nn.Parameter(torch.zeros(4))]})
    assert len(m.param_groups) == 1
    with pytest.raises(ValueError, match="steps"):
        Muon([torch.nn.Parameter(torch.zeros(4, 4))], steps=0)


def test_muon_state_keeps_fp32_momentum():
    from lic_amd.optim import Muon
    p = torch.nn.Parameter(torch.zeros(8, 8, dtype=torch.bfloat16))
    a, b = Muon([p]), Muon([p])
    a.state[p]["momentum"] = torch.randn(8, 8) * 1.2345678
    b.load_state_dict(a.state_dict())
    got = b.state[p]["momentum"]
    assert got.dtype == torch.float32 and torch.equal(got, a.state[p]["momentum"])
    assert got.data_ptr() != a.state[p]["momentum"].data_ptr()


def test_int8_context_is_nested_and_thread_local():
    import threading
    assert not Fn.int8_mode()
    seen = []
    with Fn.int8_linears():
        t = threading.Thread(target=lambda: seen.append(Fn.int8_mode()))
        t.start()
        t.join()
        with Fn.int8_linears(False):
            assert not Fn.int8_mode()
        assert Fn.int8_mode()
    assert not Fn.int8_mode() and seen == [False]


def test_rotary_block_refusal():
    from lic_amd.layers import WinBasedAttention
    with pytest.raises(ValueError, match="even head"):
        WinBasedAttention(24, 8, 8, rotary=100.0)
    plain, turned = WinBasedAttention(32, 4, 8), WinBasedAttention(32, 4, 8, rotary=100.0)
    assert plain.state_dict().keys() == turned.state_dict().keys()


def test_together_takes_no_groups_of_its_own():
    """A group that no optimiser would step is refused; one given to an optimiser is stepped, and the whole's scheduler,
    zero_grad and GradScaler see it."""
    from lic_amd.optim import Together
    p, q, r = (torch.nn.Parameter(torch.ones(3)) for _ in range(3))
    opt = Together(torch.optim.Adam([p], lr=0.5), torch.optim.SGD([q], lr=0.25))
    with pytest.raises(ValueError, match="one of its optimisers"):
        opt.add_param_group({"params": [r]})
    assert len(opt.param_groups) == 2
    opt.optimizers[1].add_param_group({"params": [r], "lr": 0.5})
    assert [g["lr"] for g in opt.param_groups] == [0.5, 0.25, 0.5] and opt.param_groups[2]["params"][0] is r
    sch = torch.optim.lr_scheduler.MultiStepLR(opt, [1], 0.5)
    r.grad = torch.ones(3)
    opt.step()
    sch.step()
    assert torch.equal(r, torch.full((3,), 0.5)) and opt.optimizers[1].param_groups[1]["lr"] == 0.25
    scaler = torch.amp.GradScaler("cpu", init_scale=4.0)
    scaler.scale(torch.ones(()))
    scaler.unscale_(opt)
    assert torch.equal(r.grad, torch.full((3,), 0.25))
    opt.zero_grad(set_to_none=True)
    assert r.grad is None
    with pytest.raises(ValueError, match="more than one"):
        Together(torch.optim.SGD([p], lr=0.1), torch.optim.SGD([p], lr=0.1))


@pytest.mark.parametrize("how", ["deepcopy", "pickle"])
def test_together_copies_whole(how):
    """A copy steps its own parameters with its own optimisers, whose groups and state are the copy's."""
    import copy
    import pickle
    from lic_amd.optim import Together
    p, q = (torch.nn.Parameter(torch.ones(3)) for _ in range(2))
    opt = Together(torch.optim.Adam([p], lr=0.5), torch.optim.SGD([q], lr=0.25, momentum=0.5))
    p.grad, q.grad = torch.ones(3), torch.ones(3)
    opt.step()
    twin = copy.deepcopy(opt) if how == "deepcopy" else pickle.loads(pickle.dumps(opt))
    assert [type(o) for o in twin.optimizers] == [torch.optim.Adam, torch.optim.SGD]
    (p2,), (q2,) = (g["params"] for g in twin.param_groups)
    assert p2 is not p and torch.equal(p2, p) and torch.equal(q2, q)
    assert twin.optimizers[0].state[p2]["step"] == 1
    p2.grad, q2.grad = torch.ones(3), torch.ones(3)
    torch.optim.lr_scheduler.MultiStepLR(twin, [1], 0.5)
    for g in twin.param_groups:
        g["lr"] = 0.125
    twin.step()
    assert torch.equal(q2, torch.full((3,), 0.75 - 0.125 * 1.5)) and torch.equal(q, torch.full((3,), 0.75))
    assert [g["lr"] for g in opt.param_groups] == [0.5, 0.25] and twin.optimizers[0].state[p2]["step"] == 2
    twin.load_state_dict(opt.state_dict())
    assert [g["lr"] for g in twin.param_groups] == [0.5, 0.25]


def test_rotary_plan_follows_the_block():
    """The plan is that of the block's present base and heads, also after a run with others; equal ones are kept."""
    from lic_amd.layers import WinBasedAttention
    blk = WinBasedAttention(32, 4, 8, rotary=100.0)
    first = blk.rotary_plan("cpu")
    assert blk.rotary_plan("cpu") is first
    blk.rotary = 10000.0
    fresh = WinBasedAttention(32, 4, 8, rotary=10000.0).rotary_plan("cpu")
    assert torch.equal(blk.rotary_plan("cpu").table, fresh.table) and not torch.equal(fresh.table, first.table)
    blk.num_heads = 2
    assert blk.rotary_plan("cpu").head_dim == 16
    blk.num_heads, blk.rotary = 4, 100.0
    assert blk.rotary_plan("cpu") is first
    blk.rotary = -1.0
    with pytest.raises(ValueError, match="base has to be positive"):
        blk.rotary_plan("cpu")


def test_block_stored_whole_before_it_had_rotary():
    """A block pickled as a module when the attribute did not exist runs as one without rotary positions."""
    from lic_amd.layers import WinBasedAttention
    blk = WinBasedAttention(32, 4, 8)
    del blk.__dict__["rotary"]
    assert blk.rotary is None


def test_rotary_base_travels_with_a_state():
    """The keys are those of a block without rotary positions, so the base is in the state's metadata: a strict load into a
    block of another base, or of none, is refused, also through a file.  A load that is not strict goes through and says so;
    so does a state that names no base: a block without one (whose weights may be turned from then on), another program's."""
    import collections
    import io
    from lic_amd.layers import WinBasedAttention, Win_noShift_Attention
    plain, turned, other = (WinBasedAttention(32, 4, 8, rotary=r) for r in (None, 100.0, 10000.0))
    file = io.BytesIO()
    torch.save(turned.state_dict(), file)
    file.seek(0)
    stored = torch.load(file, weights_only=True)
    for state in (turned.state_dict(), stored):
        with pytest.raises(RuntimeError, match="rotary"):
            plain.load_state_dict(state)
        with pytest.raises(RuntimeError, match="rotary"):
            other.load_state_dict(state)
        WinBasedAttention(32, 4, 8, rotary=100.0).load_state_dict(state)
        assert "rotary" in plain.load_state_dict(state, strict=False).unexpected_keys[0]
        plain.load_state_dict(collections.OrderedDict(state.items()))   # no metadata: other programs' files
    turned.load_state_dict(plain.state_dict())
    WinBasedAttention(32, 4, 8).load_state_dict(plain.state_dict())
    # nested blocks, named by their place
    a, b = Win_noShift_Attention(32, 4, 8, 4, rotary=100.0), Win_noShift_Attention(32, 4, 8, 4)
    with pytest.raises(RuntimeError, match=r"conv_b\.0.*rotary"):
        b.load_state_dict(a.state_dict())
    b.load_state_dict(Win_noShift_Attention(32, 4, 8, 4).state_dict())


def test_int8_linears_scope(monkeypatch):
    """Inside the context the window-attention blocks' qkv and proj products run in 8 bits and no other Linear: not the
    generator of the decoder's filters, nor the entropy parameters' blocks and MLPs.  A layer of one's own opts in."""
    import bench
    from lic_amd.layers import Linear, WinBasedAttention
    net = bench.build_net("net_ga", "fp16", 256, 1, "cpu")
    blocks = {n for n, m in net.named_modules() if isinstance(m, WinBasedAttention)}
    linears = {n: m for n, m in net.named_modules() if isinstance(m, Linear)}
    inside = {n for b in blocks for n in (b + ".attn.qkv", b + ".attn.proj")}
    assert inside < linears.keys()
    seen = []
    monkeypatch.setattr(Linear, "packed", lambda self, dtype: None)
    monkeypatch.setattr(Linear, "packed_int8", lambda self: None)
    monkeypatch.setattr(Fn, "conv", lambda *a, **k: None)
    monkeypatch.setattr(Fn, "linear_int8", lambda *a, **k: seen.append(True))

    def eighth(m):
        seen.clear()
        m.run(Act(torch.zeros(1, 1, 1, m.in_features)))
        return bool(seen)
    assert not any(eighth(m) for m in linears.values())
    with Fn.int8_linears():
        assert {n for n, m in linears.items() if eighth(m)} == inside
        own = Linear(16, 16)
        assert not eighth(own)
        own.int8 = True
        assert eighth(own)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tensor_lr", [False, True])
@pytest.mark.parametrize("wd", [0.01, 1.0, 30.0])
def test_muon_decay_rounds_with_the_update(monkeypatch, dtype, tensor_lr, wd):
    """w <- w - (lr scale X + lr wd w) rounded once to w's type, decays far below its step included (lr wd 1e-5 of w here
    at the least, a bf16 step is 2^-7 of it).  X is given here in multiples that put w - update next to borders.
    Tolerance: half a step of the result, and the update's few fp32 roundings, 4 * 2^-24 of its terms; for fp32 weights, whose
    decay is a product of its own, three roundings of the weight."""
    from lic_amd.optim import Muon
    g = torch.Generator().manual_seed(3)
    w, x = torch.randn(16, 24, generator=g).to(dtype), torch.randn(16, 24, generator=g)
    # with this, lr * 0.2 sqrt(24) * x is an odd number of half steps of w, and the decay decides
    step = torch.finfo(dtype).eps * torch.exp2(torch.floor(torch.log2(w.float().abs())))
    lr, scale = 1e-3, 0.2 * math.sqrt(24)
    x[::2] = (step * 0.5 / (lr * scale))[::2] * torch.sign(w.float()[::2])
    monkeypatch.setattr(Fn, "orthogonalize", lambda mats, **k: [x.clone() for _ in mats])
    monkeypatch.setattr(Fn, "_on_current_device", lambda *a: None)
    p = torch.nn.Parameter(w.clone())
    p.grad = torch.ones_like(p)
    Muon([p], lr=torch.tensor(lr) if tensor_lr else lr, weight_decay=wd).step()
    lr64 = float(torch.tensor(lr)) if tensor_lr else lr
    upd, decay = lr64 * scale * x.double(), lr64 * wd * w.double()
    want = w.double() - upd - decay
    eps = torch.finfo(dtype).eps
    tol = eps / 2 * want.abs() + 4 * 2.0 ** -24 * (upd.abs() + decay.abs())
    if dtype == torch.float32:
        tol = tol + eps * w.double().abs()
    assert ((p.detach().double() - want).abs() <= tol).all()
    assert p.dtype == dtype
    if dtype != torch.float32:   # the decay is there: without it, the even rows' ties would round elsewhere
        off = (p.detach() != (w.double() - upd).to(dtype)).double().mean()
        assert off > 0.05


def test_muon_captured_without_a_step_before_is_refused(monkeypatch):
    """A graph that created the momentum would set it to zero at every replay."""
    from lic_amd.optim import Muon
    monkeypatch.setattr(Fn, "orthogonalize", lambda mats, **k: [m.clone() for m in mats])
    monkeypatch.setattr(Fn, "_on_current_device", lambda *a: None)
    p = torch.nn.Parameter(torch.ones(8, 8))
    p.grad = torch.ones(8, 8)
    opt = Muon([p], lr=0.5)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="eager step"):
        opt.step()
    assert torch.equal(p, torch.ones(8, 8)) and not opt.state[p]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    opt.step()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    opt.step()


def test_sizes_beyond_32_bits_are_refused():
    """The C entries take 32-bit sizes, and a call by ctypes cuts longer ones off: 2^32 + 1 tokens would be one."""
    def meta(*shape, dtype=torch.float16):
        return torch.empty(shape, dtype=dtype, device="meta")
    long = Act(meta(1, 2, 2 ** 31 + 1, 2))
    pk = Fn.Int8Pack(meta(4, 64, dtype=torch.int8), meta(4, dtype=torch.float32), None, 2)
    q = Fn.Int8Act(meta(1, 2, 2 ** 31 + 1, 64, dtype=torch.int8), meta(1, 2, 2 ** 31 + 1, dtype=torch.float32), 2,
                   torch.float16)
    with pytest.raises(ValueError, match="out of range"):
        Fn.rotary(long, _plan(2, (1,)), 1)
    with pytest.raises(ValueError, match="out of range"):
        Fn.rotary(Act(meta(1, 1, 1, 2 ** 32 + 64), 0, 2), _plan(2, (1,)), 1)
    with pytest.raises(ValueError, match="out of range"):
        Fn.rotary(Act(meta(1, 1, 1, 2)), _plan(2, (1,)), 1, out=Act(meta(1, 1, 1, 2 ** 32 + 64), 0, 2))
    for x in (long, q):
        with pytest.raises(ValueError, match="out of range"):
            Fn.linear_int8(x, pk)
    with pytest.raises(ValueError, match="out of range"):
        Fn.quantize_tokens(long)
    with pytest.raises(ValueError, match="out of range"):
        Fn.pack_linear_int8(meta(2 ** 32 + 1, 2))
    for shape in ((2 ** 32 + 1, 2), (2, 2 ** 32 + 1)):
        with pytest.raises(ValueError, match="out of range"):
            Fn.orthogonalize([meta(*shape)])


def test_c_entries_refuse_what_no_launch_takes():
    """A launch has less than 2^32 threads: products and lists of matrices beyond that are refused before anything runs."""
    lib = lic_amd.load_library()
    f = 4096

    def lin(m, n, kpad=128):
        return lib.lic_linear_int8(0, None, 0, f, f, m, 100, f, kpad, f, None, n, 0, 0.0, None, 0, f, n, None, 0, None)
    _refused(lin(2 ** 31 - 255, 8), "m out of range")
    _refused(lin(2 ** 31 - 1, 8), "m out of range")
    _refused(lin(8, 2 ** 27 - 15), "n out of range")
    _refused(lin(2 ** 30, 257), "m x n out of range")
    _refused(lin(2 ** 20, 2 ** 19), "m x n out of range")

    def tiles(rows, cols, count=1):
        m = (_ffi.OrthoMat * count)()
        for d in m:
            d.g, d.rs, d.cs, d.out, d.rows, d.cols = f, cols, 1, f, rows, cols
        return lib.lic_orthogonalize_workspace(0, count, m)
    assert tiles(64, 2 ** 24) > 0 and tiles(64 * 63, 2 ** 24) > 0     # 63 * 2^18 tiles
    assert tiles(64 * 64, 2 ** 24) == -1 and tiles(64, 2 ** 24, 64) == -1


def test_int8_scope_of_blocks_stored_whole():
    """Blocks pickled as modules before the layers had the attribute are taken as new ones are; a choice made is kept."""
    import pickle
    from lic_amd.layers import WinBasedAttention
    blk = WinBasedAttention(32, 4, 8)
    del blk.attn.qkv.__dict__["int8"]
    blk.attn.proj.int8 = False
    old = pickle.loads(pickle.dumps(blk))
    assert old.attn.qkv.int8 is True and old.attn.proj.int8 is False


def test_long_empty_matrices_are_not_refused_for_their_length():
    """An empty matrix has nothing to compute, however long its other side is."""
    with pytest.raises(ValueError, match="not on the GPU"):   # the next check
        Fn.orthogonalize([torch.empty(0, 2 ** 32 + 1)])
