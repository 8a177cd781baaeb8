"""The rotary, 8-bit and orthogonalising operators together, as a window-attention block uses them: positions in its
forward and backward, a Muon step on its weights, then the block served with 8-bit Linears."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _block(rotary=100.0, shift=4):
    from lic_amd.layers import WinBasedAttention
    torch.manual_seed(3)
    return WinBasedAttention(96, 4, 8, shift, rotary=rotary).to(DEV)


def _oracle(blk, x, quant=False):
    """The block in 64 bits from its definition: [B, H, W, C] -> x + proj(attention(rotated q, k; v))."""
    from oracle import ref_cpu as R
    C, heads, ws, sh = blk.dim, blk.num_heads, blk.window_size, blk.shift_size
    B, H, W, _ = x.shape
    d = C // heads
    P = {k: v.detach().cpu().double() for k, v in blk.state_dict().items()}

    def linear(t, name):
        w, b = P[name + ".weight"], P[name + ".bias"]
        if not quant:
            return t @ w.t() + b
        tt, tw = t.abs().amax(-1, keepdim=True), w.abs().amax(-1, keepdim=True)
        return (torch.round(127 * t / tt) @ torch.round(127 * w / tw).t()) * (tt / 127) * (tw[:, 0] / 127) + b
    qkv = linear(x, "attn.qkv")
    if blk.rotary is not None:
        p0 = d // 4
        p1 = d // 2 - p0
        f = torch.cat([blk.rotary ** -(torch.arange(n, dtype=torch.float64) / n) for n in (p0, p1)])
        yy, xx = torch.meshgrid(torch.arange(H), torch.arange(W), indexing="ij")
        at = torch.cat([yy[..., None].expand(-1, -1, p0), xx[..., None].expand(-1, -1, p1)], -1).double()
        turn = torch.polar(torch.ones(H, W, d // 2, dtype=torch.float64), at * f)[None, :, :, None]
        qk = qkv[..., :2 * C].reshape(B, H, W, 2 * heads, d)
        z = torch.complex(qk[..., :d // 2], qk[..., d // 2:]) * turn
        qkv = torch.cat([torch.cat([z.real, z.imag], -1).reshape(B, H, W, 2 * C), qkv[..., 2 * C:]], -1)
    if sh:
        qkv = torch.roll(qkv, (-sh, -sh), (1, 2))
    win = R.window_partition(qkv.contiguous(), ws).view(-1, ws * ws, 3, heads, d).permute(2, 0, 3, 1, 4)
    s = (win[0] * d ** -0.5) @ win[1].transpose(-2, -1)
    bias = P["attn.relative_position_bias_table"][R.relative_position_index(ws).view(-1)]
    s = s + bias.view(ws * ws, ws * ws, heads).permute(2, 0, 1)
    if sh:
        m = R.wba_mask(H, W, ws, sh).double()
        s = (s.view(B, m.shape[0], heads, ws * ws, ws * ws) + m[None, :, None]).view_as(s)
    o = (torch.softmax(s, -1) @ win[2]).transpose(1, 2).reshape(-1, ws, ws, C)
    o = R.window_reverse(o, ws, H, W)
    if sh:
        o = torch.roll(o, (sh, sh), (1, 2))
    return x + linear(o, "attn.proj")


@pytest.mark.parametrize("rotary", [None, 100.0])
@pytest.mark.parametrize("shift", [0, 4])
def test_block_forward(rotary, shift):
    """fp32: within 1e-5 of the 64-bit block's size (its products sum up to 384 terms in fp32: 384 * 2^-24 = 2.3e-5 of
    the terms' sum at worst, the softmax and the outputs are averages of such)."""
    import lic_amd.functional as Fn
    blk = _block(rotary, shift)
    x = torch.randn(2, 16, 24, 96, generator=torch.Generator().manual_seed(1))
    want = _oracle(blk, x.double())
    with torch.no_grad():
        got = blk.run(Fn.Act(x.to(DEV))).t.cpu().double()
    assert (got - want).abs().max() <= 2.3e-5 * want.abs().max()


def test_rotary_block_is_position_relative():
    """Scores see position differences only: moving the map by a window moves the output by a window."""
    import lic_amd.functional as Fn
    blk = _block(shift=0)
    x = torch.randn(1, 32, 32, 96, device=DEV)
    with torch.no_grad():
        y = blk.run(Fn.Act(x)).t
        moved = blk.run(Fn.Act(torch.roll(x, (8, 16), (1, 2)).contiguous())).t
    assert (torch.roll(y, (8, 16), (1, 2)) - moved).abs().max() <= 2.3e-5 * y.abs().max()


def test_block_gradients():
    """Training path with rotary positions: gradients of the input and the qkv weight against differences of the 64-bit
    block in random directions (central, step 1e-4: error 1e-8 relative; fp32 backward 1e-4 of the gradient's norm)."""
    from lic_amd import train_net
    blk = _block()
    g = torch.Generator().manual_seed(2)
    x, dy = torch.randn(1, 16, 16, 96, generator=g), torch.randn(1, 16, 16, 96, generator=g)
    leaf = x.to(DEV).requires_grad_(True)
    y = train_net.wba(blk, leaf)
    gx, gw = torch.autograd.grad(y, (leaf, blk.attn.qkv.weight), dy.to(DEV))
    vx, vw = torch.randn(x.shape, generator=g).double(), torch.randn(gw.shape, generator=g).double()

    def along(direction_x, direction_w, h):
        with torch.no_grad():
            keep = blk.attn.qkv.weight.detach().clone()
            P = blk.state_dict
            sd = {k: v.detach().cpu().double() for k, v in P().items()}
            sd["attn.qkv.weight"] = sd["attn.qkv.weight"] + h * direction_w

            class Blk:
                dim, num_heads, window_size, shift_size, rotary = (blk.dim, blk.num_heads, blk.window_size,
                                                                   blk.shift_size, blk.rotary)

                @staticmethod
                def state_dict():
                    return sd
            return (_oracle(Blk, x.double() + h * direction_x) * dy.double()).sum()
    for got, dx, dw in ((gx, vx, 0 * vw), (gw, 0 * vx, vw)):
        slope = (along(dx, dw, 1e-4) - along(dx, dw, -1e-4)) / 2e-4
        v = dx if got is gx else dw
        have = (got.cpu().double() * v).sum()
        assert abs(slope - have) <= 1e-4 * got.cpu().double().norm() * v.norm()


def test_block_trains_with_muon_then_serves_in_int8():
    """One run of the operators: forward and backward with rotary positions, a Muon step on the block's matrices, the
    updated block with 8-bit Linears.  Served against the 64-bit block with the same quantisation: proj's input codes may
    differ by one where the attention's fp32 output lies within its error of a border, one step of the token's scale
    (max / 127) times one weight each."""
    import lic_amd.functional as Fn
    from lic_amd import train_net
    from lic_amd.optim import Muon, split_muon_params
    blk = _block()
    mats, others = split_muon_params(blk, blk.parameters())
    assert len(mats) == 2
    opt = Muon(mats, lr=0.01)
    before = [p.detach().clone() for p in mats]
    x = torch.randn(2, 16, 16, 96, generator=torch.Generator().manual_seed(5))
    y = train_net.wba(blk, x.to(DEV))
    (y.float() ** 2).mean().backward()
    opt.step()
    for p, b in zip(mats, before):
        # the update of matrix p: lr * 0.2 sqrt(max(rows, cols)) * X, X with singular values up to 1.21
        step = torch.linalg.matrix_norm((b - p.detach()).double(), 2)
        assert 0 < step <= 0.01 * 0.2 * max(p.shape) ** 0.5 * 1.21
    with torch.no_grad():
        plain = blk.run(Fn.Act(x.to(DEV))).t.cpu().double()
        with Fn.int8_linears():
            served = blk.run(Fn.Act(x.to(DEV))).t.cpu().double()
            again = blk.run(Fn.Act(x[1:].to(DEV).contiguous())).t.cpu().double()
    assert torch.equal(served[1:], again)       # a token's result does not depend on the batch
    want = _oracle(blk, x.double(), quant=True)
    off = (served - want).abs()
    wmax = blk.attn.proj.weight.detach().abs().max().item()
    step = 3 * want.abs().max() / 127 * wmax    # a token with three codes at a border
    assert off.max() <= step and (off > 2.3e-5 * want.abs().max()).double().mean() <= 0.05
    assert not torch.equal(served, plain)


def test_int8_linears_in_the_codec():
    """The whole codec inside the context: finite results near the fp16 ones, and two runs alike."""
    import bench
    import lic_amd.functional as Fn
    net = bench.build_net("net_ga", "fp16", 256, 1, "cpu").cuda()
    x = bench.bench_input(1, 256, 0).cuda()
    plain = [t.clone() for t in net(x, "test")]
    with Fn.int8_linears():
        a = [t.clone() for t in net(x, "test")]
        b = [t.clone() for t in net(x, "test")]
    assert all(torch.isfinite(t).all() for t in a) and all(torch.equal(u, v) for u, v in zip(a, b))
    assert not torch.equal(a[2], plain[2])
    assert all(torch.equal(u, v) for u, v in zip(plain, net(x, "test")))    # nothing of it stays


def test_wnsa_with_rotary():
    import lic_amd.functional as Fn
    from lic_amd.layers import Win_noShift_Attention
    torch.manual_seed(0)
    m = Win_noShift_Attention(96, 4, 8, 4, rotary=100.0).to(DEV)
    x = torch.randn(1, 16, 16, 96, device=DEV)
    with torch.no_grad():
        a = m.run(Fn.Act(x)).t.clone()
        for blk in m.conv_b:
            if hasattr(blk, "rotary"):
                blk.rotary = None
        b = m.run(Fn.Act(x)).t
    assert torch.isfinite(a).all() and not torch.equal(a, b)


def test_wnsa_blocks_with_rotary(monkeypatch):
    """Each of the four window-attention blocks of Win_noShift_Attention(rotary=), in its place with the input that it
    meets there, against its definition in 64 bits (test_block_forward's tolerance)."""
    import lic_amd.functional as Fn
    from lic_amd.layers import WinBasedAttention, Win_noShift_Attention
    torch.manual_seed(0)
    m = Win_noShift_Attention(96, 4, 8, 4, rotary=100.0).to(DEV)
    run, seen = WinBasedAttention.run, []

    def recorded(self, x, out=None, **kw):
        assert not kw
        before = x.nchw().permute(0, 2, 3, 1).cpu()
        y = run(self, x, out)
        seen.append((self, before, y.nchw().permute(0, 2, 3, 1).cpu()))
        return y
    monkeypatch.setattr(WinBasedAttention, "run", recorded)
    with torch.no_grad():
        m.run(Fn.Act(torch.randn(1, 16, 24, 96, generator=torch.Generator().manual_seed(7)).to(DEV)))
    assert [b for b, _, _ in seen] == [m.conv_b[i] for i in (0, 2, 5, 8)]
    for blk, x, y in seen:
        assert blk.rotary == 100.0
        want = _oracle(blk, x.double())
        assert (y.double() - want).abs().max() <= 2.3e-5 * want.abs().max()


def test_int8_linears_of_the_codec_match_64_bits(monkeypatch):
    """Every product that the codec runs in 8 bits, with the input, shortcut and weights that it meets there, against the
    quantised product in 64 bits (test_gpu_int8's tolerance): they are the window-attention blocks' qkv and proj, all of
    them."""
    import bench
    import lic_amd.functional as Fn
    from lic_amd.layers import Linear, WinBasedAttention
    from tests.test_gpu_int8 import _check, _codes, _result
    net = bench.build_net("net_ga", "fp16", 256, 1, "cpu").cuda()
    x = bench.bench_input(1, 256, 0).cuda()
    blocks = [b for b in net.modules() if isinstance(b, WinBasedAttention)]
    layers = {id(m): m for b in blocks for m in (b.attn.qkv, b.attn.proj)}
    product, run, at, calls, ran = Fn.linear_int8, Linear.run, [], [], set()

    def of_layer(self, *a, **k):
        at.append(self)
        try:
            return run(self, *a, **k)
        finally:
            at.pop()

    def recorded(a, pk, out=None, **kw):
        rows = lambda v: v.t[..., v.c0:v.c0 + v.c].reshape(-1, v.c).clone()
        r1, before = kw.get("r1"), rows(a)
        shortcut = rows(r1) if r1 is not None else None
        y = product(a, pk, out, **kw)
        ran.add(id(at[-1]))
        calls.append((at[-1], before, shortcut, kw.get("act", 0), rows(y)))
        return y
    monkeypatch.setattr(Linear, "run", of_layer)
    monkeypatch.setattr(Fn, "linear_int8", recorded)
    with torch.no_grad(), Fn.int8_linears():
        net(x, "test")
    used = [b for b in blocks if id(b.attn.qkv) in ran]
    assert len(used) >= 8 and len(calls) == 2 * len(used) and ran <= layers.keys()
    assert ran == {id(m) for b in used for m in (b.attn.qkv, b.attn.proj)}
    for layer, a, r1, act, y in calls:
        assert act == 0 and y.dtype == torch.float16
        codes, scale = _codes(a.cpu())
        wc, ws = _codes(layer.weight.detach().cpu())
        _check(y, *_result(codes, scale, wc, ws, layer.bias.detach().cpu().double(), 0, 0,
                           r1.cpu().double() if r1 is not None else None))


def test_eval_cli_with_int8_linears(capsys):
    """eval_net.py --int8-linear: the sweep inside the context, named in its line; nothing of it stays."""
    import json
    import eval_net
    import lic_amd.functional as Fn
    args = ["--synthetic-kodak", "--lambdas", "0.0067", "--precision", "fp16", "--graph"]
    lines = []
    for extra in ([], ["--int8-linear"]):
        eval_net.main(args + extra)
        lines.append(json.loads(capsys.readouterr().out.strip().splitlines()[-1]))
        assert not Fn.int8_mode()
    plain, eight = lines
    assert plain["precision"] == "fp16" and eight["precision"] == "fp16+int8_linear"
    with Fn.int8_linears():
        want, _, _ = eval_net.rd_sweep([0.0067], "", arch="net_ga", precision="fp16", graph=False, batched=True)
    for key in ("bpp", "psnr", "images"):
        assert eight["rd"][0][key] == want[0][key]
    assert eight["rd"][0]["psnr"] != plain["rd"][0]["psnr"]
    print("\n[int8 linears] fp16", plain["rd"], "8-bit", eight["rd"])
