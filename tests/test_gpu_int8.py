"""Products in 8-bit integers (lic_quantize_int8, lic_linear_int8): codes exactly, results against 64 bits.

Tolerance of a result: the integer sum is exact; its conversion, the two scales (each rounded once), their product, the
product with the sum and the bias' addition round to fp32 (6 roundings of values up to |sum * scales| + |bias|), GELU adds
8 fp32 roundings of its value's size (erf within 4 ulp, three products), r1 one more; the result rounds to its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24


def _codes(x):
    """The codes' definition in 64 bits: nearest integer to 127 x / max|x| (fp64 quotients of 24-bit values cannot
    round onto a border k + 1/2 that is not exact)."""
    x = x.double()
    top = x.abs().amax(1, keepdim=True)
    return torch.where(top > 0, torch.round(127 * x / top), torch.zeros_like(x)), top[:, 0] / 127


def _result(codes, scale, wc, ws, bias, act, slope, r1):
    acc = codes @ wc.t()
    y = acc * scale[:, None] * ws + bias
    size = (acc * scale[:, None] * ws).abs() + bias.abs()
    extra = 0
    if act == 1:
        y = y.clamp(min=0)
    elif act == 2:
        y = torch.where(y > 0, y, slope * y)
    elif act == 3:
        y, extra = torch.nn.functional.gelu(y), 8
    if r1 is not None:
        y, size = y + r1, size + r1.abs()
    return y, (7 + extra) * U * size


def _check(got, want, tol):
    dt = got.dtype
    tol = tol * 1.2 + want.abs() * torch.finfo(dt).eps / 2 + (2.0 ** -25 if dt == torch.float16 else 1e-37)
    err = (got.cpu().double() - want).abs()
    assert (err <= tol).all(), (err - tol).max()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 4096), (3, 7), (5, 64), (130, 192), (67, 333), (2, 8200), (9, 1000)])
def test_codes_are_exact(dtype, m, k):
    import lic_amd.functional as Fn
    g = torch.Generator().manual_seed(m * 1000 + k)
    x = (torch.randn(m, k, generator=g) * torch.exp(torch.randn(m, 1, generator=g) * 3)).to(dtype)
    q = Fn.quantize_tokens(Fn.Act(x.to(DEV).view(1, 1, m, k)))
    codes, scale = _codes(x)
    got = q.codes.view(m, -1).cpu()
    assert torch.equal(got[:, :k].double(), codes)
    assert (got[:, k:] == 0).all() and got.shape[1] % 64 == 0
    assert ((q.scale.view(m).cpu().double() - scale).abs() <= U * scale).all()


def test_codes_at_borders_and_extremes():
    """Exact halves go to even; rows of zeros, of the largest and the smallest values, of one value; NaN and infinity
    poison their own row only."""
    import lic_amd.functional as Fn
    halves = torch.arange(-126.5, 127.0, 1.0)
    rows = torch.zeros(10, 256)
    rows[0, :halves.numel()], rows[0, 255] = halves, 127.0            # scale 1: every border exactly
    rows[1, :halves.numel()], rows[1, 255] = halves * 2.0 ** -20, 127.0 * 2.0 ** -20
    rows[2, 5] = 1e-42                                               # subnormal
    rows[3, :2] = torch.tensor([3.4e38, -1.7e38])
    rows[4] = -0.37
    rows[6, 7] = float("nan")
    rows[7, 7] = float("-inf")
    rows[8, :3] = torch.tensor([1.0, 0.5, -0.5])                      # 63.5 -> 64
    rows[9, 0], rows[9, 1:] = 1.0, torch.nextafter(torch.tensor(0.5), torch.tensor(0.0))
    q = Fn.quantize_tokens(Fn.Act(rows.to(DEV).view(1, 2, 5, 256)))
    got, scale = q.codes.view(10, 256).cpu().double(), q.scale.view(10).cpu()
    fine = [0, 1, 2, 3, 4, 5, 8, 9]
    codes, want = _codes(rows[fine])
    assert torch.equal(got[fine], codes)
    assert ((scale[fine].double() - want).abs() <= U * want + 2.0 ** -150).all()
    assert torch.isnan(scale[6:8]).all() and (got[6:8] == 0).all()
    assert got[8, 0] == 127 and got[8, 1] == 64 and got[8, 2] == -64 and got[9, 1] == 63
    pk = Fn.pack_linear_int8(torch.randn(40, 256, device=DEV), torch.randn(40, device=DEV))
    y = Fn.linear_int8(Fn.Act(rows.to(DEV).view(1, 2, 5, 256)), pk).t.view(10, 40)
    assert torch.isnan(y[6:8]).all() and torch.isfinite(y[[0, 1, 2, 4, 5, 8, 9]]).all()
    assert torch.equal(y[5], pk.bias)


SIZES = [(1, 1, 1), (1, 64, 16), (1, 4096, 512), (2, 200, 33), (7, 333, 517), (16, 1024, 100), (17, 96, 64), (33, 4100, 70),
         (64, 192, 576), (100, 64, 1000), (129, 130, 257), (300, 2048, 300), (513, 192, 193), (1037, 333, 517)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear_int8_matches_64_bits(dtype, m, k, n):
    import lic_amd.functional as Fn
    g = torch.Generator().manual_seed(m + 7 * k + 13 * n)
    x = (torch.randn(m, k, generator=g) * torch.exp(0.7 * torch.randn(1, k, generator=g))).to(dtype)
    w, b = torch.randn(n, k, generator=g), torch.randn(n, generator=g)
    r1 = torch.randn(m, n, generator=g).to(dtype)
    pk = Fn.pack_linear_int8(w.to(DEV), b.to(DEV))
    wc, ws = _codes(w)
    assert torch.equal(pk.w.cpu()[:, :k].double(), wc)
    codes, scale = _codes(x)
    xa, ra = Fn.Act(x.to(DEV).view(1, 1, m, k)), Fn.Act(r1.to(DEV).view(1, 1, m, n))
    got = Fn.linear_int8(xa, pk).t
    _check(got.view(m, n), *_result(codes, scale, wc, ws, b.double(), 0, 0, None))
    act = 1 + (m + n) % 3
    y = Fn.linear_int8(xa, pk, act=act, slope=0.2, r1=ra).t
    _check(y.view(m, n), *_result(codes, scale, wc, ws, b.double(), act, 0.2, r1.double()))
    # quantised beforehand: the same bits
    assert torch.equal(Fn.linear_int8(Fn.quantize_tokens(xa), pk).t, got)


# whole rows in one launch (many tokens of few aligned channels; fp32 from 16384 tokens on) and the large tiles (with one to
# five steps of k, whole and ragged columns)
LARGE = [(16384, 64, 64), (16401, 128, 32), (16390, 192, 576), (16399, 200, 96), (16384, 256, 160), (16500, 320, 64),
         (16389, 384, 384), (16384, 8, 32), (2048, 40, 2048), (2050, 100, 2050), (2100, 190, 2047), (2048, 300, 2080),
         (4096, 40, 4096), (4103, 100, 4100), (4096, 190, 4097), (4100, 300, 4096)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", LARGE)
def test_linear_int8_large(dtype, m, k, n):
    import lic_amd.functional as Fn
    g = torch.Generator(device=DEV).manual_seed(m + 7 * k + 13 * n)
    x = (torch.randn(m, k, generator=g, device=DEV) * 3).to(dtype)
    x[7], x[9, 3] = 0, float("nan")
    w, b = torch.randn(n, k, generator=g, device=DEV), torch.randn(n, generator=g, device=DEV)
    r1 = torch.randn(m, n, generator=g, device=DEV).to(dtype)
    pk = Fn.pack_linear_int8(w, b)
    finite = torch.ones(m, dtype=torch.bool, device=DEV)
    finite[9] = False
    codes, scale = _codes(x[finite])
    wc, ws = _codes(w)

    def check(got, act, r):
        assert torch.isnan(got[9]).all()
        want, tol = _result(codes, scale, wc, ws, b.double(), act, 0.2, None if r is None else r[finite].double())
        dt = got.dtype
        tol = tol * 1.2 + want.abs() * torch.finfo(dt).eps / 2 + (2.0 ** -25 if dt == torch.float16 else 1e-37)
        assert ((got[finite].double() - want).abs() <= tol).all()
    xa = Fn.Act(x.view(1, 1, m, k))
    got = Fn.linear_int8(xa, pk).t
    check(got.view(m, n), 0, None)
    assert torch.equal(Fn.linear_int8(Fn.quantize_tokens(xa), pk).t.nan_to_num(), got.nan_to_num())
    act = (0, 2, 3)[(m + n) % 3]   # not a ReLU, which ends a NaN
    y = Fn.linear_int8(xa, pk, act=act, slope=0.2, r1=Fn.Act(r1.view(1, 1, m, n))).t
    check(y.view(m, n), act, r1)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_int8_rows_views(dtype):
    """The launch that takes whole rows, on channel windows (also out = r1): the bits of the quantised map's product,
    what lies beside and behind the windows left as it was, and a token's bits the same as alone."""
    import lic_amd.functional as Fn
    g = torch.Generator(device=DEV).manual_seed(4)
    m, c, n = 16401, 192, 96
    x = torch.randn(1, 1, m, c + 32, generator=g, device=DEV).to(dtype)
    r = torch.randn(1, 1, m, n + 24, generator=g, device=DEV).to(dtype)
    for bias in (None, torch.randn(n, generator=g, device=DEV)):
        pk = Fn.pack_linear_int8(torch.randn(n, c, generator=g, device=DEV), bias)
        xa, ra = Fn.Act(x, 16, c), Fn.Act(r, 8, n)
        want = Fn.linear_int8(Fn.quantize_tokens(xa), pk, r1=ra, act=2, slope=0.1).t
        buf = torch.full((1, 2, m, n + 16), 9.0, dtype=dtype, device=DEV)
        Fn.linear_int8(xa, pk, Fn.Act(buf[:, :1], 8, n), r1=ra, act=2, slope=0.1)
        assert torch.equal(buf[:, :1, :, 8:8 + n], want)
        buf[:, :1, :, 8:8 + n] = 9.0
        assert (buf == 9.0).all()
        own = r.clone()
        view = Fn.Act(own, 8, n)
        Fn.linear_int8(xa, pk, view, r1=view, act=2, slope=0.1)
        assert torch.equal(own[..., 8:8 + n], want)
        own[..., 8:8 + n] = r[..., 8:8 + n]
        assert torch.equal(own, r)
        for a, b in ((0, 1), (100, 103), (300, 340), (16000, 16401)):
            part = Fn.linear_int8(Fn.Act(x[:, :, a:b, 16:16 + c].contiguous()), pk, act=2, slope=0.1,
                                  r1=Fn.Act(r[:, :, a:b, 8:8 + n].contiguous())).t
            assert torch.equal(part, want[:, :, a:b])


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_int8_few_tokens_any_alignment(dtype):
    """One to six tokens, aligned or not, up to and beyond the channels that one launch quantises: the same bits as
    quantised beforehand."""
    import lic_amd.functional as Fn
    g = torch.Generator(device=DEV).manual_seed(5)
    for k in (1, 100, 512, 4095, 4096, 4100, 9000):
        pk = Fn.pack_linear_int8(torch.randn(40, k, generator=g, device=DEV), torch.randn(40, generator=g, device=DEV))
        x = torch.randn(1, 1, 6, k + 9, generator=g, device=DEV).to(dtype)
        for m in (1, 2, 3, 4, 5, 6):
            for c0 in (0, 1, 8):
                xa = Fn.Act(x[:, :, :m], c0, k)
                codes, _ = _codes(xa.t[0, 0, :, c0:c0 + k])
                q = Fn.quantize_tokens(xa)
                assert torch.equal(q.codes.view(m, -1)[:, :k].double(), codes)
                assert torch.equal(Fn.linear_int8(xa, pk).t, Fn.linear_int8(q, pk).t), (k, m, c0)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_int8_one_launch(dtype):
    """Few tiles of few channels, quantised inside the product: every row length around the vectors' and the steps', at odd
    addresses, with a NaN row: the bits of the product of the codes made apart, which are exact."""
    import lic_amd.functional as Fn
    g = torch.Generator(device=DEV).manual_seed(6)
    for k in (1, 2, 3, 4, 5, 7, 8, 9, 15, 63, 64, 65, 127, 190, 192, 250, 257, 320, 333, 383, 384, 385):
        for m, n in ((5, 33), (64, 64), (70, 200), (333, 65)):
            x = torch.randn(1, 1, m, k + 3, generator=g, device=DEV).to(dtype)
            x[0, 0, 1, 1:] = 0
            x[0, 0, 3, 1] = float("inf")
            pk = Fn.pack_linear_int8(torch.randn(n, k, generator=g, device=DEV), torch.randn(n, generator=g, device=DEV))
            r = Fn.Act(torch.randn(1, 1, m, n, generator=g, device=DEV).to(dtype))
            xa = Fn.Act(x, 1, k)
            q = Fn.quantize_tokens(xa)
            ok = torch.ones(m, dtype=torch.bool, device=DEV)
            ok[3] = False
            codes, _ = _codes(x[0, 0, :, 1:1 + k][ok])
            got = q.codes.view(m, -1)
            assert torch.equal(got[ok][:, :k].double(), codes) and (got[:, k:] == 0).all() and (got[3] == 0).all()
            y = Fn.linear_int8(xa, pk, act=2, r1=r).t
            assert torch.isnan(y[0, 0, 3]).all() and torch.isfinite(y[0, 0, ok]).all()
            assert torch.equal(y.nan_to_num(), Fn.linear_int8(q, pk, act=2, r1=r).t.nan_to_num()), (k, m, n)


def test_linear_int8_rows_do_not_depend_on_the_batch():
    """Integer sums: a token's result is the same bits alone and in any batch, in every form the sizes select."""
    import lic_amd.functional as Fn
    for k, n in ((192, 576), (1000, 257), (4096, 1024)):
        x = torch.randn(1, 1, 2500, k, device=DEV).to(torch.bfloat16)
        pk = Fn.pack_linear_int8(torch.randn(n, k, device=DEV), torch.randn(n, device=DEV))
        full = Fn.linear_int8(Fn.Act(x), pk).t
        for a, b in ((0, 1), (5, 8), (100, 116), (200, 233), (600, 728), (1000, 1700)):
            part = Fn.linear_int8(Fn.Act(x[:, :, a:b].contiguous()), pk).t
            assert torch.equal(part, full[:, :, a:b]), (k, n, a, b)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_int8_views(dtype):
    """Channel windows with odd offsets and strides for x, out and r1 (also out = r1): the same bits as packed, the
    rest of out untouched, rows behind the last token left as they were."""
    import lic_amd.functional as Fn
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 5, 9, 131, generator=g).to(dtype).to(DEV)
    r = torch.randn(2, 5, 9, 77, generator=g).to(dtype).to(DEV)
    for c0, c, n, o0 in ((3, 100, 70, 2), (0, 64, 64, 0), (2, 128, 65, 1)):
        pk = Fn.pack_linear_int8(torch.randn(n, c, generator=g).to(DEV))
        rr = Fn.Act(r, 77 - n, n)
        want = Fn.linear_int8(Fn.Act(x[..., c0:c0 + c].contiguous()), pk,
                              r1=Fn.Act(r[..., 77 - n:].contiguous())).t
        buf = torch.full((3, 5, 9, n + 5), 9.0, dtype=dtype, device=DEV)
        Fn.linear_int8(Fn.Act(x, c0, c), pk, Fn.Act(buf[:2], o0, n), r1=rr)
        assert torch.equal(buf[:2, ..., o0:o0 + n], want)
        buf[:2, ..., o0:o0 + n] = 9.0
        assert (buf == 9.0).all()
        own = r.clone()
        view = Fn.Act(own, 77 - n, n)
        Fn.linear_int8(Fn.Act(x, c0, c), pk, view, r1=view)
        assert torch.equal(own[..., 77 - n:], want) and torch.equal(own[..., :77 - n], r[..., :77 - n])


def test_linear_int8_refusals():
    import lic_amd.functional as Fn
    x = Fn.Act(torch.zeros(1, 2, 2, 64, device=DEV))
    pk = Fn.pack_linear_int8(torch.randn(32, 32, device=DEV))
    with pytest.raises(ValueError, match="channels"):
        Fn.linear_int8(x, pk)
    with pytest.raises(ValueError, match="overlaps x"):
        Fn.linear_int8(x.ch(0, 32), pk, x.ch(16, 48))
    with pytest.raises(ValueError, match="overlaps r1"):
        Fn.linear_int8(Fn.Act(torch.zeros(1, 2, 2, 32, device=DEV)), pk, x.ch(0, 32), r1=x.ch(8, 40))
    with pytest.raises(ValueError, match="out must be"):
        Fn.linear_int8(x.ch(0, 32), pk, Fn.Act(torch.zeros(1, 2, 2, 33, device=DEV)))
    with pytest.raises(ValueError, match="act"):
        Fn.linear_int8(x.ch(0, 32), pk, act=4)
    assert Fn.linear_int8(Fn.Act(torch.zeros(0, 2, 2, 32, device=DEV)), pk).t.shape == (0, 2, 2, 32)


def test_linear_int8_streams_and_graph():
    """Two streams at once on one pack, and a captured call replayed with new inputs."""
    import lic_amd.functional as Fn
    pk = Fn.pack_linear_int8(torch.randn(300, 256, device=DEV), torch.randn(300, device=DEV))
    xs = [torch.randn(1, 1, m, 256, device=DEV) for m in (3, 700)]
    want = [Fn.linear_int8(Fn.Act(x), pk).t.clone() for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in xs], [None, None]
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            got[i] = Fn.linear_int8(Fn.Act(xs[i]), pk).t
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [Fn.linear_int8(Fn.Act(x), pk).t for x in xs]
    for k in range(3):
        for x in xs:
            x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        for x, o in zip(xs, outs):
            assert torch.equal(o, Fn.linear_int8(Fn.Act(x), pk).t)


def test_codes_of_more_workgroups_than_a_grid_dimension():
    """From 2^26 rows of more than 512 channels on (four a workgroup of 256 threads) a launch takes a second dimension:
    rows on both sides of its own, zeros everywhere else (69 GB of rows)."""
    import lic_amd.functional as Fn
    m, k = (1 << 26) + 5, 513
    at = torch.tensor([0, 3, 4, (1 << 24) - 1, 1 << 24, (1 << 26) - 1, 1 << 26, m - 2, m - 1], device=DEV)
    x = torch.zeros(1, 1, m, k, dtype=torch.bfloat16, device=DEV)
    rows = torch.randn(at.numel(), k, generator=torch.Generator().manual_seed(2)).bfloat16()
    x.view(m, k)[at] = rows.to(DEV)
    q = Fn.quantize_tokens(Fn.Act(x))
    codes, scale = q.codes.view(m, -1), q.scale.view(m)
    got, gots = codes[at].cpu(), scale[at].cpu()
    codes[at], scale[at] = 0, 0
    assert all(int(torch.count_nonzero(part)) == 0 for part in codes.split(1 << 21))
    assert int(torch.count_nonzero(scale)) == 0
    del x, q, codes, scale
    torch.cuda.empty_cache()
    want, wants = _codes(rows)
    assert torch.equal(got[:, :k].double(), want) and (got[:, k:] == 0).all()
    assert ((gots.double() - wants).abs() <= U * wants).all()
