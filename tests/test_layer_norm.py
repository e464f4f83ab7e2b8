"""Layer norm and its gradients against the formulas in 64 bits, and what is refused."""
import numpy as np
import pytest

import tlcuda
from rows_util import U, guarded, laid_out, refused, view

torch = pytest.importorskip("torch")

# Additions that one sum of a row goes through: at most 64 in a thread (rows up to 65536), 10
# across the block, and the products around them.
SUM = 80
# Across rows: a thread's rows, the block's warps, the blocks.
ROWS = 100


def reference(x, w, b, eps):
    """(y, mean, rstd, bound of y's error, bound of the mean's) in 64 bits."""
    x = x.astype(np.float64)
    w = np.ones(x.shape[-1]) if w is None else w.astype(np.float64)
    bb = np.zeros(x.shape[-1]) if b is None else b.astype(np.float64)
    mean = x.mean(-1, keepdims=True)
    var = ((x - mean) ** 2).mean(-1, keepdims=True)
    rstd = 1 / np.sqrt(var + eps)
    y = (x - mean) * rstd * w + bb
    d_mean = SUM * U * np.abs(x).mean(-1, keepdims=True)
    # the squares go by the rounded mean (its error's square comes in) and lose SUM + 4 roundings
    rel = 0.5 * ((SUM + 4) * U + d_mean ** 2 / (var + eps)) + 3 * U
    tol = rstd * np.abs(w) * (d_mean + np.abs(x - mean) * (rel + 4 * U)) + 2 * U * (np.abs(y) + np.abs(bb))
    return y, mean, rstd, tol, d_mean, rel


def reference_backward(g, x, stats, w):
    g, x, stats = (t.astype(np.float64) for t in (g, x, stats))
    w = np.ones(x.shape[-1]) if w is None else w.astype(np.float64)
    mean, rstd = stats[..., :1], stats[..., 1:]
    hat = (x - mean) * rstd
    gw = g * w
    c0, c1 = gw.mean(-1, keepdims=True), (gw * hat).mean(-1, keepdims=True)
    dx = rstd * (gw - c0 - hat * c1)
    rows = tuple(range(x.ndim - 1))
    dw, db = (g * hat).sum(rows), g.sum(rows)
    tol = (SUM + 10) * U * rstd * (np.abs(gw) + np.abs(gw).mean(-1, keepdims=True)
                                   + np.abs(hat) * np.abs(gw * hat).mean(-1, keepdims=True))
    return (dx, dw, db), (tol, (ROWS + 4) * U * np.abs(g * hat).sum(rows), ROWS * U * np.abs(g).sum(rows))


def data(shape, seed, offset=0.0):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal(shape) * (0.5 + rng.random(shape[-1])) + offset).astype(np.float32)
    w = (1 + 0.3 * rng.standard_normal(shape[-1])).astype(np.float32)
    b = rng.standard_normal(shape[-1]).astype(np.float32)
    g = rng.standard_normal(shape).astype(np.float32)
    return x, w, b, g


def dev(a):
    return torch.from_numpy(a).cuda()


def host(t):
    return t.detach().cpu().numpy()


# one element, one row, sizes on both sides of each kernel's limits, odd ones, long rows
SHAPES = [(1, 1), (3, 1), (5, 2), (1, 3), (2, 3, 31), (7, 32), (9, 33), (4, 128), (5, 129), (17, 257), (3, 512),
          (3, 513), (40, 768), (2, 1001), (6, 1024), (3, 1025), (5, 1028), (2, 2048), (3, 2052), (2, 4097),
          (3, 5001), (2, 8192), (2, 8196), (2, 8191), (3, 16384), (2, 16385), (2, 40000), (1500, 24), (700, 768),
          (2000, 8), (333, 2049), (64, 16400),
          # the ends of the backward's ranges of columns a thread, and of the forward's
          (5, 769), (4, 1536), (4, 1537), (3, 4096), (3, 6148), (2, 10001), (3, 12288), (2, 12289), (2, 16380), (2, 32768),
          (2, 32772), (1200, 130), (700, 260), (400, 515), (310, 1540)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("affine", [True, False])
def test_against_the_formulas(shape, affine):
    x, w, b, g = data(shape, 3 * len(shape) + shape[-1], offset=1.5)
    w, b = (w, b) if affine else (None, None)
    dx_, dw_, db_ = dev(x), dev(w) if affine else None, dev(b) if affine else None
    y, stats = tlcuda.layer_norm(dx_, dw_, db_, 1e-5)
    ref, mean, rstd, tol, d_mean, rel = reference(x, w, b, 1e-5)
    assert (np.abs(host(y) - ref) <= tol).all()
    st = host(stats).astype(np.float64)
    assert (np.abs(st[..., :1] - mean) <= d_mean + U * np.abs(mean)).all()
    assert (np.abs(st[..., 1:] / rstd - 1) <= rel).all()
    got = tlcuda.layer_norm_backward(dev(g), dx_, stats, dw_)
    refs, tols = reference_backward(g, x, host(stats), w)
    for a, r, t in zip(got, refs, tols):
        assert a.shape == r.shape and (np.abs(host(a) - r) <= t).all()


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["dense", "gap", "odd gap", "columns", "shift"])
@pytest.mark.parametrize("d", [12, 768, 1030, 2048])
def test_layouts(how, d):
    x, w, b, g = data((3, 5, d), d, offset=-0.5)
    vx, vg = laid_out(dev(x), how), laid_out(dev(g), how)
    y, stats = tlcuda.layer_norm(vx, dev(w), dev(b))
    ref, *_, tol, _, _ = reference(x, w, b, 1e-5)
    assert (np.abs(host(y) - ref) <= tol).all()
    wide = torch.zeros(3, 5, 4, device="cuda")
    wide[..., 1:3] = stats
    wv = laid_out(dev(np.stack([w, w])), "columns")[0]  # a weight of stride 2
    got = tlcuda.layer_norm_backward(vg, vx, wide[..., 1:3], wv)
    refs, tols = reference_backward(g, x, host(stats), w)
    for a, r, t in zip(got, refs, tols):
        assert (np.abs(host(a) - r) <= t).all()


@pytest.mark.gpu
def test_broadcast_gradient():
    """A gradient of stride 0, as a sum's backward gives it."""
    x, w, _, _ = data((37, 100), 5)
    _, stats = tlcuda.layer_norm(dev(x), dev(w))
    got = tlcuda.layer_norm_backward(torch.ones((), device="cuda").expand(37, 100), dev(x), stats, dev(w))
    refs, tols = reference_backward(np.ones((37, 100), np.float32), x, host(stats), w)
    for a, r, t in zip(got, refs, tols):
        assert (np.abs(host(a) - r) <= t).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d,off", [(768, 0), (768, 1), (769, 0), (2048, 3), (16388, 0), (17000, 2)])
def test_stays_inside_its_outputs(d, off):
    x, w, b, g = data((6, d), d)
    out, ok_out = guarded((6, d), off)
    stats, ok_st = guarded((6, 2), off)
    tlcuda.layer_norm(dev(x), dev(w), dev(b), out=out, stats=stats)
    ref, *_, tol, _, _ = reference(x, w, b, 1e-5)
    assert (np.abs(host(out) - ref) <= tol).all() and ok_out() and ok_st()
    dx, ok_dx = guarded((6, d), off)
    dw, ok_dw = guarded((d,), off)
    db, ok_db = guarded((d,), off)
    tlcuda.layer_norm_backward(dev(g), dev(x), stats, dev(w), dx=dx, dweight=dw, dbias=db)
    refs, tols = reference_backward(g, x, host(stats), w)
    for a, r, t in zip((dx, dw, db), refs, tols):
        assert (np.abs(host(a) - r) <= t).all()
    assert ok_dx() and ok_dw() and ok_db()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(50, 768), (9, 1030), (5, 4096), (3, 20000)], ids=str)
def test_accumulate_and_parts(shape):
    x, w, _, g = data(shape, 11)
    _, stats = tlcuda.layer_norm(dev(x), dev(w))
    whole = tlcuda.layer_norm_backward(dev(g), dev(x), stats, dev(w))
    old = [torch.randn_like(t) for t in whole]
    new = [t.clone() for t in old]
    tlcuda.layer_norm_backward(dev(g), dev(x), stats, dev(w), dx=new[0], dweight=new[1], dbias=new[2],
                               accumulate=True)
    for a, o, t in zip(new, old, whole):
        assert torch.equal(a, o + t)
    for i in range(3):  # each gradient alone: the same bits
        need = [j == i for j in range(3)]
        alone = tlcuda.layer_norm_backward(dev(g), dev(x), stats, dev(w), need=need)
        assert torch.equal(alone[i], whole[i]) and sum(a is None for a in alone) == 2


@pytest.mark.gpu
def test_against_differences():
    """The gradient of sum(g y) by central differences of the 64-bit formula."""
    x, w, b, g = data((4, 9), 21)
    _, stats = tlcuda.layer_norm(dev(x), dev(w), dev(b))
    dx, dw, db = (host(t) for t in tlcuda.layer_norm_backward(dev(g), dev(x), stats, dev(w)))

    def f(x, w, b):
        mean = x.mean(-1, keepdims=True)
        hat = (x - mean) / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + 1e-5)
        return ((hat * w + b) * g).sum()

    args = [t.astype(np.float64) for t in (x, w, b)]
    for k, grad in enumerate((dx, dw, db)):
        for i in np.ndindex(grad.shape):
            h = 1e-5
            up, down = [t.copy() for t in args], [t.copy() for t in args]
            up[k][i] += h
            down[k][i] -= h
            # the difference is off by h^2 / 6 times third derivatives of order 10, the gradient by some roundings
            assert abs((f(*up) - f(*down)) / (2 * h) - grad[i]) <= 1e-5 * max(1, abs(grad[i]))


@pytest.mark.gpu
def test_values_at_the_edges():
    # a constant row has variance 0: y = b; with eps = 0 the formula is 0 * inf = NaN
    x = torch.full((2, 100), 3.0, device="cuda")
    b = torch.randn(100, device="cuda")
    y, stats = tlcuda.layer_norm(x, None, b, 1e-5)
    assert torch.equal(y, b.expand(2, 100)) and torch.equal(stats[:, 0], x[:, 0])
    assert torch.isnan(tlcuda.layer_norm(x, None, b, 0.0)[0]).all()
    # NaN and infinity stay in their row
    x = torch.randn(5, 300, device="cuda")
    clean = tlcuda.layer_norm(x)[0]
    x[1, 7], x[3, 299] = float("nan"), float("inf")
    y = tlcuda.layer_norm(x)[0]
    assert torch.isnan(y[1]).all() and torch.isnan(y[3]).all()
    assert torch.equal(y[[0, 2, 4]], clean[[0, 2, 4]])
    # a large common offset: the differences are exact, nothing cancels
    base = torch.arange(64, device="cuda", dtype=torch.float32)
    y, _ = tlcuda.layer_norm(torch.stack([base, base + 2 ** 18]), eps=0.0)
    ref = (base.double() - 31.5) / (base.double() - 31.5).square().mean().sqrt()
    assert (y.double() - ref).abs().max() <= SUM * U * 2


@pytest.mark.gpu
@pytest.mark.parametrize("d", [7, 300, 1000, 5001, 8192, 40000])
def test_means_that_are_not_finite(d):
    """stats holds the mean that the row has: infinite with infinities of one sign, NaN with both or a NaN."""
    inf, nan = float("inf"), float("nan")
    x = torch.randn(5, d, device="cuda")
    x[0, d // 2], x[1, 0], x[2, d - 1], x[3, 1], x[3, 2] = inf, -inf, nan, inf, -inf
    y, stats = tlcuda.layer_norm(x)
    assert stats[0, 0] == inf and stats[1, 0] == -inf and torch.isnan(stats[2:4, 0]).all()
    assert torch.isnan(stats[:4, 1]).all() and torch.isnan(y[:4]).all()
    assert torch.isfinite(stats[4]).all() and torch.isfinite(y[4]).all()


@pytest.mark.gpu
def test_no_rows():
    w = torch.ones(16, device="cuda")
    y, stats = tlcuda.layer_norm(torch.empty(0, 16, device="cuda"), w, w)
    assert y.shape == (0, 16) and stats.shape == (0, 2)
    x = torch.empty(0, 16, device="cuda")
    dx, dw, db = tlcuda.layer_norm_backward(x, x, stats, w)
    assert dx.shape == (0, 16) and not dw.any() and not db.any()
    old = torch.ones(16, device="cuda")
    tlcuda.layer_norm_backward(x, x, stats, w, dx=dx, dweight=old, dbias=old.clone(), accumulate=True)
    assert torch.equal(old, w)


@pytest.mark.gpu
def test_rows_beyond_32_bits():
    """Rows whose offsets pass 2^31 elements."""
    step = 2 ** 31 + 8
    buf = torch.empty(2 * step + 800, device="cuda")
    x = buf.as_strided((3, 768), (step, 1))
    vals, w, b, g = data((3, 768), 8)
    x.copy_(dev(vals))
    y, stats = tlcuda.layer_norm(x, dev(w), dev(b))
    ref, *_, tol, _, _ = reference(vals, w, b, 1e-5)
    assert (np.abs(host(y) - ref) <= tol).all()
    got = tlcuda.layer_norm_backward(dev(g), x, stats, dev(w))
    refs, tols = reference_backward(g, vals, host(stats), w)
    for a, r, t in zip(got, refs, tols):
        assert (np.abs(host(a) - r) <= t).all()


@pytest.mark.gpu
def test_streams_and_graphs():
    x, w, b, g = (dev(t) for t in data((300, 1030), 9))
    y0, s0 = tlcuda.layer_norm(x, w, b)
    b0 = tlcuda.layer_norm_backward(g, x, s0, w)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in side:  # two calls at once
        for _ in range(3):
            got.append((tlcuda.layer_norm(x, w, b, stream=s), tlcuda.layer_norm_backward(g, x, s0, w, stream=s)))
    torch.cuda.synchronize()
    for (y, st), back in got:
        assert torch.equal(y, y0) and torch.equal(st, s0)
        assert all(torch.equal(p, q) for p, q in zip(back, b0))
    graphs, outs = [], []
    for _ in range(2):  # two graphs, replayed side by side
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            yy, ss = tlcuda.layer_norm(x, w, b)
            outs.append((yy, ss, *tlcuda.layer_norm_backward(g, x, ss, w)))
        graphs.append(gr)
    for _ in range(3):
        for s, gr in zip(side, graphs):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(p, q) for p, q in zip(o, (y0, s0, *b0)))


def around_the_mean(x, w, b, eps):
    """What `reference` gives, with the bounds of a mean that the differences to a first one correct.

    The first mean is off by at most SUM roundings of mean |x|, which is `first`; the sum of the
    differences to it loses SUM roundings of their mean, at most mean |x - mean| + first."""
    x = x.astype(np.float64)
    w, bb = w.astype(np.float64), b.astype(np.float64)
    mean = x.mean(-1, keepdims=True)
    var = ((x - mean) ** 2).mean(-1, keepdims=True)
    rstd = 1 / np.sqrt(var + eps)
    y = (x - mean) * rstd * w + bb
    first = SUM * U * np.abs(x).mean(-1, keepdims=True)
    d_mean = (SUM + 4) * U * (np.abs(x - mean).mean(-1, keepdims=True) + first)
    # the squares of the differences, whose mean is at most 2 (var + first^2), lose SUM + 6 roundings
    rel = 0.5 * (SUM + 6) * U * 2 * (var + first ** 2) / (var + eps) + 3 * U
    tol = rstd * np.abs(w) * (d_mean + (np.abs(x - mean) + first) * 4 * U + np.abs(x - mean) * rel) + 2 * U * (
        np.abs(y) + np.abs(bb))
    return y, mean, rstd, tol, U * np.abs(mean) + d_mean, rel


@pytest.mark.gpu
@pytest.mark.parametrize("d", [5, 100, 768, 1030, 5001, 8192, 12001, 40000])
@pytest.mark.parametrize("off", [0, 3], ids=["aligned", "off 16 bytes"])
def test_rows_far_from_zero(d, off):
    """Rows of one value, whose partial sums round, and rows whose mean is 1e3 to 1e5 times their spread."""
    rng = np.random.default_rng(d)
    spread = rng.standard_normal((4, d))
    rows = [np.full(d, v) for v in (0.1, 1000.1, -98765.43, 1e-3)]
    rows += [v + spread[i] * s for i, (v, s) in enumerate([(1e3, 1.0), (-1e4, 1.0), (1e5, 1.0), (98765.43, 0.01)])]
    x = np.stack(rows).astype(np.float32)
    w = (1 + 0.3 * rng.standard_normal(d)).astype(np.float32)
    b = rng.standard_normal(d).astype(np.float32)
    buf = torch.empty(x.size + off, device="cuda")
    vx = buf[off:].view(x.shape)
    vx.copy_(dev(x))
    y, stats = tlcuda.layer_norm(vx, dev(w), dev(b), 1e-5)
    ref, mean, rstd, tol, d_mean, rel = around_the_mean(x, w, b, 1e-5)
    assert (np.abs(host(y) - ref) <= tol).all()
    st = host(stats).astype(np.float64)
    assert (np.abs(st[..., :1] - mean) <= d_mean).all() and (np.abs(st[..., 1:] / rstd - 1) <= rel).all()


# Rows enough that each group of threads takes more than twice as many as the gradient's ring of rows
# has places, for every number of threads a row and of columns a thread; on 16 bytes and off them.
MANY = [(90000, 128), (90000, 101), (60000, 256), (60000, 130), (30000, 512), (30000, 260), (25000, 768), (25000, 515),
        (12000, 1024), (12000, 1022), (8000, 1536), (8000, 1535), (8000, 2048), (8000, 1999), (4000, 4096), (4000, 2051),
        (1500, 6144), (1500, 5001), (2400, 8192), (1500, 8191), (1000, 12288), (1000, 10001), (1000, 16384), (1000, 16383)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", MANY, ids=str)
def test_many_rows_a_group(shape):
    n, d = shape
    gen = torch.Generator(device="cuda")
    gen.manual_seed(n + d)
    x = torch.randn(n, d, generator=gen, device="cuda") + torch.randn(n, 1, generator=gen, device="cuda")
    g = torch.randn(n, d, generator=gen, device="cuda") * (0.5 + torch.rand(n, 1, generator=gen, device="cuda"))
    w = 1 + 0.3 * torch.randn(d, generator=gen, device="cuda")
    y, stats = tlcuda.layer_norm(x, w)
    dx, dw, db = tlcuda.layer_norm_backward(g, x, stats, w)
    dw64, db64, dw_abs, db_abs = (torch.zeros(d, dtype=torch.float64, device="cuda") for _ in range(4))
    for at in range(0, n, 1000):
        part = slice(at, at + 1000)
        xx, gg, st, ww = x[part].double(), g[part].double(), stats[part].double(), w.double()
        hat = (xx - st[:, :1]) * st[:, 1:]
        # the row's own statistics, and the forward with them: 4 roundings behind these
        mean = xx.mean(-1)
        assert ((st[:, 0] - mean).abs() <= SUM * U * xx.abs().mean(-1) + U * mean.abs()).all()
        assert ((y[part].double() - hat * ww).abs() <= 4 * U * ((hat * ww).abs() + st[:, 1:] * ww.abs() * SUM * (
            xx.abs().mean(-1, keepdim=True)))).all()
        gw = gg * ww
        ref = st[:, 1:] * (gw - gw.mean(-1, keepdim=True) - hat * (gw * hat).mean(-1, keepdim=True))
        tol = (SUM + 10) * U * st[:, 1:] * (gw.abs() + gw.abs().mean(-1, keepdim=True)
                                            + hat.abs() * (gw * hat).abs().mean(-1, keepdim=True))
        assert ((dx[part].double() - ref).abs() <= tol).all(), at
        dw64 += (gg * hat).sum(0)
        db64 += gg.sum(0)
        dw_abs += (gg * hat).abs().sum(0)
        db_abs += gg.abs().sum(0)
    # a group's rows (at most 30), a block's groups (64), a sixteenth of the blocks and the sixteen sums
    adds = 30 + 64 + 10 + 16
    assert ((dw.double() - dw64).abs() <= (adds + 4) * U * dw_abs).all()
    assert ((db.double() - db64).abs() <= adds * U * db_abs).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [16400, 20001])
def test_sums_of_many_long_rows(d):
    """dw and db over 100,000 rows of more than 16384 columns: x and grad are one row each, repeated, so
    that every rounding of a running sum goes the same way."""
    n = 100_000
    x, _, _, g = data((1, d), d)
    vx, vg = dev(x).expand(n, d), dev(g).expand(n, d)
    _, stats = tlcuda.layer_norm(dev(x))
    _, dw, db = tlcuda.layer_norm_backward(vg, vx, stats.expand(n, 2), need=(False, True, True))
    mean, rstd = (host(stats)[0].astype(np.float64))
    hat = (x[0].astype(np.float64) - mean) * rstd
    # 128 rows in a running sum, a sixteenth of these 782 sums in the next, 16 in the last; 4 roundings
    # in each product
    adds = 128 + 49 + 16
    for got, one, more in ((dw, g[0] * hat, 4), (db, g[0].astype(np.float64), 0)):
        assert (np.abs(host(got) - n * one) <= (adds + more) * U * n * np.abs(one)).all()


F = "tlc_layer_norm"
B = "tlc_layer_norm_backward"
A, Z = 1 << 20, 1 << 30  # addresses far apart


def test_refusals():
    x, y, st, w = view((4, 8)), view((4, 8), data=Z), view((4, 2), data=2 * Z), view((8,), data=3 * Z)
    cases = [
        ((None, w, w, 1e-5, y, st), "x is NULL"),
        ((x, w, w, 1e-5, None, st), "out is NULL"),
        ((view(()), w, w, 1e-5, y, st), "ndim must be 1..8"),
        ((x, view((9,)), w, 1e-5, y, st), "weight: wrong shape"),
        ((x, w, view((1, 8)), 1e-5, y, st), "bias: wrong shape"),
        ((x, w, w, -1.0, y, st), "eps"),
        ((x, w, w, float("nan"), y, st), "eps"),
        ((x, w, w, float("inf"), y, st), "eps"),
        ((x, w, w, 1e-5, view((4, 9), data=Z), st), "out: wrong shape"),
        ((x, w, w, 1e-5, view((4, 8), (16, 1), Z), st), "out must be contiguous"),
        ((x, w, w, 1e-5, y, view((4, 1), data=2 * Z)), "stats: wrong shape"),
        ((x, w, w, 1e-5, view((4, 8)), st), "out overlaps x"),
        ((x, w, w, 1e-5, view((4, 8), data=A + 124), st), "out overlaps x"),
        ((x, w, w, 1e-5, y, view((4, 2), data=Z + 4)), "stats overlaps out"),
        ((x, w, w, 1e-5, view((4, 8), data=3 * Z - 16), st), "out overlaps weight"),
        ((view((4, 8), data=0), w, w, 1e-5, y, st), "x: NULL data"),
        ((view((4, 8), data=A + 2), w, w, 1e-5, y, st), "x: misaligned"),
        ((view((4, 8), (-8, 1)), w, w, 1e-5, y, st), "negative stride"),
        ((view((4, -8), (8, 1)), w, w, 1e-5, y, st), "negative size"),
        ((view((1 << 40, 1 << 40), (1, 1)), w, w, 1e-5, y, st), "too large"),
    ]
    for args, msg in cases:
        text, status = refused(F, *args)
        assert status == 1 and msg in text, (msg, text)
    d = 1 << 30
    assert refused(F, view((1, d)), None, None, 1e-5, view((1, d), data=1 << 40), None)[1] == 2


def test_refusals_backward():
    x, g, st, w = view((4, 8)), view((4, 8), data=Z), view((4, 2), data=2 * Z), view((8,), data=3 * Z)
    dx, dw, db = view((4, 8), data=4 * Z), view((8,), data=5 * Z), view((8,), data=6 * Z)
    cases = [
        ((None, x, st, w, dx, dw, db, 0), "grad is NULL"),
        ((g, None, st, w, dx, dw, db, 0), "x is NULL"),
        ((g, x, None, w, dx, dw, db, 0), "stats is NULL"),
        ((view((4, 9)), x, st, w, dx, dw, db, 0), "grad: wrong shape"),
        ((g, x, view((8,)), w, dx, dw, db, 0), "stats: wrong shape"),
        ((g, x, st, w, dx, view((4, 8), data=5 * Z), db, 0), "dweight: wrong shape"),
        ((g, x, st, w, dx, dw, view((8,), (2,), 6 * Z), 0), "dbias must be contiguous"),
        ((g, x, st, w, view((4, 8), data=Z), dw, db, 0), "dx overlaps grad"),
        ((g, x, st, w, dx, dw, view((8,), data=5 * Z + 28), 0), "dbias overlaps dweight"),
        ((g, x, st, w, dx, view((8,), data=3 * Z), db, 0), "dweight overlaps weight"),
    ]
    for args, msg in cases:
        text, status = refused(B, *args)
        assert status == 1 and msg in text, (msg, text)


def test_binding_refusals():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError):
        tlcuda.layer_norm(torch.zeros(()))
    with pytest.raises(ValueError, match="float32"):
        tlcuda.layer_norm(x.double())
    with pytest.raises(ValueError, match="current CUDA device"):
        tlcuda.layer_norm(x)
    with pytest.raises(ValueError, match="accumulate needs"):
        tlcuda.layer_norm_backward(x, x, x, accumulate=True)
