"""Embedding lookup with scaling and its gradient: the lookup bit for bit, the gradient against
sums in 64 bits, and what is refused."""
import numpy as np
import pytest

import tlcuda
from rows_util import U, guarded, index, laid_out, refused, view

torch = pytest.importorskip("torch")


def lookup(w, t, scale):
    out = np.zeros((*t.shape, w.shape[1]), np.float32)
    ok = (t >= 0) & (t < w.shape[0])
    out[ok] = np.float32(scale) * w[t[ok]]  # one rounding
    out[~ok & (t != -1)] = np.nan
    return out


def gradient(g, t, rows, scale, old=None):
    """(dweight, the bound of its error) in 64 bits: a token that occurs c times goes through at
    most c additions, then the scale and the old value are one rounding each."""
    g = g.reshape(-1, g.shape[-1]).astype(np.float64)
    t = t.reshape(-1)
    ok = (t >= 0) & (t < rows)
    d, m = np.zeros((rows, g.shape[1])), np.zeros((rows, g.shape[1]))
    np.add.at(d, t[ok], g[ok])
    np.add.at(m, t[ok], np.abs(g[ok]))
    count = np.bincount(t[ok], minlength=rows)[:, None]
    tol = abs(scale) * m * U * (count + 2)
    d = d * float(np.float32(scale))
    if old is not None:
        tol = tol + 2 * U * (np.abs(old) + np.abs(d)) * (count > 0)
        d = d + old
    return d, tol


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host(t):
    return t.detach().cpu().numpy()


def same(a, b):
    return np.array_equal(a, b, equal_nan=True)


CASES = [  # tokens' shape, rows, D
    ((1,), 1, 1), ((1,), 7, 4), ((), 5, 8), ((3,), 2, 3), ((48, 1), 320, 768), ((2, 5), 100, 33), ((31,), 10, 129),
    ((32,), 10, 128), ((33,), 3, 130), ((2, 3, 4), 50, 512), ((64,), 1000, 516), ((1000,), 513, 65), ((8191,), 300, 5),
    ((8193,), 70000, 4), ((20000,), 40, 20), ((70000,), 3, 8), ((70001,), 300000, 4), ((5, 4000), 2 ** 18, 12),
    ((513,), 2 ** 18 + 3, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape,rows,d", CASES, ids=str)
@pytest.mark.parametrize("bits", [32, 64])
def test_against_the_sums(shape, rows, d, bits):
    rng = np.random.default_rng(rows + d)
    w = rng.standard_normal((rows, d)).astype(np.float32)
    t = np.exp(rng.random(shape) * np.log(rows + 1)) - 1  # falls off as 1 / rank
    t = np.minimum(t.astype(np.int64), rows - 1)
    t = np.where(rng.random(shape) < 0.1, -1, t).astype(np.int32 if bits == 32 else np.int64)
    tok = torch.as_tensor(t).cuda()
    scale = 1.7
    assert same(host(tlcuda.embedding(dev(w), tok, scale)), lookup(w, t, scale))
    g = rng.standard_normal((*shape, d)).astype(np.float32)
    got = tlcuda.embedding_backward(dev(g), tok, rows, scale)
    ref, tol = gradient(g, t, rows, scale)
    assert (np.abs(host(got) - ref) <= tol).all()
    old = rng.standard_normal((rows, d)).astype(np.float32)
    new = dev(old)
    assert tlcuda.embedding_backward(dev(g), tok, scale=scale, dweight=new, accumulate=True) is new
    ref, tol = gradient(g, t, rows, scale, old)
    assert (np.abs(host(new) - ref) <= tol).all()
    absent = np.setdiff1d(np.arange(rows), t[t >= 0])
    assert same(host(new)[absent], old[absent])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["one", "two", "runs", "all padding", "ascending", "descending"])
@pytest.mark.parametrize("n", [31, 32, 33, 4097, 100000])
def test_lopsided_tokens(kind, n):
    """Every position on one token, long runs that end inside and on chunk borders, no token at all."""
    rows, d = 5000, 36
    i = np.arange(n)
    t = {"one": np.full(n, 4321), "two": np.where(i % 2 == 0, 17, 4999), "runs": (i // 64) % rows,
         "all padding": np.full(n, -1), "ascending": i % rows, "descending": (n - 1 - i) % rows}[kind]
    g = np.random.default_rng(n).standard_normal((n, d)).astype(np.float32)
    got = host(tlcuda.embedding_backward(dev(g), dev(t), rows))
    ref, tol = gradient(g, t, rows, 1.0)
    assert (np.abs(got - ref) <= tol).all()


@pytest.mark.gpu
def test_padding_and_strange_tokens():
    rows, d = 10, 24
    w = torch.randn(rows, d, device="cuda")
    t = np.array([-1, 0, 9, 10, -2, 2 ** 31 - 1, -2 ** 31, 3], np.int64)
    far = np.concatenate([t, [2 ** 40 + 3, -2 ** 63, 2 ** 32]])  # 2^32 + 0 must not pass for token 0
    for tokens in (t.astype(np.int32), far):
        out = host(tlcuda.embedding(w, dev(tokens)))
        assert same(out, lookup(host(w), tokens, 1.0))
        g = np.random.default_rng(1).standard_normal((len(tokens), d)).astype(np.float32)
        g[(tokens < 0) | (tokens >= rows)] = np.nan  # takes no part
        got = host(tlcuda.embedding_backward(dev(g), dev(tokens), rows))
        ref, tol = gradient(g, tokens, rows, 1.0)
        assert (np.abs(got - ref) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["dense", "gap", "odd gap", "columns", "shift"])
@pytest.mark.parametrize("d", [16, 200, 33])
def test_layouts(how, d):
    rng = np.random.default_rng(d)
    w = rng.standard_normal((90, d)).astype(np.float32)
    g = rng.standard_normal((6, 11, d)).astype(np.float32)
    t = rng.integers(-1, 90, (6, 12))
    tok = dev(t)[:, 1:]  # a strided view
    wv = laid_out(dev(w), how) if how != "shift" else dev(w)
    assert same(host(tlcuda.embedding(wv, tok, 0.5)), lookup(w, t[:, 1:], 0.5))
    assert same(host(tlcuda.embedding(wv, tok.t(), 0.5)), lookup(w, t[:, 1:].T, 0.5))
    ref, tol = gradient(g, t[:, 1:], 90, 2.0)
    got = host(tlcuda.embedding_backward(laid_out(dev(g), how), tok, 90, 2.0))
    assert (np.abs(got - ref) <= tol).all()
    one = torch.ones((), device="cuda").expand(6, 11, d)  # as a sum's backward gives it
    ref, tol = gradient(np.ones((6, 11, d), np.float32), t[:, 1:], 90, 1.0)
    assert (np.abs(host(tlcuda.embedding_backward(one, tok, 90)) - ref) <= tol).all()
    same_tok = torch.full((), 5, device="cuda").expand(6, 11)
    ref, tol = gradient(g, np.full((6, 11), 5), 90, 1.0)
    assert (np.abs(host(tlcuda.embedding_backward(dev(g), same_tok, 90)) - ref) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d,off", [(8, 0), (8, 1), (131, 0), (1024, 2), (1030, 0)])
def test_stays_inside_its_outputs(d, off):
    rng = np.random.default_rng(d)
    w, g = rng.standard_normal((70, d)).astype(np.float32), rng.standard_normal((45, d)).astype(np.float32)
    t = rng.integers(-1, 70, 45)
    out, ok = guarded((45, d), off)
    tlcuda.embedding(dev(w), dev(t), out=out)
    assert same(host(out), lookup(w, t, 1.0)) and ok()
    dw, ok = guarded((70, d), off)
    tlcuda.embedding_backward(dev(g), dev(t), dweight=dw)
    ref, tol = gradient(g, t, 70, 1.0)
    assert (np.abs(host(dw) - ref) <= tol).all() and ok()


@pytest.mark.gpu
def test_beyond_32_bits():
    step = 2 ** 31 + 4
    buf = torch.empty(2 * step + 64, device="cuda")
    w = buf.as_strided((3, 64), (step, 1))  # rows whose offsets pass 2^31 elements
    w.copy_(torch.randn(3, 64))
    t = torch.tensor([2, 0, 1, 2, -1], device="cuda")
    assert same(host(tlcuda.embedding(w, t)), lookup(host(w.contiguous()), host(t), 1.0))
    got = tlcuda.embedding_backward(w, torch.tensor([4, 0, 4], device="cuda"), 5)
    ref, tol = gradient(host(w.contiguous()), np.array([4, 0, 4]), 5, 1.0)
    assert (np.abs(host(got) - ref) <= tol).all()
    del buf, w
    # an output of more than 2^31 elements
    n, d = 530000, 4100
    table = torch.randn(11, d, device="cuda")
    t = torch.arange(n, device="cuda") % 11
    out = tlcuda.embedding(table, t)
    for at in (0, 1, 523776, 523777, n - 1):
        assert torch.equal(out[at], table[at % 11])
    got = tlcuda.embedding_backward(out, t, 11)  # and as a gradient
    count = torch.bincount(t, minlength=11).unsqueeze(1)
    assert ((got.double() - table.double() * count).abs() <= table.double().abs() * count * U * (n // 11 + 2)).all()


@pytest.mark.gpu
def test_a_table_of_many_rows():
    """More rows than the marks of all blocks hold at once (65536 a block), and three digits a token."""
    rows, d = 9_700_000, 3
    t = torch.tensor([0, rows - 1, 4_000_000, rows - 1, 7_340_031, 7_340_032, -1, 8_000_001, rows], device="cuda")
    g = torch.arange(1, 28, device="cuda", dtype=torch.float32).view(9, 3)
    got = tlcuda.embedding_backward(g, t, dweight=torch.full((rows, d), 5.0, device="cuda"))
    want = torch.zeros(rows, d, device="cuda")
    for i, v in enumerate(t.tolist()):
        if 0 <= v < rows:
            want[v] += g[i]  # whole numbers: exact
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_same_bits_streams_and_graphs():
    rng = np.random.default_rng(4)
    t = dev(np.minimum(np.exp(rng.random(9000) * np.log(2000)).astype(np.int64), 1999))
    w, g = torch.randn(2000, 260, device="cuda"), torch.randn(9000, 260, device="cuda")
    out, dw = tlcuda.embedding(w, t, 3.0), tlcuda.embedding_backward(g, t, 2000, 3.0)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = [(tlcuda.embedding(w, t, 3.0, stream=s), tlcuda.embedding_backward(g, t, 2000, 3.0, stream=s))
           for _ in range(4) for s in side]
    torch.cuda.synchronize()
    assert all(torch.equal(a, out) and torch.equal(b, dw) for a, b in got)
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append((tlcuda.embedding(w, t, 3.0), tlcuda.embedding_backward(g, t, 2000, 3.0)))
        graphs.append(gr)
    for _ in range(3):
        for s, gr in zip(side, graphs):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, out) and torch.equal(b, dw) for a, b in outs)
    # new tokens in the same memory: a replay goes by what is there then
    t.copy_((t * 7 + 3) % 2000)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], tlcuda.embedding(w, t, 3.0))
    assert torch.equal(outs[0][1], tlcuda.embedding_backward(g, t, 2000, 3.0))


@pytest.mark.gpu
def test_nothing_to_do():
    w = torch.randn(5, 8, device="cuda")
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert tlcuda.embedding(w, none).shape == (0, 8)
    assert not tlcuda.embedding_backward(torch.empty(0, 8, device="cuda"), none, 5).any()
    new = w.clone()
    tlcuda.embedding_backward(torch.empty(0, 8, device="cuda"), none, dweight=new, accumulate=True)
    assert torch.equal(new, w)
    t = torch.tensor([0, -1], device="cuda")
    assert torch.isnan(tlcuda.embedding(torch.empty(0, 8, device="cuda"), t)[0]).all()  # a table without rows
    assert tlcuda.embedding(torch.empty(5, 0, device="cuda"), t).shape == (2, 0)
    assert tlcuda.embedding_backward(torch.empty(2, 0, device="cuda"), t, 5).shape == (5, 0)


A, Z = 1 << 20, 1 << 30


def test_refusals():
    w, t, y = view((10, 8)), index((3, 2), data=Z), view((3, 2, 8), data=2 * Z)
    cases = [
        ((None, t, 1.0, y), "weight is NULL"), ((w, None, 1.0, y), "tokens is NULL"), ((w, t, 1.0, None), "out is NULL"),
        ((view((2, 5, 8)), t, 1.0, y), "weight must be 2-D"), ((view((8,)), t, 1.0, y), "weight must be 2-D"),
        ((w, index((3, 2), data=Z, bits=16), 1.0, y), "bits must be 32 or 64"),
        ((w, index((3, 2), data=Z + 4), 1.0, y), "tokens: misaligned"),
        ((w, index((3, 2), data=0), 1.0, y), "tokens: NULL data"),
        ((w, t, float("nan"), y), "scale"), ((w, t, float("inf"), y), "scale"),
        ((w, t, 1.0, view((3, 2, 9), data=2 * Z)), "out: wrong shape"),
        ((w, t, 1.0, view((6, 8), data=2 * Z)), "out: wrong shape"),
        ((w, t, 1.0, view((3, 2, 8), (32, 16, 1), 2 * Z)), "out must be contiguous"),
        ((w, t, 1.0, view((3, 2, 8), data=A + 316)), "out overlaps weight"),
        ((w, t, 1.0, view((3, 2, 8), data=Z + 40)), "out overlaps tokens"),
        ((w, index((1,) * 8, data=Z), 1.0, y), "too many dims"),
        ((w, index((3, 2), (-2, 1), Z), 1.0, y), "negative stride"),
    ]
    for args, msg in cases:
        text, status = refused("tlc_embedding", *args)
        assert status == 1 and msg in text, (msg, text)
    assert refused("tlc_embedding", view((2 ** 31, 1)), t, 1.0, view((3, 2, 1), data=1 << 40))[1] == 2


def test_refusals_backward():
    g, t, d = view((3, 2, 8)), index((3, 2), data=Z), view((10, 8), data=2 * Z)
    cases = [
        ((None, t, 1.0, d, 0), "grad is NULL"), ((g, None, 1.0, d, 0), "tokens is NULL"),
        ((g, t, 1.0, None, 0), "dweight is NULL"), ((g, t, 1.0, view((10, 9), data=2 * Z), 0), "grad: wrong shape"),
        ((g, t, 1.0, view((10, 8), (16, 1), 2 * Z), 0), "dweight must be contiguous"),
        ((g, t, float("nan"), d, 0), "scale"), ((g, t, 1.0, view((10, 8)), 0), "dweight overlaps grad"),
        ((g, t, 1.0, view((10, 8), data=Z - 16), 0), "dweight overlaps tokens"),
    ]
    for args, msg in cases:
        text, status = refused("tlc_embedding_backward", *args)
        assert status == 1 and msg in text, (msg, text)
    n = 2 ** 31 - 100
    assert refused("tlc_embedding_backward", view((n, 8), (0, 1)), index((n,), (0,), Z), 1.0, d, 0)[1] == 2


def test_binding_refusals():
    w = torch.zeros(4, 8)
    t = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="current CUDA device"):
        tlcuda.embedding(w, t)
    with pytest.raises(ValueError, match="2-D"):
        tlcuda.embedding(w[0], t)
    with pytest.raises(ValueError, match="accumulate needs"):
        tlcuda.embedding_backward(w, t, 4, accumulate=True)
    with pytest.raises(ValueError, match="rows"):
        tlcuda.embedding_backward(w, t)
    with pytest.raises(ValueError, match="another number of rows"):
        tlcuda.embedding_backward(w, t, 5, dweight=w)
    with pytest.raises(ValueError, match="int32 or int64"):
        tlcuda.embedding(w, w)
