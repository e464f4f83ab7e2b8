"""Log-probabilities of given tokens, entropy, alternatives and the gradient to the logits,
against the formulas in 64 bits, and what is refused."""
import numpy as np
import pytest

import tlcuda
from rows_util import U, guarded, index, laid_out, refused, view

torch = pytest.importorskip("torch")

NINF = -np.inf


def reference(x, t, scale):
    """The results in 64 bits and the bounds of their errors.

    A probability's exponent loses 4 roundings relative to itself (the difference, the constant,
    the two products), again as much when the running maximum moves, the power 4; the sum goes
    through an addition for each of a thread's values (at most V / 256 + 32) and a rescaling of at
    most 5 more for each, and the trees."""
    x = x.astype(np.float64)
    V = x.shape[-1]
    m = x.max(-1, keepdims=True)
    none = ~np.isfinite(m[..., 0])
    with np.errstate(invalid="ignore"):
        z = np.where(none[..., None], NINF, (x - m) * float(np.float32(scale)))
    e = np.exp(z)
    total = np.where(none, 1.0, e.sum(-1))
    log_l = np.log(total)
    p = e / total[..., None]
    zz = np.where(e > 0, z, 0.0)
    E, E2 = (p * -zz).sum(-1), (p * zz * zz).sum(-1)
    H = np.where(none, 0.0, log_l + E)
    n = V // 256 + 32
    rel = U * (6 * n + 100 + 8 * E)
    tol_l = rel + 2 * U * np.abs(log_l)
    tol_H = rel * (1 + E) * 2 + 8 * U * E2 + 4 * U * (np.abs(log_l) + E)
    lp = z - log_l[..., None]
    with np.errstate(invalid="ignore"):
        tol_lp = tol_l[..., None] + 2 * U * np.abs(zz) + U * np.abs(np.where(np.isfinite(lp), lp, 0))
    return dict(m=m[..., 0], log_l=log_l, H=H, lp=lp, p=p, none=none, tol_l=tol_l, tol_H=tol_H, tol_lp=tol_lp)


def picked(ref, t):
    """(log p of the tokens, the bound of its error): 0 for -1, NaN outside."""
    V = ref["lp"].shape[-1]
    ok = (t >= 0) & (t < V)
    at = np.where(ok, t, 0)[..., None]
    lp = np.take_along_axis(ref["lp"], at, -1)[..., 0]
    tol = np.take_along_axis(ref["tol_lp"], at, -1)[..., 0]
    return np.where(ok, lp, np.where(t == -1, 0.0, np.nan)), tol


def near(got, ref, tol):
    got = got.astype(np.float64)
    # a value beyond the largest float32 by more than half a step rounds to infinity: 1.5 (low - 1)
    # is -5.1e38, the type ends at 3.4e38
    ref = np.where(np.abs(ref) >= 2.0 ** 128, np.copysign(np.inf, ref), ref)
    same = (got == ref) | (np.isnan(got) & np.isnan(ref))
    with np.errstate(invalid="ignore"):
        return bool((same | (np.abs(got - ref) <= tol)).all())


def gradient(x, t, stats, H, g, h, scale):
    """The gradient from the forward's own statistics, and its bound: the exponent loses 3
    roundings, e^x two of its last places, the products one each."""
    x, stats, H, g, h = (a.astype(np.float64) for a in (x, stats, H, g, h))
    s = float(np.float32(scale))
    m, log_l = stats[..., :1], stats[..., 1:]
    none = np.isneginf(m)
    with np.errstate(invalid="ignore"):
        z = np.where(none, NINF, (x - m) * s)
    lp = z - log_l
    p = np.exp(lp)
    V = x.shape[-1]
    g = np.where(t == -1, 0.0, np.where((t < -1) | (t >= V), np.nan, g))[..., None]
    h, H = h[..., None], H[..., None]
    fin = np.where(p > 0, lp, 0.0)
    one = np.arange(V) == t[..., None]
    d = s * (g * one - p * (g + h * (fin + H)))
    d = np.where(none, 0.0, d)
    d_lp = U * (3 * np.abs(np.where(p > 0, z, 0)) + np.abs(log_l) + np.abs(fin))
    part = np.abs(g) + np.abs(h) * (np.abs(fin) + np.abs(H))
    tol = s * (p * (part * (d_lp + 8 * U) + np.abs(h) * d_lp) + 4 * U * np.abs(g) * one) + 1e-44
    return d, tol


def best(x, top):
    """Indices of the largest logits: NaN first, equal ones by the lower index."""
    key = np.where(np.isnan(x), np.inf, x.astype(np.float64))
    order = np.argsort(-key, axis=-1, kind="stable")
    nan_first = np.argsort(~np.isnan(np.take_along_axis(x, order, -1)), axis=-1, kind="stable")
    return np.take_along_axis(order, nan_first, -1)[..., :top]


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host(t):
    return t.detach().cpu().numpy()


def check(x, t, scale=1.0, top=0, vx=None, vt=None, entropy_grad=True, seed=0):
    """All results and gradients of logits x (numpy; `vx`, `vt`: views of the same values)."""
    vx = dev(x) if vx is None else vx
    vt = torch.as_tensor(np.array(t)).cuda() if vt is None else vt
    ref = reference(x, t, scale)
    logp, H, stats, top_lp, top_tok = tlcuda.token_logprobs(vx, vt, scale=scale, top=top)
    want, tol = picked(ref, t)
    assert near(host(logp), want, tol)
    assert near(host(H), ref["H"], ref["tol_H"])
    st = host(stats)
    assert np.array_equal(st[..., 0], x.max(-1)) and near(st[..., 1], ref["log_l"], ref["tol_l"])
    if top:
        idx = best(x, top)
        assert np.array_equal(host(top_tok), idx) and top_tok.dtype == vt.dtype
        assert near(host(top_lp), np.take_along_axis(ref["lp"], idx, -1), np.take_along_axis(ref["tol_lp"], idx, -1))
    rng = np.random.default_rng(seed)
    g, h = (rng.standard_normal(t.shape).astype(np.float32) for _ in range(2))
    h = h if entropy_grad else 0 * h
    got = tlcuda.token_logprobs_backward(vx, vt, stats, dev(g).view(t.shape),
                                         dev(h).view(t.shape) if entropy_grad else None, H, scale=scale)
    d, tol = gradient(x, t, st, host(H), g, h, scale)
    assert near(host(got), d, tol)
    return logp, H, stats, top_lp, top_tok, got


def logits(shape, seed, spread=3.0):
    return (np.random.default_rng(seed).standard_normal(shape) * spread).astype(np.float32)


# rows for a warp (to 1024), for a block, for clusters of blocks (few rows, long)
SHAPES = [((1,), 1), ((), 5), ((3,), 2), ((2, 3), 31), ((5,), 32), ((9,), 33), ((4,), 128), ((7,), 129), ((3,), 512),
          ((3,), 513), ((17,), 1000), ((3,), 1024), ((4,), 1025), ((2,), 1026), ((300,), 1030), ((2, 3), 2047),
          ((1,), 4096), ((1,), 5001), ((2,), 8193), ((40,), 9999), ((160,), 4103), ((1,), 32000), ((3,), 50001),
          ((1,), 131072), ((1,), 262147), ((5,), 100003)]


@pytest.mark.gpu
@pytest.mark.parametrize("lead,V", SHAPES, ids=str)
@pytest.mark.parametrize("scale,top", [(1.0, 0), (0.7, 1), (1.3, 5), (1.0, 20), (1.0, 32)])
def test_against_the_formulas(lead, V, scale, top):
    x = logits((*lead, V), V)
    t = np.random.default_rng(V).integers(-1, V, lead)
    check(x, t.astype(np.int32 if top == 5 else np.int64), scale, min(top, V))


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["dense", "gap", "odd gap", "columns", "shift"])
@pytest.mark.parametrize("V", [40, 1000, 1028, 5003, 40000])
def test_layouts(how, V):
    x = logits((3, 4, V), V)
    t = np.random.default_rng(V).integers(0, V, (3, 4))
    tokens = torch.zeros(3, 5, dtype=torch.int64, device="cuda")
    tokens[:, 1:] = dev(t)
    check(x, t, 0.9, 7, laid_out(dev(x), how), tokens[:, 1:])


@pytest.mark.gpu
@pytest.mark.parametrize("V", [64, 700, 3000, 50001, 200000])
def test_masked_rows(V):
    """Rows with -inf or the lowest number in most places, in all, or in all but one."""
    low = np.finfo(np.float32).min
    x = logits((9, V), V)
    rng = np.random.default_rng(V)
    x[0, rng.random(V) < 0.9] = NINF
    x[1] = NINF
    x[2] = NINF
    x[2, V - 1] = 4.0
    x[3, rng.random(V) < 0.9] = low
    x[4] = low
    x[5] = low
    x[5, 0] = 1.0
    x[6, :] = 0.25
    x[7, : V // 2] = NINF
    x[7, V // 2:] = low
    t = np.array([int(np.argmax(x[0])), 3, V - 1, 5, 6, 1, 7, V - 1, -1])
    logp, H, stats, top_lp, top_tok, got = check(x, t, 1.5, 20)
    assert host(logp)[1] == NINF and host(H)[1] == 0 and not host(got)[1].any()
    assert np.isneginf(host(top_lp)[1]).all() and host(H)[2] == 0 and host(logp)[2] == 0
    # a masked token that is asked for
    t2 = np.array([int(np.argmin(x[0])), -1, 0, 1, 2, V - 1, 0, 0, 0])
    check(x, t2, 1.0, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [33, 1000, 2500, 30000])
@pytest.mark.parametrize("pattern", ["equal", "two values", "ascending", "descending", "halves", "signed zeros"])
def test_ties_and_orders(V, pattern):
    i = np.arange(V)
    x = {"equal": np.zeros(V), "two values": (i % 3 == 0) * 1.0, "ascending": i * (8.0 / V), "descending": -i * (8.0 / V),
         "halves": (i >= V // 2) * 2.0, "signed zeros": np.where(i % 2 == 0, -0.0, 0.0)}[pattern].astype(np.float32)
    rows = np.stack([x, np.roll(x, 1), x[::-1]])
    for top in (1, 31, 32):
        check(rows, np.array([0, V - 1, V // 2]), 1.0, top)


# More rows than the grid has warps (8000 x 200, 4000 x 3001) or blocks (1000 x 20001), so that one takes
# several in turn; rows of several batches for a warp (1300 x 2001 to 16384).
MANY = [(1300, 2001, 0), (1300, 2001, 5), (1300, 2001, 32), (1300, 16384, 20), (1300, 16383, 5), (4000, 3001, 0),
        (4000, 3001, 20), (4000, 3001, 32), (8000, 200, 0), (8000, 200, 5), (8000, 200, 20), (8000, 201, 32), (1000, 20001, 0),
        (1000, 20001, 5), (1000, 20004, 20), (1000, 20001, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,V,top", MANY)
def test_many_rows_in_turn(rows, V, top):
    """Rows of all kinds, one after another: what one row leaves behind must not reach the next."""
    x = logits((rows, V), rows + V)
    rng = np.random.default_rng(V)
    kind = rng.integers(0, 12, rows)
    x[kind == 0] = 0.5  # all equal
    x[kind == 1] = NINF
    x[np.ix_(kind == 2, rng.random(V) < 0.9)] = NINF
    few = np.flatnonzero(kind == 3)  # fewer logits than alternatives
    x[few, :] = NINF
    for k in range(3):
        x[few, rng.integers(0, V, len(few))] = rng.standard_normal(len(few))
    x[kind == 4] += 100.0
    x[kind == 5] -= 100.0
    x[kind == 6] = np.sort(x[kind == 6], -1)
    t = rng.integers(-1, V, rows)
    clean = [None if a is None else host(a) for a in check(x, t, 1.0, top)]
    # the same with NaN in every 17th row: the others' bits stay
    x[::17, V // 2] = np.nan
    out = [None if a is None else host(a) for a in tlcuda.token_logprobs(dev(x), dev(t), top=top)]
    other = np.arange(rows) % 17 != 0
    for a, c in zip(out, clean):
        assert a is None or np.array_equal(a[other], c[other])
    assert np.isnan(out[1][~other]).all() and np.isnan(out[0][~other & (t >= 0)]).all()
    if top:
        assert np.array_equal(out[4][~other], best(x[~other], top))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [100, 5000, 70001])
def test_nan_and_infinity_stay_in_their_rows(V):
    x = logits((6, V), V)
    clean = [host(a) for a in tlcuda.token_logprobs(dev(x), dev(np.arange(6)), top=4)]
    x[1, V // 3] = np.nan
    x[3, V - 2] = np.inf
    x[4, 5] = -np.nan
    out = [host(a) for a in tlcuda.token_logprobs(dev(x), dev(np.arange(6)), top=4)]
    for a, c in zip(out, clean):
        assert np.array_equal(a[[0, 2, 5]], c[[0, 2, 5]])
    for row in (1, 3, 4):
        assert np.isnan(out[0][row]) and np.isnan(out[1][row]) and np.isnan(out[3][row]).all()
    assert out[4][1, 0] == V // 3 and out[4][3, 0] == V - 2 and out[4][4, 0] == 5
    assert np.array_equal(out[4][[1, 3, 4]], best(x, 4)[[1, 3, 4]])
    one = torch.ones(6, device="cuda")
    d = host(tlcuda.token_logprobs_backward(dev(x), dev(np.arange(6)), dev(out[2]), one, one, dev(out[1])))
    assert np.isnan(d[[1, 3, 4]]).all() and np.isfinite(d[[0, 2, 5]]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [50, 3001])
def test_strange_tokens(V):
    x = logits((8, V), V)
    t = np.array([-1, 0, V - 1, V, -2, 2 ** 40, -2 ** 63, 2 ** 32])
    _, H, stats, _, _, got = check(x, t)
    assert np.isnan(host(got)[3:]).all() and np.isfinite(host(got)[:3]).all()
    # without a gradient of the log-probabilities the token does not matter
    h = torch.ones(8, device="cuda")
    a = tlcuda.token_logprobs_backward(dev(x), dev(t), stats, None, h, H)
    assert torch.isfinite(a).all()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [300, 1030, 20001])
def test_outputs_and_gradients_left_out(V):
    x, t = dev(logits((5, V), 1)), torch.arange(5, device="cuda")
    logp, H, stats, tl, tt = tlcuda.token_logprobs(x, t, top=3)
    alone = tlcuda.token_logprobs(x, top=3, need_entropy=False, need_stats=False)
    assert alone[:3] == (None, None, None) and torch.equal(alone[3], tl) and torch.equal(alone[4], tt)
    only = tlcuda.token_logprobs(x, t, need_entropy=False, need_stats=False)
    assert torch.equal(only[0], logp) and only[1:] == (None, None, None, None)
    check(host(x), host(t), entropy_grad=False)
    assert not tlcuda.token_logprobs_backward(x, t, stats).any()
    # broadcast gradients, and statistics inside a wider tensor
    g = torch.full((), 0.5, device="cuda").expand(5)
    wide = torch.zeros(5, 3, device="cuda")
    wide[:, 1:] = stats
    a = tlcuda.token_logprobs_backward(x, t, wide[:, 1:], g, g, H)
    assert torch.equal(a, tlcuda.token_logprobs_backward(x, t, stats, g.contiguous(), g.contiguous(), H))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [77, 1028, 9001])
def test_in_place_and_inside_its_outputs(V):
    x, t = dev(logits((7, V), 2)), torch.arange(7, device="cuda")
    _, H, stats, _, _ = tlcuda.token_logprobs(x, t)
    g = torch.randn(7, device="cuda")
    want = tlcuda.token_logprobs_backward(x, t, stats, g, g, H)
    for off in (0, 1, 3):
        out, ok = guarded((7, V), off)
        tlcuda.token_logprobs_backward(x, t, stats, g, g, H, out=out)
        assert torch.equal(out, want) and ok()
        buf, ok = guarded((7, V), off)  # in the logits' own memory
        buf.copy_(x)
        assert tlcuda.token_logprobs_backward(buf, t, stats, g, g, H, out=buf) is buf
        assert torch.equal(buf, want) and ok()


@pytest.mark.gpu
def test_large_and_small_logits():
    """Differences count: a common offset of 2^16 changes nothing, and a scale of 1e-3 is exact too."""
    x = np.round(logits((4, 3000), 3) * 16) / 16
    t = np.array([0, 5, 7, 2999])
    a = check(x, t, 1.0, 10)
    b = check(x + np.float32(2 ** 16), t, 1.0, 10)
    for i in (0, 1, 3, 4, 5):
        assert torch.equal(a[i], b[i])
    check(logits((3, 2000), 4, spread=1000.0), np.array([1, 2, 3]), 1e-3, 5)
    check(logits((3, 2000), 4, spread=1e30), np.array([1, 2, 3]), 100.0, 5)


@pytest.mark.gpu
def test_against_differences():
    x, t = logits((3, 11), 6), np.array([4, 0, 10])
    rng = np.random.default_rng(0)
    g, h = (rng.standard_normal(3).astype(np.float32) for _ in range(2))
    _, H, stats, _, _ = tlcuda.token_logprobs(dev(x), dev(t), scale=0.8)
    got = host(tlcuda.token_logprobs_backward(dev(x), dev(t), stats, dev(g), dev(h), H, scale=0.8))

    def f(x):
        z = x * float(np.float32(0.8))
        lp = z - np.log(np.exp(z).sum(-1, keepdims=True))
        return (g * lp[np.arange(3), t] - h * (np.exp(lp) * lp).sum(-1)).sum()

    for i in np.ndindex(x.shape):
        up, down = x.astype(np.float64), x.astype(np.float64)
        up[i] += 1e-5
        down[i] -= 1e-5
        # the difference is off by 1e-10 / 6 times third derivatives of order 10, the gradient by some roundings
        assert abs((f(up) - f(down)) / 2e-5 - got[i]) <= 1e-5 * max(1, abs(got[i]))


@pytest.mark.gpu
def test_rows_beyond_32_bits():
    step = 2 ** 31 + 12
    buf = torch.empty(2 * step + 6000, device="cuda")
    x = logits((3, 5001), 7)
    vx = buf.as_strided((3, 5001), (step, 1))
    vx.copy_(dev(x))
    check(x, np.array([5000, 1, 77]), 1.0, 4, vx)
    del buf, vx
    n, V = 66000, 33000  # more than 2^31 logits in all
    row = dev(logits((V,), 8))
    big = row.repeat(n, 1)
    t = torch.arange(n, device="cuda") % V
    logp, H, stats, tl, tt = tlcuda.token_logprobs(big, t, top=2)
    want = tlcuda.token_logprobs(row.expand(2, V), t[-2:], top=2)
    for a, b in zip((logp, H, stats, tl, tt), want):
        assert torch.equal(a[-2:], b) and (a.dim() == 1 or torch.equal(a[0], b[1]))
    g = torch.ones(n, device="cuda")
    out = tlcuda.token_logprobs_backward(big, t, stats, g, out=big)
    want = tlcuda.token_logprobs_backward(row.expand(2, V), t[-2:], stats[-2:], g[:2])
    assert torch.equal(out[-2:], want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,V", [(1, 131072), (40, 30001), (2000, 3000), (500, 200)])
def test_same_bits_streams_and_graphs(rows, V):
    x, t = dev(logits((rows, V), 9)), torch.arange(rows, device="cuda") % V
    g = torch.randn(rows, device="cuda")

    def run(s=None):
        f = tlcuda.token_logprobs(x, t, top=8, stream=s)
        return (*f, tlcuda.token_logprobs_backward(x, t, f[2], g, g, f[1], stream=s))

    want = run()
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = [run(s) for _ in range(3) for s in side]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in got for a, b in zip(o, want))
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(run())
        graphs.append(gr)
    for _ in range(3):
        for s, gr in zip(side, graphs):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))


@pytest.mark.gpu
def test_no_rows():
    x, t = torch.empty(0, 7, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    logp, H, stats, tl, tt = tlcuda.token_logprobs(x, t, top=3)
    assert logp.shape == (0,) and stats.shape == (0, 2) and tt.shape == (0, 3) and tt.dtype == torch.int32
    assert tlcuda.token_logprobs_backward(x, t, stats, logp).shape == (0, 7)


A, Z = 1 << 20, 1 << 30


def test_refusals():
    x, t, lp, H, st = view((4, 50)), index((4,), data=Z), view((4,), data=2 * Z), view((4,), data=3 * Z), view(
        (4, 2), data=4 * Z)
    tl, tt = view((4, 3), data=5 * Z), index((4, 3), data=6 * Z)
    cases = [
        ((None, t, 1.0, lp, H, st, 0, None, None), "logits is NULL"),
        ((view(()), t, 1.0, lp, H, st, 0, None, None), "ndim must be 1..8"),
        ((x, None, 1.0, lp, H, st, 0, None, None), "tokens is NULL"),
        ((x, index((5,), data=Z), 1.0, lp, H, st, 0, None, None), "tokens: wrong shape"),
        ((x, index((4,), data=Z, bits=8), 1.0, lp, H, st, 0, None, None), "bits must be 32 or 64"),
        ((x, t, 0.0, lp, H, st, 0, None, None), "scale"), ((x, t, -1.0, lp, H, st, 0, None, None), "scale"),
        ((x, t, float("nan"), lp, H, st, 0, None, None), "scale"),
        ((x, t, float("inf"), lp, H, st, 0, None, None), "scale"),
        ((x, t, 1.0, lp, H, st, -1, None, None), "top must be"), ((x, t, 1.0, lp, H, st, 51, tl, tt), "top must be"),
        ((x, t, 1.0, lp, H, st, 3, None, tt), "top_logprobs is NULL"),
        ((x, t, 1.0, lp, H, st, 3, tl, None), "top_tokens is NULL"),
        ((x, t, 1.0, lp, H, st, 4, tl, tt), "top_logprobs: wrong shape"),
        ((x, t, 1.0, lp, H, st, 3, tl, index((4, 2), data=6 * Z)), "top_tokens: wrong shape"),
        ((x, t, 1.0, lp, H, st, 3, tl, index((4, 3), (4, 1), 6 * Z)), "top_tokens must be contiguous"),
        ((x, t, 1.0, view((4, 1), data=2 * Z), H, st, 0, None, None), "logprobs: wrong shape"),
        ((x, t, 1.0, lp, view((4,), (2,), 3 * Z), st, 0, None, None), "entropy must be contiguous"),
        ((x, t, 1.0, lp, H, view((4,), data=4 * Z), 0, None, None), "stats: wrong shape"),
        ((x, t, 1.0, view((4,), data=A + 8), H, st, 0, None, None), "logprobs overlaps logits"),
        ((x, t, 1.0, lp, view((4,), data=2 * Z), st, 0, None, None), "entropy overlaps logprobs"),
        ((x, t, 1.0, lp, H, view((4, 2), data=Z), 0, None, None), "stats overlaps tokens"),
        ((view((4, 0)), t, 1.0, lp, H, st, 0, None, None), "rows without logits"),
    ]
    for args, msg in cases:
        text, status = refused("tlc_token_logprobs", *args)
        assert status == 1 and msg in text, (msg, text)
    tl, tt = view((4, 33), data=5 * Z), index((4, 33), data=6 * Z)
    assert refused("tlc_token_logprobs", x, t, 1.0, lp, H, st, 33, tl, tt)[1] == 2


@pytest.mark.parametrize("scale", [2.0 ** 100 * (1 + 2.0 ** -23), 1e31, 2.0 ** 127, 2.4e38, 3.4e38, 1e-46, -0.0])
def test_scales_out_of_range(scale):
    """Above 2^100 scale * log2 e, or scale times a gradient, would leave float32; 1e-46 is 0 in it."""
    x, t, lp, st, H = view((4, 50)), index((4,), data=Z), view((4,), data=2 * Z), view((4, 2), data=3 * Z), view((4,), data=4 * Z)
    text, status = refused("tlc_token_logprobs", x, t, scale, lp, H, st, 0, None, None)
    assert status == 1 and "scale" in text
    text, status = refused("tlc_token_logprobs_backward", x, t, st, H, lp, H, scale, view((4, 50), data=6 * Z))
    assert status == 1 and "scale" in text


@pytest.mark.gpu
@pytest.mark.parametrize("V", [40, 2000, 30001])
@pytest.mark.parametrize("scale", [2.0 ** 100, 1e20, 2.0 ** -100])
def test_scales_at_the_ends_of_the_range(V, scale):
    """A huge scale leaves the largest logit and its equals (differences are 1/2 at least), a tiny one all alike."""
    x = np.round(logits((5, V), V) * 2) / 2
    x[3, V // 2] = NINF
    check(x, np.array([int(np.argmax(x[0])), 0, V - 1, V // 2, -1]), scale, 5)


def test_refusals_backward():
    x, t, st, H = view((4, 50)), index((4,), data=Z), view((4, 2), data=2 * Z), view((4,), data=3 * Z)
    g, h, d = view((4,), data=4 * Z), view((4,), data=5 * Z), view((4, 50), data=6 * Z)
    cases = [
        ((None, t, st, H, g, h, 1.0, d), "logits is NULL"), ((x, None, st, H, g, h, 1.0, d), "tokens is NULL"),
        ((x, t, None, H, g, h, 1.0, d), "stats is NULL"), ((x, t, st, None, g, h, 1.0, d), "entropy is NULL"),
        ((x, t, st, H, g, h, 1.0, None), "dlogits is NULL"), ((x, t, st, H, view((5,)), h, 1.0, d), "grad_logprobs: wrong"),
        ((x, t, st, H, g, view((4, 1)), 1.0, d), "grad_entropy: wrong"), ((x, t, st, H, g, h, 0.0, d), "scale"),
        ((x, t, st, H, g, h, 1.0, view((4, 50), (60, 1), 6 * Z)), "dlogits must be contiguous"),
        ((x, t, st, H, g, h, 1.0, view((4, 50), data=A + 4)), "dlogits overlaps logits"),
        ((view((4, 50), (51, 1)), t, st, H, g, h, 1.0, view((4, 50))), "dlogits overlaps logits"),
        ((x, t, st, H, g, h, 1.0, view((4, 50), data=2 * Z)), "dlogits overlaps stats"),
    ]
    for args, msg in cases:
        text, status = refused("tlc_token_logprobs_backward", *args)
        assert status == 1 and msg in text, (msg, text)


def test_binding_refusals():
    x, t = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="current CUDA device"):
        tlcuda.token_logprobs(x, t)
    with pytest.raises(ValueError, match="at least 1-D"):
        tlcuda.token_logprobs(x.sum())
    with pytest.raises(ValueError, match="needs the forward's entropy"):
        tlcuda.token_logprobs_backward(x, t, x, grad_entropy=x)
