"""One training step of a small language model through the binding: embedding, layer norm,
flash attention, Linear and token log-probabilities, forward and backward, against autograd in 64
bits; alone, captured into a graph and replayed on other tokens, and beside an eager step."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import tlcuda  # noqa: E402

B, S, D, H, V = 3, 33, 64, 2, 203
EMB, TEMP = 8.0, 0.9
# Each gradient comes through at most 8 products of up to 203 terms, whose roundings (2^-24 each, of
# random sign) add up to 8 sqrt(203) 2^-24, times what the norms and the softmax magnify them by (10).
TOL = 8 * math.sqrt(203) * 2.0 ** -24 * 10


def make():
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)

    def normal(*shape, size=1.0):
        return torch.randn(shape, generator=gen, device="cuda") * size

    p = {"emb": normal(V, D, size=0.3), "w1": 1 + normal(D, size=0.2), "b1": normal(D, size=0.2),
         "wq": normal(D, D, size=0.2), "wk": normal(D, D, size=0.2), "wv": normal(D, D, size=0.2), "bv": normal(D),
         "w2": 1 + normal(D, size=0.2), "b2": normal(D, size=0.2), "wo": normal(D, V, size=0.3)}
    tokens = torch.randint(0, V, (B, S + 1), generator=gen, device="cuda")
    tokens[1, 20:] = -1  # a shorter sequence
    return p, tokens


def heads(x):
    return x.view(B, S, H, D // H).transpose(1, 2).contiguous()


def unheads(x):
    return x.transpose(1, 2).contiguous().view(B, S, D)


def step(p, tokens):
    """Loss terms and gradients, as a user's program calls the operators."""
    tl, sm = tlcuda, 1.0 / math.sqrt(D // H)
    now, nxt = tokens[:, :-1], tokens[:, 1:]
    h = tl.embedding(p["emb"], now, scale=EMB)
    a, st1 = tl.layer_norm(h, p["w1"], p["b1"])
    q, k = heads(tl.matmul(a, p["wq"])), heads(tl.matmul(a, p["wk"]))
    v = heads(tl.matmul_fused(a, p["wv"], bias=p["bv"]))
    o, lse = tl.flash_attention(q, k, v, sm)
    r = tl.add_tensors(h, unheads(o))
    y, st2 = tl.layer_norm(r, p["w2"], p["b2"])
    logits = tl.matmul(y, p["wo"])
    logp, ent, stats, best, which = tl.token_logprobs(logits, nxt, scale=TEMP, top=3)
    g_lp = torch.full((), -1.0, device="cuda").expand(B, S)
    g_ent = torch.full((), -0.1, device="cuda").expand(B, S)
    d_logits = tl.token_logprobs_backward(logits, nxt, stats, g_lp, g_ent, ent, scale=TEMP)
    g = {}
    dy, g["wo"] = tl.matmul_backward(d_logits, y, p["wo"])
    dr, g["w2"], g["b2"] = tl.layer_norm_backward(dy, r, st2, p["w2"])
    dq, dk, dv = tl.flash_attention_backward(heads(dr), q, k, v, o, lse, sm)
    da, g["wq"] = tl.matmul_backward(unheads(dq), a, p["wq"])
    da, g["wk"] = tl.matmul_backward(unheads(dk), a, p["wk"], da=da, db=torch.zeros_like(p["wk"]), accumulate=True)
    da, g["wv"] = tl.matmul_backward(unheads(dv), a, p["wv"], da=da, db=torch.zeros_like(p["wv"]), accumulate=True)
    g["bv"] = tl.sum_to(unheads(dv), (D,))
    # the residual branch's gradient is in dr already: the norm's is added to it
    dh, g["w1"], g["b1"] = tl.layer_norm_backward(da, h, st1, p["w1"], dx=dr, dweight=torch.zeros_like(p["w1"]),
                                                  dbias=torch.zeros_like(p["b1"]), accumulate=True)
    g["emb"] = tl.embedding_backward(dh, now, V, scale=EMB)
    return (logp, ent, best, which), g


def reference(p, tokens):
    q = {k: v.double().requires_grad_() for k, v in p.items()}
    now, nxt = tokens[:, :-1], tokens[:, 1:]
    h = torch.where((now >= 0).unsqueeze(-1), q["emb"][now.clamp(min=0)] * EMB, 0.0)

    def norm(x, w, b):
        m = x.mean(-1, keepdim=True)
        return (x - m) / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + 1e-5) * w + b

    a = norm(h, q["w1"], q["b1"])

    def split(x):
        return x.view(B, S, H, D // H).transpose(1, 2)

    s = split(a @ q["wq"]) @ split(a @ q["wk"]).transpose(-1, -2) / math.sqrt(D // H)
    o = torch.softmax(s, -1) @ split(a @ q["wv"] + q["bv"])
    r = h + o.transpose(1, 2).reshape(B, S, D)
    logits = norm(r, q["w2"], q["b2"]) @ q["wo"]
    every = torch.log_softmax(logits * float(torch.tensor(TEMP)), -1)
    logp = torch.where(nxt >= 0, every.gather(-1, nxt.clamp(min=0).unsqueeze(-1))[..., 0], 0.0)
    ent = -(every.exp() * every).sum(-1)
    (-logp.sum() - 0.1 * ent.sum()).backward()
    best = every.topk(3, -1)
    return (logp, ent, best.values, best.indices), {k: v.grad for k, v in q.items()}


def check(got, want):
    for i, (a, b) in enumerate(zip(got[0], (w.detach() for w in want[0]))):
        if i == 3:
            assert torch.equal(a, b)
        else:
            assert float((a.double() - b).norm() / b.norm()) <= TOL, i
    for k, b in want[1].items():
        assert float((got[1][k].double() - b).norm() / b.norm()) <= TOL, k


def test_training_step():
    p, tokens = make()
    check(step(p, tokens), reference(p, tokens))


def test_training_step_in_a_graph():
    p, tokens = make()
    eager = step(p, tokens)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(p, tokens)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip((*out[0], *out[1].values()), (*eager[0], *eager[1].values())):
        assert torch.equal(a, b)
    # other tokens in the same memory, replayed while an eager step runs on another stream
    other = torch.roll(tokens, 1, 0).flip(1).contiguous()
    other[0, :3] = -1
    tokens.copy_(other)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph.replay()
    again = step(p, other)
    torch.cuda.synchronize()
    check(out, reference(p, other))
    check(again, reference(p, other))


FIRST = """
import sys
sys.path.insert(0, {pkg!r})
import torch, tlcuda
x, w = torch.randn(40, 5001, device="cuda"), torch.randn(5001, device="cuda")
t = torch.arange(40, device="cuda") % 7
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y, st = tlcuda.layer_norm(x, w, w)
    back = tlcuda.layer_norm_backward(y, x, st, w)
    e = tlcuda.embedding(x, t, 2.0)
    d = tlcuda.embedding_backward(e, t, 7)
    f = tlcuda.token_logprobs(x, t, top=5)
    b = tlcuda.token_logprobs_backward(x, t, f[2], f[0], f[1], f[1])
graph.replay()
torch.cuda.synchronize()
got = [y, st, *back, e, d, *f, b]
y, st = tlcuda.layer_norm(x, w, w)
f = tlcuda.token_logprobs(x, t, top=5)
want = [y, st, *tlcuda.layer_norm_backward(y, x, st, w), tlcuda.embedding(x, t, 2.0),
        tlcuda.embedding_backward(tlcuda.embedding(x, t, 2.0), t, 7), *f,
        tlcuda.token_logprobs_backward(x, t, f[2], f[0], f[1], f[1])]
assert all(torch.equal(a, c) for a, c in zip(got, want))
print("captured first")
"""


def test_first_calls_of_a_process_captured():
    """The set-up of a first call (kernel attributes, occupancy, the memory pool) inside a capture."""
    import os
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", FIRST.format(pkg=os.path.dirname(os.path.abspath(tlcuda.__file__)))],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stdout + r.stderr


def test_two_host_threads():
    """Calls from two threads, each on its own stream, give each thread's own results."""
    import threading
    p, tokens = make()
    inputs = [tokens, torch.roll(tokens, 2, 1).contiguous()]
    want = [step(p, t) for t in inputs]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(5):
                got[i] = step(p, inputs[i])
        s.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        for x, y in zip((*a[0], *a[1].values()), (*b[0], *b[1].values())):
            assert torch.equal(x, y)


def test_views_that_repeat_memory():
    """Inputs of stride 0 (one row for all, one value for all) and the same token everywhere."""
    row = torch.randn(300, device="cuda")
    w = torch.randn(300, device="cuda")
    x = row.expand(20, 300)
    y, st = tlcuda.layer_norm(x, w)
    assert torch.equal(y, tlcuda.layer_norm(x.contiguous(), w)[0])
    one = torch.ones((), device="cuda").expand(300)
    assert torch.equal(tlcuda.layer_norm(x, one, one)[0], tlcuda.layer_norm(x, one.contiguous(), one.contiguous())[0])
    for a, b in zip(tlcuda.layer_norm_backward(x, x, st[:1].expand(20, 2), w),
                    tlcuda.layer_norm_backward(x.contiguous(), x.contiguous(), st, w)):
        assert torch.equal(a, b)
    t = torch.full((), 7, device="cuda").expand(20)
    assert torch.equal(tlcuda.embedding(x, t), x)
    for a, b in zip(tlcuda.token_logprobs(x, t, top=3), tlcuda.token_logprobs(x.contiguous(), t.contiguous(), top=3)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("top", [-1, -2 ** 31, 204, 2 ** 31, 2 ** 32, 2 ** 40])
def test_alternatives_out_of_range(top):
    """Refused before their outputs are made (2^32 wraps to 0 in an int, and would take 48 GB)."""
    x, t = torch.zeros(1, V, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    with pytest.raises(ValueError, match="top must be 0 to the vocabulary's size"):
        tlcuda.token_logprobs(x, t, top=top)
    with pytest.raises(tlcuda.TLCError, match="top is at most 32"):
        tlcuda.token_logprobs(x, t, top=33)
    # the three other outputs, twice
    assert torch.cuda.memory_stats()["allocation.all.allocated"] - before <= 6


def test_a_table_of_less_than_no_rows():
    g, t = torch.zeros(1, 8, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="rows must not be negative"):
        tlcuda.embedding_backward(g, t, -1)


def test_views_that_torch_negates_lazily():
    """The imaginary part of a conjugate holds the values' negatives and a mark that says so: what is
    behind its address is not what it means."""
    x = torch.randn(6, 40, dtype=torch.complex64, device="cuda").conj().imag
    assert x.is_neg() and x.dtype is torch.float32
    y, st = tlcuda.layer_norm(x.resolve_neg())
    t = torch.arange(6, device="cuda")
    for call in (lambda: tlcuda.layer_norm(x), lambda: tlcuda.layer_norm(y, None, x[0]),
                 lambda: tlcuda.layer_norm_backward(x, y, st), lambda: tlcuda.embedding(x, t),
                 lambda: tlcuda.embedding_backward(x, t, 6), lambda: tlcuda.token_logprobs(x, t),
                 lambda: tlcuda.token_logprobs_backward(y, t, st, x[:, 0])):
        with pytest.raises(ValueError, match="resolve_neg"):
            call()
