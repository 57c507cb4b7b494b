"""Token scores (scoring.token_logprobs) against log-softmax in 64 bits, and the refusals."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def reference(x, ids, k):
    """x [n, V] float64 (the values that the kernel reads), ids [n]: scores row by row."""
    lp_all = np.empty_like(x)
    for r, row in enumerate(x):
        m = row.max()
        if m == -math.inf:
            lp_all[r] = -math.inf
        else:
            lp_all[r] = row - m - math.log(np.exp(row - m).sum())
    p = np.exp(lp_all)
    ent = -np.where(p > 0, p * np.where(p > 0, lp_all, 0), 0).sum(-1)
    lp = lp_all[np.arange(len(x)), ids]
    rank = 1 + (x > x[np.arange(len(x)), ids][:, None]).sum(-1)
    order = np.argsort(-x, axis=-1, kind="stable")[:, :k]
    return lp, ent, rank, order, np.take_along_axis(lp_all, order, -1)


def check(dev, x, ids, k, dtype):
    """Bounds: every sum of at most 2^17 positive fp32 terms is taken in shares of at most 2^9
    terms and a tree, the exponent of a term carries an error of 2^-23 (|x| log2 e + 1), exp2 and
    log2 are good to 2^-21; so ln l is within 2^-22 (2^9 + ...) only in the worst case and, as
    roundings do not all point one way, 4e-6 (1 + |x|max / 16) is kept as the bound here; the
    difference x - m is exact to 2^-24 of its value."""
    from knlp_b200 import scoring
    xd = x.to(dtype).to(dev)
    r = scoring.token_logprobs(xd, ids.to(dev), top_k=k)
    xv = xd.double().cpu().numpy()
    lp, ent, rank, order, top = reference(xv, ids.numpy(), k)
    finite = np.abs(xv[np.isfinite(xv)])
    tol = 4e-6 * (1 + (finite.max() if finite.size else 0) / 16)

    def near(a, b, t):
        a = a.double().cpu().numpy()
        fin = np.isfinite(b)
        assert np.array_equal(np.isfinite(a), fin) and np.array_equal(a[~fin], b[~fin])
        assert np.all(np.abs(a - b)[fin] <= t + 2.0 ** -23 * np.abs(b[fin]))

    near(r.logprob, lp, tol)
    near(r.entropy, ent, tol * (1 + ent.max(initial=0)))
    assert np.array_equal(r.rank.cpu().numpy(), rank)
    assert r.top_ids.shape == r.top_logprobs.shape == (len(xv), k)
    if k:
        assert np.array_equal(r.top_ids.cpu().numpy(), order)
        near(r.top_logprobs, top, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (1, 7, 7), (3, 33, 5), (2, 64, 64), (5, 1000, 20),
                                          (1, 50257, 8), (4, 50257, 64), (37, 20011, 1),
                                          (300, 4099, 3), (2, 131072, 32), (700, 513, 0)])
def test_random_rows(dt, rows, vocab, k, cuda_device):
    g = torch.Generator().manual_seed(rows * 7 + vocab)
    x = torch.randn(rows, vocab, generator=g) * 3
    ids = torch.randint(0, vocab, (rows,), generator=g)
    check(cuda_device, x, ids, k, DT[dt])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["equal", "two values", "rising", "falling", "one share",
                                  "masked but 5", "masked", "all masked", "lowest", "large"])
def test_rows_that_are_hard_to_rank(kind, dt, cuda_device):
    """Ties, sorted rows, rows whose large values fall into the shares of few threads, masks."""
    n, V, k = 3, 30011, 40
    g = torch.Generator().manual_seed(3)
    x = torch.randn(n, V, generator=g)
    if kind == "equal":
        x = torch.full((n, V), 1.25)
    elif kind == "two values":
        x = torch.where(x > 2.5, 1.0, 0.0)
    elif kind == "rising":
        x = torch.arange(V).float()[None].expand(n, V) / 1000
    elif kind == "falling":
        x = -torch.arange(V).float()[None].expand(n, V) / 1000
    elif kind == "one share":  # every value of a few vector columns is large
        x = x * 0.1 + 40.0 * ((torch.arange(V) % 4096) < 100)
    elif kind == "masked but 5":
        keep = torch.zeros(n, V, dtype=torch.bool)
        keep[:, [3, 17, 9000, 9001, V - 1]] = True
        x = x.masked_fill(~keep, -math.inf)
    elif kind == "masked":
        x = x.masked_fill(torch.rand(n, V, generator=g) < 0.97, -math.inf)
    elif kind == "all masked":
        x = torch.full((n, V), -math.inf)
    elif kind == "lowest":  # masks of the type's lowest value
        x = x.masked_fill(torch.rand(n, V, generator=g) < 0.9, torch.finfo(DT[dt]).min)
    elif kind == "large":
        x = x * 1e30
    ids = torch.tensor([0, 17, V - 1])
    if kind in ("lowest", "large"):  # beyond the derived bound's range: the integers, and finite sums
        from knlp_b200 import scoring
        xd = x.to(DT[dt]).to(cuda_device)
        r = scoring.token_logprobs(xd, ids.to(cuda_device), top_k=k)
        lp, ent, rank, order, _ = reference(xd.double().cpu().numpy(), ids.numpy(), k)
        assert np.array_equal(r.rank.cpu().numpy(), rank)
        assert np.array_equal(r.top_ids.cpu().numpy(), order)
        assert np.allclose(r.logprob.cpu().numpy(), lp, rtol=1e-6, atol=1e-5)
        assert np.allclose(r.entropy.cpu().numpy(), ent, rtol=1e-5, atol=1e-5)
        return
    check(cuda_device, x, ids, k, DT[dt])


@pytest.mark.gpu
def test_nan_and_infinity(cuda_device):
    from knlp_b200 import scoring
    V = 9000
    x = torch.randn(4, V)
    x[0, 77] = math.nan
    x[1, 5000] = math.inf
    x[2, 8999], x[2, 4] = math.nan, math.inf
    x[3, :] = math.nan
    ids = torch.tensor([77, 3, 4, 9])
    r = scoring.token_logprobs(x.to(cuda_device), ids.to(cuda_device), top_k=3)
    assert torch.isnan(r.logprob).all() and torch.isnan(r.entropy).all()
    assert r.top_ids[0, 0] == 77 and r.top_ids[1, 0] == 5000
    assert r.top_ids[2, :2].tolist() == [8999, 4] and r.top_ids[3].tolist() == [0, 1, 2]
    # comparisons with a NaN are false
    want = [1, 1 + int((x[1] > x[1, 3]).sum()), 1, 1]
    assert r.rank.tolist() == want


@pytest.mark.gpu
def test_ids_outside_and_shapes(cuda_device):
    from knlp_b200 import scoring
    dev = cuda_device
    x = torch.randn(2, 3, 501, device=dev).to(torch.float16)
    ids = torch.tensor([[0, -100, 501], [500, 2, -1]], device=dev)
    r = scoring.token_logprobs(x, ids, top_k=2)
    assert r.logprob.shape == (2, 3) and r.top_ids.shape == (2, 3, 2)
    want = torch.log_softmax(x.double(), -1)
    for i, j in ((0, 0), (1, 0), (1, 1)):
        assert abs(float(r.logprob[i, j]) - float(want[i, j, ids[i, j]])) < 1e-5
    assert r.logprob[0, 1] == 0 and r.logprob[1, 2] == 0 and torch.isnan(r.logprob[0, 2])
    assert r.rank[0, 1] == 0 and r.rank[0, 2] == 0
    # rows of a wider buffer, a transposed view, a vocabulary cut off at odd places
    wide = torch.randn(6, 700, device=dev)
    for view in (wide[:, 1:502], wide[::2, 3:504], torch.randn(501, 3, device=dev).t(),
                 torch.randn(1, 501, device=dev).expand(4, 501)):
        t = torch.arange(view.shape[0], device=dev)
        a = scoring.token_logprobs(view, t, top_k=4)
        b = scoring.token_logprobs(view.clone().contiguous(), t, top_k=4)
        assert all(torch.equal(p, q) for p, q in zip(a[2:4], b[2:4]))
        assert torch.allclose(a.logprob, b.logprob, atol=4e-6) and torch.allclose(
            a.entropy, b.entropy, atol=1e-5)
    empty = scoring.token_logprobs(x[:0], ids[:0], top_k=2)
    assert empty.logprob.shape == (0, 3) and empty.top_ids.shape == (0, 3, 2)


@pytest.mark.gpu
def test_repeated_and_captured_calls_agree(cuda_device):
    from knlp_b200 import scoring
    dev = cuda_device
    x = torch.randn(5, 50257, device=dev).to(torch.bfloat16)
    ids = torch.randint(0, 50257, (5,), device=dev)
    first = scoring.token_logprobs(x, ids, top_k=8)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = scoring.token_logprobs(x, ids, top_k=8)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = scoring.token_logprobs(x, ids, top_k=8)
    g.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(first, again, captured):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_refusals_of_the_library():
    from knlp_b200 import _lib
    lib = _lib.load()
    buf = C.create_string_buffer(64)
    p = C.cast(buf, C.c_void_p).value

    def call(**kw):
        a = dict(x=p, dt=0, stride=10, ids=p, rows=1, vocab=10, k=2, lp=p, ent=p, rank=p, ti=p, tl=p)
        a.update(kw)
        return lib.knlp_b200_token_score(*a.values(), None)

    assert call(dt=3) == -3
    for bad in (dict(rows=-1), dict(vocab=0), dict(k=-1), dict(k=11)):
        assert call(**bad) == -2
    assert call(k=65, vocab=100) == -9
    assert call(rows=0, x=None, ids=None) == 0
    for missing in ("x", "ids", "lp", "ent", "rank", "ti", "tl"):
        assert call(**{missing: None}) == -1, missing
    assert call(x=p + 2) == -5 and call(x=p + 1, dt=2) == -5


@pytest.mark.gpu
def test_refusals_of_the_wrapper(cuda_device):
    from knlp_b200 import scoring
    x, ids = torch.zeros(2, 9, device=cuda_device), torch.zeros(2, dtype=torch.long, device=cuda_device)
    with pytest.raises(RuntimeError):
        scoring.token_logprobs(x.cpu(), ids)
    with pytest.raises(TypeError):
        scoring.token_logprobs(x.double(), ids)
    with pytest.raises(TypeError):
        scoring.token_logprobs(x, ids.int())
    for a in ((x, ids[:1]), (x[:, :0], ids)):
        with pytest.raises(ValueError):
            scoring.token_logprobs(*a)
    for k in (-1, 10):
        with pytest.raises(ValueError):
            scoring.token_logprobs(x, ids, top_k=k)
