"""Tokens drawn from logits against a draw in 64 bits (ids have to be equal).

The kernel sums integers that are within half a unit of 2^-44 of the weights (plus the error
of its exponential, of the same order); the oracle sums doubles.  A draw or a top-p edge can
only differ where the target lies within about 2^-44 * vocab of a running sum; the oracle
measures that distance, and no input here comes near it (asserted, not skipped).
"""
import numpy as np
import pytest


def _draw(x, u, temp, k, p, mp):
    """One row in float64; returns (token, smallest relative distance of a decision)."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    best = x.max()
    if best == -np.inf:
        return 0, 1.0
    if not temp > 0:
        return int(np.argmax(x)), 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp((x - best) / np.float64(temp))
    w = np.where(x == best, 1.0, np.where((x == -np.inf) | (best == np.inf), 0.0, w))
    order = np.lexsort((np.arange(x.size), -x))
    margin = 1.0
    if 0 < k < x.size:
        order = order[:k]
    if p < 1:
        cum = np.cumsum(w[order])
        before = np.concatenate([[0.0], cum[:-1]])
        target = max(p, 0.0) * cum[-1]
        n = max(1, int((before < target).sum()))
        if p > 0:
            margin = min(margin, np.abs(before - target).min() / cum[-1])
        order = order[:n]
    if mp > 0:
        order = order[w[order] >= min(mp, 1.0)]
    ids = np.sort(order)
    cum = np.cumsum(w[ids])
    u = min(max(u, 0.0), 1.0 - 2.0 ** -24) if u == u else 0.0
    target = u * cum[-1]
    if u > 0:
        margin = min(margin, np.abs(cum - target).min() / cum[-1])
    return int(ids[np.nonzero(cum > target)[0][0]]), margin


def _run(pkg, logits, u, temp=None, k=None, p=None, mp=None, pos=None, stream=None):
    import torch

    dev = logits.device
    out = torch.full((logits.shape[0],), -7, dtype=torch.int32, device=dev)

    def put(v, dtype):
        return None if v is None else torch.as_tensor(v, dtype=dtype).to(dev)

    pkg.sample_tokens(logits, put(u, torch.float32), out, temperature=put(temp, torch.float32),
                      top_k=put(k, torch.int32), top_p=put(p, torch.float32),
                      min_p=put(mp, torch.float32), pos=put(pos, torch.int32),
                      stream=torch.cuda.current_stream().cuda_stream if stream is None else stream)
    torch.cuda.synchronize()
    return out.cpu().numpy()


def _check(pkg, logits, u, temp=None, k=None, p=None, mp=None, near=1e-11):
    got = _run(pkg, logits, u, temp, k, p, mp)
    x = logits.double().cpu().numpy()
    n = x.shape[0]
    f = lambda v, d: np.full(n, d) if v is None else np.asarray(v)  # noqa: E731
    f32 = lambda v, d: f(v, d).astype(np.float32).astype(np.float64)  # noqa: E731
    uu, tt, pp, mm, kk = f32(u, 0), f32(temp, 1.0), f32(p, 1.0), f32(mp, 0.0), f(k, 0)
    for r in range(n):
        want, margin = _draw(x[r], uu[r], tt[r], int(kk[r]), pp[r], mm[r])
        assert margin > near, f"row {r}: the oracle itself is within {margin:.2e} of a border"
        assert got[r] == want, f"row {r}: {got[r]}, expected {want} (margin {margin:.2e})"
    return got


VOCABS = [1, 2, 31, 32, 33, 777, 1024, 4097, 50257, 131071, 201088, 262144]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_every_filter(pkg, vocab, dtype):
    import torch

    dev = torch.device("cuda:0")
    rng = np.random.default_rng(vocab)
    n = 13
    x = rng.standard_normal((n, vocab)) * rng.choice([0.3, 2.0, 5.0], size=(n, 1))
    logits = torch.from_numpy(x).to(getattr(torch, dtype)).to(dev)
    u = rng.random(n, dtype=np.float32)
    temp = rng.uniform(0.3, 1.6, n)
    temp[5] = 0.0
    k = rng.integers(1, max(2, min(vocab, 3000)), n)
    k[6:8] = 0, vocab
    p = rng.uniform(0.05, 0.999, n)
    mp = rng.uniform(0.001, 0.3, n)
    _check(pkg, logits, u)
    _check(pkg, logits, u, temp)
    _check(pkg, logits, u, temp, k=k)
    _check(pkg, logits, u, temp, p=p)
    _check(pkg, logits, u, temp, mp=mp)
    _check(pkg, logits, u, temp, k, p, mp)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [40, 5000, 201088])
def test_ties(pkg, vocab):
    """Few distinct values: the edges of top-k and top-p fall among equal logits, where the
    lowest ids are kept."""
    import torch

    rng = np.random.default_rng(7)
    n = 12
    x = rng.integers(0, 4, (n, vocab)) * 0.5
    x[8:] = 1.25  # all equal
    x[10, ::3] = -0.0
    x[10, 1::3] = 0.0
    x[10, 2::3] = -5.0
    u = np.concatenate([rng.random(10), [0.0, 0.99999994]]).astype(np.float32)
    k = rng.integers(1, vocab, n)
    p = rng.uniform(0.1, 0.95, n)
    logits = torch.from_numpy(x).float().to("cuda:0")
    _check(pkg, logits, u, k=k)
    _check(pkg, logits, u, p=p)
    _check(pkg, logits, u, k=k, p=p, mp=np.full(n, 0.5))


@pytest.mark.gpu
def test_filter_limits(pkg):
    """Values that switch a filter off, that leave one token, or that are out of range."""
    import torch

    rng = np.random.default_rng(9)
    x = rng.standard_normal((11, 3001)) * 2
    logits = torch.from_numpy(x).float().to("cuda:0")
    u = rng.random(11, dtype=np.float32)
    best = x.astype(np.float32).argmax(1)
    full = _check(pkg, logits, u)
    assert (_run(pkg, logits, u, k=np.ones(11)) == best).all()
    assert (_run(pkg, logits, u, p=np.zeros(11)) == best).all()
    assert (_run(pkg, logits, u, p=np.full(11, -1.0)) == best).all()
    assert (_run(pkg, logits, u, mp=np.ones(11)) == best).all()
    assert (_run(pkg, logits, u, mp=np.full(11, 5.0)) == best).all()
    for off in (dict(k=np.full(11, -3)), dict(k=np.full(11, 1 << 30)), dict(p=np.ones(11)),
                dict(p=np.full(11, np.nan)), dict(mp=np.full(11, -1.0)), dict(mp=np.full(11, np.nan))):
        assert (_run(pkg, logits, u, **off) == full).all(), off
    for temp in (np.zeros(11), np.full(11, -1.0), np.full(11, np.nan)):
        assert (_run(pkg, logits, u, temp) == best).all()
    # u at and outside its range
    first = _run(pkg, logits, np.zeros(11))
    assert (_run(pkg, logits, np.full(11, np.nan)) == first).all()
    assert (_run(pkg, logits, np.full(11, -2.0)) == first).all()
    last = _check(pkg, logits, np.full(11, 1 - 2.0 ** -24, np.float32))
    assert (_run(pkg, logits, np.full(11, 1.0)) == last).all()
    assert (_run(pkg, logits, np.full(11, np.inf)) == last).all()
    # extreme temperatures
    _check(pkg, logits, u, np.full(11, 1e-6))
    assert (_run(pkg, logits, u, np.full(11, 1e-45)) == best).all()
    _check(pkg, logits, u, np.full(11, 1e30))
    _check(pkg, logits, u, np.full(11, 50.0), k=np.full(11, 2999), p=np.full(11, 0.9999))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [100, 201088])
def test_infinities_and_nan(pkg, vocab):
    import torch

    rng = np.random.default_rng(2)
    x = rng.standard_normal((9, vocab)).astype(np.float32) * 3
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 5:] = -np.inf            # most tokens masked
    x[3, ::2] = np.finfo(np.float32).min
    x[4, 7] = np.inf
    x[5, [3, 50, 99]] = np.inf
    x[6, 1::2] = np.nan
    x[7, :] = -np.inf
    x[7, 42] = -3e38              # one token left
    x[8, 10:] = np.finfo(np.float32).min
    logits = torch.from_numpy(x).to("cuda:0")
    u = rng.random(9, dtype=np.float32)
    for kw in (dict(), dict(k=np.full(9, 20)), dict(p=np.full(9, 0.9)), dict(mp=np.full(9, 0.1)),
               dict(k=np.full(9, 30), p=np.full(9, 0.7), mp=np.full(9, 0.01))):
        got = _check(pkg, logits, u, np.full(9, 0.9), **kw)
        assert got[0] == 0 and got[1] == 0 and got[4] == 7 and got[7] == 42
    greedy = _run(pkg, logits, u, np.zeros(9))
    assert greedy[5] == 3 and greedy[0] == 0 and greedy[1] == 0


@pytest.mark.gpu
def test_strides_inactive_rows_and_rows_behind(pkg):
    import torch

    dev = torch.device("cuda:0")
    rng = np.random.default_rng(4)
    for dtype, off in ((torch.float32, 1), (torch.bfloat16, 3), (torch.float16, 8)):
        store = torch.from_numpy(rng.standard_normal((40, 1240)) * 3).to(dtype).to(dev)
        store[:, 1237:] = 1e4  # beyond every row's vocabulary
        logits = store[:, off:off + 1237 - off]
        u = rng.random(40, dtype=np.float32)
        want = _check(pkg, logits, u, p=np.full(40, 0.9))
        pos = np.arange(40) % 3 - 1
        got = _run(pkg, logits, u, p=np.full(40, 0.9), pos=pos)
        assert (got[pos < 0] == -1).all() and (got[pos >= 0] == want[pos >= 0]).all()
    # the first rows of a larger buffer; the others stay
    nxt = torch.full((6,), -7, dtype=torch.int32, device=dev)
    pkg.sample_tokens(logits[:4], torch.zeros(4, device=dev), nxt[:4],
                      stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (nxt[4:] == -7).all() and (nxt[:4] >= 0).all()


@pytest.mark.gpu
def test_many_rows(pkg):
    """More rows than run at once, each with its own settings, small and large vocabulary."""
    import torch

    rng = np.random.default_rng(8)
    for n, vocab in ((700, 1500), (90, 120001)):
        x = torch.randn(n, vocab, generator=torch.Generator().manual_seed(n)) * 2.5
        kind = np.arange(n) % 5
        temp = np.where(kind == 0, 0.0, rng.uniform(0.5, 1.2, n))
        k = np.where((kind == 1) | (kind == 2), rng.integers(1, 200, n), 0)
        p = np.where((kind == 1) | (kind == 3), rng.uniform(0.5, 0.99, n), 1.0)
        mp = np.where(kind == 1, rng.uniform(0.01, 0.1, n), 0.0)
        _check(pkg, x.to("cuda:0"), rng.random(n, dtype=np.float32), temp, k, p, mp)


@pytest.mark.gpu
def test_drawn_frequencies(pkg):
    """Stratified u over one row: counts are the probabilities to within one draw per edge."""
    import torch

    n, vocab = 4096, 50
    row = torch.randn(vocab, generator=torch.Generator().manual_seed(1)).double()
    logits = row.float().repeat(n, 1).to("cuda:0")
    u = (np.arange(n) + 0.5) / n
    got = _run(pkg, logits, u)
    w = np.exp(row.float().double().numpy())
    counts = np.bincount(got, minlength=vocab)
    assert np.abs(counts - n * w / w.sum()).max() <= 1.0


@pytest.mark.gpu
def test_streams_and_graphs(pkg):
    import torch

    dev = torch.device("cuda:0")
    logits = torch.randn(64, 50257, device=dev) * 2
    u = torch.rand(64, device=dev)
    p = torch.full((64,), 0.9, device=dev)
    outs = [torch.zeros(64, dtype=torch.int32, device=dev) for _ in range(4)]
    pkg.sample_tokens(logits, u, outs[0], top_p=p, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    pkg.sample_tokens(logits, u, outs[1], top_p=p, stream=s1.cuda_stream)
    pkg.sample_tokens(logits, u, outs[2], top_p=p, stream=s2.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.sample_tokens(logits, u, outs[3], top_p=p, stream=torch.cuda.current_stream().cuda_stream)
    u.copy_(1 - u)
    graph.replay()
    pkg.sample_tokens(logits, u, outs[1], top_p=p, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(outs[3], outs[1]) and not torch.equal(outs[3], outs[0])


def _c_args(pkg, **change):
    base = dict(logits=0x1000, u=0x2000, temperature=None, top_k=None, top_p=None, min_p=None,
                pos=None, next=0x3000, stride=100, n_rows=4, vocab=100, dtype=2)
    base.update(change)
    a = pkg.SampleArgs()
    for name, value in base.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change", [
    dict(n_rows=-1), dict(vocab=0), dict(vocab=-5), dict(dtype=3), dict(dtype=-1), dict(stride=99),
    dict(stride=-100), dict(logits=None), dict(u=None), dict(next=None), dict(logits=0x1002),
    dict(dtype=0, logits=0x1001),
], ids=str)
def test_refusals(pkg, change):
    import ctypes

    lib = pkg.load_library()
    rc = lib.gptoss_decode_sample(ctypes.byref(_c_args(pkg, **change)), None)
    assert rc == pkg.GPTOSS_E_INVALID
    assert b"sample" in lib.gptoss_decode_last_error(None)


def test_vocabulary_limit_and_no_rows(pkg):
    import ctypes

    lib = pkg.load_library()
    assert lib.gptoss_decode_sample(None, None) == pkg.GPTOSS_E_INVALID
    a = _c_args(pkg, vocab=(1 << 18) + 1, stride=1 << 19)
    assert lib.gptoss_decode_sample(ctypes.byref(a), None) == pkg.GPTOSS_E_CAPACITY
    a = _c_args(pkg, n_rows=0, logits=None, u=None, next=None)
    assert lib.gptoss_decode_sample(ctypes.byref(a), None) == pkg.GPTOSS_OK
