"""Attention of packed prompts, prompt pieces and single tokens against 64-bit softmax.

Tolerance.  With p_t the normalised probabilities, A = sum p_t |v_t| and u half a step of the
16-bit type relative to a value (bf16 2^-8, fp16 2^-11): rounding each probability to the type
moves the sum by at most u A.  The scores are fp32 sums of head_dim exact products: their
error is at most head_dim * 2^-24 * sum |q_i k_i| * scale, below 2^-14 for the inputs here, the
exponential adds at most 2^-13 and the sum and the accumulation of up to 20000 terms of one
sign at most 2^-24 * 20000 / 2 < 2^-10 in the worst case and far less in the tiled sums here:
2^-11 A covers them together for bf16; for fp16 it is of the size of u itself.  The
result's rounding adds u |o|.  fp16 probabilities below 2^-14 are subnormal: each may be off by
2^-25 against the row's maximum of 1, hence the last term with the number of keys.
"""
import math

import numpy as np
import pytest

U = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def _reference(q, k, v, q_lens, kv_start, kv_lens, sinks, scale, window, q_first=0):
    """(out, A, visible keys) in float64; rows outside the sequences stay NaN."""
    import torch

    tokens, hq, d = q.shape
    hkv = k.shape[1]
    out = torch.full((tokens, hq, d), math.nan, dtype=torch.float64, device=q.device)
    mag, keys = torch.zeros_like(out), torch.zeros(tokens, 1, 1, dtype=torch.float64, device=q.device)
    at = q_first
    for n, start, length in zip(q_lens, kv_start, kv_lens):
        kk = k[start:start + length].double().repeat_interleave(hq // hkv, 1)
        vv = v[start:start + length].double().repeat_interleave(hq // hkv, 1)
        p = torch.arange(n, device=q.device) + (length - n)
        t = torch.arange(length, device=q.device)
        seen = t[None] <= p[:, None]
        if window:
            seen &= t[None] > p[:, None] - window
        # what no query sees takes part in nothing
        some = seen.any(0)
        kk = torch.where(some[:, None, None], kk, 0.0)
        vv = torch.where(some[:, None, None], vv, 0.0)
        s = torch.einsum("qhd,khd->hqk", q[at:at + n].double(), kk) * scale
        s = s.masked_fill(~seen[None], -math.inf)
        if sinks is not None:
            s = torch.cat([s, sinks.double()[:, None, None].expand(hq, n, 1)], 2)
        pr = torch.softmax(s, -1)[..., :length]
        pr = torch.where(seen[None], pr, 0.0)
        out[at:at + n] = torch.einsum("hqk,khd->qhd", pr, vv)
        mag[at:at + n] = torch.einsum("hqk,khd->qhd", pr, vv.abs())
        keys[at:at + n, 0, 0] = seen.sum(1).double()
        at += n
    return out, mag, keys


def _check(got, want, mag, keys, dtype, v_max):
    u = U[dtype]
    limit = mag * (u + 2.0 ** -11) + want.abs() * u + 1e-30
    if dtype == "float16":
        limit = limit + keys * 2.0 ** -25 * v_max + 2.0 ** -25
    err = (got.double() - want).abs()
    worst = (err / limit).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3f} of the limit, max error {err.max().item():.3e}"


def _make(torch, dev, seed, q_lens, kv_lens, hq, hkv, d, dtype, pad=0, gap=5, q_tail=0, v_pad=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = getattr(torch, dtype)
    starts, at = [], gap
    for n in kv_lens:
        starts.append(at)
        at += n + gap
    tokens = sum(q_lens) + q_tail
    q = torch.randn(tokens, hq * d + pad, generator=gen, device=dev).to(dt)
    k = torch.full((at, hkv * d + pad), math.nan, dtype=dt, device=dev)
    v = torch.full((at, hkv * d + pad + v_pad), math.nan, dtype=dt, device=dev)
    for s, n in zip(starts, kv_lens):
        k[s:s + n] = torch.randn(n, k.shape[1], generator=gen, device=dev).to(dt)
        v[s:s + n] = torch.randn(n, v.shape[1], generator=gen, device=dev).to(dt)
    sinks = torch.randn(hq, generator=gen, device=dev) * 2

    def view(x, h):
        return x[:, :h * d].unflatten(1, (h, d))

    out = torch.full((tokens, hq * d + pad), 9.0, dtype=dt, device=dev)
    return (view(q, hq), view(k, hkv), view(v, hkv), sinks, view(out, hq), out, starts)


def _index(torch, dev, q_lens, starts, kv_lens):
    return (torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32, device=dev),
            torch.tensor(starts, dtype=torch.int64, device=dev),
            torch.tensor(kv_lens, dtype=torch.int32, device=dev))


# q_lens, kv_lens, q heads, kv heads, head_dim, window, sinks, dtype, pad
CASES = [
    ([1], [1], 64, 8, 64, 0, True, "bfloat16", 0),
    ([7], [7], 8, 1, 64, 0, False, "bfloat16", 0),
    ([16, 17, 1, 33], [16, 17, 1, 33], 64, 8, 64, 128, True, "bfloat16", 0),
    ([129, 1, 300], [129, 1, 300], 8, 8, 64, 0, True, "float16", 8),
    ([500], [500], 8, 2, 64, 128, True, "bfloat16", 16),
    ([500], [500], 8, 2, 64, 1, False, "bfloat16", 0),        # every query its own key only
    ([257], [1000], 6, 2, 64, 100, True, "float16", 0),
    ([1025], [1025], 2, 1, 128, 0, False, "bfloat16", 0),
    ([65, 640], [2048, 700], 16, 4, 128, 0, True, "float16", 24),
    ([40, 3], [333, 3], 7, 1, 128, 77, True, "bfloat16", 0),  # group of 7
    ([200, 50], [200, 1700], 12, 4, 32, 0, True, "bfloat16", 0),
    ([90], [90], 3, 3, 32, 31, False, "float16", 8),
    ([5, 9], [5, 900], 128, 1, 64, 0, True, "bfloat16", 0),   # 128 heads on one
    ([3], [640], 96, 1, 32, 0, False, "float16", 0),
    ([1] * 9, [1, 2, 127, 128, 129, 255, 1000, 4096, 5001], 64, 8, 64, 0, True, "bfloat16", 0),
    ([1] * 5, [1, 130, 128, 2049, 7000], 16, 2, 128, 0, False, "bfloat16", 0),
    ([1, 1, 2], [20000, 19999, 300], 8, 1, 64, 0, True, "float16", 0),
    ([1, 1, 2], [9000, 128, 300], 8, 2, 64, 128, True, "bfloat16", 0),
    ([2000, 1, 31, 2], [2500, 4000, 31, 4001], 16, 2, 64, 0, True, "bfloat16", 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_against_64_bits(pkg, case):
    import torch

    q_lens, kv_lens, hq, hkv, d, window, with_sinks, dtype, pad = case
    dev = torch.device("cuda:0")
    q, k, v, sinks, out, whole, starts = _make(torch, dev, 11, q_lens, kv_lens, hq, hkv, d, dtype,
                                               pad, q_tail=3, v_pad=8)
    sinks = sinks if with_sinks else None
    q_start, kv_start, kv_len = _index(torch, dev, q_lens, starts, kv_lens)
    want, mag, keys = _reference(q, k, v, q_lens, starts, kv_lens, sinks, d ** -0.5, window)
    n = sum(q_lens)
    v_max = v.double().nan_to_num(0).abs().max().item()
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    stream = torch.cuda.current_stream().cuda_stream
    first = None
    for bound in (max(kv_lens), 0):  # however the work is split
        whole.fill_(9.0)
        pkg.prompt_attention(q, k, v, q_start, kv_start, kv_len, out, sinks=sinks, window=window,
                             max_kv_len=bound, status=status, stream=stream)
        torch.cuda.synchronize()
        assert status.item() == 0
        _check(out[:n], want[:n], mag[:n], keys[:n], dtype, v_max)
        assert (out[n:] == 9.0).all(), "rows behind the last sequence were written"
        assert (whole[:, hq * d:] == 9.0).all(), "padding was written"
        again = out.clone()
        pkg.prompt_attention(q, k, v, q_start, kv_start, kv_len, out, sinks=sinks, window=window,
                             max_kv_len=bound, status=status, stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(out, again), "two calls differ"
        first = again if first is None else first


@pytest.mark.gpu
@pytest.mark.parametrize("with_sinks", [True, False])
def test_rows_without_keys_and_empty_sequences(pkg, with_sinks):
    """kv_len 0, kv_len below the number of queries, and a sequence without queries."""
    import torch

    dev = torch.device("cuda:0")
    q_lens, kv_lens = [4, 0, 40, 6, 0], [0, 50, 25, 6, 0]
    q, k, v, sinks, out, whole, starts = _make(torch, dev, 3, q_lens, kv_lens, 8, 2, 64, "bfloat16")
    sinks = sinks if with_sinks else None
    q_start, kv_start, kv_len = _index(torch, dev, q_lens, starts, kv_lens)
    pkg.prompt_attention(q, k, v, q_start, kv_start, kv_len, out, sinks=sinks,
                         stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (out[:4] == 0).all() and (out[4:19] == 0).all()
    # the queries that do see keys: 25 of the third sequence, all of the fourth
    want, mag, keys = _reference(q, k, v, [25, 6], [starts[2], starts[3]], [25, 6], sinks, 0.125, 0,
                                 q_first=19)
    _check(out[19:], want[19:], mag[19:], keys[19:], "bfloat16", 10.0)


@pytest.mark.gpu
def test_what_no_query_sees_may_hold_anything(pkg):
    """NaN and infinities in keys before every window and after the last key."""
    import torch

    dev = torch.device("cuda:0")
    q_lens, kv_lens, window = [3, 40], [500, 700], 64
    q, k, v, sinks, out, whole, starts = _make(torch, dev, 4, q_lens, kv_lens, 16, 2, 64, "float16")
    for s, n, length in zip(starts, q_lens, kv_lens):
        unseen = length - n - window + 1
        k[s:s + unseen] = math.inf
        v[s:s + unseen] = math.nan
    q_start, kv_start, kv_len = _index(torch, dev, q_lens, starts, kv_lens)
    want, mag, keys = _reference(q, k, v, q_lens, starts, kv_lens, sinks, 0.125, window)
    for bound in (0, 700):
        pkg.prompt_attention(q, k, v, q_start, kv_start, kv_len, out, sinks=sinks, window=window,
                             max_kv_len=bound, stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        _check(out, want, mag, keys, "float16", 10.0)


@pytest.mark.gpu
def test_extreme_scores(pkg):
    """Large scores of both signs, equal scores, a sink far above and far below them."""
    import torch

    dev = torch.device("cuda:0")
    q_lens, kv_lens = [200], [900]
    q, k, v, _, out, whole, starts = _make(torch, dev, 6, q_lens, kv_lens, 8, 2, 64, "bfloat16")
    s0 = starts[0]
    q[:50] *= 8
    k[s0:s0 + 300] *= 4  # scores beyond +-100
    q[50:100] = 0  # all scores equal
    # rising scores: the running maximum moves at every block
    k[s0 + 300:s0 + 900] = (torch.arange(600, device=dev)[:, None, None] / 50.0).to(k.dtype)
    q[100:150] = 1.0
    sinks = torch.tensor([-math.inf, -300.0, 300.0, 0.0, 5.0, -5.0, 60.0, 90.0], device=dev)
    q_start, kv_start, kv_len = _index(torch, dev, q_lens, starts, kv_lens)
    want, mag, keys = _reference(q, k, v, q_lens, starts, kv_lens, sinks, 0.125, 0)
    pkg.prompt_attention(q, k, v, q_start, kv_start, kv_len, out, sinks=sinks, max_kv_len=900,
                         stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    # scores of up to 1500: 64 * 2^-24 * sum |q k| * scale is up to 2^-7 there, on the
    # exponent and so relative to A; probabilities below the rounded sum's reach vanish
    err = (out.double() - want).abs()
    limit = mag * (U["bfloat16"] + 2.0 ** -7) + want.abs() * U["bfloat16"] + 1e-12
    assert (err <= limit).all(), (err / limit).max().item()


@pytest.mark.gpu
def test_bad_sequences_are_reported_and_left_alone(pkg):
    import torch

    dev = torch.device("cuda:0")
    q_lens, kv_lens = [5, 6, 7, 8], [50, 60, 70, 80]
    q, k, v, sinks, out, whole, starts = _make(torch, dev, 8, q_lens, kv_lens, 8, 2, 64, "bfloat16")
    q_start, kv_start, kv_len = _index(torch, dev, q_lens, starts, kv_lens)
    stream = torch.cuda.current_stream().cuda_stream
    want, mag, keys = _reference(q, k, v, q_lens, starts, kv_lens, None, 0.125, 0)
    for field, value in (("start", -1), ("start", k.shape[0] - 59), ("start", 1 << 40), ("len", -3),
                         ("len", 1 << 30)):
        ks, kl = kv_start.clone(), kv_len.clone()
        (ks if field == "start" else kl)[1] = value
        status = torch.zeros(1, dtype=torch.int32, device=dev)
        whole.fill_(9.0)
        pkg.prompt_attention(q, k, v, q_start, ks, kl, out, status=status, stream=stream)
        torch.cuda.synchronize()
        assert status.item() == 104
        assert (out[5:11] == 9.0).all()
        for a, b in ((0, 5), (11, 26)):
            _check(out[a:b], want[a:b], mag[a:b], keys[a:b], "bfloat16", 10.0)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(pkg):
    """A cache whose rows lie past 2^31 elements."""
    import torch

    dev = torch.device("cuda:0")
    rows = 4_300_000
    k = torch.empty(rows, 8, 64, dtype=torch.bfloat16, device=dev)
    v = torch.empty(rows, 8, 64, dtype=torch.bfloat16, device=dev)
    assert k.numel() > 2 ** 31
    gen = torch.Generator(device=dev).manual_seed(1)
    q_lens, kv_lens, starts = [20, 1], [300, 1000], [rows - 300, rows - 100_000]
    for s, n in zip(starts, kv_lens):
        k[s:s + n] = torch.randn(n, 8, 64, generator=gen, device=dev).bfloat16()
        v[s:s + n] = torch.randn(n, 8, 64, generator=gen, device=dev).bfloat16()
    q = torch.randn(21, 64, 64, generator=gen, device=dev).bfloat16()
    out = torch.zeros_like(q)
    q_start, kv_start, kv_len = _index(torch, dev, q_lens, starts, kv_lens)
    want, mag, keys = _reference(q, k, v, q_lens, starts, kv_lens, None, 0.125, 0)
    pkg.prompt_attention(q, k, v, q_start, kv_start, kv_len, out, max_kv_len=1000,
                         stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    _check(out, want, mag, keys, "bfloat16", 10.0)


@pytest.mark.gpu
def test_streams_graphs_and_two_calls_at_once(pkg):
    import torch

    dev = torch.device("cuda:0")
    q_lens, kv_lens = [1, 300], [5000, 900]
    sets = [_make(torch, dev, s, q_lens, kv_lens, 16, 2, 64, "bfloat16") for s in (1, 2)]
    index = _index(torch, dev, q_lens, sets[0][6], kv_lens)

    def call(s, out, stream):
        pkg.prompt_attention(s[0], s[1], s[2], *index, out, sinks=s[3], max_kv_len=5000, stream=stream)

    want = [torch.zeros_like(s[4]) for s in sets]
    for s, w in zip(sets, want):
        call(s, w, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    got = [torch.zeros_like(s[4]) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        for s, g, st in zip(sets, got, streams):
            call(s, g, st.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph, rep = torch.cuda.CUDAGraph(), torch.zeros_like(want[0])
    with torch.cuda.graph(graph):
        call(sets[0], rep, torch.cuda.current_stream().cuda_stream)
    sets[0][0].copy_(sets[1][0])  # new queries and lengths for the replay
    index[2][0] = 4000
    graph.replay()
    other = torch.zeros_like(rep)
    call(sets[0], other, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(rep, other) and not torch.equal(rep, want[0])


def _c_args(pkg, **change):
    base = dict(q=0x1000, k=0x2000, v=0x3000, out=0x4000, q_start=0x5000, kv_start=0x6000,
                kv_len=0x7000, sinks=None, status=None, q_stride=512, k_stride=128, v_stride=128,
                out_stride=512, n_kv_rows=100, scale=0.125, n_tokens=10, n_seqs=2, n_q_heads=8,
                n_kv_heads=2, head_dim=64, window=0, max_kv_len=50, dtype=0)
    base.update(change)
    a = pkg.AttentionArgs()
    for name, value in base.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change", [
    dict(n_tokens=-1), dict(n_seqs=-1), dict(n_kv_rows=-1), dict(window=-1), dict(max_kv_len=-1),
    dict(dtype=2), dict(dtype=7), dict(head_dim=96), dict(head_dim=0), dict(n_q_heads=7),
    dict(n_q_heads=0), dict(n_kv_heads=0), dict(n_q_heads=258), dict(scale=0.0), dict(scale=-1.0),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(q_stride=511), dict(out_stride=0),
    dict(k_stride=120), dict(v_stride=64), dict(q_stride=516), dict(k_stride=132),
    dict(v_stride=1 << 40), dict(q=None), dict(out=None), dict(k=None), dict(v=None),
    dict(q_start=None), dict(kv_start=None), dict(kv_len=None), dict(q=0x1008), dict(k=0x2002),
    dict(v=0x3008), dict(out=0x4004),
], ids=str)
def test_refusals(pkg, change):
    import ctypes

    lib = pkg.load_library()
    rc = lib.gptoss_decode_prompt_attention(ctypes.byref(_c_args(pkg, **change)), None)
    assert rc == pkg.GPTOSS_E_INVALID
    assert b"prompt_attention" in lib.gptoss_decode_last_error(None)


def test_too_many_rows_and_nothing_to_do(pkg):
    import ctypes

    lib = pkg.load_library()
    assert lib.gptoss_decode_prompt_attention(None, None) == pkg.GPTOSS_E_INVALID
    a = _c_args(pkg, n_kv_rows=(1 << 31) - 256)
    assert lib.gptoss_decode_prompt_attention(ctypes.byref(a), None) == pkg.GPTOSS_E_CAPACITY
    for change in (dict(n_tokens=0, q=None, out=None), dict(n_seqs=0, q_start=None)):
        a = _c_args(pkg, **change)
        assert lib.gptoss_decode_prompt_attention(ctypes.byref(a), None) == pkg.GPTOSS_OK


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,window", [("bfloat16", 64, 0), ("bfloat16", 64, 100), ("float16", 32, 0),
                                            ("bfloat16", 128, 0)])
def test_huge_values_behind_a_query_have_no_weight(pkg, dtype, d, window):
    """A key that a query may not see weighs exactly nothing, even where its value is near the
    type's largest: the queries before it match as if it were not there."""
    import torch

    dev = torch.device("cuda:0")
    q_lens, kv_lens, seen = [300], [300], 250
    q, k, v, sinks, out, whole, starts = _make(torch, dev, 14, q_lens, kv_lens, 8, 1, d, dtype)
    v[starts[0] + seen:starts[0] + 300] = torch.finfo(v.dtype).max / 2
    q_start, kv_start, kv_len = _index(torch, dev, q_lens, starts, kv_lens)
    want, mag, keys = _reference(q, k, v, q_lens, starts, kv_lens, sinks, d ** -0.5, window)
    pkg.prompt_attention(q, k, v, q_start, kv_start, kv_len, out, sinks=sinks, window=window,
                         stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    _check(out[:seen], want[:seen], mag[:seen], keys[:seen], dtype, 10.0)


@pytest.mark.gpu
@pytest.mark.parametrize("most", [2, 6])
def test_thousands_of_sequences(pkg, most):
    """More sequences than one look at their starts covers, some without a query; a bad one late
    in the list is reported and the others stand."""
    import torch

    dev = torch.device("cuda:0")
    rng = np.random.default_rng(most)
    q_lens = [int(n) for n in rng.integers(0, most + 1, 2900)]
    kv_lens = [n + int(rng.integers(0, 9)) for n in q_lens]
    q, k, v, sinks, out, whole, starts = _make(torch, dev, 15, q_lens, kv_lens, 8, 1, 32, "bfloat16", gap=1)
    q_start, kv_start, kv_len = _index(torch, dev, q_lens, starts, kv_lens)
    bad = max(i for i, n in enumerate(q_lens) if n)
    kv_len[bad] = -1
    want, mag, keys = _reference(q, k, v, q_lens, starts, kv_lens, sinks, 32 ** -0.5, 0)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    pkg.prompt_attention(q, k, v, q_start, kv_start, kv_len, out, sinks=sinks, status=status,
                         stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert status.item() == 104
    at = sum(q_lens[:bad])
    assert (out[at:at + q_lens[bad]] == 9.0).all()
    _check(out[:at], want[:at], mag[:at], keys[:at], "bfloat16", 10.0)


@pytest.mark.gpu
@pytest.mark.parametrize("starts_of", [[0, 5, 3, 10, 12], [0, -4, 3, 8, 12], [2, 5, 8, 10, 12], [0, 5, 8, 40, 12]])
@pytest.mark.parametrize("group", [1, 32])
def test_starts_that_do_not_ascend(pkg, starts_of, group):
    """Reported, and nothing is written outside the rows."""
    import torch

    dev = torch.device("cuda:0")
    q, k, v, sinks, out, whole, starts = _make(torch, dev, 16, [3, 3, 3, 3], [30, 30, 30, 30], group, 1, 64,
                                               "bfloat16", pad=8)
    q_start, kv_start, kv_len = _index(torch, dev, [3, 3, 3, 3], starts, [30, 30, 30, 30])
    q_start.copy_(torch.tensor(starts_of, dtype=torch.int32))
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    pkg.prompt_attention(q, k, v, q_start, kv_start, kv_len, out, status=status,
                         stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert status.item() == (0 if starts_of[0] == 2 else 104)
    assert (whole[:, group * 64:] == 9.0).all()
    assert torch.isfinite(out.float()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    ([1500], [1500], 8, 2, 64, 600, True, "bfloat16", 0),
    ([700, 3], [2000, 1300], 4, 4, 32, 513, False, "float16", 8),
    ([900, 300], [900, 2100], 8, 1, 64, 512, True, "bfloat16", 0),
    ([1100], [1400], 4, 1, 128, 700, True, "float16", 0),
], ids=str)
def test_wide_windows(pkg, case):
    test_against_64_bits(pkg, case)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv", [(8, 1), (2, 2)])
def test_entries_of_a_sequence_without_queries_do_not_count(pkg, hq, hkv):
    """Places that a batch of fixed size leaves empty may hold any kv_start and kv_len."""
    import torch

    dev = torch.device("cuda:0")
    q_lens, kv_lens = [0, 5, 0, 7, 0], [30, 50, 30, 60, 30]
    q, k, v, sinks, out, whole, starts = _make(torch, dev, 21, q_lens, kv_lens, hq, hkv, 64, "bfloat16")
    q_start, kv_start, kv_len = _index(torch, dev, q_lens, starts, kv_lens)
    want, mag, keys = _reference(q, k, v, q_lens, starts, kv_lens, sinks, 0.125, 0)
    kv_start[0], kv_len[2], kv_start[4], kv_len[4] = 1 << 40, -9, -1, 1 << 30
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    pkg.prompt_attention(q, k, v, q_start, kv_start, kv_len, out, sinks=sinks, status=status,
                         stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert status.item() == 0
    _check(out, want, mag, keys, "bfloat16", 10.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,window", [("bfloat16", 64, 0), ("float16", 64, 0), ("float16", 64, 100),
                                            ("bfloat16", 128, 0), ("float16", 128, 0), ("bfloat16", 32, 0)])
@pytest.mark.parametrize("tokens", [1, 150])
def test_scores_near_the_documented_limit(pkg, dtype, d, window, tokens):
    """Scores of up to 2^25.5.  Queries and keys are signs times a power of two, so every score is
    exact: equal patterns tie, others are millions apart, and the result is a mean of values (or
    nothing, where the sink is above them)."""
    import torch

    dev = torch.device("cuda:0")
    q_lens, kv_lens = [tokens, tokens], [700, tokens]
    q, k, v, sinks, out, whole, starts = _make(torch, dev, 22, q_lens, kv_lens, 8, 2, d, dtype)
    gen = torch.Generator(device=dev).manual_seed(23)
    signs = torch.randint(0, 2, (6, d), generator=gen, device=dev).to(q.dtype) * 2 - 1
    q.copy_(signs[torch.randint(0, 6, q.shape[:2], generator=gen, device=dev)] * 2.0 ** 11)
    k.copy_(signs[torch.randint(0, 6, k.shape[:2], generator=gen, device=dev)] * 2.0 ** 11)
    q_start, kv_start, kv_len = _index(torch, dev, q_lens, starts, kv_lens)
    want, mag, keys = _reference(q, k, v, q_lens, starts, kv_lens, sinks, d ** -0.5, window)
    for bound in (0, 700):
        pkg.prompt_attention(q, k, v, q_start, kv_start, kv_len, out, sinks=sinks, window=window,
                             max_kv_len=bound, stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        _check(out, want, mag, keys, dtype, 10.0)


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    ([300] + [0] * 200, [2000] + [0] * 200, 16, 2, 64, 100, True, "bfloat16", 0),
    ([0] * 200 + [300], [5] * 200 + [2000], 16, 2, 64, 0, False, "float16", 8),
    ([40, 3, 0, 0], [3000, 700, 9, 0], 4, 4, 64, 0, True, "bfloat16", 0),
    ([40, 3, 0, 0], [3000, 700, 9, 0], 4, 4, 32, 500, True, "float16", 0),
    ([10, 0, 2], [5000, 10, 300], 3, 1, 128, 0, False, "bfloat16", 0),
    ([0, 10, 2], [10, 5000, 300], 3, 1, 128, 77, True, "float16", 0),
    ([3, 0, 0], [900, 0, 0], 16, 1, 64, 0, True, "bfloat16", 0),
], ids=str)
def test_batches_padded_with_empty_sequences(pkg, case):
    """Few rows on average, many in one sequence: several jobs of the kernel for single tokens."""
    test_against_64_bits(pkg, case)
