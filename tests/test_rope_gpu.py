"""Rotary positions with the append to the KV cache against the formula in 64 bits.

Tolerance: the result is formed in fp32 and rounded once to the type.  With inputs of
magnitude X a rotated element is a sum of two products of an input with a cosine or sine;
the cosine and sine of the fp64 angle carry at most a few units of 2^-24 (4 ulp taken),
the concentration multiplies with 2^-24 more and the two products and the sum add three
roundings, so the fp32 value is within 2 * X * c * 8 * 2^-24 of the exact one; the rounding
to the type adds half a step of the value.  Copied elements are equal.
"""
import numpy as np
import pytest

HALF_STEP = {"bfloat16": 2.0 ** -9, "float16": 2.0 ** -12, "float32": 2.0 ** -25}


def _formula(x, pos, inv_freq, conc, rotary, interleaved):
    """x [rows, heads, D] float64 -> rotated."""
    half = rotary // 2
    ang = pos.astype(np.float64)[:, None] * inv_freq.astype(np.float64)[None, :]
    c, s = np.cos(ang)[:, None] * conc, np.sin(ang)[:, None] * conc
    out = x.copy()
    i1 = np.arange(half) * 2 if interleaved else np.arange(half)
    i2 = i1 + 1 if interleaved else i1 + half
    out[..., i1] = x[..., i1] * c - x[..., i2] * s
    out[..., i2] = x[..., i2] * c + x[..., i1] * s
    return out


def _check(got, want, x_max, conc, dtype, what):
    err = np.abs(got.double().cpu().numpy() - want)
    tiny = 2.0 ** -25 if dtype == "float16" else 0.0  # half a step of fp16's subnormals
    limit = (2 * x_max * conc * 8 * 2.0 ** -24) * (1 + 2 ** -8) + np.abs(want) * 2 * HALF_STEP[dtype] + tiny
    assert (err <= limit).all(), f"{what}: {err.max():.3e}, {(err / limit).max():.2f} of the limit"


# rows, q heads, kv heads, head_dim, rotary_dim, interleaved, dtype, pad (elements between rows)
CASES = [
    (1, 64, 8, 64, 64, False, "bfloat16", 0),
    (3, 8, 1, 64, 64, True, "bfloat16", 8),
    (129, 7, 7, 32, 32, False, "float16", 0),
    (5, 3, 1, 128, 96, False, "bfloat16", 4),      # 8-byte accesses
    (17, 4, 2, 32, 24, False, "float16", 0),       # half of 12
    (17, 4, 2, 32, 24, True, "bfloat16", 0),
    (9, 5, 5, 80, 2, False, "float32", 1),         # odd row stride: scalar accesses
    (9, 5, 5, 80, 2, True, "float16", 1),
    (33, 2, 2, 7, 6, True, "bfloat16", 3),         # odd head
    (33, 2, 2, 7, 6, False, "float32", 0),
    (5000, 4, 2, 64, 32, False, "bfloat16", 16),   # several rows per CTA
    (2501, 2, 2, 128, 128, True, "float32", 0),
    (2, 1, 1, 1024, 1024, False, "float16", 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(str(v) for v in c))
def test_against_the_formula(pkg, case):
    import torch

    rows, hq, hkv, d, rotary, inter, dtype, pad = case
    dev = torch.device("cuda:0")
    gen = torch.Generator().manual_seed(sum(case[:5]))
    dt = getattr(torch, dtype)
    ld = (hq + 2 * hkv) * d + pad
    store = torch.randn(rows, ld, generator=gen).to(dt).to(dev)
    qkv = store[:, :(hq + 2 * hkv) * d].unflatten(1, (hq + 2 * hkv, d))
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    pos = torch.randint(0, 1 << 20, (rows,), generator=gen, dtype=torch.int32)
    pos[rows // 2::5] = -1
    pos[0] = 0 if rows > 1 else (1 << 20) - 1
    n_slots = rows + 9
    slots = torch.randperm(n_slots, generator=gen)[:rows].to(torch.int64)
    if rows > 4:  # rows that are rotated but not stored
        slots[1], slots[2] = -1, n_slots
    inv, conc = pkg.rope_table(rotary, 150000.0, 32.0, 4096)
    q_out = torch.full((rows, hq, d), 7.0, dtype=dt, device=dev)
    k_cache = torch.full((n_slots, hkv, d), 7.0, dtype=dt, device=dev)
    v_cache = torch.full((n_slots, hkv, d), 7.0, dtype=dt, device=dev)
    pkg.rope_append(q, k, v, pos.to(dev), torch.from_numpy(inv).to(dev), q_out, k_cache, v_cache,
                    slots=slots.to(dev), concentration=conc, interleaved=inter,
                    stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    x = qkv.double().cpu().numpy()
    p, sl = pos.numpy(), slots.numpy()
    want = _formula(x, p, inv, conc, rotary, inter)
    x_max = np.abs(x).max()
    live = p >= 0
    want_q = np.where(live[:, None, None], want[:, :hq], 7.0)
    _check(q_out, want_q, x_max, conc, dtype, "q")
    want_k = np.full((n_slots, hkv, d), 7.0)
    want_v = want_k.copy()
    kept = live & (sl >= 0) & (sl < n_slots)
    want_k[sl[kept]] = want[kept, hq:hq + hkv]
    want_v[sl[kept]] = x[kept, hq + hkv:]
    _check(k_cache, want_k, x_max, conc, dtype, "k")
    assert (v_cache.double().cpu().numpy() == want_v).all()
    if rotary < d:  # what is not rotated is copied
        assert (q_out.double().cpu().numpy()[..., rotary:] == want_q[..., rotary:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("inter", [False, True])
def test_in_place_and_parts(pkg, inter):
    """q and k rotated where they are, without a cache; k alone; v alone."""
    import torch

    dev = torch.device("cuda:0")
    gen = torch.Generator().manual_seed(5)
    q0 = torch.randn(40, 6, 64, generator=gen).bfloat16()
    k0 = torch.randn(40, 2, 64, generator=gen).bfloat16()
    pos = torch.arange(40, dtype=torch.int32) * 1000 - 3000
    inv, conc = pkg.rope_table(64, 10000.0)
    assert conc == 1.0
    inv_d = torch.from_numpy(inv).to(dev)
    q, k = q0.to(dev), k0.to(dev)
    pkg.rope_append(q, k, None, pos.to(dev), inv_d, q_out=q, k_cache=k, interleaved=inter,
                    stream=torch.cuda.current_stream().cuda_stream)
    k2, v2 = torch.zeros_like(k), torch.zeros_like(k)
    pkg.rope_append(None, k0.to(dev), None, pos.to(dev), inv_d, k_cache=k2, interleaved=inter,
                    stream=torch.cuda.current_stream().cuda_stream)
    pkg.rope_append(None, None, k0.to(dev), pos.to(dev), inv_d, v_cache=v2, interleaved=inter,
                    stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    p = pos.numpy()
    live = (p >= 0)[:, None, None]
    for got, x in ((q, q0), (k, k0)):
        x = x.double().numpy()
        want = np.where(live, _formula(x, p, inv, conc, 64, inter), x)
        _check(got, want, np.abs(x).max(), conc, "bfloat16", "in place")
    assert torch.equal(k2[3:], k[3:]) and (k2[:3] == 0).all()
    assert torch.equal(v2[3:].cpu(), k0[3:]) and (v2[:3] == 0).all()


@pytest.mark.gpu
def test_fp32_angle_is_the_decode_steps(pkg):
    """angle_f32 rounds pos * inv_freq to fp32 before the cosine, as the reference does."""
    import torch

    dev = torch.device("cuda:0")
    inv, conc = pkg.rope_table(64, 150000.0, 32.0, 4096)
    pos = np.array([0, 1, 4097, 131071, 1000003], np.int32)
    x = np.random.default_rng(3).standard_normal((5, 2, 64)).astype(np.float32)
    ang = pos.astype(np.float32)[:, None] * inv[None, :]
    c = np.cos(ang.astype(np.float64))[:, None] * conc
    s = np.sin(ang.astype(np.float64))[:, None] * conc
    want = np.concatenate([x[..., :32] * c - x[..., 32:] * s, x[..., 32:] * c + x[..., :32] * s], -1)
    got = torch.zeros(5, 2, 64, device=dev)
    pkg.rope_append(torch.from_numpy(x).to(dev), None, None, torch.from_numpy(pos).to(dev),
                    torch.from_numpy(inv).to(dev), q_out=got, concentration=conc, angle_f32=True,
                    stream=torch.cuda.current_stream().cuda_stream)
    _check(got, want, np.abs(x).max(), conc, "float32", "fp32 angle")
    exact = torch.zeros(5, 2, 64, device=dev)
    pkg.rope_append(torch.from_numpy(x).to(dev), None, None, torch.from_numpy(pos).to(dev),
                    torch.from_numpy(inv).to(dev), q_out=exact, concentration=conc,
                    stream=torch.cuda.current_stream().cuda_stream)
    _check(exact, _formula(x.astype(np.float64), pos, inv, conc, 64, False), np.abs(x).max(), conc,
           "float32", "fp64 angle")


@pytest.mark.gpu
def test_another_stream_and_a_captured_call(pkg):
    import torch

    dev = torch.device("cuda:0")
    q = torch.randn(300, 8, 64, device=dev).bfloat16()
    pos = torch.arange(300, dtype=torch.int32, device=dev)
    inv, conc = pkg.rope_table(64, 10000.0)
    inv = torch.from_numpy(inv).to(dev)
    want, got, rep = (torch.zeros_like(q) for _ in range(3))
    pkg.rope_append(q, None, None, pos, inv, q_out=want,
                    stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        pkg.rope_append(q, None, None, pos, inv, q_out=got, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.rope_append(q, None, None, pos, inv, q_out=rep,
                        stream=torch.cuda.current_stream().cuda_stream)
    assert (rep == 0).all()
    pos += 17  # a replay reads what the buffers hold then
    graph.replay()
    pkg.rope_append(q, None, None, pos, inv, q_out=want,
                    stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(rep, want)


def test_table_is_the_yarn_formula(pkg):
    """Host function: bases, interpolation ramp and concentration in 64 bits."""
    for rotary, theta, factor, ctx in ((64, 150000.0, 32.0, 4096), (32, 10000.0, 1.0, 4096),
                                       (96, 500000.0, 8.0, 8192)):
        inv, conc = pkg.rope_table(rotary, theta, factor, ctx)
        half = rotary // 2
        freq = theta ** (np.arange(half) * 2.0 / rotary)
        want = 1 / freq
        if factor > 1:
            low = half * np.log(ctx / (32 * 2 * np.pi)) / np.log(theta)
            high = half * np.log(ctx / (2 * np.pi)) / np.log(theta)
            ramp = np.clip((np.arange(half) - low) / (high - low), 0, 1)
            want = ramp / (factor * freq) + (1 - ramp) / freq
            assert abs(conc - (0.1 * np.log(factor) + 1)) < 1e-6
        else:
            assert conc == 1.0
        # fp32 throughout; powf's error grows with its result's exponent, the ramp's
        # difference of two fp32 numbers of size `half` costs half * 2^-23 / (high - low)
        np.testing.assert_allclose(inv, want, rtol=3e-5)
    for bad in ((63, 1e4, 1.0, 4096), (0, 1e4, 1.0, 4096), (2048, 1e4, 1.0, 4096), (64, 0.5, 1.0, 4096),
                (64, float("nan"), 1.0, 4096), (64, 1e4, 2.0, 0)):
        with pytest.raises(pkg.MoeError) as ei:
            pkg.rope_table(*bad)
        assert ei.value.code == pkg.GPTOSS_E_INVALID


def _c_args(pkg, **change):
    base = dict(q=0x1000, k=0x2000, v=0x3000, q_out=0x4000, k_cache=0x5000, v_cache=0x6000,
                pos=0x7000, slots=0x8000, inv_freq=0x9000, q_stride=512, k_stride=128, v_stride=128,
                q_out_stride=512, k_cache_stride=128, v_cache_stride=128, n_slots=100,
                concentration=1.0, n_rows=10, n_q_heads=8, n_kv_heads=2, head_dim=64, rotary_dim=64,
                interleaved=0, angle_f32=0, dtype=0)
    base.update(change)
    a = pkg.RopeArgs()
    for name, value in base.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change", [
    dict(n_rows=-1), dict(n_slots=-1), dict(dtype=3), dict(dtype=-1), dict(head_dim=0),
    dict(head_dim=1025), dict(rotary_dim=66), dict(rotary_dim=63), dict(rotary_dim=0),
    dict(q=None), dict(q_out=None), dict(k_cache=None), dict(v=None), dict(n_q_heads=0),
    dict(n_q_heads=1025), dict(n_kv_heads=0), dict(q_stride=511), dict(k_stride=127),
    dict(v_cache_stride=1), dict(q_out_stride=0), dict(slots=None, n_slots=9), dict(pos=None),
    dict(inv_freq=None), dict(k_cache=0x2000), dict(v_cache=0x3000),
    dict(k_cache=0x2000, slots=None, k_cache_stride=256), dict(q_out=0x1000, q_out_stride=1024),
    dict(q=0x1001), dict(k_cache=0x5001), dict(dtype=2, v=0x3002),
    dict(q=None, q_out=None, k=None, k_cache=None, v=None, v_cache=None),
], ids=str)
def test_refusals(pkg, change):
    """Checked on the host before CUDA is touched: the pointers here point nowhere."""
    import ctypes

    lib = pkg.load_library()
    rc = lib.gptoss_decode_rope_append(ctypes.byref(_c_args(pkg, **change)), None)
    assert rc == pkg.GPTOSS_E_INVALID
    assert b"rope_append" in lib.gptoss_decode_last_error(None)
    assert lib.gptoss_decode_rope_append(None, None) == pkg.GPTOSS_E_INVALID


def test_no_rows_is_no_work(pkg):
    import ctypes

    lib = pkg.load_library()
    a = _c_args(pkg, n_rows=0, pos=None, inv_freq=None)
    assert lib.gptoss_decode_rope_append(ctypes.byref(a), None) == pkg.GPTOSS_OK


def test_binding_refuses_tensors_it_cannot_pass(pkg):
    import torch

    q = torch.zeros(4, 2, 8)
    with pytest.raises(ValueError, match="GPU"):
        pkg.rope_append(q, None, None, torch.zeros(4, dtype=torch.int32), torch.zeros(4), q_out=q)
    with pytest.raises(ValueError, match="all None"):
        pkg.rope_append(None, None, None, None, None)


@pytest.mark.gpu
def test_binding_refusals_on_the_gpu(pkg):
    import torch

    dev = torch.device("cuda:0")
    q = torch.zeros(4, 2, 8, device=dev)
    pos, inv = torch.zeros(4, dtype=torch.int32, device=dev), torch.zeros(4, device=dev)
    with pytest.raises(ValueError, match="contiguous"):
        pkg.rope_append(q.transpose(0, 1), None, None, pos, inv, q_out=q)
    with pytest.raises(TypeError, match="q_out"):
        pkg.rope_append(q, None, None, pos, inv, q_out=q.half())
    with pytest.raises(TypeError, match="int32"):
        pkg.rope_append(q, None, None, pos.long(), inv, q_out=q)
    with pytest.raises(ValueError, match="cpu"):
        pkg.rope_append(q, None, None, pos.cpu(), inv, q_out=q)
    with pytest.raises(TypeError, match="not supported"):
        pkg.rope_append(q.double(), None, None, pos, inv, q_out=q.double())
    with pytest.raises(pkg.MoeError) as ei:  # rotary_dim 8 of a head of 8, an output missing
        pkg.rope_append(q, None, None, pos, inv)
    assert ei.value.code == pkg.GPTOSS_E_INVALID
