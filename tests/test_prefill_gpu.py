"""Prompts brought in by the prefill against the same prompts fed token by token, against the
reference's recorded logits, and drawn tokens against a draw from the step's own logits.

Tolerances.  Prefill and step run the same GEMMs row by row; their attention sums in another
order with probabilities rounded to bf16 in both, so the residual stream differs by roundings
to bf16 that fall the other way: the limits of the decode tests for logits against the fp32
reference (2e-2 largest, 2e-3 mean, logits of std 0.23) hold for each side, and twice that
between the two.
"""
import numpy as np
import pytest

from test_decode_gpu import LOGIT_MAX_ABS, LOGIT_MEAN_ABS, _golden
from test_sample_gpu import _draw


def _engine(pkg, cfg, seed, tmp_path, max_batch, max_tokens=None):
    from gpt_oss_b200 import synth

    path = tmp_path / "model.bin"
    if not path.exists():
        synth.write_model_bin(path, cfg, seed)
    eng = pkg.DecodeEngine(cfg, max_batch, max_tokens=max_tokens)
    eng.load_bin(np.asarray(np.memmap(path, dtype=np.uint8, mode="r")))
    return eng


def _close(a, b):
    err = np.abs(a.astype(np.float64) - b)
    assert err.max() <= 2 * LOGIT_MAX_ABS and err.mean() <= 2 * LOGIT_MEAN_ABS, (err.max(), err.mean())


def _feed(eng, tokens, row, pos0=0):
    nxt = None
    for i, t in enumerate(tokens):
        tok, pos = np.full(eng.max_batch, -1, np.int32), np.full(eng.max_batch, -1, np.int32)
        tok[row], pos[row] = t, pos0 + i
        nxt = eng.step(tok, pos)[row]
    return int(nxt), eng.logits(row)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["tiny", "mini"])
@pytest.mark.parametrize("max_tokens", [None, 5, 64])
def test_prefill_matches_reference_logits(pkg, tmp_path, name, max_tokens):
    """The golden tokens up to several positions, in one or more passes, then a step."""
    from gpt_oss_b200 import synth

    g = _golden(name)
    cfg = synth.TINY_MODEL if name == "tiny" else synth.MINI_MODEL
    eng = _engine(pkg, cfg, int(g["seed"]), tmp_path, 4, max_tokens)
    tokens, probes = g["tokens"], g["probes"]
    for n in (1, 2, 13, len(tokens) - 1):
        eng.prefill([tokens[:n]], [2])
        err = np.abs(eng.logits(0)[probes].astype(np.float64) - g["probe_logits"][n - 1])
        assert err.max() <= LOGIT_MAX_ABS and err.mean() <= LOGIT_MEAN_ABS
        tok, pos = np.full(4, -1, np.int32), np.full(4, -1, np.int32)
        tok[2], pos[2] = tokens[n], n  # the step goes on from the cache that the prefill left
        eng.step(tok, pos)
        err = np.abs(eng.logits(2)[probes].astype(np.float64) - g["probe_logits"][n])
        assert err.max() <= LOGIT_MAX_ABS and err.mean() <= LOGIT_MEAN_ABS
    eng.close()


@pytest.mark.gpu
@pytest.mark.parametrize("max_tokens", [8, 37, 400])
def test_several_prompts_and_continuations(pkg, tmp_path, max_tokens):
    """Prompts of different lengths beyond the window, two of them continued, in passes of
    several sizes; a row outside the call keeps its cache."""
    import torch

    from gpt_oss_b200 import synth

    # every expert is selected, so no near-tie in the router separates the two ways
    cfg = dict(synth.MINI_MODEL, vocab_size=900, sliding_window=21, n_layers=3, seq_len=160, n_attn_heads=6,
               n_kv_heads=2, n_experts=4, experts_per_token=4)
    rng = np.random.default_rng(1)
    lens = [70, 1, 33, 100]
    prompts = [rng.integers(0, 900, n, dtype=np.int32) for n in lens]
    more = [rng.integers(0, 900, n, dtype=np.int32) for n in (17, 2)]
    steps = _engine(pkg, cfg, 5, tmp_path, 6)
    want = [_feed(steps, p, r) for p, r in zip(prompts, (4, 0, 2, 5))]
    want_more = [_feed(steps, m, r, p0) for m, r, p0 in zip(more, (4, 2), (70, 33))]
    eng = _engine(pkg, cfg, 5, tmp_path, 6, max_tokens)
    dev, dkv = torch.device("cuda:0"), cfg["n_kv_heads"] * cfg["head_dim"]
    marks = [torch.randn(1, 8, dkv, device=dev).bfloat16() for _ in range(2)]
    eng.set_kv(1, 3, 0, *marks)
    nxt = eng.prefill(prompts, [4, 0, 2, 5])
    for i, (token, logits) in enumerate(want):
        _close(eng.logits(i), logits)
        assert nxt[i] == token or logits[token] - logits[nxt[i]] <= 4 * LOGIT_MAX_ABS
    nxt = eng.prefill(more, [4, 2], pos0=[70, 33])
    for i, (token, logits) in enumerate(want_more):
        _close(eng.logits(i), logits)
    # caches: the first layer's keys and values come from the same projection rows; a rotated
    # key is rounded to bf16 once, after fp32 sums that may be contracted differently
    for layer in range(3):
        for row, n in ((4, 87), (0, 1), (2, 35), (5, 100)):
            a = [torch.zeros(1, n, dkv, dtype=torch.bfloat16, device=dev) for _ in range(4)]
            steps.get_kv(layer, row, 0, a[0], a[1])
            eng.get_kv(layer, row, 0, a[2], a[3])
            for x, y in ((a[0], a[2]), (a[1], a[3])):
                diff = (x.float() - y.float()).abs()
                if layer == 0:
                    assert (diff <= x.float().abs() * 2.0 ** -7 + 1e-6).all()
                else:
                    assert diff.max() <= 0.05 * x.float().abs().max()
    kept = [torch.zeros(1, 8, dkv, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    eng.get_kv(1, 3, 0, *kept)
    assert torch.equal(kept[0], marks[0]) and torch.equal(kept[1], marks[1])
    steps.close()
    eng.close()


@pytest.mark.gpu
def test_full_chain_of_prompt_steps_and_draws(pkg, tmp_path):
    """Prefill with drawn tokens, then sampled steps: every token is the draw from the logits
    that the engine reports, and settings that leave one token give the greedy one."""
    from gpt_oss_b200 import synth

    cfg = dict(synth.MINI_MODEL, vocab_size=1200, n_layers=2)
    eng = _engine(pkg, cfg, 9, tmp_path, 4, 48)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, 1200, n, dtype=np.int32) for n in (20, 3, 41)]
    greedy = eng.prefill(prompts, [0, 1, 3])
    one = eng.prefill(prompts, [0, 1, 3], sampling=dict(u=rng.random(3), top_k=[1, 1, 1]))
    assert (greedy == one).all()

    def settings(n):
        return dict(u=rng.random(n, dtype=np.float32), temperature=rng.uniform(0.3, 1.2, n).astype(np.float32),
                    top_k=rng.integers(0, 60, n), top_p=rng.uniform(0.3, 1.0, n).astype(np.float32),
                    min_p=rng.uniform(0.0, 0.1, n).astype(np.float32))

    def check(rows, got, s):
        for i, r in enumerate(rows):
            f = lambda k: float(np.float64(np.float32(s[k][r])))  # noqa: E731
            want, margin = _draw(eng.logits(r), f("u"), f("temperature"), int(s["top_k"][r]), f("top_p"), f("min_p"))
            assert margin > 1e-11 and got[r] == want

    s = settings(3)
    nxt = eng.prefill(prompts, [0, 1, 3], sampling=s)
    check([0, 1, 2], nxt, s)
    where = {0: 20, 1: 3, 3: 41}
    token = {0: nxt[0], 1: nxt[1], 3: nxt[2]}
    for _ in range(4):
        tok, pos = np.full(4, -1, np.int32), np.full(4, -1, np.int32)
        for r in where:
            tok[r], pos[r] = token[r], where[r]
        s = settings(4)
        out = eng.step(tok, pos, sampling=s)
        assert out[2] == -1
        check([0, 1, 3], out, s)
        for r in where:
            where[r] += 1
            token[r] = out[r]
    # the same step again, greedy: sampling leaves the plain step as it was
    plain = eng.step(tok, pos)
    assert all(plain[r] == eng.logits(r).argmax() for r in where)
    assert (eng.step(tok, pos, sampling=dict(u=np.zeros(4), temperature=np.zeros(4))) == plain).all()
    eng.close()


@pytest.mark.gpu
def test_refusals_change_nothing(pkg, tmp_path):
    from gpt_oss_b200 import synth

    cfg = dict(synth.MINI_MODEL, vocab_size=300, n_layers=1, seq_len=64)
    eng = _engine(pkg, cfg, 2, tmp_path, 3, 16)
    ok = np.arange(10, dtype=np.int32)
    want = eng.prefill([ok], [1])
    for args, code in (((([ok], [3])), pkg.GPTOSS_E_INVALID), ((([ok], [-1])), pkg.GPTOSS_E_INVALID),
                       ((([ok, ok], [1, 1])), pkg.GPTOSS_E_INVALID),
                       ((([ok, ok[:0]], [0, 1])), pkg.GPTOSS_E_INVALID),
                       ((([ok], [1], [-1])), pkg.GPTOSS_E_INVALID),
                       ((([ok], [1], [55])), pkg.GPTOSS_E_CAPACITY),
                       ((([ok, ok, ok, ok], [0, 1, 2, 0])), pkg.GPTOSS_E_CAPACITY),
                       ((([ok, np.array([5, 300])], [0, 1])), pkg.GPTOSS_E_INVALID),
                       ((([np.array([-1])], [1])), pkg.GPTOSS_E_INVALID)):
        with pytest.raises(pkg.MoeError) as ei:
            eng.prefill(*args)
        assert ei.value.code == code
    with pytest.raises(pkg.MoeError, match="u"):
        eng.prefill([ok], [1], sampling=dict(temperature=[1.0]))
    with pytest.raises(ValueError, match="unknown"):
        eng.prefill([ok], [1], sampling=dict(u=[0.5], topk=[1]))
    with pytest.raises(ValueError, match="entries"):
        eng.step(ok[:2], np.array([0, 1]), sampling=dict(u=[0.5]))
    assert eng.prefill([], []).shape == (0,)
    # the row still continues where it was: the next step gives what a fresh engine gives
    tok, pos = np.array([-1, 7, -1], np.int32), np.array([-1, 10, -1], np.int32)
    after = eng.step(tok, pos)[1]
    other = _engine(pkg, cfg, 2, tmp_path, 3, 16)
    assert (other.prefill([ok], [1]) == want).all() and other.step(tok, pos)[1] == after
    eng.close()
    other.close()


def test_create_refuses_fewer_tokens_than_rows(pkg):
    from gpt_oss_b200 import synth

    with pytest.raises(pkg.MoeError) as ei:
        pkg.DecodeEngine(synth.MINI_MODEL, 8, max_tokens=4)
    assert ei.value.code == pkg.GPTOSS_E_INVALID
    with pytest.raises(ValueError, match="local"):
        pkg.DecodeEngine(synth.MINI_MODEL, 8, ep_size=2, max_tokens=64)


def test_null_handles(pkg):
    lib = pkg.load_library()
    assert lib.gptoss_decode_prefill(None, None, None, None, None, 0, None, None, None) == pkg.GPTOSS_E_INVALID
    assert lib.gptoss_decode_step_sample(None, None, None, 1, None, None, None) == pkg.GPTOSS_E_INVALID


UNFINISHED = """
import ctypes, sys
sys.path[:0] = [{root!r}]
ctypes.CDLL({blas!r}, mode=ctypes.RTLD_GLOBAL)  # answers every cublasCreate with an error
import numpy as np
import __graft_entry__ as entry
pkg = entry.load_package()
from gpt_oss_b200 import synth
cfg = dict(synth.MINI_MODEL, vocab_size=901, n_layers=1)  # (logits of such rows go to cuBLAS)
eng = pkg.DecodeEngine(cfg, 2, max_tokens=16)
eng.load_bin(np.fromfile({model!r}, dtype=np.uint8))
cuda = ctypes.CDLL("libcuda.so.1")
big, size = ctypes.c_uint64(), 4 << 30
assert cuda.cuMemAlloc_v2(ctypes.byref(big), ctypes.c_size_t(size)) == 0
before = ctypes.c_void_p()
assert cuda.cuEventCreate(ctypes.byref(before), 0) == 0
step = {step!r}
for again in range(2):  # the second call builds no schedule, which would wait for the stream
    for i in range(40):
        assert cuda.cuMemsetD8Async(big, ctypes.c_ubyte(i), ctypes.c_size_t(size), None) == 0
    assert cuda.cuEventRecord(before, None) == 0  # what the call's copies have to wait for
    try:
        if step:
            eng.step([3, 4], [0, 0], sampling=dict(u=[0.5, 0.5]))
        else:
            eng.prefill([np.arange(10), np.arange(6)], [0, 1])
        raise SystemExit("the call did not fail")
    except pkg.MoeError as e:
        assert "cublasCreate" in str(e), e
    pending = cuda.cuEventQuery(before)
    assert cuda.cuCtxSynchronize() == 0
print("still to be read" if pending else "inputs read")
"""


@pytest.mark.gpu
@pytest.mark.parametrize("step", [False, True])
def test_a_failed_call_has_read_its_pinned_inputs(pkg, tmp_path, step):
    """A call that fails after its copies were queued waits for them: the next call writes the
    same pinned memory.  The failure is cuBLAS refusing to start (a stand-in library)."""
    import pathlib
    import subprocess
    import sys

    from gpt_oss_b200 import synth

    src, lib = tmp_path / "blas.c", tmp_path / "libcublas.so.12"
    src.write_text("int cublasCreate_v2(void **h) { (void)h; return 1; }\nint cublasDestroy_v2(void *h) { (void)h; return 0; }\n"
                   "int cublasSetStream_v2(void *h, void *s) { (void)h; (void)s; return 1; }\nint cublasGemmEx(void) { return 1; }\n")
    subprocess.run(["gcc", "-shared", "-fPIC", "-Wl,-soname,libcublas.so.12", "-o", str(lib), str(src)], check=True)
    model = tmp_path / "model.bin"
    synth.write_model_bin(model, dict(synth.MINI_MODEL, vocab_size=901, n_layers=1), 3)
    code = UNFINISHED.format(root=str(pathlib.Path(__file__).resolve().parents[1]), blas=str(lib),
                             model=str(model), step=step)
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "inputs read" in res.stdout, res.stdout + res.stderr


@pytest.mark.gpu
def test_a_reported_status_is_not_taken_for_a_token_id_alone(pkg, tmp_path):
    """The engine's kernels share a status word; the error's text names what its values mean."""
    from gpt_oss_b200 import synth

    cfg = dict(synth.MINI_MODEL, vocab_size=300, n_layers=1)
    eng = _engine(pkg, cfg, 2, tmp_path, 2, 16)
    want = eng.prefill([[5, 6]], [1])
    with pytest.raises(pkg.MoeError) as ei:
        eng.step([300, 5], [0, 0])
    text = str(ei.value)
    assert ei.value.code == pkg.GPTOSS_E_DEVICE and "status 104" in text
    assert "101-103" in text and "wait" in text and "token id" in text and "keys of a prompt" in text
    assert (eng.prefill([[5, 6]], [1]) == want).all()  # reported once
    eng.close()


@pytest.mark.gpu
@pytest.mark.parametrize("lens,max_tokens", [((600, 257, 1), 1000), ((600, 257, 1), 512), ((600, 257, 1), 300),
                                             ((256,), 513), ((257,), 513), ((513,), 513)], ids=str)
def test_passes_of_more_rows_than_a_tile(pkg, tmp_path, lens, max_tokens):
    """Passes of one to four row tiles in the projections, the schedule rebuilt between them and
    for the few rows of the logits, against the same prompts fed token by token."""
    import torch

    from gpt_oss_b200 import synth

    cfg = dict(synth.MINI_MODEL, vocab_size=900, sliding_window=200, n_layers=2, seq_len=700, n_attn_heads=6,
               n_kv_heads=2, n_experts=4, experts_per_token=4)
    rng = np.random.default_rng(17)
    prompts = [rng.integers(0, 900, n, dtype=np.int32) for n in lens]
    steps = _engine(pkg, cfg, 6, tmp_path, 4)
    logits = {}
    for p in range(max(lens)):  # all sequences side by side, sequence i in row i + 1
        tok, pos = np.full(4, -1, np.int32), np.full(4, -1, np.int32)
        for i, prompt in enumerate(prompts):
            if p < len(prompt):
                tok[i + 1], pos[i + 1] = prompt[p], p
        steps.step(tok, pos)
        for i, prompt in enumerate(prompts):
            if p == len(prompt) - 1:
                logits[i] = steps.logits(i + 1)
    eng = _engine(pkg, cfg, 6, tmp_path, 4, max_tokens)
    rows = list(range(1, len(lens) + 1))
    for _ in range(2):  # the second call meets the schedule that the first one left
        nxt = eng.prefill(prompts, rows)
        for i, want in logits.items():
            _close(eng.logits(i), want)
            assert want.max() - want[nxt[i]] <= 4 * LOGIT_MAX_ABS
    # Caches.  The two sides' projections may round the other way: a step of bf16, 2^-7 of the
    # element (1e-5 for sums near zero: 128 products of rows of norm 1 and weights of 0.02, at
    # 2^-24 each).  Rotation takes two of them to at most 2^-7 of the pair's length (Cauchy), and
    # both sides round once more, 2^-8 of the element each.
    dev, d, dkv = torch.device("cuda:0"), cfg["head_dim"], cfg["n_kv_heads"] * cfg["head_dim"]
    for layer in range(2):
        for row, n in zip(rows, lens):
            a = [torch.zeros(1, n, dkv, dtype=torch.bfloat16, device=dev) for _ in range(4)]
            steps.get_kv(layer, row, 0, a[0], a[1])
            eng.get_kv(layer, row, 0, a[2], a[3])
            k0, v0, k1, v1 = (x[0].float().reshape(n, -1, 2, d // 2) for x in a)
            if layer == 0:
                length = k0.pow(2).sum(2, keepdim=True).sqrt()
                assert ((k0 - k1).abs() <= length * 2.0 ** -6 + 2e-5).all()
                assert ((v0 - v1).abs() <= v0.abs() * 2.0 ** -7 + 1e-5).all()
            else:
                assert (k0 - k1).abs().max() <= 0.05 * k0.abs().max()
                assert (v0 - v1).abs().max() <= 0.05 * v0.abs().max()
    steps.close()
    eng.close()
