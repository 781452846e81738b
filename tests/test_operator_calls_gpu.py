"""How the handle-free operators may be called: from several host threads at once, after a
failed call of something else, and captured before they have ever run."""
import ctypes
import pathlib
import subprocess
import sys
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ROOT = pathlib.Path(__file__).resolve().parents[1]


def _at_once(jobs):
    """Runs the functions in a thread each, started together; returns what they raised."""
    start, raised = threading.Barrier(len(jobs)), []

    def run(job):
        try:
            start.wait(60)
            job()
        except Exception as e:  # noqa: BLE001
            raised.append(e)

    threads = [threading.Thread(target=run, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return raised


def _sample_args(pkg, logits, u, out, p):
    a = pkg.SampleArgs()
    a.logits, a.u, a.next, a.top_p = logits.data_ptr(), u.data_ptr(), out.data_ptr(), p.data_ptr()
    a.stride, a.n_rows, a.vocab, a.dtype = logits.stride(0), logits.shape[0], logits.shape[1], 2
    return a


def test_two_threads_two_vocabularies(pkg):
    """Rows of 201088 and of 50257 logits are cut over eight CTAs alike, so both threads launch
    one kernel with different amounts of shared memory."""
    import torch

    dev = torch.device("cuda:0")
    lib = pkg.load_library()
    sets = []
    for vocab in (201088, 50257):
        logits = torch.randn(4, vocab, device=dev) * 2
        u, p = torch.rand(4, device=dev), torch.full((4,), 0.9, device=dev)
        out, stream = torch.zeros(4, dtype=torch.int32, device=dev), torch.cuda.Stream()
        sets.append((_sample_args(pkg, logits, u, out, p), out, stream, (logits, u, p)))
    torch.cuda.synchronize()
    want = []
    for args, out, stream, _ in sets:
        assert lib.gptoss_decode_sample(ctypes.byref(args), stream.cuda_stream) == 0
        torch.cuda.synchronize()
        want.append(out.clone())
        out.fill_(-7)
    torch.cuda.synchronize()

    def job(args, stream):
        for _ in range(1500):
            rc = lib.gptoss_decode_sample(ctypes.byref(args), stream)
            if rc:
                raise pkg.MoeError(rc, lib.gptoss_decode_last_error(None).decode())

    raised = _at_once([lambda s=s: job(s[0], s[2].cuda_stream) for s in sets])
    torch.cuda.synchronize()
    assert not raised, raised[0]
    assert all(torch.equal(s[1], w) for s, w in zip(sets, want))


def test_all_operators_from_threads_of_their_own(pkg):
    """Each operator with two shapes at once, through the bindings; the results are those of
    calls one after the other."""
    import torch

    dev = torch.device("cuda:0")
    calls = []
    for hq, hkv, d, q_lens, kv_lens in ((16, 2, 64, [300, 1], [900, 5000]), (4, 4, 32, [1] * 5, [700] * 5)):
        q = torch.randn(sum(q_lens), hq, d, device=dev).bfloat16()
        k, v = (torch.randn(sum(kv_lens), hkv, d, device=dev).bfloat16() for _ in range(2))
        index = (torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32, device=dev),
                 torch.tensor(np.cumsum([0] + kv_lens[:-1]), dtype=torch.int64, device=dev),
                 torch.tensor(kv_lens, dtype=torch.int32, device=dev))
        calls.append((torch.zeros_like(q), lambda out, st, q=q, k=k, v=v, index=index: pkg.prompt_attention(
            q, k, v, *index, out, max_kv_len=5000, stream=st)))
        pos = torch.arange(q.shape[0], dtype=torch.int32, device=dev) + 7
        inv = torch.from_numpy(pkg.rope_table(d, 10000.0)[0]).to(dev)
        calls.append((torch.zeros_like(q), lambda out, st, q=q, pos=pos, inv=inv: pkg.rope_append(
            q, None, None, pos, inv, q_out=out, stream=st)))
        logits, u = torch.randn(sum(q_lens), 50 * d, device=dev), torch.rand(sum(q_lens), device=dev)
        calls.append((torch.zeros(sum(q_lens), dtype=torch.int32, device=dev),
                      lambda out, st, x=logits, u=u: pkg.sample_tokens(x, u, out, stream=st)))
    torch.cuda.synchronize()
    want = []
    for out, call in calls:
        call(out, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        want.append(out.clone())
        out.zero_()
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()

    def job(out, call, st):
        for _ in range(100):
            call(out, st)

    raised = _at_once([lambda c=c, s=s: job(*c, s.cuda_stream) for c, s in zip(calls, streams)])
    torch.cuda.synchronize()
    assert not raised, raised[0]
    assert all(torch.equal(c[0], w) for c, w in zip(calls, want))


def _small_calls(pkg):
    """name -> (output, function that fills it on a stream), with fixed inputs."""
    import torch

    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(5)
    q = torch.randn(40, 8, 64, generator=gen, device=dev).bfloat16()
    k, v = (torch.randn(90, 2, 64, generator=gen, device=dev).bfloat16() for _ in range(2))
    one = torch.tensor([0], dtype=torch.int64, device=dev)
    length = torch.tensor([90], dtype=torch.int32, device=dev)
    pos = torch.arange(40, dtype=torch.int32, device=dev)
    inv = torch.from_numpy(pkg.rope_table(64, 10000.0)[0]).to(dev)
    logits, u = torch.randn(6, 900, generator=gen, device=dev), torch.rand(6, generator=gen, device=dev)

    def attend(n):
        start = torch.tensor([0, n], dtype=torch.int32, device=dev)
        return torch.zeros_like(q[:n]), lambda out, st: pkg.prompt_attention(q[:n], k, v, start, one, length, out,
                                                                             stream=st)

    return {"prompt": attend(40), "token": attend(1),
            "rope": (torch.zeros_like(q), lambda out, st: pkg.rope_append(q, None, None, pos, inv, q_out=out, stream=st)),
            "sample": (torch.zeros(6, dtype=torch.int32, device=dev),
                       lambda out, st: pkg.sample_tokens(logits, u, out, stream=st))}


def _failed_create(pkg):
    """An engine whose cache no GPU holds: its allocation is refused."""
    from gpt_oss_b200 import synth

    with pytest.raises(pkg.MoeError) as ei:
        pkg.DecodeEngine(dict(synth.MINI_MODEL, seq_len=1 << 30), 64)
    assert ei.value.code == pkg.GPTOSS_E_CUDA and "allocation" in str(ei.value)


@pytest.mark.parametrize("which", ["prompt", "token", "rope", "sample"])
def test_an_earlier_failure_is_not_the_operators(pkg, which):
    """An error that another call left on the thread does not make a launched operator fail."""
    import torch

    out, call = _small_calls(pkg)[which]
    st = torch.cuda.current_stream().cuda_stream
    call(out, st)
    torch.cuda.synchronize()
    want = out.clone()
    out.zero_()
    _failed_create(pkg)
    call(out, st)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("kind", ["decode", "moe"])
def test_an_engine_outlives_the_failed_creation_of_another(pkg, tmp_path, kind):
    """The creation that fails leaves no error behind for the calls of an engine that is there."""
    from gpt_oss_b200 import synth

    cfg = dict(synth.MINI_MODEL, vocab_size=300, n_layers=1)
    synth.write_model_bin(tmp_path / "m.bin", cfg, 1)
    eng = pkg.DecodeEngine(cfg, 2)
    eng.load_bin(np.fromfile(tmp_path / "m.bin", dtype=np.uint8))
    want = eng.step([5, 7], [0, 0])
    if kind == "decode":
        _failed_create(pkg)
    else:
        with pytest.raises(pkg.MoeError) as ei:
            pkg.MoeEngine(1 << 16, 128, 8, 4, max_tokens=1 << 24)  # rows of 9 TB
        assert ei.value.code == pkg.GPTOSS_E_CUDA
    assert (eng.step([5, 7], [0, 0]) == want).all()
    eng.close()


FIRST_CALL = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import torch
import __graft_entry__ as entry
import test_operator_calls_gpu as calls
out, call = calls._small_calls(entry.load_package())[{which!r}]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    call(out, torch.cuda.current_stream().cuda_stream)
graph.replay()
torch.cuda.synchronize()
got = out.clone()
out.zero_()
call(out, torch.cuda.current_stream().cuda_stream)
torch.cuda.synchronize()
assert out.any() and torch.equal(got, out)
print("captured")
"""


@pytest.mark.parametrize("which", ["prompt", "token", "rope", "sample"])
def test_the_first_call_may_be_a_captured_one(which):
    """In a process of its own, so that nothing of the operator has been loaded before."""
    code = FIRST_CALL.format(root=str(ROOT), tests=str(ROOT / "tests"), which=which)
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "captured" in res.stdout, res.stdout + res.stderr
