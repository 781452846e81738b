"""How the handle-free operators may be called: from several host threads at once."""
import ctypes
import threading

import pytest

pytestmark = pytest.mark.gpu


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
