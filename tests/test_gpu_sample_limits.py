"""GPU: sampling calls of different sizes beside each other, and rows at the ends of its lists."""
import threading

import pytest

torch = pytest.importorskip("torch")

from test_gpu_sample import logits, run, want  # noqa: E402

pytestmark = pytest.mark.gpu


def test_threads_with_different_vocabularies(pkg):
    """Calls from host threads, each with a stream and a vocabulary of its own: none is refused
    because another's needs less shared memory, and each draws its own tokens."""
    vocabs = (262144, 512, 200000, 513, 600, 1000)
    calls, out, failed = 6000, {}, []
    gate = threading.Barrier(len(vocabs))

    def work(vocab):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                x = logits(1, vocab, seed=vocab)
                u = torch.tensor([0.37], device="cuda")
                k = torch.tensor([40], dtype=torch.int32, device="cuda")
                tok = torch.full((1,), -9, dtype=torch.int32, device="cuda")
            st.synchronize()
            args = dict(logits=x.data_ptr(), rows=1, vocab=vocab, uniform=u.data_ptr(), tokens=tok.data_ptr(),
                        top_k=k.data_ptr(), stream=st.cuda_stream)
            gate.wait(60)
            for _ in range(calls):
                pkg.sample(**args)
            st.synchronize()
            out[vocab] = (tok.tolist(), want(x, [0.37], k=[40]))
        except Exception as e:  # noqa: BLE001 (reported by the test's thread)
            failed.append(f"{vocab}: {e}")

    threads = [threading.Thread(target=work, args=(v,)) for v in vocabs]
    for t in threads:
        t.start()
    for t in threads:
        t.join(300)
    assert not failed
    for got, ref in out.values():
        assert got == ref


@pytest.mark.parametrize("vocab", [16000, 60000, 151936])
@pytest.mark.parametrize("allowed", [2049, 5000, 10000])
@pytest.mark.parametrize("mask", [-1e9, -1e4, float("-inf")])
def test_top_k_above_the_tokens_that_weigh(pkg, vocab, allowed, mask):
    """Thousands of tokens allowed, the rest masked with finite values far below, top_k between
    the allowed ones and the vocabulary: all allowed tokens stay."""
    rows = 8
    x = torch.full((rows, vocab), mask, device="cuda")
    at = torch.randperm(vocab, generator=torch.Generator("cuda").manual_seed(allowed), device="cuda")[:allowed]
    x[:, at] = logits(rows, allowed, seed=vocab, spread=1.0)
    u = [0.0, 0.1, 0.3, 0.5, 0.7, 0.9, 0.99, 0.9999]
    for k in (allowed - 1, allowed, allowed + 1, (allowed + vocab) // 2, vocab - 1):
        for kw in (dict(), dict(p=[0.9] * rows), dict(floor=[0.05] * rows), dict(p=[0.7] * rows, temp=[0.6] * rows)):
            kw = dict(kw, k=[k] * rows)
            assert run(pkg, x, u, **kw) == want(x, u, **kw), (k, kw)
