"""GPU: sampling calls of different sizes beside each other, and rows at the ends of its lists."""
import threading

import pytest

torch = pytest.importorskip("torch")

from test_gpu_sample import logits, want  # noqa: E402

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
