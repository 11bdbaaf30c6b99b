"""GPU: waits of the paged kernels that run out.

With the limit at 0 cycles a wait gives up at its first unsuccessful check: the kernel records it
in the error words, lets its own copies land and returns. (Short histories may find every tile
there already; their output is right then.) With the limit restored the next call is right.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_paged import Pool, check_attention, queries, run_decode, run_prompt  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def world(pkg, synth):
    ws = synth.WeightSet(synth.PRESETS["tiny"], seed=12, norm_jitter=0.1)
    return ws, synth.audio_embeddings(ws.cfg, 40, seed=4), pkg.Model(ws, device=0, mask_eos=True)


class limit:
    """The data waits' limit, in cycles, inside a with block."""

    def __init__(self, model, cycles):
        self.model, self.cycles = model, cycles

    def __enter__(self):
        torch.cuda.synchronize()
        self.model.set_wait_limit(self.cycles)

    def __exit__(self, *_):
        torch.cuda.synchronize()
        self.model.set_wait_limit(-1)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,lens", [(4, [404]), (16, [700, 0, 33, 5000]), (32, [20000, 17] + [300] * 40)])
def test_decode_wait_runs_out(pkg, world, dtype, heads, lens):
    model = world[2]
    pool = Pool(pkg, lens, 2, 16, dtype, seed=heads)
    q = queries(len(lens), heads, dtype)
    for _ in range(3):
        with limit(model, 0):
            out = run_decode(pkg, pkg.PagedWorkspace(), pool, q)
        if pool.err.tolist()[0] == 0 and sum(lens) < 10000:  # (no more than a tile or two per warp)
            check_attention(pool, q, out, [1] * len(lens))
        else:
            assert pool.err.tolist()[0] == 1
        pool.err.zero_()
        check_attention(pool, q, run_decode(pkg, pkg.PagedWorkspace(), pool, q), [1] * len(lens))


def test_paged_session_recovers(pkg, world):
    """Through the model: the step fails with the wait named, and the next one is right (the joins'
    counters start again from zero)."""
    ws, emb, model = world
    pool = pkg.PagePool(model, 64, 16)
    a, b, one = pool.session(400), pool.session(), model.session(64)
    for s in (a, b, one):
        s.prefill(emb[:20], 0)
    x = np.stack([emb[20]] * 2)
    _, want = pkg.forward_batch([one, one], x, [20, 20], want_logits=True)
    for _ in range(3):
        with limit(model, 0):
            with pytest.raises(pkg.QdbError, match="bounded wait"):
                pkg.forward_batch([a, b], x, [20, 20])
            with pytest.raises(pkg.QdbError, match="bounded wait"):
                pkg.decode_greedy_batch([a, b], [3, 4], [20, 20], 6)
        _, got = pkg.forward_batch([a, b], x, [20, 20], want_logits=True)
        assert np.abs(got - want).max() <= 2e-2


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,lens,q_lens", [
    (4, 2, [1], [1]), (16, 8, [404], [404]), (4, 4, [900, 0, 3000], [900, 0, 5]), (16, 1, [300] * 40, [70] * 40),
    (8, 4, [40] * 300, [13] * 300), (16, 8, [9000, 4000], [3000, 4000])], ids=str)
def test_prompt_wait_runs_out(pkg, world, dtype, heads, kv_heads, lens, q_lens):
    model = world[2]
    pool = Pool(pkg, lens, kv_heads, 32, dtype, seed=heads)
    q = queries(sum(q_lens), heads, dtype)
    for _ in range(3):
        with limit(model, 0):
            run_prompt(pkg, pool, q, q_lens)
        assert pool.err.tolist()[0] == 1
        pool.err.zero_()
        check_attention(pool, q, run_prompt(pkg, pool, q, q_lens), q_lens)


@pytest.mark.parametrize("cycles", [1, 300, 1000, 3000, 10000, 30000])
def test_prompt_gives_up_anywhere(pkg, world, cycles):
    """Limits between the shortest and the longest wait: roles give up at different places, some
    after their last copy; either the error is recorded or the output is right."""
    model = world[2]
    lens, q_lens = [700, 1, 90, 4000, 129], [700, 1, 33, 300, 129]
    pool = Pool(pkg, lens, 2, 16, "bf16", seed=cycles)
    q = queries(sum(q_lens), 8, "bf16")
    for _ in range(5):
        with limit(model, cycles):
            out = run_prompt(pkg, pool, q, q_lens)
        if pool.err.tolist()[0] == 0:
            check_attention(pool, q, out, q_lens)
        else:
            assert pool.err.tolist()[0] == 1
        pool.err.zero_()
        check_attention(pool, q, run_prompt(pkg, pool, q, q_lens), q_lens)


def test_paged_prefill_recovers(pkg, world):
    ws, emb, model = world
    pool = pkg.PagePool(model, 64, 16)
    a, one = pool.session(), model.session(64)
    one.prefill(emb[:30], 0)
    _, _, want = one.forward(emb[30], 30, want_logits=True)
    for _ in range(3):
        with limit(model, 0):
            with pytest.raises(pkg.QdbError, match="bounded wait"):
                a.prefill(emb[:30], 0)
        a.prefill(emb[:30], 0)
        _, _, got = a.forward(emb[30], 30, want_logits=True)
        assert np.abs(got - want).max() <= 2e-2


def test_failed_steps_followed_at_once(pkg, world):
    """The error words and the joins' counters are cleared ahead of the call that follows."""
    ws, emb, model = world
    pool = pkg.PagePool(model, 128, 16)
    a, one = pool.session(1500), model.session(64)
    for s in (a, one):
        s.prefill(emb[:20], 0)
    _, _, want = one.forward(emb[20], 20, want_logits=True)
    for _ in range(100):
        model.set_wait_limit(0)
        try:
            with pytest.raises(pkg.QdbError, match="bounded wait"):
                a.forward(emb[20], 1200)
        finally:
            model.set_wait_limit(-1)
        _, _, got = a.forward(emb[20], 20, want_logits=True)
        assert np.abs(got - want).max() <= 2e-2


def test_error_names_the_row_kernels(pkg, world):
    """The words are shared by the GEMMs and the attention kernels: the message does not single one out."""
    ws, emb, model = world
    s = pkg.PagePool(model, 64, 16).session()
    with limit(model, 0):
        with pytest.raises(pkg.QdbError, match=r"in the row kernels \(a bounded wait ran out\)"):
            s.prefill(emb[:30], 0)
