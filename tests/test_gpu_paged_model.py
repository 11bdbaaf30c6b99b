"""GPU: paged sessions and sampled decoding through the model API: against the CPU
oracle and the contiguous sessions, in every call that takes them."""
import numpy as np
import pytest

from conftest import MARGIN, MAX_ABS, assert_logits_close
from oracle.pyoracle import Oracle, margin_top2
from test_gpu_sample import sample64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def world(pkg, synth):
    cfg = synth.PRESETS["small"]
    ws = synth.WeightSet(cfg, seed=0, norm_jitter=0.1)
    return ws, pkg.Model(ws, device=0, mask_eos=True)


def prompts(synth, ws, lens, seed=3):
    return [synth.prompt_embeddings(ws, synth.audio_embeddings(ws.cfg, n, seed=seed + n))[:n] for n in lens]


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_paged_session_matches_oracle(pkg, synth, world, page):
    """Prefill in chunks, steps, and a rewind, teacher-forced on the oracle."""
    ws, model = world
    pool = pkg.PagePool(model, 4096 // page, page)
    s = pool.session()
    emb = prompts(synth, ws, [150])[0]
    orc = Oracle(ws, max_pos=256)
    s.prefill(emb[:37], 0)
    s.prefill(emb[37:129], 37)
    orc.prefill(emb[:129])
    pos, e = 129, emb[129]
    for _ in range(8):
        tok, hid, log = s.forward(e, pos, want_hidden=True, want_logits=True)
        otok, ohid, olog = orc.forward(e)
        assert_logits_close(log, olog, f"pos {pos}")
        assert np.abs(hid - ohid).max() <= 2e-2
        assert tok == otok or margin_top2(olog) <= MARGIN
        e = synth.embed_rows(ws, [otok])[0]
        pos += 1
    # rewind to 100 and go on with other rows: what was cached behind counts no more
    s.prefill(emb[100:120], 100)
    orc.kv_cache_len = 100
    orc.prefill(emb[100:120])
    tok, _, log = s.forward(emb[120], 120, want_logits=True)
    otok, _, olog = orc.forward(emb[120])
    assert_logits_close(log, olog, "after the rewind")


def test_paged_batches_match_contiguous(pkg, synth, world):
    ws, model = world
    lens = [3, 70, 16, 129, 1, 33]
    pool = pkg.PagePool(model, 200, 16)
    a = [pool.session() for _ in lens]
    b = [model.session(512) for _ in lens]
    pr = prompts(synth, ws, lens)
    pkg.prefill_batch(a, pr, [0] * len(lens))
    pkg.prefill_batch(b, pr, [0] * len(lens))
    e = np.stack([p[-1] for p in pr])
    ta, la = pkg.forward_batch(a, e, lens, want_logits=True)
    tb, lb = pkg.forward_batch(b, e, lens, want_logits=True)
    for i in range(len(lens)):
        assert_logits_close(la[i], lb[i], f"row {i}")
        assert ta[i] == tb[i] or margin_top2(lb[i]) <= MARGIN
    # the captured step replayed with other sessions and positions
    for k in range(1, 4):
        order = np.roll(np.arange(len(lens)), k)
        sa, sb = [a[i] for i in order], [b[i] for i in order]
        pos = [lens[i] + 1 + (k - 1) for i in order]
        _, la = pkg.forward_batch(sa, e, pos, want_logits=True)
        _, lb = pkg.forward_batch(sb, e, pos, want_logits=True)
        for i in range(len(lens)):
            assert_logits_close(la[i], lb[i], f"turn {k} row {i}")
    first = [5, 6, 7, 8, 9, 10]
    ga = pkg.decode_greedy_batch(a, first, lens, 20)
    gb = pkg.decode_greedy_batch(b, first, lens, 20)
    # a near tie may send a row another way: from there on it is no longer comparable
    same = (ga == gb).all(0)
    for i in np.flatnonzero(~same):
        k = int(np.flatnonzero(ga[:, i] != gb[:, i])[0])
        toks = [first[i]] + list(gb[:k, i])
        b[i].prefill(np.stack([synth.embed_rows(ws, [t])[0] for t in toks[:-1]]) if k else np.zeros((0, ws.cfg.hidden)), lens[i])
        _, _, log = b[i].forward(synth.embed_rows(ws, [toks[-1]])[0], lens[i] + k, want_logits=True)
        assert margin_top2(log) <= MARGIN, (i, k)
    assert same.sum() >= len(lens) - 2


def test_paged_greedy_single_equals_batch_of_one(pkg, synth, world):
    ws, model = world
    pool = pkg.PagePool(model, 40, 16)
    s, t = pool.session(), pool.session()
    emb = prompts(synth, ws, [40])[0]
    for x in (s, t):
        x.prefill(emb, 0)
    assert list(s.decode_greedy(11, 40, 9)) == list(pkg.decode_greedy_batch([t], [11], [40], 9)[:, 0])


def test_many_rows_take_the_wide_path(pkg, synth, world):
    """More than 64 rows in one step."""
    ws, model = world
    n = 70
    pool = pkg.PagePool(model, 300, 32)
    ss = [pool.session() for _ in range(n)]
    pr = prompts(synth, ws, [5 + i % 40 for i in range(n)])
    pkg.prefill_batch(ss, pr, [0] * n)
    e = np.stack([p[-1] for p in pr])
    pos = [len(p) for p in pr]
    _, la = pkg.forward_batch(ss, e, pos, want_logits=True)
    one = model.session(256)
    for i in (0, 33, 69):
        one.prefill(pr[i], 0)
        _, _, log = one.forward(e[i], pos[i], want_logits=True)
        assert_logits_close(la[i], log, f"row {i}")


def test_pool_accounting(pkg, synth, world):
    ws, model = world
    pool = pkg.PagePool(model, 10, 16)
    a = pool.session(33)
    assert pool.free_pages == 7 and a.capacity == 48
    b = pool.session()
    assert pool.free_pages == 7 and b.capacity == 0
    emb = prompts(synth, ws, [150])[0]
    with pytest.raises(pkg.QdbError, match="page pool exhausted"):
        b.prefill(emb, 0)
    assert pool.free_pages == 7 and b.capacity == 0
    # a batch that does not fit leaves every session as it was
    c = pool.session()
    with pytest.raises(pkg.QdbError, match="page pool exhausted"):
        pkg.prefill_batch([a, b, c], [emb[:40], emb[:60], emb[:70]], [0, 0, 0])
    assert pool.free_pages == 7 and (a.capacity, b.capacity, c.capacity) == (48, 0, 0)
    with pytest.raises(pkg.QdbError, match="page pool exhausted"):
        pkg.decode_greedy_batch([a, b], [1, 2], [40, 100], 50)
    assert pool.free_pages == 7 and b.capacity == 0
    with pytest.raises(pkg.QdbError, match="page pool exhausted"):
        pool.session(200)
    b.prefill(emb[:100], 0)
    assert pool.free_pages == 0
    b.close()
    assert pool.free_pages == 7
    c.prefill(emb[:112], 0)  # pages that another session has used
    orc = Oracle(ws, max_pos=256)
    orc.prefill(emb[:112])
    _, _, olog = orc.forward(emb[112])
    a.close()
    _, _, log = c.forward(emb[112], 112, want_logits=True)
    assert_logits_close(log, olog, "reused pages")


def test_pool_refusals_and_lifetimes(pkg, synth, world):
    ws, model = world
    for n, page, match in ((0, 16, "pages"), (4, 24, "page size"), (4, 0, "page size"), (-1, 32, "pages"),
                           (1 << 28, 256, "pages")):
        with pytest.raises(pkg.QdbError, match=match):
            pkg.PagePool(model, n, page)
    emb = prompts(synth, ws, [20])[0]
    pool, other = pkg.PagePool(model, 8, 16), pkg.PagePool(model, 8, 16)
    a, b, c = pool.session(), other.session(), model.session(64)
    for mix in ([a, b], [a, c], [c, a]):
        with pytest.raises(pkg.QdbError, match="one page pool"):
            pkg.prefill_batch(mix, [emb, emb], [0, 0])
        with pytest.raises(pkg.QdbError, match="one page pool"):
            pkg.forward_batch(mix, np.stack([emb[0], emb[0]]), [0, 0])
    a.prefill(emb, 0)
    with pytest.raises(pkg.QdbError, match="paged"):
        a.trace_step(1, 20)
    with pytest.raises(pkg.QdbError, match="paged"):
        pkg.trace_batch_step([a], emb[:1], [20])
    assert pkg.lib.qdb_forward_noalloc(a.h, 256, 20, 256) == -1 and b"paged" in pkg.lib.qdb_last_error()
    pool.close()
    with pytest.raises(pkg.QdbError, match="freed"):
        a.forward(emb[0], 20)
    a.close()
    b.prefill(emb, 0)
    m2 = pkg.Model(ws, device=0)
    p2 = pkg.PagePool(m2, 4, 16)
    d = p2.session(16)
    m2.close()
    with pytest.raises(pkg.QdbError, match="freed"):
        d.forward(emb[0], 0)
    assert p2.free_pages == 0
    with pytest.raises(pkg.QdbError, match="freed"):
        p2.session()
    d.close()
    p2.close()


def test_pool_in_a_freed_ones_place(pkg, synth, world):
    """A captured step must not outlive its pool, though a new pool of another
    page size may get the same memory."""
    ws, model = world
    emb = prompts(synth, ws, [70])[0]
    one = model.session(128)
    one.prefill(emb, 0)
    _, _, want = one.forward(emb[3], 70, want_logits=True)
    for page in (16, 64, 32, 128, 16):
        pool = pkg.PagePool(model, 1024 // page, page)
        s = [pool.session(), pool.session()]
        pkg.prefill_batch(s, [emb[:40], emb], [0, 0])
        for _ in range(3):  # (the second call captures, the third replays)
            _, log = pkg.forward_batch(s, emb[[40, 3]], [40, 70], want_logits=True)
            assert_logits_close(log[1], want, f"page {page}")
        for x in s:
            x.close()
        pool.close()


def test_sessions_without_rows_in_a_prefill(pkg, synth, world):
    """No rows from any position: nothing happens to that session."""
    ws, model = world
    emb = prompts(synth, ws, [40])[0]
    pool = pkg.PagePool(model, 16, 16)
    a, b, c = pool.session(), pool.session(), pool.session()
    pkg.prefill_batch([a, b, c], [emb[:0], emb, emb[:0]], [500, 0, 7])
    assert (a.capacity, b.capacity, c.capacity) == (0, 48, 0)
    one = model.session(64)
    one.prefill(emb, 0)
    _, _, want = one.forward(emb[3], 40, want_logits=True)
    _, _, log = b.forward(emb[3], 40, want_logits=True)
    assert_logits_close(log, want, "beside sessions without rows")


def test_one_session_in_several_rows(pkg, synth, world):
    """Two pieces of one session in one prefill, two of its positions in one step."""
    ws, model = world
    emb = prompts(synth, ws, [60])[0]
    pool = pkg.PagePool(model, 16, 16)
    s, one = pool.session(), model.session(64)
    pkg.prefill_batch([s, s], [emb[:25], emb[25:50]], [0, 25])
    one.prefill(emb[:50], 0)
    _, log = pkg.forward_batch([s, s], emb[50:52], [50, 51], want_logits=True)
    for i in range(2):
        _, _, want = one.forward(emb[50 + i], 50 + i, want_logits=True)
        assert_logits_close(log[i], want, f"row {i}")


def test_injected_failures_leave_paged_calls_usable(pkg, synth, world, monkeypatch):
    ws, model = world
    pool = pkg.PagePool(model, 16, 16)
    s = pool.session()
    emb = prompts(synth, ws, [20])[0]
    monkeypatch.setenv("QWEN_ASR_B200_FAULT", "launch")
    with pytest.raises(pkg.QdbError, match="injected"):
        s.prefill(emb, 0)
    monkeypatch.setenv("QWEN_ASR_B200_FAULT", "alloc")
    with pytest.raises(pkg.QdbError, match="injected"):
        pkg.PagePool(model, 4, 16)
    monkeypatch.delenv("QWEN_ASR_B200_FAULT")
    s.prefill(emb, 0)
    assert s.forward(emb[0], 20)[0] >= 0


# ---------------------------------------------------------------- sampled decoding
@pytest.mark.parametrize("paged", [False, True])
def test_sampled_loop_draws_from_the_step_logits(pkg, synth, world, paged):
    """Each drawn token against the definition's draw from the logits of the same
    step run by itself.

    Both runs' logits are within MAX_ABS of the reference's (the parity bar), so
    they differ by at most d = 2 MAX_ABS, and every weight by a factor of at most
    e^(d / T). A running sum F of normalised weights then moves by at most
    F (1 - F) (e^(2 d / T) - 1) <= (e^(2 d / T) - 1) / 4, and the mass that top_p
    keeps by as much again, which moves F by at most that over top_p. So the token
    lies, in index order, between the definition's draws at uniform -+ the sum of
    the two. Rows with a token within 2 d of a border of top_k or min_p, whose
    place in the set is open, are left out."""
    ws, model = world
    lens = [20, 33, 7, 50]
    n = len(lens)
    pool = pkg.PagePool(model, 100, 16)
    make = (lambda: pool.session()) if paged else (lambda: model.session(256))
    a, b = [make() for _ in lens], [make() for _ in lens]
    pr = prompts(synth, ws, lens)
    for ss in (a, b):
        pkg.prefill_batch(ss, pr, [0] * n)
    steps = 12
    rng = np.random.default_rng(4)
    u = rng.random((steps, n)).astype(np.float32)
    kw = dict(temperature=[0.7, 1.0, 0.0, 1.5], top_k=[40, 0, 0, 7], top_p=[0.95, 0.9, 1.0, 1.0], min_p=[0, 0, 0, 0.05])
    first = np.array([3, 4, 5, 6], np.int32)
    got = pkg.decode_sample_batch(a, first, lens, u, **kw)
    assert got.shape == (steps, n)
    temp, top_p, min_p = [np.float64(np.asarray(kw[k], np.float32)) for k in ("temperature", "top_p", "min_p")]
    d = 2 * MAX_ABS
    tok, checked = first, 0
    for s in range(steps):
        e = np.stack([synth.embed_rows(ws, [t])[0] for t in tok])
        _, log = pkg.forward_batch(b, e, [p + s for p in lens], want_logits=True)
        for i in range(n):
            x = log[i].astype(np.float64)
            for eos in (151643, 151645):
                if eos < len(x):
                    x[eos] = -np.inf
            if temp[i] == 0:
                if margin_top2(log[i]) > 2 * d:
                    checked += 1
                    assert got[s, i] == int(x.argmax()), (s, i)
                continue
            order = np.sort(x)[::-1]
            k = kw["top_k"][i]
            if k and order[k - 1] - order[k] <= 2 * d:
                continue
            if min_p[i] > 0 and (np.abs(x - x.max() - temp[i] * np.log(min_p[i])) <= 2 * d).any():
                continue
            move = (np.exp(2 * d / temp[i]) - 1) / 4
            move += move / top_p[i] if top_p[i] < 1 else 0
            lo, hi = [sample64(x, temp[i], k, top_p[i], min_p[i], v)
                      for v in (max(u[s, i] - move, 0.0), min(u[s, i] + move, 1 - 1e-9))]
            checked += 1
            assert lo <= got[s, i] <= hi, (s, i, lo, got[s, i], hi)
        tok = got[s]
    assert checked >= 12  # (at least the rows without top_k and min_p)


def test_sampled_loop_greedy_and_repeatable(pkg, synth, world):
    ws, model = world
    emb = prompts(synth, ws, [30])[0]
    u = np.random.default_rng(0).random((10, 1))
    outs = []
    for _ in range(2):
        s = model.session(128)
        s.prefill(emb, 0)
        outs.append(pkg.decode_sample_batch([s], [3], [30], u, temperature=0.0)[:, 0].tolist())
    s = model.session(128)
    s.prefill(emb, 0)
    assert outs[0] == outs[1] == pkg.decode_greedy_batch([s], [3], [30], 10)[:, 0].tolist()
    assert pkg.decode_sample_batch([s], [3], [30], np.zeros((0, 1))).shape == (0, 1)


def test_sampled_loop_refusals(pkg, synth, world):
    ws, model = world
    s = model.session(64)
    f = np.zeros(1, np.int32)
    out = np.zeros(4, np.int32)
    import ctypes
    i32 = ctypes.POINTER(ctypes.c_int)
    args = (f.ctypes.data_as(i32), f.ctypes.data_as(i32), 2)
    h = (ctypes.c_void_p * 1)(s.h)
    assert pkg.lib.qdb_decode_sample_batch(h, 1, *args, None, out.ctypes.data_as(i32)) == -1
    assert pkg.lib.qdb_decode_sample_batch(h, 1, *args, pkg.QdbSampling(), out.ctypes.data_as(i32)) == -1
    assert b"random numbers" in pkg.lib.qdb_last_error()
    with pytest.raises(pkg.QdbError, match="out of range"):
        pkg.decode_sample_batch([s], [-1], [0], [[0.5]])
    with pytest.raises(pkg.QdbError, match="negative position"):
        pkg.decode_sample_batch([s], [1], [-1], [[0.5]])
