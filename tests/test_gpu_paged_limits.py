"""GPU: the paged-cache operators and paged sessions at the ends of what they hold."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_paged import (D, T, Pool, append64, half_step, queries, rope_table, run_decode, starts_of,  # noqa: E402
                            stream)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- rows behind the page table
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("rope", [True, False])
@pytest.mark.parametrize("over,new", [(1, 1), (1, 9), (40, 9), (40, 60), (1 << 20, 3)])
def test_append_leaves_out_rows_behind_the_table(pkg, dtype, layout, rope, over, new):
    """A sequence that has outgrown its page table by `over` positions: of its `new` newest rows
    those the table still holds go where they belong, the others nowhere (neither to an earlier
    position nor, where the table is padded with a valid id, to another sequence's page), and the
    first of them is recorded. The sequences beside it are served."""
    page, heads, hk = 16, 4, 2
    full = 3 * page
    pool = Pool(pkg, [full, 30, full], hk, page, dtype, layout, seed=over)
    tab = torch.tensor(pool.tab[:, :3], device="cuda")
    tab[1, 2] = tab[0, 0]  # padded with a valid id
    tab = tab.contiguous()
    lens = [full + over, full + over, full]
    q_lens = [new, 1, 1]
    starts = starts_of(q_lens)
    lens_dev = torch.tensor(lens, dtype=torch.int32, device="cuda")
    rows = sum(q_lens)
    qkv = torch.randn(rows, (heads + 2 * hk) * D, generator=torch.Generator("cuda").manual_seed(3), device="cuda")
    q = torch.full((rows, heads, D), 7.0, device="cuda", dtype=T[dtype])
    table = rope_table((1 << 20) + 64 if over > 40 else 256) if rope else None
    batch = pkg.PagedBatch(3, rows, lens_dev.data_ptr(), tab.data_ptr(), 3, q_starts=starts.data_ptr(),
                           err=pool.err.data_ptr())
    k0, v0 = pool.k.clone(), pool.v.clone()
    pkg.paged_append(pool.kv(), batch, qkv.data_ptr(), q.data_ptr(), heads, rope=table.data_ptr() if rope else 0,
                     rope_len=len(table) if rope else 0, stream=stream())
    torch.cuda.synchronize()
    pos = np.concatenate([np.arange(n - m, n) for m, n in zip(q_lens, lens)])
    inside = torch.tensor(pos < full, device="cuda")
    at = torch.tensor(np.minimum(pos, full - 1), device="cuda")
    wq, wk, wv, size = append64(qkv, heads, hk, at, table, None, None, 1e-6)
    u = half_step(dtype)
    near = lambda got, want, sz: ((got.double() - want).abs() <= u * want.abs() + 2.0 ** -20 * sz + 2.0 ** -25).all()  # noqa: E731
    assert (q[~inside] == 7.0).all()
    assert near(q[inside], wq[inside], size[inside][:, :heads])
    for r in torch.nonzero(inside).flatten().tolist():
        b = int(np.searchsorted(np.cumsum(q_lens), r, side="right"))
        pg, sl = int(pool.tab[b, pos[r] // page]), int(pos[r] % page)
        for c, c0, w in ((pool.k, k0, wk), (pool.v, v0, wv)):
            got = c[pg, :, sl] if layout == "hnd" else c[pg, sl]
            assert near(got, w[r], size[r, heads:] if c is pool.k else 0.0)
            got.copy_(c0[pg, :, sl] if layout == "hnd" else c0[pg, sl])  # (put back: the rest is untouched)
    for c, c0 in ((pool.k, k0), (pool.v, v0)):
        assert torch.equal(c.view(torch.int16), c0.view(torch.int16))
    err = pool.err.tolist()
    assert err[:2] == [3, 2] and err[2] in (0, 1) and err[3] in pos[pos >= full]


# ---------------------------------------------------------------- positions behind what an int holds
@pytest.fixture(scope="module")
def world(pkg, synth):
    ws = synth.WeightSet(synth.PRESETS["small"], seed=0, norm_jitter=0.1)
    return ws, pkg.Model(ws, device=0, mask_eos=True)


@pytest.mark.parametrize("paged", [False, True])
def test_positions_behind_the_limit_are_refused(pkg, synth, world, paged):
    """Positions whose sum with the steps or rows passes 2^30 or 31 bits: refused before any launch,
    the session's capacity as it was, and the session still of use."""
    ws, model = world
    pool = pkg.PagePool(model, 16, 16)
    make = (lambda: pool.session(32)) if paged else (lambda: model.session(256))
    s, t = make(), make()
    cap, free = s.capacity, pool.free_pages
    emb = synth.prompt_embeddings(ws, synth.audio_embeddings(ws.cfg, 30, seed=2))[:30]
    top = (1 << 31) - 1
    limit = "limit of 2\\^30"
    for pos in (1 << 30, top - 9, top - 1, top):
        for steps in (1, 8, 10, 200):
            with pytest.raises(pkg.QdbError, match=limit):
                s.decode_greedy(3, pos, steps)
            with pytest.raises(pkg.QdbError, match=limit):
                pkg.decode_greedy_batch([s, t], [3, 4], [pos, 0], steps)
            with pytest.raises(pkg.QdbError, match=limit):
                pkg.decode_sample_batch([t, s], [3, 4], [0, pos], np.full((steps, 2), 0.5))
        with pytest.raises(pkg.QdbError, match=limit):
            s.forward(emb[0], pos)
        with pytest.raises(pkg.QdbError, match=limit):
            pkg.forward_batch([s, t], emb[:2], [pos, 0])
        with pytest.raises(pkg.QdbError, match=limit):
            s.prefill(emb, pos)
        with pytest.raises(pkg.QdbError, match=limit):
            pkg.prefill_batch([t, s], [emb[:3], emb], [0, pos])
    with pytest.raises(pkg.QdbError, match=limit):
        s.decode_greedy(3, (1 << 30) - 4, 5)
    with pytest.raises(pkg.QdbError, match=limit):
        s.prefill(emb, (1 << 30) - 29)
    for n in ((1 << 30) + 1, top):
        assert pkg.lib.qdb_session_reserve(s.h, n) == -1
    assert (s.capacity, pool.free_pages) == (cap, free)
    s.prefill(emb, 0)
    assert s.forward(emb[3], 30)[0] >= 0


# ---------------------------------------------------------------- values that are not finite
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,n", [(4, 300), (32, 300), (4, 20)])
@pytest.mark.parametrize("scale", [0.0, 1e-3])
def test_decode_infinite_values(pkg, dtype, heads, n, scale):
    """An infinite V gives an infinite output of its sign to the heads that see it, NaN gives NaN,
    and the other dims and heads stay as they were (f16: a weight below its smallest value, 2^-32 of
    the largest, gives NaN)."""
    ws = pkg.PagedWorkspace()
    pool = Pool(pkg, [n, n], 2, 16, dtype, seed=n)
    q = queries(2, heads, dtype)
    clean = run_decode(pkg, ws, pool, q, scale=scale)
    inf = float("inf")
    for key, dim, x in ((0, 3, inf), (n - 1, 127, -inf), (n // 2, 9, float("nan"))):
        pg, sl = pool.where(0, n)
        pool.v[pg[key], 1, sl[key], dim] = x
    out = run_decode(pkg, ws, pool, q, scale=scale)
    g = heads // 2
    assert torch.equal(out[1], clean[1]) and torch.equal(out[0, :g], clean[0, :g])
    bad = out[0, g:]
    k = pool.get(0, n)[0][:, 1].double()
    p = torch.softmax((q[0, g:].double() @ k.T) * (scale or 128 ** -0.5), -1)
    least = (2.0 ** -31 if dtype == "f16" else 0.0) * p.max(-1)[0]
    for key, dim, x in ((0, 3, inf), (n - 1, 127, -inf)):
        assert ((bad[:, dim] == x) | (torch.isnan(bad[:, dim]) & (p[:, key] <= least))).all()
    assert torch.isnan(bad[:, 9]).all()
    rest = [d for d in range(128) if d not in (3, 9, 127)]
    assert torch.equal(bad[:, rest], clean[0, g:][:, rest])
