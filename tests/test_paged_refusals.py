"""CPU: the paged-cache operators and sampling refuse bad arguments before any launch."""
import ctypes

import pytest

from conftest import has_gpu

P = 1 << 20  # an aligned, never dereferenced address


def kv(pkg, **o):
    a = dict(k=P, v=P, n_pages=8, page_size=16, kv_heads=2, dtype="f16")
    a.update(o)
    return pkg.PagedKV(**a)


def batch(pkg, **o):
    a = dict(n_seqs=3, rows=3, kv_lens=P, tables=P, table_stride=4)
    a.update(o)
    return pkg.PagedBatch(**a)


KV_BAD = [
    (dict(k=0), "null cache"), (dict(v=None), "null cache"), (dict(k=P + 8), "16-byte"), (dict(v=P + 2), "16-byte"),
    (dict(dtype="f32"), "cache type"), (dict(n_pages=0), "pool"), (dict(n_pages=-4), "pool"),
    (dict(page_size=8), "page size"), (dict(page_size=24), "page size"), (dict(page_size=512), "page size"),
    (dict(page_size=0), "page size"), (dict(strides=(4096, 2048, 64)), "stride"),
    (dict(strides=(4096, 2048, 132)), "stride"), (dict(strides=(-4096, 2048, 128)), "stride"),
    (dict(strides=(1 << 40, 2048, 128)), "stride"),
]
BATCH_BAD = [
    (dict(n_seqs=-1), "negative"), (dict(rows=-1), "negative"), (dict(rows=(1 << 22) + 1), "rows"),
    (dict(n_seqs=(1 << 20) + 1, rows=(1 << 20) + 1), "sequences"), (dict(kv_lens=0), "null"),
    (dict(tables=0), "null"), (dict(table_stride=0), "page tables"), (dict(rows=4), "q_starts"),
]


def ops(pkg):
    ws = type("W", (), {"h": 1})()

    def append(k, b, heads=4, q=P, o=P, **x):
        pkg.paged_append(k, b, q, o, heads, **x)

    def decode(k, b, heads=4, q=P, o=P, **x):
        pkg.paged_decode(k, b, q, o, heads, ws, **x)

    def prompt(k, b, heads=4, q=P, o=P, **x):
        pkg.paged_prompt(k, b, q, o, heads, **x)

    return append, decode, prompt


@pytest.mark.parametrize("change,match", KV_BAD)
def test_bad_cache(pkg, change, match):
    for op in ops(pkg):
        with pytest.raises(pkg.QdbError, match=match):
            op(kv(pkg, **change), batch(pkg))


@pytest.mark.parametrize("change,match", BATCH_BAD)
def test_bad_batch(pkg, change, match):
    for op in ops(pkg):
        with pytest.raises(pkg.QdbError, match=match):
            op(kv(pkg), batch(pkg, **change))


@pytest.mark.parametrize("heads", [0, -4, 3, 34, 64])
def test_bad_heads(pkg, heads):
    for op in ops(pkg):
        with pytest.raises(pkg.QdbError, match="heads"):
            op(kv(pkg), batch(pkg), heads=heads)


def test_bad_rows(pkg):
    append, decode, prompt = ops(pkg)
    for op in (decode, prompt):
        for x, match in ((dict(q=0), "null"), (dict(o=0), "null"), (dict(q=P + 8), "16-byte"), (dict(o=P + 8), "16-byte"),
                         (dict(q_stride=511), "stride"), (dict(q_stride=516), "stride"), (dict(out_stride=-512), "stride"),
                         (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
                         (dict(scale=float("inf")), "scale")):
            with pytest.raises(pkg.QdbError, match=match):
                op(kv(pkg), batch(pkg), **x)
    for x, match in ((dict(q=0), "null"), (dict(o=0), "null"), (dict(q=P + 4), "16-byte"), (dict(row_stride=1023), "stride"),
                     (dict(row_stride=1026), "stride"), (dict(q_stride=500), "stride"), (dict(q_norm=P + 4), "16-byte"),
                     (dict(rope=P, rope_len=0), "rotation"), (dict(rope=P + 8, rope_len=9), "16-byte"),
                     (dict(dtype="int8"), "type")):
        with pytest.raises(pkg.QdbError, match=match):
            append(kv(pkg), batch(pkg), **x)
    with pytest.raises(pkg.QdbError, match="q_starts must be null"):
        decode(kv(pkg), batch(pkg, q_starts=P))
    with pytest.raises(pkg.QdbError, match="layout"):
        kv(pkg, layout="dhn")


@pytest.mark.parametrize("off", [1, 2, 3])
def test_misaligned_arrays(pkg, off):
    append, decode, prompt = ops(pkg)
    for name in ("kv_lens", "tables", "err", "q_starts"):
        for op in (append, prompt) if name == "q_starts" else (append, decode, prompt):
            with pytest.raises(pkg.QdbError, match=f"{name} is not aligned"):
                op(kv(pkg), batch(pkg, **{name: P + off}))
    for name in ("temperature", "top_k", "top_p", "min_p", "uniform", "tokens"):
        with pytest.raises(pkg.QdbError, match="is not aligned"):
            pkg.sample(**{**dict(logits=P, rows=2, vocab=100, uniform=P, tokens=P), name: P + off})


def test_null_structs(pkg):
    b, k = batch(pkg).c, kv(pkg).c
    assert pkg.lib.qdb_paged_decode(None, b, P, 0, 4, 0.0, P, 0, 1, None) == -1
    assert pkg.lib.qdb_paged_decode(k, None, P, 0, 4, 0.0, P, 0, 1, None) == -1
    assert pkg.lib.qdb_paged_decode(k, b, P, 0, 4, 0.0, P, 0, None, None) == -1
    assert b"workspace" in pkg.lib.qdb_last_error()
    assert pkg.lib.qdb_paged_prompt(None, None, P, 0, 4, 0.0, P, 0, None) == -1
    assert pkg.lib.qdb_paged_append(None, None, P, 0, 0, 4, None, None, 0.0, None, 0, P, 0, None) == -1


def test_empty_batches_are_done(pkg):
    for op in ops(pkg):
        op(kv(pkg), batch(pkg, n_seqs=0, rows=0, kv_lens=0, tables=0), q=0, o=0)
    _, _, prompt = ops(pkg)
    prompt(kv(pkg), batch(pkg, rows=0, q_starts=P))
    pkg.sample(0, 0, 10, 0, 0)


def test_bad_sampling(pkg):
    ok = dict(logits=P, rows=2, vocab=100, uniform=P, tokens=P)
    for x, match in ((dict(logits=0), "null"), (dict(uniform=0), "null"), (dict(tokens=0), "null"), (dict(rows=-1), "rows"),
                     (dict(vocab=0), "vocabulary"), (dict(vocab=262145), "vocabulary"), (dict(row_stride=99), "stride"),
                     (dict(logits=P + 2), "aligned"), (dict(dtype="f64"), "type")):
        with pytest.raises(pkg.QdbError, match=match):
            pkg.sample(**{**ok, **x})
    assert pkg.lib.qdb_sample(P, 0, 0, 1, 10, None, P, None) == -1
    assert pkg.lib.qdb_sample(P, 7, 0, 1, 10, pkg.QdbSampling(), P, None) == -1


def test_workspace_of_a_missing_device(pkg):
    with pytest.raises(pkg.QdbError, match="not available"):
        pkg.PagedWorkspace(device=99)
    with pytest.raises(pkg.QdbError, match="not available"):
        pkg.PagedWorkspace(device=-1)


def test_host_pointers_are_refused(pkg):
    """Without a device every launch is refused; with one, a host buffer is."""
    buf = ctypes.create_string_buffer(1 << 16)
    host = (ctypes.addressof(buf) + 255) // 256 * 256
    for op in ops(pkg):
        with pytest.raises(pkg.QdbError, match="not a device pointer" if has_gpu() else "CUDA"):
            op(kv(pkg, k=host, v=host), batch(pkg, kv_lens=host, tables=host), q=host, o=host)
    with pytest.raises(pkg.QdbError, match="not a device pointer" if has_gpu() else "CUDA"):
        pkg.sample(host, 1, 100, host, host)


def test_sampled_loop_arrays_of_other_lengths(pkg):
    """One first token, position and column of random numbers per session: nothing shorter is read
    behind its end, nothing longer is cut."""
    two = [type("S", (), {"h": None})()] * 2
    for f, p, u, kw in (([1], [0, 0], [[0.5, 0.5]], {}), ([1, 2], [0], [[0.5, 0.5]], {}), ([1, 2, 3], [0, 0], [[0.5, 0.5]], {}),
                        ([1, 2], [0, 0], [[0.5]], {}), ([1, 2], [0, 0], [[0.5] * 4], {}), ([1, 2], [0, 0], [0.5] * 3, {}),
                        ([1, 2], [0, 0], [[0.5, 0.5]], dict(top_k=[1, 2, 3])), (1, [0, 0], [[0.5, 0.5]], {})):
        with pytest.raises((pkg.QdbError, ValueError), match="shape|broadcast|sessions"):
            pkg.decode_sample_batch(two, f, p, u, **kw)
    with pytest.raises(pkg.QdbError, match="session"):  # (of the right lengths: the library's own check)
        pkg.decode_sample_batch(two, [1, 2], [0, 0], [[0.5, 0.5]] * 3)
