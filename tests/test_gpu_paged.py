"""GPU: the paged-cache operators against their definitions in 64 bits.

Every slot that no position owns (behind a sequence's end, unused pages) holds
NaN, and every table entry behind a sequence's pages an id outside the pool.

Tolerances. u = eps / 2 of the 16-bit type is the largest relative error of one
rounding. An attention output carries the rounding of the weights (at most u
each, so u * A with A = sum p |v|), the score and exponential errors (scores of
up to 2^6 in f32 and an exponential to 2^-16: below 2^-14 * A), weights under
the 16-bit type's smallest step (2^-30 of the largest weight each) and its own
rounding u * |o|. An appended value carries f32 arithmetic on its own pair of
dims (a norm and a rotation: below 2^-20 of the pair's length) and one rounding.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

D = 128
T = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def half_step(dtype):
    return torch.finfo(T[dtype]).eps / 2


class Pool:
    """A paged cache of given lengths: pages in random order, NaN wherever no position lives."""

    def __init__(self, pkg, lens, kv_heads, page, dtype="f16", layout="hnd", seed=0, fill=True, spread=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.pkg, self.lens, self.hk, self.page, self.dtype, self.layout = pkg, list(lens), kv_heads, page, dtype, layout
        need = [(max(n, 0) + page - 1) // page for n in lens]
        self.pages = sum(need) + 2
        order = torch.randperm(self.pages, generator=g, device="cuda").to(torch.int32).cpu().numpy()
        self.width = max(max(need), 1) + 1
        tab = np.full((len(lens), self.width), 1 << 30, np.int32)
        at = 0
        for b, m in enumerate(need):
            tab[b, :m] = order[at:at + m]
            at += m
        self.tab = tab
        self.tables = torch.tensor(tab, device="cuda")
        shape = (self.pages, kv_heads, page, D) if layout == "hnd" else (self.pages, page, kv_heads, D)
        self.k = torch.full(shape, float("nan"), device="cuda", dtype=T[dtype])
        self.v = self.k.clone()
        if fill:
            for b, n in enumerate(lens):
                if n > 0:
                    kk = torch.randn(n, kv_heads, D, generator=g, device="cuda") * spread
                    self.put(b, kk, torch.randn(n, kv_heads, D, generator=g, device="cuda"))
        self.lens_dev = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.err = torch.zeros(4, dtype=torch.int32, device="cuda")

    def where(self, b, n):
        pos = np.arange(n)
        return (torch.tensor(self.tab[b, pos // self.page], device="cuda").long(),
                torch.tensor(pos % self.page, device="cuda"))

    def put(self, b, k, v):
        pg, sl = self.where(b, k.shape[0])
        for c, x in ((self.k, k), (self.v, v)):
            if self.layout == "hnd":
                c[pg, :, sl] = x.to(c.dtype)
            else:
                c[pg, sl] = x.to(c.dtype)

    def get(self, b, n):
        pg, sl = self.where(b, n)
        return [(c[pg, :, sl] if self.layout == "hnd" else c[pg, sl]) for c in (self.k, self.v)]

    def kv(self):
        return self.pkg.PagedKV(self.k.data_ptr(), self.v.data_ptr(), self.pages, self.page, self.hk, self.dtype,
                                layout=self.layout)

    def batch(self, rows=None, starts=None):
        n = len(self.lens)
        return self.pkg.PagedBatch(n, n if rows is None else rows, self.lens_dev.data_ptr(), self.tables.data_ptr(),
                                   self.width, q_starts=0 if starts is None else starts.data_ptr(),
                                   err=self.err.data_ptr())


def starts_of(q_lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32, device="cuda")


def attention64(pool, q, q_lens, scale):
    """(outputs, A = sum p |v|, keys seen, largest |v|) of every row, in 64 bits."""
    rows, hq = q.shape[:2]
    grp = hq // pool.hk
    out = torch.zeros(rows, hq, D, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    tiny = torch.zeros(rows, 1, 1, dtype=torch.float64, device="cuda")
    r = 0
    for b, n in enumerate(q_lens):
        kv = max(pool.lens[b], 0)
        k, v = [x.double().repeat_interleave(grp, dim=1).transpose(0, 1) for x in pool.get(b, kv)]
        for i0 in range(0, n, 512):
            m = min(512, n - i0)
            if kv == 0:
                continue
            z = torch.matmul(q[r + i0:r + i0 + m].double().transpose(0, 1), k.transpose(1, 2)) * scale
            pos = torch.arange(kv - n + i0, kv - n + i0 + m, device="cuda")
            z.masked_fill_((torch.arange(kv, device="cuda")[None] > pos[:, None])[None], -float("inf"))
            p = torch.softmax(z, -1).nan_to_num(0.0)
            out[r + i0:r + i0 + m] = torch.matmul(p, v).transpose(0, 1)
            mag[r + i0:r + i0 + m] = torch.matmul(p, v.abs()).transpose(0, 1)
            tiny[r + i0:r + i0 + m, 0, 0] = (pos + 1).clamp_min(0) * 2.0 ** -30 * v.abs().max()
        r += n
    return out, mag, tiny


def check_attention(pool, q, out, q_lens, scale=D ** -0.5, what=""):
    want, mag, tiny = attention64(pool, q, q_lens, scale)
    rows = want.shape[0]
    u = half_step(pool.dtype)
    tol = u * want.abs() + (u + 2.0 ** -14) * mag + tiny + 2.0 ** -24
    d = (out[:rows].double() - want).abs()
    assert torch.isfinite(out[:rows]).all(), what
    worst = (d / tol).max().item() if rows else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} of the tolerance, at {torch.nonzero(d > tol)[:4].tolist()}"
    assert pool.err.tolist() == [0, 0, 0, 0]


def queries(rows, heads, dtype, seed=1, scale=1.2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, heads, D, generator=g, device="cuda") * scale).to(T[dtype])


@pytest.fixture(scope="module")
def ws(pkg):
    return pkg.PagedWorkspace()


def stream():
    return torch.cuda.current_stream().cuda_stream


def run_decode(pkg, ws, pool, q, **kw):
    out = torch.full_like(q, 7.0)
    pkg.paged_decode(pool.kv(), pool.batch(), q.data_ptr(), out.data_ptr(), q.shape[1], ws, stream=stream(), **kw)
    torch.cuda.synchronize()
    return out


def run_prompt(pkg, pool, q, q_lens, pad=0, **kw):
    out = torch.full_like(q, 7.0)
    st = starts_of(q_lens)
    pkg.paged_prompt(pool.kv(), pool.batch(rows=q.shape[0], starts=st), q.data_ptr(), out.data_ptr(), q.shape[1],
                     stream=stream(), **kw)
    torch.cuda.synchronize()
    if pad:
        assert (out[-pad:] == 7.0).all()  # rows behind the last sequence stay as they were
    return out


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 700]


# ---------------------------------------------------------------- one new token
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_decode_edges(pkg, ws, dtype, layout, page):
    pool = Pool(pkg, EDGES, 2, page, dtype, layout, seed=page)
    q = queries(len(EDGES), 4, dtype)
    check_attention(pool, q, run_decode(pkg, ws, pool, q), [1] * len(EDGES))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (16, 8), (12, 4), (6, 2), (5, 1), (32, 4), (7, 1), (16, 1),
                                            (18, 2), (33, 3), (64, 4)])
def test_decode_head_groups(pkg, ws, heads, kv_heads):
    pool = Pool(pkg, [333, 1, 0, 90], kv_heads, 16, "f16", seed=heads)
    q = queries(4, heads, "f16")
    check_attention(pool, q, run_decode(pkg, ws, pool, q), [1] * 4)


@pytest.mark.parametrize("lens", [[1], [16], [404], [5000], [20000], [1] * 300, [3, 20000, 1, 0, 40], [0] * 5,
                                  [17] * 200 + [9000]], ids=str)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_decode_lengths(pkg, ws, lens, dtype):
    pool = Pool(pkg, lens, 2, 32, dtype, seed=3)
    q = queries(len(lens), 16, dtype)
    check_attention(pool, q, run_decode(pkg, ws, pool, q), [1] * len(lens))


def test_decode_random_batches(pkg, ws):
    rng = np.random.default_rng(5)
    for it in range(12):
        n = int(rng.integers(1, 120))
        lens = np.exp(rng.uniform(0, np.log(3000), n)).astype(int).tolist()
        hk, grp = int(rng.choice([1, 2, 3, 8])), int(rng.choice([1, 2, 3, 8, 11]))
        dt = ["f16", "bf16"][it % 2]
        pool = Pool(pkg, lens, hk, int(rng.choice([16, 32, 64, 128])), dt, ["hnd", "nhd"][it // 2 % 2], seed=it)
        q = queries(n, hk * grp, dt, seed=it)
        check_attention(pool, q, run_decode(pkg, ws, pool, q), [1] * n, what=f"batch {it}")


@pytest.mark.parametrize("dtype,heads,kv_heads", [("f16", 8, 4), ("bf16", 32, 4), ("bf16", 16, 1)])
def test_decode_long_histories(pkg, ws, dtype, heads, kv_heads):
    """Long enough that shares of the tile list begin and end anywhere in a history."""
    lens = [60000, 50001, 0, 44443] if kv_heads > 1 else [200000, 131073, 17]
    pool = Pool(pkg, lens, kv_heads, 64, dtype, seed=14)
    q = queries(len(lens), heads, dtype)
    check_attention(pool, q, run_decode(pkg, ws, pool, q), [1] * len(lens))


def test_decode_large_scores(pkg, ws):
    """One key far above the rest, and late: the running maximum moves by hundreds."""
    for dtype in ("f16", "bf16"):
        pool = Pool(pkg, [900, 350], 2, 16, dtype, seed=9, spread=3.0)
        q = queries(2, 4, dtype, scale=3.0)
        check_attention(pool, q, run_decode(pkg, ws, pool, q, scale=0.25), [1, 1], scale=0.25)


def test_decode_repeats_bit_for_bit(pkg, ws):
    pool = Pool(pkg, [1, 6000, 37, 900, 15000], 2, 16, "bf16", seed=4)
    q = queries(5, 16, "bf16")
    first = run_decode(pkg, ws, pool, q)
    for _ in range(20):
        assert torch.equal(first, run_decode(pkg, ws, pool, q))


def strided(x, pad):
    """The same rows in a buffer with `pad` more elements between them."""
    rows, w = x.shape[0], x[0].numel()
    buf = torch.full((rows, w + pad), 3.0, device="cuda", dtype=x.dtype)
    buf[:, :w] = x.reshape(rows, w)
    return buf


def test_strided_rows_and_pools(pkg, ws):
    lens, q_lens = [70, 33, 300], [9, 33, 40]
    base = Pool(pkg, lens, 2, 32, "f16", seed=8)
    # K and V of one page side by side, pages of a larger allocation
    big = torch.full((base.pages, 2, 2, 32 + 3, D + 8), float("nan"), device="cuda", dtype=torch.float16)
    big[:, 0, :, :32, :D] = base.k
    big[:, 1, :, :32, :D] = base.v
    s = big.stride()
    kv = pkg.PagedKV(big[0, 0].data_ptr(), big[0, 1].data_ptr(), base.pages, 32, 2, "f16", strides=(s[0], s[2], s[3]))
    q = queries(sum(q_lens), 4, "f16")
    for one in (True, False):
        x = q[:3] if one else q
        n = [1] * 3 if one else q_lens
        qs, out = strided(x, 24), strided(torch.zeros_like(x), 40)
        if one:
            pkg.paged_decode(kv, base.batch(), qs.data_ptr(), out.data_ptr(), 4, ws, q_stride=qs.shape[1],
                             out_stride=out.shape[1], stream=stream())
        else:
            st = starts_of(q_lens)
            pkg.paged_prompt(kv, base.batch(rows=len(x), starts=st), qs.data_ptr(), out.data_ptr(), 4,
                             q_stride=qs.shape[1], out_stride=out.shape[1], stream=stream())
        torch.cuda.synchronize()
        assert (out[:, 4 * D:] == 3.0).all()
        check_attention(base, x, out[:, :4 * D].reshape(-1, 4, D), n)


# ---------------------------------------------------------------- packed prompts
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_prompt_edges(pkg, dtype, layout, page):
    lens = EDGES
    q_lens = [min(n, [n, 1, 7, 40, 130][i % 5]) for i, n in enumerate(lens)]
    pool = Pool(pkg, lens, 2, page, dtype, layout, seed=page + 1)
    q = queries(sum(q_lens) + 3, 4, dtype)
    out = run_prompt(pkg, pool, q, q_lens, pad=3)
    check_attention(pool, q[:-3], out, q_lens)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (16, 8), (12, 4), (6, 2), (5, 1), (32, 4), (7, 1), (16, 1),
                                            (18, 2), (33, 3), (64, 4)])
def test_prompt_head_groups(pkg, heads, kv_heads):
    lens, q_lens = [333, 1, 0, 290], [333, 1, 0, 77]
    pool = Pool(pkg, lens, kv_heads, 16, "bf16", seed=heads)
    q = queries(sum(q_lens), heads, "bf16")
    check_attention(pool, q, run_prompt(pkg, pool, q, q_lens), q_lens)


@pytest.mark.parametrize("lens,q_lens", [([1], [1]), ([404], [404]), ([2500], [2500]), ([9000], [5]), ([9000], [600]),
                                         ([5, 0, 60], [9, 4, 70]), ([0], [3]), ([0, 0], [0, 0]),
                                         ([40] * 100, [13] * 100), ([1000, 3, 2000], [0, 0, 1])], ids=str)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_prompt_lengths(pkg, lens, q_lens, dtype):
    """Among them more rows than positions: the first rows see nothing and are zero."""
    pool = Pool(pkg, lens, 2, 32, dtype, seed=6)
    q = queries(sum(q_lens) + 1, 4, dtype)
    out = run_prompt(pkg, pool, q, q_lens, pad=1)
    check_attention(pool, q[:-1], out, q_lens)


def test_prompt_random_batches(pkg):
    rng = np.random.default_rng(6)
    for it in range(12):
        n = int(rng.integers(1, 30))
        q_lens = np.exp(rng.uniform(0, np.log(900), n)).astype(int).tolist()
        lens = [m + int(rng.integers(0, 600)) * int(rng.integers(0, 2)) for m in q_lens]
        hk, grp = int(rng.choice([1, 2, 3, 8])), int(rng.choice([1, 2, 3, 8, 11]))
        dt = ["f16", "bf16"][it % 2]
        pool = Pool(pkg, lens, hk, int(rng.choice([16, 32, 64, 128])), dt, ["hnd", "nhd"][it // 2 % 2], seed=it)
        q = queries(sum(q_lens), hk * grp, dt, seed=it)
        check_attention(pool, q, run_prompt(pkg, pool, q, q_lens), q_lens, what=f"batch {it}")


def test_prompt_large_scores(pkg):
    for dtype in ("f16", "bf16"):
        pool = Pool(pkg, [900, 350], 2, 16, dtype, seed=9, spread=3.0)
        q = queries(900 + 100, 4, dtype, scale=3.0)
        check_attention(pool, q, run_prompt(pkg, pool, q, [900, 100], scale=0.25), [900, 100], scale=0.25)


def test_prompt_rising_scores(pkg):
    """Keys sorted so that every tile raises the maximum: each rescale of the sums is taken."""
    for dtype in ("f16", "bf16"):
        n = 1400
        pool = Pool(pkg, [n], 1, 64, dtype, fill=False)
        base = torch.ones(n, 1, D, device="cuda")
        k = base * (torch.arange(n, device="cuda")[:, None, None] / 40.0)
        g = torch.Generator(device="cuda").manual_seed(3)
        pool.put(0, k, torch.randn(n, 1, D, generator=g, device="cuda"))
        q = torch.full((n, 2, D), 1.0, device="cuda").to(T[dtype])
        check_attention(pool, q, run_prompt(pkg, pool, q, [n], scale=1 / 64), [n], scale=1 / 64)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("key,q_len", [(100, 300), (0, 300), (299, 300), (5, 40), (270, 40), (128, 172)])
def test_prompt_non_finite_values_reach_only_rows_that_see_them(pkg, dtype, key, q_len):
    n = 300
    pool = Pool(pkg, [n], 2, 32, dtype, seed=6)
    q = queries(q_len, 4, dtype)
    clean = run_prompt(pkg, pool, q, [q_len])
    pg, sl = pool.where(0, n)
    pool.v[pg[key], 1, sl[key], 3] = float("inf")
    pool.v[pg[key], 1, sl[key], 9] = float("nan")
    pool.v[pg[key], 1, sl[key], 127] = -float("inf")
    out = run_prompt(pkg, pool, q, [q_len])
    sees = torch.arange(n - q_len, n, device="cuda") >= key
    assert torch.equal(out[~sees], clean[~sees])
    assert torch.equal(out[:, :2], clean[:, :2])
    bad = out[sees][:, 2:]
    # inf times a weight: inf, or NaN where the weight is below the type's smallest
    assert ((bad[..., 3] == float("inf")) | torch.isnan(bad[..., 3])).all()
    assert ((bad[..., 127] == -float("inf")) | torch.isnan(bad[..., 127])).all()
    assert torch.isnan(bad[..., 9]).all()
    rest = [d for d in range(D) if d not in (3, 9, 127)]
    assert torch.equal(bad[..., rest], clean[sees][:, 2:][..., rest])


def test_prompt_equals_decode(pkg, ws):
    """The last row of a prompt is the decode row of the same cache."""
    pool = Pool(pkg, [500, 31, 1], 2, 16, "f16", seed=2)
    q = queries(3, 8, "f16")
    a, b = run_decode(pkg, ws, pool, q), run_prompt(pkg, pool, q, [1, 1, 1])
    assert (a.double() - b.double()).abs().max() <= 2 ** -9


# ---------------------------------------------------------------- append
def append64(qkv, heads, hk, pos, rope, q_norm, k_norm, eps):
    x = qkv.double().reshape(len(qkv), heads + 2 * hk, D)
    y = x[:, :heads + hk].clone()
    if q_norm is not None:
        y[:, :heads] *= q_norm.double() / torch.sqrt(y[:, :heads].square().mean(-1, keepdim=True) + eps)
    if k_norm is not None:
        y[:, heads:] *= k_norm.double() / torch.sqrt(y[:, heads:].square().mean(-1, keepdim=True) + eps)
    a, b = y[..., :64], y[..., 64:]
    size = torch.sqrt(a * a + b * b)
    if rope is not None:
        c, s = rope[pos].double()[:, None].unbind(-1)
        a, b = a * c - b * s, b * c + a * s
    y = torch.cat([a, b], -1)
    return y[:, :heads], y[:, heads:], x[:, heads + hk:], torch.cat([size, size], -1)


def rope_table(n):
    ang = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * (1e6 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D))
    return torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()


def run_append(pkg, pool, q_lens, heads, src, norm="qk", rope=True, pad=0, seed=1, stride_pad=0, one=False):
    hk = pool.hk
    rows = sum(q_lens)
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = (torch.randn(rows + pad, (heads + 2 * hk) * D, generator=g, device="cuda") * 1.5).to(T[src])
    qn = 1 + 0.2 * torch.randn(D, generator=g, device="cuda") if "q" in norm else None
    kn = 1 + 0.2 * torch.randn(D, generator=g, device="cuda") if "k" in norm else None
    tab = rope_table(max(max(pool.lens), 1)) if rope else None
    st = starts_of(q_lens)
    buf = strided(qkv, stride_pad)
    q = torch.full((rows + pad, heads, D), 7.0, device="cuda", dtype=T[pool.dtype])
    p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    k0, v0 = pool.k.clone(), pool.v.clone()
    pkg.paged_append(pool.kv(), pool.batch() if one else pool.batch(rows=rows + pad, starts=st), buf.data_ptr(),
                     q.data_ptr(), heads, dtype=src, row_stride=buf.shape[1] if stride_pad else 0, q_norm=p(qn),
                     k_norm=p(kn), rope=p(tab), rope_len=len(tab) if rope else 0, stream=stream())
    torch.cuda.synchronize()
    assert pool.err.tolist() == [0, 0, 0, 0]
    pos = torch.tensor(np.concatenate([np.arange(n - m, n) for m, n in zip(q_lens, pool.lens)]).astype(np.int64),
                       device="cuda")
    real = pos >= 0  # rows at negative positions are left out
    wq, wk, wv, size = append64(qkv[:rows], heads, hk, pos.clamp_min(0), tab, qn, kn, 1e-6)
    u = half_step(pool.dtype)
    close = lambda got, want, sz: ((got.double() - want).abs() <= u * want.abs() + 2.0 ** -20 * sz + 2.0 ** -25).all()  # noqa: E731
    assert close(q[:rows][real], wq[real], size[real][:, :heads])
    assert (q[:rows][~real] == 7.0).all()
    if pad:
        assert (q[rows:] == 7.0).all()
    r = 0
    for b, (m, n) in enumerate(zip(q_lens, pool.lens)):
        lo = max(0, m - n)
        if m > lo:
            pg, sl = pool.where(b, n)
            pg, sl = pg[n - m + lo:], sl[n - m + lo:]
            k, v = [(c[pg, :, sl] if pool.layout == "hnd" else c[pg, sl]) for c in (pool.k, pool.v)]
            assert close(k, wk[r + lo:r + m], size[r + lo:r + m][:, heads:])
            assert close(v, wv[r + lo:r + m], 0.0)
            for c, c0 in ((pool.k, k0), (pool.v, v0)):  # put the old values back: everything else is untouched
                if pool.layout == "hnd":
                    c[pg, :, sl] = c0[pg, :, sl]
                else:
                    c[pg, sl] = c0[pg, sl]
        r += m
    for c, c0 in ((pool.k, k0), (pool.v, v0)):
        assert torch.equal(c.view(torch.int16), c0.view(torch.int16))


@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("norm", ["", "q", "qk"])
def test_append_forms(pkg, src, dtype, layout, norm):
    lens, q_lens = [5, 64, 200, 17, 0, 33], [5, 1, 70, 17, 0, 2]
    pool = Pool(pkg, lens, 2, 16, dtype, layout, seed=3)
    run_append(pkg, pool, q_lens, 4, src, norm=norm, rope=norm != "q", pad=2, stride_pad=8 if norm else 0)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (16, 8), (7, 1), (32, 4), (33, 3), (16, 1), (64, 4)])
@pytest.mark.parametrize("page", [16, 256])
def test_append_heads_and_pages(pkg, heads, kv_heads, page):
    pool = Pool(pkg, [700, 3, 90], kv_heads, page, "f16", seed=heads)
    run_append(pkg, pool, [300, 3, 1], heads, "f32")


def test_append_one_row_per_sequence(pkg):
    pool = Pool(pkg, [1, 16, 17, 4000], 8, 16, "bf16", "nhd", seed=1)
    run_append(pkg, pool, [1, 1, 1, 1], 16, "f32", one=True)


def test_append_more_rows_than_positions(pkg):
    pool = Pool(pkg, [3, 0, 20], 2, 16, "f16", seed=1)
    run_append(pkg, pool, [8, 4, 20], 4, "f32")


def test_append_saturates_f16_and_keeps_nan(pkg):
    pool = Pool(pkg, [1], 1, 16, "f16", fill=False)
    qkv = torch.zeros(1, 3 * D, device="cuda")
    qkv[0, D] = 1e6
    qkv[0, 2 * D] = -1e6
    qkv[0, 2 * D + 1] = float("nan")
    q = torch.zeros(1, 1, D, device="cuda", dtype=torch.float16)
    pkg.paged_append(pool.kv(), pool.batch(), qkv.data_ptr(), q.data_ptr(), 1, stream=stream())
    torch.cuda.synchronize()
    k, v = pool.get(0, 1)
    assert k[0, 0, 0] == 65504 and v[0, 0, 0] == -65504 and torch.isnan(v[0, 0, 1])


# ---------------------------------------------------------------- bad device data stays in bounds
def test_bad_pages_are_recorded(pkg, ws):
    for what, bad in (("page", -1), ("page", 1 << 30)):
        pool = Pool(pkg, [100, 100], 2, 16, "f16", seed=3)
        pool.tables[0, 2] = bad
        q = queries(2, 4, "f16")
        out = run_decode(pkg, ws, pool, q)
        assert pool.err.tolist()[:3] == [3, 1, 0]
        pool.err.zero_()
        good = Pool(pkg, [100, 100], 2, 16, "f16", seed=3)
        check_attention(Sub(good, 1), q[1:], out[1:], [1])
        out = run_prompt(pkg, pool, q, [1, 1])
        assert pool.err.tolist()[:3] == [3, 1, 0]
        check_attention(Sub(good, 1), q[1:], out[1:], [1])


class Sub:
    """One sequence of a pool."""

    def __init__(self, pool, b):
        self.hk, self.dtype, self.lens, self.err = pool.hk, pool.dtype, [pool.lens[b]], torch.zeros(4)
        self.err = torch.zeros(4, dtype=torch.int32)
        self.get = lambda _, n: pool.get(b, n)


def test_bad_lengths_and_starts_are_recorded(pkg, ws):
    pool = Pool(pkg, [100, 100], 2, 16, "f16", seed=3)
    pool.tables.fill_(1)
    pool.lens_dev[0] = 1 << 20
    q = queries(2, 4, "f16")
    run_decode(pkg, ws, pool, q)
    assert pool.err.tolist()[:3] == [3, 2, 0]
    for st in ([0, 5, 2], [-3, 1, 2], [0, 1, 9], [4, 1, 2]):
        pool = Pool(pkg, [100, 100], 2, 16, "f16", seed=3)
        t = torch.tensor(st, dtype=torch.int32, device="cuda")
        out = torch.full_like(q, 7.0)
        pkg.paged_prompt(pool.kv(), pool.batch(rows=2, starts=t), q.data_ptr(), out.data_ptr(), 4, stream=stream())
        torch.cuda.synchronize()
        assert pool.err.tolist()[:2] == [3, 4]


def test_append_outside_is_recorded(pkg):
    pool = Pool(pkg, [40], 1, 16, "f16", fill=False)
    qkv, q = torch.ones(1, 3 * D, device="cuda"), torch.zeros(1, 1, D, device="cuda", dtype=torch.float16)
    tab = rope_table(20)
    pkg.paged_append(pool.kv(), pool.batch(), qkv.data_ptr(), q.data_ptr(), 1, rope=tab.data_ptr(), rope_len=20,
                     stream=stream())
    torch.cuda.synchronize()
    assert pool.err.tolist() == [3, 3, 0, 39]
    pool.err.zero_()
    pool.tables[0, 2] = -7
    pkg.paged_append(pool.kv(), pool.batch(), qkv.data_ptr(), q.data_ptr(), 1, stream=stream())
    torch.cuda.synchronize()
    assert pool.err.tolist() == [3, 1, 0, -7]
    assert torch.isnan(pool.k).all() and torch.isnan(pool.v).all()


# ---------------------------------------------------------------- streams, graphs, far offsets
def test_side_stream_and_graph(pkg):
    """The three operators captured together and replayed on other contents and lengths."""
    ws2 = pkg.PagedWorkspace()
    lens = [40, 700, 1]
    pool = Pool(pkg, lens, 2, 16, "f16", seed=5)
    qkv = torch.randn(3, 8 * D, device="cuda")
    tab = rope_table(1024)
    q = torch.zeros(3, 4, D, device="cuda", dtype=torch.float16)
    out, out2 = torch.zeros_like(q), torch.zeros_like(q)
    st3 = torch.arange(4, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()

    def step(s):
        pkg.paged_append(pool.kv(), pool.batch(), qkv.data_ptr(), q.data_ptr(), 4, rope=tab.data_ptr(), rope_len=1024,
                         stream=s)
        pkg.paged_decode(pool.kv(), pool.batch(), q.data_ptr(), out.data_ptr(), 4, ws2, stream=s)
        pkg.paged_prompt(pool.kv(), pool.batch(rows=3, starts=st3), q.data_ptr(), out2.data_ptr(), 4, stream=s)

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(side.cuda_stream)
    side.synchronize()
    check_attention(pool, q, out, [1] * 3)
    check_attention(pool, q, out2, [1] * 3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream().cuda_stream)
    for n in ([39, 690, 1], [17, 300, 1]):
        qkv.copy_(torch.randn(3, 8 * D, device="cuda"))
        pool.lens_dev.copy_(torch.tensor(n, dtype=torch.int32))
        pool.lens = n
        graph.replay()
        torch.cuda.synchronize()
        check_attention(pool, q, out, [1] * 3)
        check_attention(pool, q, out2, [1] * 3)


def test_calls_on_two_streams_at_once(pkg):
    """Decode and prompt calls that overlap on the GPU, each stream with its own workspace, give
    what they give alone, bit for bit."""
    sides = [torch.cuda.Stream() for _ in range(2)]
    jobs = []
    for i, side in enumerate(sides):
        lens = [900 + 13 * i, 5, 3000, 64 + i]
        q_lens = [300, 5, 700 + i, 1]
        pool = Pool(pkg, lens, 2, 16 << i, ["f16", "bf16"][i], seed=20 + i)
        q1, q2 = queries(4, 8, pool.dtype, seed=i), queries(sum(q_lens), 8, pool.dtype, seed=i)
        jobs.append((side, pkg.PagedWorkspace(), pool, q1, torch.zeros_like(q1), q2, torch.zeros_like(q2), q_lens,
                     starts_of(q_lens)))
    torch.cuda.synchronize()

    def go(job):
        side, w, pool, q1, o1, q2, o2, _, st = job
        s = side.cuda_stream
        pkg.paged_decode(pool.kv(), pool.batch(), q1.data_ptr(), o1.data_ptr(), 8, w, stream=s)
        pkg.paged_prompt(pool.kv(), pool.batch(rows=len(q2), starts=st), q2.data_ptr(), o2.data_ptr(), 8, stream=s)

    alone = []
    for job in jobs:
        go(job)
        torch.cuda.synchronize()
        check_attention(job[2], job[3], job[4], [1] * 4)
        check_attention(job[2], job[5], job[6], job[7])
        alone.append((job[4].clone(), job[6].clone()))
    for _ in range(30):
        for job in jobs:
            job[4].fill_(9), job[6].fill_(9)
        torch.cuda.synchronize()
        for _ in range(3):
            for job in jobs:
                go(job)
        torch.cuda.synchronize()
        for job, (o1, o2) in zip(jobs, alone):
            assert torch.equal(job[4], o1) and torch.equal(job[6], o2)


def test_thousands_of_short_sequences(pkg, ws):
    rng = np.random.default_rng(11)
    n = 3000
    lens = rng.integers(0, 40, n).tolist()
    pool = Pool(pkg, lens, 2, 16, "f16", seed=12)
    q = queries(n, 4, "f16")
    check_attention(pool, q, run_decode(pkg, ws, pool, q), [1] * n)
    q_lens = [int(rng.integers(0, m + 1)) for m in lens]
    q = queries(sum(q_lens), 4, "f16")
    check_attention(pool, q, run_prompt(pkg, pool, q, q_lens), q_lens)


def test_rows_ahead_of_the_first_sequence(pkg):
    """q_starts may begin above 0: the rows before belong to nobody and stay as they are."""
    lens, q_lens, ahead = [300, 0, 40], [290, 0, 3], 37
    pool = Pool(pkg, lens, 2, 16, "bf16", seed=8)
    q = queries(ahead + sum(q_lens), 4, "bf16")
    out = torch.full_like(q, 7.0)
    st = starts_of(q_lens) + ahead
    pkg.paged_prompt(pool.kv(), pool.batch(rows=len(q), starts=st), q.data_ptr(), out.data_ptr(), 4, stream=stream())
    torch.cuda.synchronize()
    assert (out[:ahead] == 7.0).all()
    check_attention(pool, q[ahead:], out[ahead:], q_lens)
    qkv = torch.randn(len(q), 8 * D, device="cuda")
    new = torch.full_like(q, 7.0)
    pkg.paged_append(pool.kv(), pool.batch(rows=len(q), starts=st), qkv.data_ptr(), new.data_ptr(), 4, stream=stream())
    torch.cuda.synchronize()
    assert (new[:ahead] == 7.0).all()
    assert torch.equal(new[ahead:].reshape(-1, 4 * D), qkv[ahead:, :4 * D].to(torch.bfloat16))
    assert torch.equal(pool.get(2, 40)[1][37:], qkv[-3:, 6 * D:].view(3, 2, D).to(torch.bfloat16))
    assert pool.err.tolist() == [0, 0, 0, 0]


def test_pool_offsets_beyond_32_bits(pkg, ws):
    """A pool of more than 2^32 elements: pages at its very end are the ones read and written."""
    hk, page = 8, 256
    pages = (1 << 32) // (hk * page * D) + 40
    k = torch.empty(pages, hk, page, D, device="cuda", dtype=torch.bfloat16)
    v = torch.empty_like(k)
    small = Pool(pkg, [600, 300], hk, page, "bf16", seed=4)
    ids = torch.arange(pages - small.pages, pages, device="cuda")
    k[ids], v[ids] = small.k, small.v
    tables = torch.where(small.tables < small.pages, small.tables + (pages - small.pages), small.tables)
    kv = pkg.PagedKV(k.data_ptr(), v.data_ptr(), pages, page, hk, "bf16")
    b = lambda st=None, rows=2: pkg.PagedBatch(2, rows, small.lens_dev.data_ptr(), tables.data_ptr(), small.width, q_starts=st.data_ptr() if st is not None else 0, err=small.err.data_ptr())  # noqa: E731
    q = queries(2, 16, "bf16")
    out = torch.zeros_like(q)
    pkg.paged_decode(kv, b(), q.data_ptr(), out.data_ptr(), 16, ws, stream=stream())
    torch.cuda.synchronize()
    check_attention(small, q, out, [1, 1])
    q = queries(400, 16, "bf16")
    out = torch.zeros_like(q)
    st = starts_of([300, 100])
    pkg.paged_prompt(kv, b(st, 400), q.data_ptr(), out.data_ptr(), 16, stream=stream())
    torch.cuda.synchronize()
    check_attention(small, q, out, [300, 100])
    qkv = torch.randn(2, 32 * D, device="cuda")
    q = queries(2, 16, "bf16")
    pkg.paged_append(kv, b(), qkv.data_ptr(), q.data_ptr(), 16, stream=stream())
    torch.cuda.synchronize()
    pg = tables[0, 599 // page].long()
    assert torch.equal(v[pg, :, 599 % page], qkv[0].view(32, D)[24:].to(torch.bfloat16))
    assert small.err.tolist() == [0, 0, 0, 0]
