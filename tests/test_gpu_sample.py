"""GPU: sampling against its definition in 64 bits (tokens have to be equal)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

T = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def sample64(x, temp, k, p, floor, u):
    """The definition: one row of logits (float64), numpy."""
    x = np.where(np.isnan(x), -np.inf, x)
    best = int(np.argmax(x))
    if x[best] == -np.inf:
        return -1
    if not temp > 0 or p <= 0 or floor > 1:
        return best
    with np.errstate(invalid="ignore"):
        w = np.where(x == x[best], 1.0, np.exp((x - x[best]) / temp))
    order = np.lexsort((np.arange(len(x)), -x))
    if k > 0:
        order = order[:k]
    ws = w[order]
    ahead = np.concatenate([[0.0], np.cumsum(ws)])
    keep = (ws >= floor) & ((ahead[:-1] < p * ahead[-1]) if p < 1 else True)
    left = np.sort(order[keep])
    run = np.cumsum(w[left])
    return int(left[np.searchsorted(run, u * run[-1], side="right")])


def run(pkg, x, u, temp=None, k=None, p=None, floor=None, dtype="f32", row_stride=0):
    dev = lambda v, t: None if v is None else torch.tensor(v, dtype=t, device="cuda")  # noqa: E731
    rows = len(u)
    keep = [dev(temp, torch.float32), dev(k, torch.int32), dev(p, torch.float32), dev(floor, torch.float32),
            dev(u, torch.float32)]
    ptr = [0 if t is None else t.data_ptr() for t in keep]
    out = torch.full((rows,), -9, dtype=torch.int32, device="cuda")
    pkg.sample(x.data_ptr(), rows, x.shape[1] if not row_stride else x.shape[1] - 5, ptr[4], out.data_ptr(), dtype=dtype,
               row_stride=row_stride, temperature=ptr[0], top_k=ptr[1], top_p=ptr[2], min_p=ptr[3],
               stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return out.tolist()


def want(x, u, temp=None, k=None, p=None, floor=None):
    n = len(u)
    f = lambda v, d: np.asarray(v, np.float32).astype(np.float64) if v is not None else np.full(n, d)  # noqa: E731
    T_, p_, m_, u_ = f(temp, 1.0), f(p, 1.0), f(floor, 0.0), f(u, 0.0)
    kk = k if k is not None else [0] * n
    return [sample64(r, T_[i], kk[i], p_[i], m_[i], u_[i]) for i, r in enumerate(x.double().cpu().numpy())]


def logits(rows, vocab, dtype="f32", seed=0, spread=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g, device="cuda") * spread
    x[:, ::97] += 4
    return x.to(T[dtype])


@pytest.mark.parametrize("vocab", [1, 2, 31, 32, 33, 1000, 1023, 1024, 1025, 4097, 32000, 50257, 151936, 262144])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_vocabularies(pkg, vocab, dtype):
    rows = 12
    rng = np.random.default_rng(vocab)
    x = logits(rows, vocab, dtype, seed=vocab)
    u = rng.random(rows).astype(np.float32).tolist()
    kw = dict(temp=rng.choice([0.0, 0.3, 1.0, 1.7], rows).tolist(), k=rng.choice([0, 1, 3, 50, 300000], rows).tolist(),
              p=rng.choice([1.0, 0.95, 0.5, 0.01], rows).tolist(), floor=rng.choice([0.0, 0.05, 0.4], rows).tolist())
    assert run(pkg, x, u, dtype=dtype, **kw) == want(x, u, **kw)
    assert run(pkg, x, u, dtype=dtype) == want(x, u)


@pytest.mark.parametrize("knob", ["temp", "k", "p", "floor"])
def test_each_parameter_alone(pkg, knob):
    vals = dict(temp=[0.05, 0.5, 1.0, 4.0, 100.0], k=[2, 7, 64, 1000, 1999], p=[0.001, 0.3, 0.9, 0.999, 1.5],
                floor=[1e-6, 0.01, 0.3, 0.9, 1.0])[knob]
    x = logits(40, 2000, seed=3)
    u = np.linspace(0, 0.9999, 40).tolist()
    kw = {knob: (vals * 8)[:40]}
    assert run(pkg, x, u, **kw) == want(x, u, **kw)


def test_ties(pkg):
    """All logits equal, and few distinct values: ties stay in index order."""
    for x in (torch.zeros(16, 5000, device="cuda"), torch.full((16, 5000), -3.5, device="cuda"),
              torch.randint(0, 3, (16, 5000), device="cuda").float() - 1,
              torch.randint(0, 2, (16, 5000), device="cuda").float() * 40):
        u = np.linspace(0, 0.999, 16).tolist()
        for kw in (dict(), dict(k=[10] * 16), dict(k=[1700] * 16), dict(p=[0.5] * 16), dict(p=[0.1234] * 16, k=[777] * 16),
                   dict(temp=[0.0] * 16), dict(floor=[1.0] * 16, k=[2500] * 16)):
            assert run(pkg, x, u, **kw) == want(x, u, **kw)
    z = torch.zeros(1, 64, device="cuda")
    z[0, ::2] = -0.0
    for kw in (dict(temp=[0.0]), dict(k=[3]), dict(p=[0.25])):
        assert run(pkg, z, [0.9], **kw) == want(z, [0.9], **kw)


def test_masked_and_special_logits(pkg):
    inf, nan = float("inf"), float("nan")
    low = torch.finfo(torch.float32).min
    rows = [[-inf] * 40, [nan] * 40, [-inf] * 39 + [2.0], [nan] * 20 + [1.0] * 20, [inf] + [0.0] * 39,
            [0.0] * 20 + [inf, inf] + [5.0] * 18, [low] * 40, [low] * 39 + [0.0], [-inf, nan] * 20, [3e38, -3e38] * 20]
    x = torch.tensor(rows, device="cuda")
    for u in (0.0, 0.4, 0.999999):
        n = [u] * len(rows)
        for kw in (dict(), dict(k=[3] * 10), dict(p=[0.6] * 10), dict(temp=[0.0] * 10), dict(floor=[0.5] * 10),
                   dict(k=[30] * 10, p=[0.9] * 10, temp=[1e-20] * 10)):
            assert run(pkg, x, n, **kw) == want(x, n, **kw)


def test_odd_parameters_are_off_or_greedy(pkg):
    x = logits(8, 300, seed=5)
    g = x.argmax(-1).tolist()
    u = [0.7] * 8
    nan = float("nan")
    assert run(pkg, x, u, temp=[nan] * 8) == g
    assert run(pkg, x, u, temp=[-1.0] * 8) == g
    assert run(pkg, x, u, p=[0.0] * 8) == g
    assert run(pkg, x, u, p=[-0.5] * 8) == g
    assert run(pkg, x, u, floor=[1.5] * 8) == g
    assert run(pkg, x, u, k=[1] * 8) == g
    free = want(x, u)
    assert run(pkg, x, u, p=[nan] * 8) == free
    assert run(pkg, x, u, floor=[nan] * 8) == free
    assert run(pkg, x, u, k=[-5] * 8) == free
    assert run(pkg, x, [1.0] * 8) == run(pkg, x, [float(np.nextafter(np.float32(1), np.float32(0)))] * 8)
    assert run(pkg, x, [-1.0] * 8) == run(pkg, x, [0.0] * 8) == run(pkg, x, [nan] * 8)


def test_row_stride_and_many_rows(pkg):
    x = logits(300, 777, seed=6)
    u = np.random.default_rng(0).random(300).astype(np.float32).tolist()
    kw = dict(k=[40] * 300, p=[0.9] * 300)
    ref = want(x[:, :772], u, **kw)
    assert run(pkg, x, u, row_stride=777, **kw) == ref
    y = logits(300, 777, "bf16", seed=6)
    assert run(pkg, y, u, row_stride=777, dtype="bf16", **kw) == want(y[:, :772], u, **kw)


@pytest.mark.parametrize("vocab,rows", [(40, 700), (20000, 333), (151936, 131)])
def test_rows_of_all_kinds_beside_each_other(pkg, vocab, rows):
    """More rows than run at once: which row is taken when depends on its parameters, its token not."""
    rng = np.random.default_rng(rows)
    x = logits(rows, vocab, seed=rows)
    u = rng.random(rows).astype(np.float32).tolist()
    kw = dict(temp=rng.choice([0.0, 0.4, 1.0, float("nan")], rows).tolist(),
              k=rng.choice([0, 1, 5, 400, 1500], rows).tolist(), p=rng.choice([1.0, 0.9, 0.5, 0.0], rows).tolist(),
              floor=rng.choice([0.0, 0.02, 2.0], rows).tolist())
    got = run(pkg, x, u, **kw)
    assert got == want(x, u, **kw)
    for one in ("temp", "k", "p", "floor"):
        assert run(pkg, x, u, **{one: kw[one]}) == want(x, u, **{one: kw[one]})


@pytest.mark.parametrize("equal", [1, 5, 31, 32, 33, 100, 1000])
def test_lists_with_groups_of_equal_logits(pkg, equal):
    """Lists of 129 to 2048 tokens whose logits come in groups."""
    rng = np.random.default_rng(equal)
    vocab, rows = 30000, 10
    level = rng.permutation(vocab) // equal
    x = torch.tensor(-0.004 * equal * level, device="cuda").float().repeat(rows, 1)
    x[1::2] += torch.tensor(rng.normal(size=(rows // 2, 1)), device="cuda").float()
    u = rng.random(rows).astype(np.float32).tolist()
    for kw in (dict(k=[129] * rows), dict(k=[700] * rows, p=[0.8] * rows), dict(k=[1900] * rows), dict(p=[0.99] * rows),
               dict(p=[0.6] * rows, temp=[3.0] * rows), dict(p=[0.9] * rows, floor=[0.01] * rows)):
        assert run(pkg, x, u, **kw) == want(x, u, **kw)


def test_frequencies(pkg):
    """Evenly spaced random numbers give each token its share of the draws, to within one draw."""
    x = torch.tensor([[0.0, 1.0, 2.0, -1.0]], device="cuda").repeat(4096, 1)
    u = ((np.arange(4096) + 0.5) / 4096).tolist()
    got = np.bincount(run(pkg, x, u), minlength=4) / 4096
    p = np.exp([0, 1, 2, -1]) / np.exp([0, 1, 2, -1]).sum()
    assert np.abs(got - p).max() <= 1 / 4096


def test_same_result_every_time_and_in_a_graph(pkg):
    x = logits(8, 151936, seed=7)
    u = torch.rand(8, device="cuda")
    p = torch.full((8,), 0.97, device="cuda")
    out = torch.zeros(8, dtype=torch.int32, device="cuda")
    call = lambda: pkg.sample(x.data_ptr(), 8, 151936, u.data_ptr(), out.data_ptr(), top_p=p.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)  # noqa: E731
    call()
    torch.cuda.synchronize()
    first = out.tolist()
    for _ in range(20):
        call()
        assert out.tolist() == first
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    u.copy_(torch.rand(8, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    assert out.tolist() == want(x, u.tolist(), p=[0.97] * 8)
