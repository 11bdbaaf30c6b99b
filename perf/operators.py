"""Cases of the paged-cache serving operators: appending rotated keys and values to a paged
cache, attention of one new token per sequence over it, causal attention of packed prompts
over it, and sampling the next token from given random numbers.

Each operator has a plain form in elementary torch operations (`own` false) and the library's
call (`own` true). Head dimension 128 throughout, as in the decoder.
"""
import importlib.util
import math
import os
import random
import sys

import numpy as np
import torch

own = False

D = 128
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
VOCAB = 151936  # the decoder's vocabulary


def listed():
    return [
        # one decode step of 64 utterances: QKV projection rows (f32, as the GEMM leaves them) into the cache
        dict(name="append_step_64", op="append", seqs=64, q_lo=1, q_hi=1, prefix=660, heads=16, kv_heads=8,
             src="f32", dtype="f16", norm=True, page=16, layout="hnd", ragged=1),
        # a long prompt (five minutes of audio) appended at once
        dict(name="append_prompt_3721", op="append", seqs=1, q_lo=3721, q_hi=3721, prefix=0, heads=16, kv_heads=8,
             src="f32", dtype="f16", norm=True, page=64, layout="hnd", ragged=2),
        # many prompts of different lengths packed into one batch, 16-bit projections, no head norms
        dict(name="append_packed_bf16", op="append", seqs=64, q_lo=30, q_hi=800, prefix=100, heads=16, kv_heads=8,
             src="bf16", dtype="bf16", norm=False, page=32, layout="nhd", ragged=3),
        # a single utterance's decode step just after a 404-position prompt: latency
        dict(name="decode_one_404", op="decode", seqs=1, lo=404, hi=404, heads=16, kv_heads=8, dtype="f16", page=16,
             layout="hnd", ragged=4),
        # the batched decode step of 64 utterances
        dict(name="decode_64_utterances", op="decode", seqs=64, lo=404, hi=660, heads=16, kv_heads=8, dtype="f16",
             page=16, layout="hnd", ragged=5),
        # 256 staggered streams with very different histories
        dict(name="decode_256_ragged", op="decode", seqs=256, lo=1, hi=1500, heads=16, kv_heads=8, dtype="bf16",
             page=32, layout="nhd", ragged=6),
        # few sequences with very long histories, eight query heads to a key head
        dict(name="decode_8_long", op="decode", seqs=8, lo=24000, hi=32768, heads=32, kv_heads=4, dtype="bf16",
             page=64, layout="hnd", ragged=7),
        # the prompt of a 30-second utterance
        dict(name="prompt_one_404", op="prompt", seqs=1, q_lo=404, q_hi=404, prefix=0, heads=16, kv_heads=8,
             dtype="f16", page=16, layout="hnd", ragged=8),
        # streaming: every stream appends a short piece behind what it has cached
        dict(name="prompt_64_pieces", op="prompt", seqs=64, q_lo=30, q_hi=130, prefix=400, heads=16, kv_heads=8,
             dtype="f16", page=32, layout="hnd", ragged=9),
        # a very long prompt: arithmetic
        dict(name="prompt_one_16384", op="prompt", seqs=1, q_lo=16384, q_hi=16384, prefix=0, heads=16, kv_heads=8,
             dtype="bf16", page=64, layout="hnd", ragged=10),
        # one row of logits, top-k and top-p: latency
        dict(name="sample_one", op="sample", rows=1, vocab=VOCAB, src="f32", mix=False, ragged=11),
        # a step of 64 utterances, every row with its own temperature, top-k, top-p and min-p
        dict(name="sample_64_mixed", op="sample", rows=64, vocab=VOCAB, src="f32", mix=True, ragged=12),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "prompt", "sample"])
    rag = rng.randrange(1 << 30)
    if op == "sample":
        return dict(op=op, rows=_log(rng, 1, 64), vocab=_log(rng, 1000, VOCAB), src=rng.choice(["f32", "f32", "bf16"]),
                    mix=rng.random() < 0.7, ragged=rag)
    heads, kv_heads = rng.choice([(16, 8), (16, 8), (8, 8), (32, 4), (12, 4), (16, 1), (6, 2)])
    c = dict(op=op, heads=heads, kv_heads=kv_heads, dtype=rng.choice(["f16", "bf16"]),
             page=rng.choice([16, 32, 64, 128]), layout=rng.choice(["hnd", "nhd"]), ragged=rag)
    if op == "decode":
        hi = _log(rng, 16, 32768)
        # no more than 8 x 32768 positions of 4 heads in all
        c.update(seqs=_log(rng, 1, max(1, min(256, 8 * 24000 * 4 // (hi * kv_heads)))), lo=rng.randint(1, hi), hi=hi)
        return c
    if op == "append":
        q_hi = rng.choice([1, _log(rng, 2, 4000)])
        seqs = _log(rng, 1, max(1, min(256, 20000 // q_hi)))
        c.update(src=rng.choice(["f32", "f16", "bf16"]), norm=rng.random() < 0.5)
        if heads > 16:
            c.update(heads=16, kv_heads=8)
    else:
        q_hi = _log(rng, 2, 12000)
        seqs = _log(rng, 1, max(1, min(64, int(16e7 * 8 / heads / (q_hi * (q_hi + 500.0))))))
    c.update(seqs=seqs, q_lo=rng.randint(1, q_hi), q_hi=q_hi, prefix=_log(rng, 1, 500) if rng.random() < 0.7 else 0)
    return c


def _lengths(case):
    """(new rows, cached positions with them) of each sequence, from the case alone."""
    r = random.Random(case["ragged"])
    if case["op"] == "decode":
        kv = [r.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
        return [1] * case["seqs"], kv
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["seqs"])]
    return q, [n + (r.randint(0, case["prefix"]) if case["prefix"] else 0) for n in q]


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * SIZE[case["src"]] + case["rows"] * 24, "flops": 4 * n}
    q, kv = _lengths(case)
    rows, hq, hk, es = sum(q), case["heads"], case["kv_heads"], SIZE[case["dtype"]]
    if case["op"] == "append":
        made = rows * (hq + 2 * hk) * D
        return {"bytes": made * (SIZE[case["src"]] + es) + rows * D * 4, "flops": rows * (hq + hk) * D * 7}
    pairs = sum(n * k - n * (n - 1) // 2 for n, k in zip(q, kv))
    return {"bytes": 2 * rows * hq * D * es + 2 * sum(kv) * hk * D * es, "flops": 4 * pairs * hq * D}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"
    if case["op"] == "sample":
        return _prepare_sample(case, g)
    q, kv = _lengths(case)
    hq, hk, page, t = case["heads"], case["kv_heads"], case["page"], TYPES[case["dtype"]]
    rows, n = sum(q), len(q)
    need = [(k + page - 1) // page for k in kv]
    width = max(need)
    pages = sum(need) + 3
    # a pool whose pages have been handed out in any order
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    tables = torch.zeros(n, width, dtype=torch.int32, device=dev)
    mask = torch.arange(width, device=dev)[None] < torch.tensor(need, device=dev)[:, None]
    tables[mask] = order[:sum(need)]
    shape = (pages, hk, page, D) if case["layout"] == "hnd" else (pages, page, hk, D)
    state = {
        "case": case, "q_lens": q, "kv_lens": kv, "rows": rows, "seqs": n, "pages": pages, "tables": tables,
        "lens_dev": torch.tensor(kv, dtype=torch.int32, device=dev),
        "starts_dev": torch.tensor(np.concatenate([[0], np.cumsum(q)]), dtype=torch.int32, device=dev),
        "row_seq": torch.tensor(np.repeat(np.arange(n), q), device=dev),
        "row_pos": torch.tensor(np.concatenate([np.arange(k - m, k) for m, k in zip(q, kv)]), device=dev),
        "k": torch.randn(shape, generator=g, device=dev, dtype=t),
        "v": torch.randn(shape, generator=g, device=dev, dtype=t),
        "handle": None,
    }
    if case["op"] == "append":
        state["qkv"] = (torch.randn(rows, (hq + 2 * hk) * D, generator=g, device=dev) * 1.5).to(TYPES[case["src"]])
        state["q_norm"] = 1 + 0.2 * torch.randn(D, generator=g, device=dev) if case["norm"] else None
        state["k_norm"] = 1 + 0.2 * torch.randn(D, generator=g, device=dev) if case["norm"] else None
        ang = torch.arange(max(kv), device=dev, dtype=torch.float64)[:, None] * (
            1e6 ** (-torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D))
        state["rope"] = torch.stack([ang.cos(), ang.sin()], dim=-1).float().contiguous()
    else:
        # queries and keys after the head norms: scores of a few units, some keys far more alike than others
        state["q"] = (torch.randn(rows, hq, D, generator=g, device=dev) * 1.2).to(t)
    return state


def _prepare_sample(case, g):
    dev, rows, vocab = "cuda", case["rows"], case["vocab"]
    r = random.Random(case["ragged"])
    # a wide body and a few tokens well above it, as a language model's head gives
    x = torch.randn(rows, vocab, generator=g, device=dev) * 2.5
    hot = torch.randint(0, vocab, (rows, 20), generator=g, device=dev)
    x.scatter_add_(1, hot, torch.rand(rows, 20, generator=g, device=dev) * 10)
    pick = lambda a, one: [r.choice(a) if case["mix"] else one for _ in range(rows)]  # noqa: E731
    f = lambda v: torch.tensor(v, dtype=torch.float32, device=dev)  # noqa: E731
    return {
        "case": case, "logits": x.to(TYPES[case["src"]]),
        "temperature": f(pick([0.0, 0.4, 0.7, 1.0, 1.3], 0.8)),
        "top_k": torch.tensor(pick([0, 0, 5, 50, 400], 50), dtype=torch.int32, device=dev),
        "top_p": f(pick([1.0, 1.0, 0.95, 0.8, 0.5], 0.95)),
        "min_p": f(pick([0.0, 0.0, 0.02, 0.1], 0.0)),
        "uniform": torch.rand(rows, generator=g, device=dev),
        "tokens": torch.empty(rows, dtype=torch.int32, device=dev),
    }


# ---------------------------------------------------------------- the library's calls
def _package():
    """The package (its folder's name has a hyphen)."""
    name = "qwen_asr_b200"
    if name not in sys.modules:
        folder = os.path.join(os.getcwd(), "qwen-asr_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"),
                                                      submodule_search_locations=[folder])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


def _handle(s):
    """What a program keeps beside the cache: its description, the batch's and the workspace."""
    if s["handle"] is None:
        pkg, c = _package(), s["case"]
        kv = pkg.PagedKV(s["k"].data_ptr(), s["v"].data_ptr(), s["pages"], c["page"], c["kv_heads"], c["dtype"],
                         layout=c["layout"])
        starts = 0 if c["op"] == "decode" else s["starts_dev"].data_ptr()
        batch = pkg.PagedBatch(s["seqs"], s["rows"], s["lens_dev"].data_ptr(), s["tables"].data_ptr(),
                               s["tables"].shape[1], q_starts=starts)
        ws = pkg.PagedWorkspace() if c["op"] == "decode" else None
        s["handle"] = (pkg, kv, batch, ws)
    return s["handle"]


def _run_own(s):
    c = s["case"]
    st = torch.cuda.current_stream().cuda_stream
    ptr = lambda x: 0 if x is None else x.data_ptr()  # noqa: E731
    if c["op"] == "sample":
        pkg = _package()
        out = torch.empty_like(s["tokens"])
        pkg.sample(s["logits"].data_ptr(), c["rows"], c["vocab"], s["uniform"].data_ptr(), out.data_ptr(),
                   dtype=c["src"], temperature=ptr(s["temperature"]), top_k=ptr(s["top_k"]), top_p=ptr(s["top_p"]),
                   min_p=ptr(s["min_p"]), stream=st)
        return out
    pkg, kv, batch, ws = _handle(s)
    if c["op"] == "append":
        q = torch.empty(s["rows"], c["heads"], D, dtype=TYPES[c["dtype"]], device="cuda")
        pkg.paged_append(kv, batch, s["qkv"].data_ptr(), q.data_ptr(), c["heads"], dtype=c["src"],
                         q_norm=ptr(s["q_norm"]), k_norm=ptr(s["k_norm"]), eps=1e-6, rope=s["rope"].data_ptr(),
                         rope_len=s["rope"].shape[0], stream=st)
        return {"q": q, "k": s["k"], "v": s["v"]}
    out = torch.empty_like(s["q"])
    if c["op"] == "decode":
        pkg.paged_decode(kv, batch, s["q"].data_ptr(), out.data_ptr(), c["heads"], ws, stream=st)
    else:
        pkg.paged_prompt(kv, batch, s["q"].data_ptr(), out.data_ptr(), c["heads"], stream=st)
    return out


# ---------------------------------------------------------------- plain forms
def _append(s):
    c = s["case"]
    hq, hk, t, page = c["heads"], c["kv_heads"], TYPES[c["dtype"]], c["page"]
    x = s["qkv"].float().view(s["rows"], hq + 2 * hk, D)
    v = x[:, hq + hk:]
    y = x[:, :hq + hk]
    if c["norm"]:
        w = torch.cat([s["q_norm"].expand(hq, D), s["k_norm"].expand(hk, D)])
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w
    cs = s["rope"][s["row_pos"]][:, None]
    a, b = y[..., :D // 2], y[..., D // 2:]
    y = torch.cat([a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1]], dim=-1)
    pg = s["tables"][s["row_seq"], s["row_pos"] // page].long()
    at = s["row_pos"] % page
    if c["layout"] == "hnd":
        s["k"][pg, :, at] = y[:, hq:].to(t)
        s["v"][pg, :, at] = v.to(t)
    else:
        s["k"][pg, at] = y[:, hq:].to(t)
        s["v"][pg, at] = v.to(t)
    return {"q": y[:, :hq].to(t), "k": s["k"], "v": s["v"]}


def _gather(s, cache, b0, b1, n):
    """Positions 0..n-1 of sequences b0..b1-1 as f32 [seqs, kv_heads, n, D]."""
    page = s["case"]["page"]
    tab = s["tables"][b0:b1, :(n + page - 1) // page].long()
    x = cache[tab]  # [seqs, pages, (heads, page | page, heads), D]
    x = x.permute(0, 2, 1, 3, 4) if s["case"]["layout"] == "hnd" else x.permute(0, 3, 1, 2, 4)
    return x.flatten(2, 3)[:, :, :n].float()


def _softmax_product(q, k, v, seen):
    """q [b, h, r, D], k and v [b, h, n, D], seen [b, 1, r, n]: a row that sees nothing is zero."""
    p = torch.matmul(q, k.transpose(2, 3)) * D ** -0.5
    p.masked_fill_(~seen, -math.inf)
    m = p.amax(-1, keepdim=True).clamp_min(-3e38)
    p.sub_(m).exp_()
    return torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp_min(1e-38)


def _attend(s):
    """Causal attention of each sequence's new rows over its cached positions, in padded groups of
    sequences (and of rows, where one sequence is long) that keep the scores within 4 GB."""
    c = s["case"]
    hq, hk = c["heads"], c["kv_heads"]
    grp, mq, mk = hq // hk, max(s["q_lens"]), max(s["kv_lens"])
    out = torch.empty_like(s["q"])
    step = max(1, int(1e9 // (mq * mk * hq + 2 * mk * hk * D)))
    rows = max(1, min(mq, int(1e9 // (mk * hq))))
    for b0 in range(0, s["seqs"], step):
        b1 = min(s["seqs"], b0 + step)
        k, v = _gather(s, s["k"], b0, b1, mk), _gather(s, s["v"], b0, b1, mk)
        # stale positions behind a sequence's end count for nothing
        kv = s["lens_dev"][b0:b1].long()
        v = v.masked_fill((torch.arange(mk, device="cuda")[None] >= kv[:, None])[:, None, :, None], 0.0)
        first, last = s["starts_dev"][b0:b1].long(), s["starts_dev"][b0 + 1:b1 + 1].long()
        for r0 in range(0, mq, rows):
            i = torch.arange(r0, min(mq, r0 + rows), device="cuda")[None]
            at = first[:, None] + i
            real = at < last[:, None]
            pos = (kv - last)[:, None] + at
            x = s["q"][at.clamp_max(s["rows"] - 1)].float()  # [b, r, hq, D]
            x = x.view(b1 - b0, -1, hk, grp, D).permute(0, 2, 3, 1, 4).flatten(2, 3)
            seen = (torch.arange(mk, device="cuda")[None, None] <= pos[..., None])[:, None]
            o = _softmax_product(x, k, v, seen.repeat(1, 1, grp, 1))
            o = o.view(b1 - b0, hk, grp, -1, D).permute(0, 3, 1, 2, 4).reshape(b1 - b0, -1, hq, D)
            out[at[real]] = o[real].to(out.dtype)
    return out


def _sample(s):
    """In 64 bits: a draw near the border between two tokens has to fall on the same side everywhere."""
    c = s["case"]
    x = s["logits"].double()
    temp = s["temperature"].double()[:, None]
    top, order = x.sort(dim=-1, descending=True, stable=True)  # ties: lowest token first
    dead = torch.isinf(top[:, 0]) & (top[:, 0] < 0)
    w = torch.exp((top - top[:, :1]) / torch.where(temp > 0, temp, 1.0))
    rank = torch.arange(c["vocab"], device="cuda")[None]
    k = s["top_k"].long()[:, None]
    w = w * ((rank < k) | (k <= 0))
    before = w.cumsum(-1) - w
    keep = (before < s["top_p"].double()[:, None] * w.sum(-1, keepdim=True)) & (w >= s["min_p"].double()[:, None])
    keep[:, 0] = True
    w = torch.zeros_like(w).scatter_(1, order, w * keep)
    total = w.cumsum(-1)
    got = (total <= s["uniform"].double()[:, None] * total[:, -1:]).sum(-1)
    got = torch.where(temp[:, 0] > 0, got, order[:, 0])
    return torch.where(dead, -1, got).to(torch.int32)


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    return _append(state) if op == "append" else _sample(state) if op == "sample" else _attend(state)


# ---------------------------------------------------------------- definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    if case["op"] == "append":
        return _exact_append(s)
    page, hk, grp = case["page"], case["kv_heads"], case["heads"] // case["kv_heads"]
    out = torch.empty(s["rows"], case["heads"], D, dtype=torch.float64, device="cuda")
    row = 0
    for b, (n, kv) in enumerate(zip(s["q_lens"], s["kv_lens"])):
        j = torch.arange(kv, device="cuda")
        pg, at = s["tables"][b, j // page].long(), j % page
        for h in range(hk):
            k = (s["k"][pg, h, at] if case["layout"] == "hnd" else s["k"][pg, at, h]).double()
            v = (s["v"][pg, h, at] if case["layout"] == "hnd" else s["v"][pg, at, h]).double()
            for r0 in range(0, n, 2048):
                m = min(2048, n - r0)
                see = kv - n + r0 + m
                q = s["q"][row + r0:row + r0 + m, h * grp:(h + 1) * grp].double().permute(1, 0, 2)
                z = q @ k[:see].T / math.sqrt(D)
                hide = j[None, :see] > torch.arange(see - m, see, device="cuda")[:, None]
                z = torch.exp(z.masked_fill(hide, -math.inf) - z.masked_fill(hide, -math.inf).max(-1, keepdim=True)[0])
                o = (z / z.sum(-1, keepdim=True)) @ v[:see]
                out[row + r0:row + r0 + m, h * grp:(h + 1) * grp] = o.permute(1, 0, 2)
        row += n
    return out


def _exact_append(s):
    c = s["case"]
    hq, hk, page = c["heads"], c["kv_heads"], c["page"]
    x = s["qkv"].double().reshape(s["rows"], hq + 2 * hk, D)
    z = torch.complex(x[:, :hq + hk, :D // 2], x[:, :hq + hk, D // 2:])
    if c["norm"]:
        ms = x[:, :hq + hk].square().sum(-1, keepdim=True) / D
        wq, wk = s["q_norm"].double(), s["k_norm"].double()
        w = torch.stack([wq] * hq + [wk] * hk)
        z = torch.complex(z.real * w[:, :D // 2], z.imag * w[:, D // 2:]) / torch.sqrt(ms + 1e-6)
    turn = torch.complex(s["rope"][..., 0].double(), s["rope"][..., 1].double())[s["row_pos"]]
    z = z * turn[:, None]
    y = torch.cat([z.real, z.imag], dim=-1)
    k, v = s["k"].double(), s["v"].double()
    if c["layout"] == "hnd":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    page_of = s["tables"][s["row_seq"], s["row_pos"] // page].long()
    k[page_of, s["row_pos"] % page] = y[:, hq:]
    v[page_of, s["row_pos"] % page] = x[:, hq + hk:]
    if c["layout"] == "hnd":
        k, v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
    return {"q": y[:, :hq].contiguous(), "k": k, "v": v}


def _exact_sample(s):
    got = []
    logits = s["logits"].float().cpu().numpy().astype(np.float64)
    knobs = [s[n].cpu().numpy().astype(np.float64) for n in ("temperature", "top_k", "top_p", "min_p", "uniform")]
    for x, temp, k, p, floor, u in zip(logits, *knobs):
        best = int(np.argmax(x))
        if x[best] == -np.inf or temp <= 0:
            got.append(-1 if x[best] == -np.inf else best)
            continue
        w = np.exp((x - x[best]) / temp)
        order = np.lexsort((np.arange(len(x)), -x))
        if k > 0:
            order = order[:int(k)]
        ahead = np.concatenate([[0.0], np.cumsum(w[order])])
        left = order[(ahead[:-1] < p * ahead[-1]) & (w[order] >= floor)]
        left = np.sort(left if len(left) else order[:1])
        run_ = np.cumsum(w[left])
        got.append(int(left[min(len(left) - 1, np.searchsorted(run_, u * run_[-1], side="right"))]))
    return torch.tensor(got, dtype=torch.int32, device="cuda")
