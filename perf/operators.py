"""Sparse entmax attention of a decoder that reads an encoder's states and keeps its own in pages, as cases that can be timed
and whose outputs can be compared.

``cross``   ``cross_attention``: queries of a decoder against an encoder's keys and values of another length, padded batches and
            grouped K/V heads; a forward pass, a training step with the gradients of q, k and v, or one new token a sequence.
``paged``   ``paged_attention``: one new token of every request against its keys in a paged cache.
``tables``  ``build_block_tables``: the pages and slots of the tokens that a step adds to the requests.
``write``   ``write_pages``: the keys and values of those tokens go to their slots in the cache.

Scores have the spread that ``q_scale`` gives: with unit-variance q and k the scaled scores have unit variance; 3 is a peaked
distribution, 0.125 a flat one.  Lengths of a batch are spread evenly over [n/4, n] in an order that the seed gives, so a case's
work does not depend on the seed.  The plain form takes the threshold of a row from its sorted values (alpha = 1.5 and 2, where it has a
closed form).
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _cross(name, B, Hq, Hkv, Nq, Nk, D, dtype, alpha, q_scale, padded, train):
    return {"name": name, "kind": "cross", "B": B, "Hq": Hq, "Hkv": Hkv, "Nq": Nq, "Nk": Nk, "D": D, "dtype": dtype, "alpha": alpha,
            "q_scale": q_scale, "padded": padded, "train": train}


def _paged(name, B, Hq, Hkv, N, D, page, dtype, alpha, q_scale):
    return {"name": name, "kind": "paged", "B": B, "Hq": Hq, "Hkv": Hkv, "N": N, "D": D, "page": page, "dtype": dtype, "alpha": alpha,
            "q_scale": q_scale}


def _tables(name, B, held, new, page):
    return {"name": name, "kind": "tables", "B": B, "held": held, "new": new, "page": page}


def _write(name, T, Hkv, D, page, dtype):
    return {"name": name, "kind": "write", "T": T, "Hkv": Hkv, "D": D, "page": page, "dtype": dtype}


def listed():
    return [
        # the smallest call: a sentence through a small translation model in single precision
        _cross("cross_1x8_q40_k57_d64_f32", 1, 8, 8, 40, 57, 64, "f32", 1.5, 1.0, False, False),
        # fine-tuning a translation or summary model on padded batches
        _cross("cross_16x12_q130_k500_d64_bf16_train", 16, 12, 12, 130, 500, 64, "bf16", 1.5, 1.0, True, True),
        # training in single precision on padded batches: transcripts of recordings
        _cross("cross_2x8_q448_k1500_d64_f32_train", 2, 8, 8, 448, 1500, 64, "f32", 1.5, 1.0, True, True),
        # a training step of a large decoder on long documents, grouped K/V heads
        _cross("cross_4x32x8_q1024_k5000_d128_bf16_train", 4, 32, 8, 1024, 5000, 128, "bf16", 1.5, 1.0, True, True),
        # one new token a sequence against the encoder's states, as a generating loop calls it
        _cross("cross_32x16_q1_k1500_d64_f16", 32, 16, 16, 1, 1500, 64, "f16", 1.5, 1.0, True, False),
        # one request of a few hundred tokens: the smallest decoding step
        _paged("paged_1x32x8_k600_d128_bf16", 1, 32, 8, 600, 128, 16, "bf16", 1.5, 1.0),
        # a batch of requests of all lengths, as a server holds them
        _paged("paged_48x32x8_k8192_d128_bf16", 48, 32, 8, 8192, 128, 16, "bf16", 1.5, 1.0),
        # two requests with very long contexts
        _paged("paged_2x32x8_k131071_d128_bf16", 2, 32, 8, 131071, 128, 64, "bf16", 1.5, 1.0),
        # a decoding step of a large batch: a token a request
        _tables("tables_256_new1_page16", 256, 4000, 1, 16),
        # prompts that enter: tens of thousands of tokens in one step
        _tables("tables_64_new1000_page16", 64, 500, 1000, 16),
        # a decoding step's keys and values
        _write("write_256x8_d128_bf16", 256, 8, 128, 16, "bf16"),
        # those of prompts
        _write("write_32000x8_d128_bf16", 32000, 8, 128, 16, "bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm, odd as often as not."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("cross", "cross", "cross", "cross", "paged", "paged", "paged", "tables", "write"))
    D = rng.choice((64, 128))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    q_scale = rng.choice((1.0, 1.0, 3.0, 0.125))
    Hkv = rng.choice((4, 8, 12, 16))
    Hq = Hkv * rng.choice((1, 1, 2, 4))
    page = rng.choice((8, 16, 32, 64, 100))
    if kind == "tables":
        new = rng.choice((1, _spread(rng, 2, 1000)))
        B = _spread(rng, 1, 256 if new == 1 else 64)
        case = _tables("", B, _spread(rng, 1, 8192), new, page)
    elif kind == "write":
        case = _write("", _spread(rng, 1, 32000), rng.choice((4, 8)), D, page, dtype)
    elif kind == "paged":
        N = _spread(rng, 1, 131071)
        B = _spread(rng, 1, 64)
        # no more than half of the largest listed case's cache, nor scores than that
        while B > 1 and (B * Hkv * N * D > (1 << 27) or B * Hq * N > (1 << 23)):
            B //= 2
        if B * Hkv * N * D > (1 << 27):
            N = (1 << 27) // (Hkv * D)
        case = _paged("", B, Hq, Hkv, N, D, page, dtype, rng.choice((1.5, 1.5, 2.0)), q_scale)
    else:
        train = rng.random() < 0.5
        Nq = 1 if not train and rng.random() < 0.3 else _spread(rng, 1, 2048)
        Nk = _spread(rng, 1, 8192)
        B = _spread(rng, 1, 32)
        # a tenth of the largest listed case's products, a quarter of that in single precision
        most = (1 << 27) if dtype != "f32" else (1 << 25)
        while B > 1 and B * Hq * Nq * Nk * D > 64 * most:
            B //= 2
        while B * Hq * Nq * Nk * D > 64 * most:
            Nk //= 2
        # (sparsemax's gradient jumps where a value crosses the threshold: in training 1.5)
        alpha = 1.5 if train else rng.choice((1.5, 1.5, 2.0))
        case = _cross("", B, Hq, Hkv, Nq, Nk, D, dtype, alpha, q_scale, rng.random() < 0.6, train)
    del case["name"]
    return case


def _lengths(B, n, padded=True):
    """Lengths of a batch in ascending order: evenly spread over [n/4, n]."""
    if not padded:
        return [n] * B
    lo = max(1, n // 4)
    return [n - (n - lo) * i // max(1, B - 1) for i in range(B)][::-1]


def _held(case):
    """Tokens that each request holds, and those that are new to it."""
    held = _lengths(case["B"], case["held"])
    return held, [1] * case["B"] if case["new"] == 1 else _lengths(case["B"], case["new"])


def _pages(tokens, page):
    return -(-tokens // page)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, state = case["kind"], {"case": case}

    def normal(shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(DTYPES[case["dtype"]])

    def shuffled(n):
        return torch.randperm(n, generator=g, device="cuda")

    def lengths(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")[shuffled(len(values))]

    if kind == "cross":
        B, D = case["B"], case["D"]
        state["q"] = normal((B, case["Hq"], case["Nq"], D), case["q_scale"]).requires_grad_(case["train"])
        state["k"] = normal((B, case["Hkv"], case["Nk"], D)).requires_grad_(case["train"])
        state["v"] = normal((B, case["Hkv"], case["Nk"], D)).requires_grad_(case["train"])
        # (a queue of single tokens has no padding among its queries)
        order = shuffled(B)
        ql, kl = _lengths(B, case["Nq"]), _lengths(B, case["Nk"])
        state["varlen_q"] = torch.tensor(ql, dtype=torch.int32, device="cuda")[order] if case["padded"] and case["Nq"] > 1 else None
        state["varlen_k"] = torch.tensor(kl, dtype=torch.int32, device="cuda")[order] if case["padded"] else None
        if case["train"]:
            state["dout"] = normal((B, case["Hq"], case["Nq"], D))
        return state
    page = case["page"]
    if kind == "write":
        T = case["T"]
        pages = _pages(T, page) + 64
        state["k_pages"] = normal((pages, case["Hkv"], page, case["D"]))
        state["v_pages"] = normal((pages, case["Hkv"], page, case["D"]))
        state["k"] = normal((T, case["Hkv"], case["D"]))
        state["v"] = normal((T, case["Hkv"], case["D"]))
        # tokens of a request lie side by side in pages that lie anywhere; one in sixty-four is padding
        taken = shuffled(pages)[: _pages(T, page)]
        at = torch.arange(T, device="cuda")
        slots = taken[at // page] * page + at % page
        state["slots"] = torch.where(torch.rand(T, generator=g, device="cuda") < 1 / 64, -1, slots)
        return state
    if kind == "paged":
        B, N = case["B"], case["N"]
        held = lengths(_lengths(B, N))
        width, pages = _pages(N, page), sum(_pages(n, page) for n in _lengths(B, N)) + 16
        state["k_pages"] = normal((pages, case["Hkv"], page, case["D"]))
        state["v_pages"] = normal((pages, case["Hkv"], page, case["D"]))
        state["q"] = normal((B, case["Hq"], 1, case["D"]), case["q_scale"])
        state["lengths"] = held
        new = held
        before = torch.zeros_like(held)
    else:
        held, new = _held(case)
        width = max(_pages(h + n, page) for h, n in zip(sorted(held), sorted(new))) + 1
        state["total"] = sum(new)
        pages = sum(_pages(h, page) + _pages(n, page) + 1 for h, n in zip(held, new))
        order = shuffled(case["B"])
        before = torch.tensor(held, dtype=torch.int32, device="cuda")[order]
        new = torch.tensor(new, dtype=torch.int32, device="cuda")[order]
        state["lengths"], state["new_tokens"] = before, new
    # pages that a request has: those behind the pages of the requests in front of it, in a shuffled pool
    pool = shuffled(pages).to(torch.int32)
    have = (new + page - 1) // page if kind == "paged" else (before + page - 1) // page
    first = have.cumsum(0) - have
    col = torch.arange(width, device="cuda")
    at = (first[:, None] + col).clamp(max=pages - 1)
    state["block_tables"] = torch.where(col < have[:, None], pool[at], -1).to(torch.int32)
    if kind == "tables":
        state["free_pages"] = pool
        state["free_range"] = torch.stack([have.sum(), torch.tensor(pages, device="cuda")]).to(torch.int64)
    return state


def _entmax(x, alpha):
    """alpha-entmax of the last dimension for alpha = 1.5 and 2, and p^(2 - alpha); a row of -inf is a row of zeros."""
    z = x * (alpha - 1.0)
    z = z - z.amax(-1, keepdim=True).clamp(min=-1e30)
    # (far below any support, and its square is still a number; sums of thousands of values in 64 bits)
    s = z.sort(-1, descending=True).values.clamp(min=-1e4).double()
    k = torch.arange(1, s.shape[-1] + 1, device=s.device, dtype=s.dtype)
    if alpha == 2.0:
        tau = (s.cumsum(-1) - 1.0) / k
    else:
        mean = s.cumsum(-1) / k
        tau = mean - ((1.0 - ((s * s).cumsum(-1) - k * mean * mean)) / k).clamp(min=0.0).sqrt()
    size = (tau < s).sum(-1, keepdim=True).clamp(min=1)
    u = (z - tau.gather(-1, size - 1).float()).clamp(min=0.0)
    return (u, (u > 0).to(u.dtype)) if alpha == 2.0 else (u * u, u)


def _below(lengths, n, B):
    """(B, n): the places in front of each length."""
    at = torch.arange(n, device="cuda")
    return (at < lengths[:, None]) if lengths is not None else torch.ones(B, n, dtype=torch.bool, device="cuda")


def _plain_cross(state):
    case = state["case"]
    B, Hq, Hkv, Nq, Nk, D = (case[x] for x in ("B", "Hq", "Hkv", "Nq", "Nk", "D"))
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(D)
    rows = _below(state["varlen_q"], Nq, B)[:, None, None, :, None]
    keys = _below(state["varlen_k"], Nk, B)[:, None, None, None, :]
    q = state["q"].detach().float().view(B, Hkv, G * Nq, D)
    k, v = state["k"].detach().float(), state["v"].detach().float()
    x = (q @ k.transpose(-1, -2)).view(B, Hkv, G, Nq, Nk) * scale
    p, u = _entmax(x.masked_fill(~keys, -math.inf), case["alpha"])
    p = (p * rows).view(B, Hkv, G * Nq, Nk)
    out = (p @ v).view(state["q"].shape).to(state["q"].dtype)
    if not case["train"]:
        return out
    do = state["dout"].float().view(B, Hkv, G * Nq, D)
    u = (u * rows).view(B, Hkv, G * Nq, Nk)
    dp = do @ v.transpose(-1, -2)
    delta = (u * dp).sum(-1, keepdim=True) / u.sum(-1, keepdim=True).clamp(min=1e-30)
    ds = u * (dp - delta) * scale
    dq, dk, dv = ds @ k, ds.transpose(-1, -2) @ q, p.transpose(-1, -2) @ do
    return [out, dq.view(state["q"].shape).to(out.dtype), dk.to(out.dtype), dv.to(out.dtype)]


def _plain_paged(state):
    case, tables = state["case"], state["block_tables"]
    B, Hq, Hkv, D, page = (case[x] for x in ("B", "Hq", "Hkv", "D", "page"))
    n = tables.shape[1] * page
    k, v = (state[x][tables.clamp(min=0).long()].transpose(1, 2).reshape(B, Hkv, n, D).float() for x in ("k_pages", "v_pages"))
    x = state["q"].float().view(B, Hkv, Hq // Hkv, D) @ k.transpose(-1, -2) / math.sqrt(D)
    keys = _below(state["lengths"], n, B)[:, None, None, :]
    p, _ = _entmax(x.masked_fill(~keys, -math.inf), case["alpha"])
    return (p @ v).view(B, Hq, 1, D).to(state["q"].dtype)


def _plain_tables(state):
    page, total = state["case"]["page"], state["total"]
    tables, free, (first, end) = state["block_tables"], state["free_pages"], state["free_range"].unbind()
    held, new = state["lengths"].long(), state["new_tokens"].long()
    width = tables.shape[1]
    have = (held + page - 1) // page
    need = ((held + new + page - 1) // page).clamp(max=width) - have
    upto = need.cumsum(0)
    got = ((end - first) - (upto - need)).clamp(min=0).minimum(need)
    col = torch.arange(width, device="cuda")
    new_col = (col >= have[:, None]) & (col < (have + got)[:, None])
    at = (first + (upto - need)[:, None] + col - have[:, None]) % free.numel()
    tables.copy_(torch.where(new_col, free[at], tables))
    after = torch.minimum(held + new, (have + got) * page)
    # the tokens of a step lie request behind request
    ends = new.cumsum(0)
    token = torch.arange(total, device="cuda")
    of = torch.searchsorted(ends, token, right=True).clamp(max=len(new) - 1)
    pos = held[of] + token - (ends - new)[of]
    there = tables[of, (pos // page).clamp(max=width - 1)].long()
    slots = torch.where((pos < after[of]) & (token < ends[-1]), there * page + pos % page, -1)
    taken = torch.minimum(upto[-1], end - first)
    return [tables, slots, after.to(torch.int32), torch.stack([first + taken, end])]


def _plain_write(state):
    slots, page = state["slots"], state["case"]["page"]
    keep = slots >= 0
    at = slots[keep]
    for new, pages in (("k", "k_pages"), ("v", "v_pages")):
        state[pages][at // page, :, at % page] = state[new][keep]
    return [state["k_pages"], state["v_pages"]]


def _own(state):
    import adasplash_amd as A

    case = state["case"]
    if case["kind"] == "cross":
        q, k, v = state["q"], state["k"], state["v"]
        out = A.cross_attention(q, k, v, alpha=case["alpha"], varlen_q=state["varlen_q"], varlen_k=state["varlen_k"])
        if not case["train"]:
            return out
        return [out.detach(), *torch.autograd.grad(out, (q, k, v), state["dout"])]
    if case["kind"] == "paged":
        return A.paged_attention(state["q"], state["k_pages"], state["v_pages"], state["block_tables"], state["lengths"], alpha=case["alpha"])
    if case["kind"] == "tables":
        slots, after, left = A.build_block_tables(state["lengths"], state["new_tokens"], state["block_tables"], state["free_pages"],
                                                  state["free_range"], page_size=case["page"], total_tokens=state["total"])
        return [state["block_tables"], slots, after, left]
    A.write_pages(state["k"], state["v"], state["slots"], state["k_pages"], state["v_pages"])
    return [state["k_pages"], state["v_pages"]]


def run(state):
    if own:
        return _own(state)
    return {"cross": _plain_cross, "paged": _plain_paged, "tables": _plain_tables, "write": _plain_write}[state["case"]["kind"]](state)


def work(case):
    kind = case["kind"]
    if kind == "tables":
        held, new = _held(case)
        pages = sum(_pages(h + n, case["page"]) - _pages(h, case["page"]) for h, n in zip(held, new))
        # lengths in and out, a free page read and an entry of a table written for each new page, a slot written for each token
        return {"bytes": 12 * case["B"] + 8 * pages + 8 * sum(new), "flops": 0}
    size = 4 if case["dtype"] == "f32" else 2
    D, Hkv = case["D"], case["Hkv"]
    if kind == "write":
        return {"bytes": 4 * size * case["T"] * Hkv * D + 8 * case["T"], "flops": 0}
    if kind == "paged":
        keys = sum(_lengths(case["B"], case["N"]))
        # every key once; of the values only the supports' rows are needed, whose number the scores decide: not counted
        return {"bytes": size * D * (Hkv * keys + 2 * case["B"] * case["Hq"]) + 4 * keys // case["page"], "flops": 2 * D * case["Hq"] * keys}
    B, Hq, Nq, Nk = case["B"], case["Hq"], case["Nq"], case["Nk"]
    ql, kl = _lengths(B, Nq, case["padded"] and Nq > 1), _lengths(B, Nk, case["padded"])
    pairs = Hq * sum(a * b for a, b in zip(ql, kl))
    q_elems, kv_elems = D * Hq * sum(ql), D * Hkv * sum(kl)
    if not case["train"]:
        values = 1 if Nq > 1 else 0  # (a single query reads its support's values only, as above)
        return {"bytes": size * (q_elems + D * Hq * B * Nq + (1 + values) * kv_elems), "flops": (2 + 2 * values) * D * pairs}
    # two products forward, four more for the gradients (dP, dV, dK, dQ); outputs and gradients are written to the end of the padding
    return {"bytes": size * (2 * q_elems + 2 * kv_elems + 2 * D * Hq * B * Nq + 2 * D * Hkv * B * Nk), "flops": 12 * D * pairs}


def _exact_rows(x, alpha):
    """alpha-entmax of the rows of x in 64 bits, and p^(2 - alpha): the threshold by bisection, and two steps of Newton's method behind it."""
    z = x * (alpha - 1.0)
    top = z.amax(-1, keepdim=True)
    some = torch.isfinite(top)
    top = torch.where(some, top, 0.0)
    power = 1.0 / (alpha - 1.0)
    lo, hi = top - 1.0, top.clone()
    for _ in range(44):
        mid = (lo + hi) / 2
        over = (z - mid).clamp(min=0).pow_(power).sum(-1, keepdim=True) > 1.0
        lo, hi = torch.where(over, mid, lo), torch.where(over, hi, mid)
    t = lo
    for _ in range(2):
        u = (z - t).clamp(min=0)
        t = t + (u.pow(power).sum(-1, keepdim=True) - 1.0) / (power * u.pow(power - 1.0).mul_(u > 0).sum(-1, keepdim=True)).clamp(min=1e-300)
    u = torch.where(some, (z - t).clamp(min=0), 0.0)
    return u.pow(power), torch.where(u > 0, u.pow((2.0 - alpha) * power), 0.0)


def exact(case, seed):
    if case["kind"] == "tables":
        return None
    state = prepare(case, seed)
    if case["kind"] == "write":
        pages = [state["k_pages"].double(), state["v_pages"].double()]
        slots = state["slots"].cpu()
        there = (slots >= 0).nonzero()[:, 0].cuda()
        for to, new in zip(pages, (state["k"], state["v"])):
            rows = to.permute(0, 2, 1, 3).reshape(-1, case["Hkv"], case["D"])
            rows.index_copy_(0, state["slots"][there], new[there].double())
            to.copy_(rows.view(to.shape[0], case["page"], case["Hkv"], case["D"]).permute(0, 2, 1, 3))
        return pages
    D, G, train = case["D"], case["Hq"] // case["Hkv"], case.get("train", False)
    outs = {x: torch.zeros(state[x].shape, dtype=torch.float64, device="cuda") for x in (("q", "k", "v") if train else ())}
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["B"]):
        if case["kind"] == "paged":
            n, m, page = int(state["lengths"][b]), 1, case["page"]
            at = torch.arange(n, device="cuda")
            where = state["block_tables"][b].long()[at // page]
            k, v = (state[x][where, :, at % page].transpose(0, 1) for x in ("k_pages", "v_pages"))
        else:
            m = case["Nq"] if state["varlen_q"] is None else int(state["varlen_q"][b])
            n = case["Nk"] if state["varlen_k"] is None else int(state["varlen_k"][b])
            k, v = state["k"].detach()[b, :, :n], state["v"].detach()[b, :, :n]
        for h in range(case["Hkv"]):
            heads = slice(h * G, (h + 1) * G)
            q = state["q"].detach()[b, heads, :m].double().reshape(G * m, D)
            kk, vv = k[h].double(), v[h].double()
            p, u = _exact_rows(q @ kk.T / math.sqrt(D), case["alpha"])
            out[b, heads, :m] = (p @ vv).view(G, m, D)
            if train:
                do = state["dout"][b, heads, :m].double().reshape(G * m, D)
                dp = do @ vv.T
                ds = u * (dp - (u * dp).sum(-1, keepdim=True) / u.sum(-1, keepdim=True)) / math.sqrt(D)
                outs["q"][b, heads, :m] = (ds @ kk).view(G, m, D)
                outs["k"][b, h, :n], outs["v"][b, h, :n] = ds.T @ q, p.T @ do
    return [out, outs["q"], outs["k"], outs["v"]] if train else out
