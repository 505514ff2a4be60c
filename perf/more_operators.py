"""What a decoder does around its attention when it answers, as cases that can be timed and whose outputs can be compared: positions
for queries and keys, one prompt that many requests go on from, and pages that change hands.

``rotary``   ``rotary``: the heads of q and k normed and turned by the positions of their tokens in one pass; of prompts, of one new
             token a request, and with its gradients in training.
``place``    ``write_pages`` with a ``Rotary``: new keys are normed and turned on the way to their slots of a paged cache.
``prefix``   ``paged_attention`` with a ``prefix_table``: one new token of every request, the pages of their common prompt computed once.
``fork``     ``fork_requests``: requests go on from others, share their pages, or end.
``compact``  ``compact_pages``: the pages that requests hold, side by side in another pool.

q and k have unit variance (scaled scores of unit variance), lengths of a batch are spread evenly in an order that the seed gives, so a
case's work does not depend on the seed.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


def _rotary(name, B, N, Hq, Hkv, D, rot, layout, norm, stretch, start, dtype, train):
    return {"name": name, "kind": "rotary", "B": B, "N": N, "Hq": Hq, "Hkv": Hkv, "D": D, "rot": rot, "layout": layout, "norm": norm,
            "stretch": stretch, "start": start, "dtype": dtype, "train": train}


def _place(name, T, Hkv, D, rot, layout, norm, page, dtype):
    return {"name": name, "kind": "place", "T": T, "Hkv": Hkv, "D": D, "rot": rot, "layout": layout, "norm": norm, "stretch": 1.0,
            "page": page, "dtype": dtype}


def _prefix(name, B, Hq, Hkv, prompt, new, D, page, dtype, alpha):
    return {"name": name, "kind": "prefix", "B": B, "Hq": Hq, "Hkv": Hkv, "prompt": prompt, "new": new, "D": D, "page": page, "dtype": dtype,
            "alpha": alpha}


def _fork(name, groups, each, prompt, new, sample, ended, Hkv, D, page, dtype):
    return {"name": name, "kind": "fork", "groups": groups, "each": each, "prompt": prompt, "new": new, "sample": sample, "ended": ended,
            "Hkv": Hkv, "D": D, "page": page, "dtype": dtype}


def _compact(name, groups, each, prompt, new, Hkv, D, page, dtype):
    return {"name": name, "kind": "compact", "groups": groups, "each": each, "prompt": prompt, "new": new, "Hkv": Hkv, "D": D, "page": page,
            "dtype": dtype}


def listed():
    return [
        # one new token of a single request, far behind the lengths of the training: the smallest call
        _rotary("rotary_1x1_32x8_d128_bf16_far", 1, 1, 32, 8, 128, 128, "half", True, 32.0, 1000003, "bf16", False),
        # a prompt: queries and keys as a projection left them, token behind token
        _rotary("rotary_1x8190_32x8_d128_bf16", 1, 8190, 32, 8, 128, 128, "half", False, 1.0, 0, "bf16", False),
        # training with norms of queries and keys on long sequences, grouped K/V heads
        _rotary("rotary_4x8192_32x8_d128_bf16_train", 4, 8192, 32, 8, 128, 128, "half", True, 1.0, 0, "bf16", True),
        # a decoding step's keys and values on the way to their slots, neighbours turned in half of the head
        _place("place_48x8_d64_r32_f16", 48, 8, 64, 32, "interleaved", False, 16, "f16"),
        # those of prompts
        _place("place_16000x8_d128_bf16", 16000, 8, 128, 128, "half", True, 16, "bf16"),
        # a few samples of one prompt
        _prefix("prefix_4x32x8_p2000_n100_bf16", 4, 32, 8, 2000, 100, 128, 16, "bf16", 1.5),
        # many requests behind one long instruction, as a server holds them
        _prefix("prefix_64x32x8_p8192_n300_bf16", 64, 32, 8, 8192, 300, 128, 16, "bf16", 1.5),
        # questions about one very long document
        _prefix("prefix_16x32x8_p65500_n500_bf16", 16, 32, 8, 65500, 500, 128, 64, "bf16", 1.5),
        # a step of a beam search over a batch, some of which has ended
        _fork("fork_16x4_beam_p1000_bf16", 16, 4, 1000, 60, False, 1, 8, 128, 16, "bf16"),
        # one long prompt goes on in many samples
        _fork("fork_1x256_sample_p8189_bf16", 1, 256, 8189, 0, True, 0, 8, 128, 64, "bf16"),
        # the cache of a few requests moves into another pool
        _compact("compact_2x2_p200_f32", 2, 2, 200, 50, 4, 64, 16, "f32"),
        # that of a server
        _compact("compact_64x2_p2000_bf16", 64, 2, 2000, 500, 8, 128, 16, "bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm, odd as often as not."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("rotary", "rotary", "rotary", "place", "prefix", "prefix", "prefix", "fork", "fork", "compact"))
    D = rng.choice((64, 128))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    Hkv = rng.choice((2, 4, 8, 12))
    Hq = Hkv * rng.choice((1, 2, 4, 8))
    page = rng.choice((8, 16, 32, 64, 100))
    layout = rng.choice(("half", "interleaved"))
    rot = rng.choice((D, D, D // 2, D // 4, 24))
    norm = rng.random() < 0.5
    if kind == "rotary":
        train = rng.random() < 0.5
        D = rng.choice((16, 32, 64, 128, 256))
        rot = rng.choice((D, D, D // 2, 8))
        B = _spread(rng, 1, 64)
        N = 1 if not train and rng.random() < 0.3 else _spread(rng, 1, 8192)
        # half of the largest listed case
        while B > 1 and B * N * (Hq + Hkv) * D > (1 << 26):
            B //= 2
        while B * N * (Hq + Hkv) * D > (1 << 26):
            N //= 2
        case = _rotary("", B, N, Hq, Hkv, D, rot, layout, norm, rng.choice((1.0, 1.0, 4.0, 32.0)), rng.choice((0, 0, _spread(rng, 1, 1000000))),
                       dtype, train)
    elif kind == "place":
        case = _place("", _spread(rng, 1, 16000), Hkv, D, rot, layout, norm, page, dtype)
    elif kind == "prefix":
        B, prompt, new = _spread(rng, 1, 64), _spread(rng, 1, 65536), _spread(rng, 1, 2000)
        # the largest listed case's scores, an eighth of that in single precision
        most = (1 << 25) if dtype != "f32" else (1 << 22)
        while B > 1 and B * Hq * (prompt + new) > most:
            B //= 2
        while B * Hq * (prompt + new) > most:
            prompt, new = prompt // 2 + 1, new // 2 + 1
        case = _prefix("", B, Hq, Hkv, prompt, new, D, page, dtype, rng.choice((1.5, 1.5, 2.0)))
    elif kind == "fork":
        groups, each = _spread(rng, 1, 32), _spread(rng, 1, 16)
        sample = rng.random() < 0.4
        case = _fork("", groups, each, _spread(rng, 1, 4000), 0 if sample else _spread(rng, 1, 200), sample, min(groups, rng.choice((0, 1, 2))), Hkv, D, page,
                     dtype)
    else:
        case = _compact("", _spread(rng, 1, 48), _spread(rng, 1, 4), _spread(rng, 1, 1000), _spread(rng, 1, 300), Hkv, D, page, dtype)
    del case["name"]
    return case


def _lengths(B, n):
    """Lengths of a batch in ascending order: evenly spread over [n/4, n]."""
    lo = min(n, max(1, n // 4))
    return [n - (n - lo) * i // max(1, B - 1) for i in range(B)][::-1]


def _pages(tokens, page):
    return -(-tokens // page)


def _frequencies(case):
    """Radians a position, and what the turned part is multiplied with.  Stretched: fast pairs keep their frequencies, slow ones, of less than a turn in 4096
    positions, have theirs divided, with a ramp up to 32 turns."""
    rot, stretch = case["rot"], case["stretch"]
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if stretch == 1.0:
        return f.cuda(), 1.0
    turns = 4096 * f / (2 * math.pi)
    keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
    return (f / stretch * (1.0 - keep) + f * keep).cuda(), 0.1 * math.log(stretch) + 1.0


def _families(case):
    """Requests of a cache with what each group has in common: total and common pages of each request, its length, and its group."""
    page, groups, each = case["page"], case["groups"], case["each"]
    own = _lengths(groups, case["new"]) if case["new"] else [0] * groups
    prompts = _lengths(groups, case["prompt"])
    length = [prompts[g] + own[g] for g in range(groups) for _ in range(each)]
    common = [prompts[g] // page for g in range(groups) for _ in range(each)]
    return length, common


def _cache(state, case, length, common, each, spare, shuffled, normal):
    """Pages of requests of which `each` in a row share their first `common`; a request of length 0 shares none."""
    page, B = case["page"], len(length)
    first, used = [], 0
    for b in range(B):
        lead = b - b % each
        n = _pages(length[b], page)
        first.append(used)
        used += n if b == lead else (n - min(n, common[b]))
    width, pages = max(_pages(n, page) for n in length) + 1, used + spare
    col = torch.arange(width)
    n = torch.tensor([_pages(x, page) for x in length])[:, None]
    b = torch.arange(B)[:, None]
    start = torch.tensor(first)
    shared = torch.tensor(common)[:, None].clamp(max=n)
    lead = b - b % each
    at = torch.where((col < shared) & (b != lead), start[lead[:, 0]][:, None] + col, start[:, None] + col - torch.where(b == lead, 0, shared))
    pool = shuffled(pages).to(torch.int32)
    state["block_tables"] = torch.where((col < n).cuda(), pool[at.clamp(max=pages - 1).cuda()], -1).to(torch.int32)
    state["lengths"] = torch.tensor(length, dtype=torch.int32, device="cuda")
    state["free_pages"], state["free_range"] = pool, torch.tensor([used, pages], device="cuda")
    held = (col < n)
    shares = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    shares.index_add_(0, state["block_tables"][held.cuda()].long(), torch.ones(int(held.sum()), dtype=torch.int32, device="cuda"))
    state["shares"] = shares.clamp(min=0)
    state["k_pages"] = normal((pages, case["Hkv"], page, case["D"]))
    state["v_pages"] = normal((pages, case["Hkv"], page, case["D"]))
    return used


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, state = case["kind"], {"case": case}
    D, dtype = case["D"], DTYPES[case["dtype"]]

    def normal(shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    def shuffled(n):
        return torch.randperm(n, generator=g, device="cuda")

    def weight():
        return (1.0 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dtype) if case["norm"] else None

    if kind == "rotary":
        B, N, train = case["B"], case["N"], case["train"]
        state["frequencies"], state["factor"] = _frequencies(case)
        # a projection's outputs, token behind token; the heads' view of them is what the call takes
        state["q"] = normal((B, N, case["Hq"], D), 2.0).requires_grad_(train)
        state["k"] = normal((B, N, case["Hkv"], D), 2.0).requires_grad_(train)
        state["q_weight"], state["k_weight"] = weight(), weight()
        if N == 1:
            state["positions"] = case["start"] + torch.randint(0, 4000, (B, 1), generator=g, device="cuda")
        else:
            state["positions"] = case["start"] + torch.arange(N, device="cuda")
        if train:
            state["dq"], state["dk"] = normal((B, case["Hq"], N, D)), normal((B, case["Hkv"], N, D))
            for x in ("q_weight", "k_weight"):
                if state[x] is not None:
                    state[x].requires_grad_(True)
        return state
    page = case["page"]
    if kind == "place":
        T = case["T"]
        pages = _pages(T, page) + 64
        state["k_pages"], state["v_pages"] = normal((pages, case["Hkv"], page, D)), normal((pages, case["Hkv"], page, D))
        state["k"], state["v"] = normal((T, case["Hkv"], D), 2.0), normal((T, case["Hkv"], D))
        state["k_weight"] = weight()
        state["frequencies"], state["factor"] = _frequencies(case)
        # tokens of a request lie side by side in pages that lie anywhere; one in sixty-four is padding
        taken = shuffled(pages)[: _pages(T, page)]
        at = torch.arange(T, device="cuda")
        slots = taken[at // page] * page + at % page
        state["slots"] = torch.where(torch.rand(T, generator=g, device="cuda") < 1 / 64, -1, slots)
        state["positions"] = at % 3001 + torch.randint(0, 2000, (1,), generator=g, device="cuda")
        if own:
            import adasplash_amd as A

            state["rotary"] = A.Rotary(state["frequencies"], layout=case["layout"], k_weight=state["k_weight"], eps=EPS, factor=state["factor"])
        return state
    if kind == "prefix":
        B = case["B"]
        new = _lengths(B, case["new"])
        _cache(state, case, [case["prompt"] + new[int(i)] for i in shuffled(B)], [case["prompt"] // page] * B, B, 16, shuffled, normal)
        state["prefix_table"] = state["block_tables"][0, : case["prompt"] // page].clone()
        state["q"] = normal((B, case["Hq"], 1, D))
        return state
    length, common = _families(case)
    B, each = len(length), case["each"]
    if kind == "fork":
        if case["sample"]:
            length = [n if b % each == 0 else 0 for b, n in enumerate(length)]
        _cache(state, case, length, common, each, 2 * B + 16, shuffled, normal)
        b = torch.arange(B, device="cuda")
        lead = b - b % each
        parents = lead if case["sample"] else lead + torch.randint(0, each, (B,), generator=g, device="cuda")
        over = shuffled(case["groups"])[: case["ended"]]
        state["parents"] = torch.where(torch.isin(b // each, over), -1, parents)
        return state
    used = _cache(state, case, length, common, each, 64, shuffled, normal)
    shape = (used + 40, case["Hkv"], page, D)
    state["k_to"], state["v_to"] = (torch.zeros(shape, dtype=dtype, device="cuda") for _ in range(2))
    return state


def _cos_sin(positions, frequencies, factor):
    angle = positions.double()[..., None] * frequencies
    return (angle.cos() * factor).float(), (angle.sin() * factor).float()


def _pairs(x, rot, layout):
    """Both elements of the turned pairs, and the rest of the head."""
    t = x[..., :rot]
    a, b = (t[..., : rot // 2], t[..., rot // 2:]) if layout == "half" else (t[..., 0::2], t[..., 1::2])
    return a, b, x[..., rot:]


def _joined(a, b, rest, layout):
    t = torch.cat([a, b], -1) if layout == "half" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([t, rest], -1)


def _turned(x, weight, cos, sin, case):
    """Heads normed (with a weight) and turned, in 32 bits; and the normed head without its weight."""
    x = x.float()
    xn = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) if weight is not None else x
    a, b, rest = _pairs(xn * weight.float() if weight is not None else xn, case["rot"], case["layout"])
    return _joined(a * cos - b * sin, b * cos + a * sin, rest, case["layout"]), xn


def _plain_rotary(state):
    case = state["case"]
    cos, sin = _cos_sin(state["positions"], state["frequencies"], state["factor"])
    outs, grads, weights = [], [], []
    for x, w, do in (("q", "q_weight", "dq"), ("k", "k_weight", "dk")):
        w = state[w].detach() if state[w] is not None else None
        x = state[x].detach().transpose(1, 2)
        c, s = (t[:, None] if t.dim() == 3 else t for t in (cos, sin))
        out, xn = _turned(x, w, c, s, case)
        outs.append(out.to(x.dtype))
        if case["train"]:
            a, b, rest = _pairs(state[do].float(), case["rot"], case["layout"])
            dn = _joined(a * c + b * s, b * c - a * s, rest, case["layout"])
            if w is not None:
                weights.append((dn * xn).sum((0, 1, 2), dtype=torch.float64).to(w.dtype))
                dn = dn * w.float()
                x = x.float()
                dn = (dn - xn * (dn * xn).mean(-1, keepdim=True)) * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
            grads.append(dn.to(out.dtype if x.dtype == torch.float32 and case["dtype"] == "f32" else DTYPES[case["dtype"]]).transpose(1, 2))
    return outs + grads + weights


def _plain_place(state):
    case = state["case"]
    cos, sin = _cos_sin(state["positions"], state["frequencies"], state["factor"])
    k = _turned(state["k"], state["k_weight"], cos[:, None], sin[:, None], case)[0].to(state["k"].dtype)
    slots, page = state["slots"], case["page"]
    keep = slots >= 0
    at = slots[keep]
    for new, pages in ((k, "k_pages"), (state["v"], "v_pages")):
        state[pages][at // page, :, at % page] = new[keep]
    return [state["k_pages"], state["v_pages"]]


def _entmax(x, alpha):
    """alpha-entmax of the last dimension for alpha = 1.5 and 2; a row of -inf is a row of zeros."""
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
    return u if alpha == 2.0 else u * u


def _plain_prefix(state):
    """The pages of the prompt against the queries of all requests at once, what lies behind them request by request."""
    case, tables = state["case"], state["block_tables"]
    B, Hq, Hkv, D, page = (case[x] for x in ("B", "Hq", "Hkv", "D", "page"))
    G, front = Hq // Hkv, state["prefix_table"].numel()
    tail = tables[:, front:]
    n = tail.shape[1] * page
    own_k, own_v = (state[x][tail.clamp(min=0).long()].transpose(1, 2).reshape(B, Hkv, n, D).float() for x in ("k_pages", "v_pages"))
    k, v = (state[x][state["prefix_table"].long()].transpose(0, 1).reshape(Hkv, front * page, D).float() for x in ("k_pages", "v_pages"))
    q = state["q"].float().view(B, Hkv, G, D)
    rows = q.transpose(0, 1).reshape(Hkv, B * G, D)
    x = (rows @ k.transpose(-1, -2).contiguous()).view(Hkv, B, G, front * page).transpose(0, 1)
    y = (q @ own_k.transpose(-1, -2).contiguous()).masked_fill(
        ~(torch.arange(n, device="cuda") < (state["lengths"] - front * page)[:, None])[:, None, None, :], -math.inf)
    p = _entmax(torch.cat([x, y], -1) / math.sqrt(D), case["alpha"])
    out = (p[..., : front * page].transpose(0, 1).reshape(Hkv, B * G, front * page) @ v).view(Hkv, B, G, D).transpose(0, 1)
    return (out + p[..., front * page:] @ own_v).reshape(B, Hq, 1, D).to(state["q"].dtype)


def _plain_fork(state):
    case = state["case"]
    page, tables, free, shares = case["page"], state["block_tables"], state["free_pages"], state["shares"]
    B, width = tables.shape
    first, end = state["free_range"].unbind()
    parents, held = state["parents"], state["lengths"].long()
    b, col = torch.arange(B, device="cuda"), torch.arange(width, device="cuda")
    has, src = parents >= 0, parents.clamp(min=0)
    count = torch.zeros_like(held).index_add_(0, src, has.long())
    full, rest = held // page, held % page
    partly = (col == full[:, None]) & (rest > 0)[:, None]
    held_cols = (col < full[:, None]) | partly
    old = tables.clone()
    # holders of each page behind the step, less one
    shares.index_add_(0, old[held_cols].long(), (torch.where(partly, count.clamp(max=1)[:, None], count[:, None]) - 1)[held_cols].to(torch.int32))
    gone = old[held_cols].long()
    gone = gone[shares[gone] < 0]
    order = torch.arange(gone.numel(), device="cuda")
    seen = torch.full((shares.numel(),), gone.numel(), device="cuda").scatter_reduce_(0, gone, order, "amin")
    gone = gone[seen[gone] == order]
    shares[gone] = 0
    free[(end + torch.arange(gone.numel(), device="cuda")) % free.numel()] = gone.to(torch.int32)
    # the last page of a request that several go on from: one keeps it, the others copy it
    heir = torch.full_like(held, B).scatter_reduce_(0, src[has], b[has], "amin")
    heir = torch.where(parents == b, b, heir)
    copies = has & (rest[src] > 0) & (heir[src] != b)
    rank = copies.cumsum(0) - 1
    got = copies & (rank < end + gone.numel() - first)
    fresh = free[(first + rank).clamp(min=0) % free.numel()]
    n = torch.where(has, full[src] + ((rest[src] > 0) & (~copies | got)).long(), 0)
    rows = torch.where(col < n[:, None], old[src], -1)
    rows = torch.where(got[:, None] & (col == full[src][:, None]), fresh[:, None], rows)
    tables.copy_(torch.where((parents == b)[:, None], old, rows))
    state["lengths"].copy_(torch.where(has, torch.where(copies & ~got, full[src] * page, held[src]), 0))
    state["free_range"].copy_(torch.stack([first + got.sum(), end + gone.numel()]))
    to, of = fresh[got].long(), old[src, full[src].clamp(max=width - 1)][got].long()
    mask = (torch.arange(page, device="cuda") < rest[src][got][:, None])[:, None, :, None]
    for x in ("k_pages", "v_pages"):
        state[x][to] = torch.where(mask, state[x][of], state[x][to])
    return _forked(state)


def _forked(state):
    return [state[x] for x in ("block_tables", "lengths", "shares", "free_pages", "free_range", "k_pages", "v_pages")]


def _plain_compact(state):
    page, tables, held, k_to, v_to = state["case"]["page"], state["block_tables"], state["lengths"], state["k_to"], state["v_to"]
    cols = torch.arange(tables.shape[1], device="cuda") < ((held + page - 1) // page)[:, None]
    pages = tables[cols].long()
    order = torch.arange(pages.numel(), device="cuda")
    seen = torch.full((state["k_pages"].shape[0],), pages.numel(), device="cuda").scatter_reduce_(0, pages, order, "amin")
    lead = seen[pages] == order
    number = torch.zeros_like(seen).index_copy_(0, pages[lead], lead.cumsum(0)[lead] - 1)
    moved = pages[lead]
    k_to[: moved.numel()], v_to[: moved.numel()] = state["k_pages"][moved], state["v_pages"][moved]
    new = torch.full_like(tables, -1)
    new[cols] = number[pages].to(torch.int32)
    room = k_to.shape[0]
    shares = torch.zeros(room, dtype=torch.int32, device="cuda").index_add_(0, number[pages], (~lead).to(torch.int32))
    free = (torch.arange(room, device="cuda") + moved.numel()) % room
    return [held.clone(), new, shares, free.to(torch.int32), torch.tensor([0, room - moved.numel()], device="cuda"), k_to, v_to]


def _own(state):
    import adasplash_amd as A

    case = state["case"]
    if case["kind"] == "rotary":
        q, k = state["q"], state["k"]
        outs = A.rotary(q.transpose(1, 2), k.transpose(1, 2), state["positions"], state["frequencies"], layout=case["layout"], q_weight=state["q_weight"],
                        k_weight=state["k_weight"], eps=EPS, factor=state["factor"])
        if not case["train"]:
            return list(outs)
        leaves = [q, k] + ([state["q_weight"], state["k_weight"]] if case["norm"] else [])
        return [x.detach() for x in outs] + list(torch.autograd.grad(outs, leaves, (state["dq"], state["dk"])))
    if case["kind"] == "place":
        A.write_pages(state["k"], state["v"], state["slots"], state["k_pages"], state["v_pages"], positions=state["positions"], rotary=state["rotary"])
        return [state["k_pages"], state["v_pages"]]
    if case["kind"] == "prefix":
        return A.paged_attention(state["q"], state["k_pages"], state["v_pages"], state["block_tables"], state["lengths"], alpha=case["alpha"],
                                 prefix_table=state["prefix_table"])
    if case["kind"] == "fork":
        A.fork_requests(state["parents"], state["lengths"], state["block_tables"], state["free_pages"], state["free_range"], state["shares"],
                        state["k_pages"], state["v_pages"])
        return _forked(state)
    return [*A.compact_pages(state["lengths"], state["block_tables"], state["k_pages"], state["v_pages"], state["k_to"], state["v_to"]), state["k_to"],
            state["v_to"]]


def run(state):
    if own:
        return _own(state)
    return {"rotary": _plain_rotary, "place": _plain_place, "prefix": _plain_prefix, "fork": _plain_fork, "compact": _plain_compact}[
        state["case"]["kind"]](state)


def work(case):
    kind, size, D = case["kind"], 4 if case["dtype"] == "f32" else 2, case["D"]
    if kind == "rotary":
        tokens, elems = case["B"] * case["N"], case["B"] * case["N"] * (case["Hq"] + case["Hkv"]) * D
        # in and out; in training the gradients of the outputs in and those of q and k out, and with norms q and k once more
        passes = 2 if not case["train"] else 4 + (1 if case["norm"] else 0)
        return {"bytes": passes * size * elems + 8 * tokens, "flops": elems * (6 + (4 if case["norm"] else 0)) * (3 if case["train"] else 1)}
    if kind == "place":
        return {"bytes": 4 * size * case["T"] * case["Hkv"] * D + 16 * case["T"], "flops": case["T"] * case["Hkv"] * D * (10 if case["norm"] else 6)}
    page, Hkv = case["page"], case["Hkv"]
    if kind == "prefix":
        B, front = case["B"], case["prompt"] // page * page
        own_keys = sum(case["prompt"] - front + n for n in _lengths(B, case["new"]))
        # every key once, the prompt's for all requests together; of the values the supports' rows only, whose number the scores decide: not counted
        return {"bytes": size * D * (Hkv * (front + own_keys) + 2 * B * case["Hq"]) + 4 * B * (case["prompt"] + case["new"]) // page,
                "flops": 2 * D * case["Hq"] * (B * front + own_keys)}
    length, common = _families(case)
    each, row = case["each"], 2 * size * Hkv * D  # K and V of a token
    if kind == "fork":
        groups = range(case["ended"] * each, len(length))
        if case["sample"]:
            copied = sum(length[b] % page for b in groups if b % each)
        else:  # (of four that choose among four, some two and a half are chosen)
            copied = sum(length[b] % page for b in groups) * (1.0 - (1.0 - (1.0 - 1.0 / each) ** each))
        entries = sum(_pages(n, page) for n in length)
        # old tables in, new ones out, holders of the pages, rows in and out
        return {"bytes": int(2 * row * copied + 16 * entries), "flops": 0}
    held = sum(_pages(n, page) - (min(c, _pages(n, page)) if b % each else 0) for b, (n, c) in enumerate(zip(length, common)))
    return {"bytes": 2 * row * page * held + 8 * sum(_pages(n, page) for n in length), "flops": 0}


def _exact_turn(x, weight, positions, case, frequencies, factor, back=False):
    """Heads (..., D) in 64 bits, normed where there is a weight and turned as complex numbers by positions (...,); back: turned the other way, not normed."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()
    rot, half = case["rot"], case["layout"] == "half"
    i = torch.arange(rot // 2, device=x.device)
    re, im = (i, i + rot // 2) if half else (2 * i, 2 * i + 1)
    turn = torch.polar(torch.full_like(frequencies, factor).expand(*positions.shape, -1).contiguous(), positions.double()[..., None] * frequencies)
    z = torch.complex(x[..., re], x[..., im]) * (turn.conj() if back else turn)
    y = x.clone()
    y[..., re], y[..., im] = z.real, z.imag
    return y


def _exact_rotary(case, state):
    outs, grads, weights = [], [], []
    at = state["positions"].expand(case["B"], case["N"])
    for name in ("q", "k"):
        x, w = state[name].detach(), state[name + "_weight"]
        w = w.detach() if w is not None else None
        y, dx = torch.empty(x.transpose(1, 2).shape, dtype=torch.float64, device="cuda"), torch.empty(x.shape, dtype=torch.float64, device="cuda")
        dw = torch.zeros(x.shape[-1], dtype=torch.float64, device="cuda")
        for h in range(x.shape[2]):  # head by head: the angles are the same
            xh = x[:, :, h]
            y[:, h] = _exact_turn(xh, w, at, case, state["frequencies"], state["factor"])
            if not case["train"]:
                continue
            dn = _exact_turn(state["d" + name][:, h], None, at, case, state["frequencies"], state["factor"], back=True)
            if w is not None:
                xd = xh.double()
                size = (xd.square().mean(-1, keepdim=True) + EPS).sqrt()
                dw += (dn * xd / size).sum((0, 1))
                dn = dn * w.double()
                dn = dn / size - xd * (dn * xd).mean(-1, keepdim=True) / size ** 3
            dx[:, :, h] = dn
        outs.append(y)
        if case["train"]:
            grads.append(dx)
            if w is not None:
                weights.append(dw)
    return outs + grads + weights


def _exact_rows(x, alpha):
    """alpha-entmax of the rows of x in 64 bits: the threshold by bisection, and two steps of Newton's method behind it."""
    z = x * (alpha - 1.0)
    top = z.amax(-1, keepdim=True)
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
    return (z - t).clamp(min=0).pow(power)


def exact(case, seed):
    kind, state = case["kind"], prepare(case, seed)
    if kind == "rotary":
        return _exact_rotary(case, state)
    page = case["page"]
    if kind == "place":
        k = _exact_turn(state["k"].transpose(0, 1), state["k_weight"], state["positions"].expand(case["Hkv"], -1), case, state["frequencies"],
                        state["factor"]).transpose(0, 1)
        pages = [state["k_pages"].double(), state["v_pages"].double()]
        there = (state["slots"].cpu() >= 0).nonzero()[:, 0].cuda()
        for to, new in zip(pages, (k, state["v"].double())):
            rows = to.permute(0, 2, 1, 3).reshape(-1, case["Hkv"], case["D"])
            rows.index_copy_(0, state["slots"][there], new[there])
            to.copy_(rows.view(to.shape[0], page, case["Hkv"], case["D"]).permute(0, 2, 1, 3))
        return pages
    if kind == "prefix":
        G, D = case["Hq"] // case["Hkv"], case["D"]
        out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
        for b in range(case["B"]):
            n = int(state["lengths"][b])
            at = torch.arange(n, device="cuda")
            where = state["block_tables"][b].long()[at // page]
            k, v = (state[x][where, :, at % page].transpose(0, 1) for x in ("k_pages", "v_pages"))
            for h in range(case["Hkv"]):
                heads = slice(h * G, (h + 1) * G)
                x = state["q"][b, heads, 0].double() @ k[h].double().T / math.sqrt(D)
                out[b, heads, 0] = _exact_rows(x, case["alpha"]) @ v[h].double()
        return out
    tables, lengths = state["block_tables"].tolist(), state["lengths"].tolist()
    k, v = state["k_pages"].double(), state["v_pages"].double()
    if kind == "compact":
        number, to = {}, [state["k_to"].double(), state["v_to"].double()]
        for b, n in enumerate(lengths):
            for p in tables[b][: _pages(n, page)]:
                number.setdefault(p, len(number))
        of = torch.tensor(list(number), device="cuda")
        to[0][: len(number)], to[1][: len(number)] = k[of], v[of]
        return [None] * 5 + to
    # the last page of a request goes to itself, or to the first that goes on from it; the others take pages in their order, those that the step frees behind the others
    parents = state["parents"].tolist()
    first, end = state["free_range"].tolist()
    ring = state["free_pages"].tolist()
    free = [ring[i % len(ring)] for i in range(first, end)]
    kept = {p for s, n in enumerate(lengths) if s in parents for p in tables[s][: _pages(n, page)]}
    for s, n in enumerate(lengths):
        for p in tables[s][: _pages(n, page)]:
            if p not in kept:
                kept.add(p)
                free.append(p)
    heir, copies = {}, []
    for b, s in enumerate(parents):
        if s >= 0:
            heir.setdefault(s, s if parents[s] == s else b)
    for b, s in enumerate(parents):
        if s >= 0 and lengths[s] % page and heir[s] != b and free:
            copies.append((tables[s][lengths[s] // page], free.pop(0), lengths[s] % page))
    for of, to, rows in copies:
        k[to, :, :rows], v[to, :, :rows] = k[of, :, :rows].clone(), v[of, :, :rows].clone()
    return [None] * 5 + [k, v]
