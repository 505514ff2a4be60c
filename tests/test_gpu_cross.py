"""Attention to keys of another length on the GPU: forward and gradients against 64 bits."""

import pytest
import torch

import adasplash_amd as A
from tests import op_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def inputs(B, Hq, Hkv, Nq, Nk, D, dtype, seed=0, q_scale=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(shape, generator=g) for shape in ((B, Hq, Nq, D), (B, Hkv, Nk, D), (B, Hkv, Nk, D), (B, Hq, Nq, D)))
    return [t.to(dtype) for t in (q * q_scale, k, v, do)]


def reference(q, k, v, do, alpha, lq, lk, train):
    """(want, tolerance) of output, dq, dk and dv."""
    B, Hq, Nq, D = q.shape
    Hkv = k.shape[1]
    G = Hq // Hkv
    res = [[torch.zeros(t.shape, dtype=torch.float64) for _ in range(2)] for t in (q, q, k, v)]
    for b in range(B):
        m, n = lq[b], lk[b]
        for h in range(Hkv):
            hs = slice(h * G, (h + 1) * G)
            qq, dd = (t[b, hs, :m].reshape(G * m, D) for t in (q, do))
            kk, vv = k[b, h, :n], v[b, h, :n]
            for to, x in zip(res[0], ref.attend(qq, kk, vv, alpha, roundings=2)):
                to[b, hs, :m] = x.view(G, m, D)
            if train:
                for i, pair in enumerate(ref.gradients(qq, kk, vv, dd, alpha)):
                    for to, x in zip(res[i + 1], pair):
                        if i == 0:
                            to[b, hs, :m] = x.view(G, m, D)
                        else:
                            to[b, h, :n] = x
    return res


def spoil(t, lens, value=float("nan")):
    """The padding holds anything."""
    t = t.clone()
    for b, n in enumerate(lens):
        t[b, :, n:] = value
    return t


def run_case(B, Hq, Hkv, Nq, Nk, D, dtype, alpha=1.5, lq=None, lk=None, q_scale=1.0, train=True, bits=torch.int32, value=float("nan"), seed=0):
    what = f"B={B} Hq={Hq} Hkv={Hkv} Nq={Nq} Nk={Nk} D={D} {dtype} alpha={alpha} lq={lq} lk={lk} q*{q_scale}"
    print(what, flush=True)
    q, k, v, do = inputs(B, Hq, Hkv, Nq, Nk, D, dtype, seed, q_scale)
    fq, fk = lq or [Nq] * B, lk or [Nk] * B
    want = reference(q, k, v, do, alpha, fq, fk, train)
    if lq:
        q, do = spoil(q, lq, value), spoil(do, lq, value)
    if lk:
        k, v = spoil(k, lk, value), spoil(v, lk, value)
    args = {"alpha": alpha}
    if lq:
        args["varlen_q"] = torch.tensor(lq, dtype=bits, device=DEV)
    if lk:
        args["varlen_k"] = torch.tensor(lk, dtype=bits, device=DEV)
    q, k, v, do = (t.to(DEV) for t in (q, k, v, do))
    out = A.cross_attention(q, k, v, **args)
    ref.check(out, *want[0], what + " out")
    assert torch.equal(out, A.cross_attention(q, k, v, **args))
    if train:
        q, k, v = (t.requires_grad_(True) for t in (q, k, v))
        out = A.cross_attention(q, k, v, **args)
        ref.check(out, *want[0], what + " out of a training step")
        grads = torch.autograd.grad(out, (q, k, v), do, retain_graph=True)
        for name, got, pair in zip(("dq", "dk", "dv"), grads, want[1:]):
            ref.check(got, *pair, what + " " + name)
        for a, b in zip(grads, torch.autograd.grad(out, (q, k, v), do)):
            assert torch.equal(a, b)
    return out


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
def test_types_and_head_dims(dtype, D):
    run_case(2, 4, 2, 70, 150, D, dtype)
    run_case(2, 2, 2, 150, 33, D, dtype, lq=[150, 7], lk=[1, 33])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("alpha", [1.05, 1.125, 1.25, 1.333, 1.75, 2.0])
def test_alphas(dtype, alpha):
    run_case(1, 2, 1, 65, 200, 64, dtype, alpha=alpha)
    run_case(1, 2, 2, 40, 90, 128, dtype, alpha=alpha, lk=[77])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Nq, Nk", [(1, 1), (1, 2), (2, 1), (1, 65), (3, 1000), (31, 32), (32, 31), (33, 33), (64, 127), (127, 64), (128, 129), (129, 128), (300, 1), (17, 513), (5, 1025),
                                    (40, 2048), (40, 2049), (600, 20)])
def test_lengths(dtype, Nq, Nk):
    run_case(1, 2, 1, Nq, Nk, 64, dtype)
    run_case(1, 1, 1, Nq, Nk, 128, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_padded_batches(dtype, D):
    lq, lk = [0, 1, 100, 64, 33, 100, 5], [130, 0, 1, 64, 129, 130, 65]
    run_case(7, 4, 2, 100, 130, D, dtype, lq=lq, lk=lk, bits=torch.int64)
    run_case(7, 2, 2, 100, 130, D, dtype, lq=lq, value=float("inf"))
    run_case(7, 2, 1, 100, 130, D, dtype, lk=lk, value=float("-inf"))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_spreads_over_many_keys(dtype):
    for q_scale in (0.03, 0.25, 1.0, 4.0):
        run_case(1, 2, 1, 130, 2500, 64, dtype, q_scale=q_scale)
        run_case(1, 1, 1, 33, 1100, 128, dtype, q_scale=q_scale, lk=[1030])


@pytest.mark.parametrize("group", [1, 2, 3, 8, 17])
def test_groups(group):
    run_case(2, group * 2, 2, 20, 90, 64, BF16, lq=[20, 3], lk=[41, 90])
    run_case(1, group, 1, 1, 300, 64, BF16, train=False)
    run_case(1, group, 1, 1, 300, 64, F32, train=False)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
def test_a_few_queries(dtype, D):
    run_case(2, 4, 2, 3, 700, D, dtype, lq=[3, 1], lk=[700, 65])
    run_case(3, 2, 2, 1, 70, D, dtype, lk=[0, 70, 1])
    run_case(1, 16, 1, 1, 300, D, dtype)
    run_case(2, 3, 1, 5, 64, D, dtype, lq=[0, 5])


@pytest.mark.parametrize("keep", ["never", "always"])
def test_a_few_queries_and_what_is_kept(keep):
    before = A.set_keep_supports(keep)
    try:
        run_case(2, 4, 2, 3, 700, 64, BF16, lq=[3, 1], lk=[700, 65])
        run_case(1, 4, 2, 2, 5000, 128, F32)
    finally:
        A.set_keep_supports(before)


@pytest.mark.parametrize("alpha", [1.05, 1.25, 1.333, 1.75, 2.0])
def test_a_few_queries_and_alphas(alpha):
    for dtype in (F32, BF16):
        run_case(1, 4, 2, 2, 5000, 64, dtype, alpha=alpha)
        run_case(1, 2, 1, 4, 900, 128, dtype, alpha=alpha, lk=[897])


@pytest.mark.parametrize("n", [600, 2049, 6000])
def test_a_few_queries_of_equal_scores(n):
    """Every key is a member, more than a list holds from some thousand on: u is the same for all, delta their mean dP."""
    for D, dtype in ((64, F32), (128, BF16)):
        q, k, v, do = inputs(1, 2, 1, 2, n, D, dtype)
        q.zero_()
        ts = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
        out = A.cross_attention(*ts)
        want = reference(q, k, v, do, 1.5, [2], [n], True)
        ref.check(out, *want[0], f"equal scores n={n} {dtype}")
        for name, got, pair in zip(("dq", "dk", "dv"), torch.autograd.grad(out, ts, do.to(DEV)), want[1:]):
            ref.check(got, *pair, f"equal scores n={n} {dtype} {name}")


SUPPORTS = 10, 4, 2, 1030, 2600, 128  # large enough, padding included, for the kernels on the supports: queries and keys of odd lengths, two query heads a key head
SUPPORTS_LENGTHS = {"lq": [1030, 77, 0, 1, 128, 129, 5, 33, 64, 200], "lk": [2599, 1400, 2600, 700, 0, 1, 2500, 65, 2048, 300]}


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("alpha", [1.125, 1.5, 1.75, 2.0])
def test_supports(dtype, alpha):
    run_case(*SUPPORTS, dtype, alpha=alpha, q_scale=2.0, **SUPPORTS_LENGTHS)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_supports_of_narrow_heads(dtype):
    run_case(12, 3, 1, 1030, 4700, 64, dtype, lq=[1030] + [40, 1] * 5 + [0], lk=[4700] + [4699, 3000] * 5 + [9])
    run_case(6, 9, 9, 1025, 1537, 64, dtype, lq=[0, 1025, 1, 128, 129, 33], lk=[1537, 0, 1537, 1, 700, 65])


def test_supports_of_many_queries_over_few_keys_and_of_few_over_many():
    run_case(2, 8, 4, 9000, 600, 128, BF16, lq=[1200, 3000])
    run_case(2, 12, 12, 65, 40000, 128, BF16, lk=[9001, 300])
    run_case(8, 70, 70, 33, 2305, 128, F16, q_scale=3.0, lq=[33, 1, 0, 2, 5, 3, 32, 4])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
def test_many_queries_over_few_keys(dtype, D):
    run_case(3, 8, 2, 700, 40, D, dtype, lq=[700, 0, 290], lk=[33, 40, 1])
    run_case(2, 2, 2, 1501, 3, D, dtype, lq=[1501, 800], lk=[3, 0])
    run_case(1, 6, 1, 400, 130, D, dtype, q_scale=0.1)


@pytest.mark.parametrize("keep", ["never", "always"])
@pytest.mark.parametrize("alpha", [1.25, 1.5, 2.0])
def test_many_row_blocks_over_few_keys(keep, alpha):
    """More row blocks than run at once: one or two waves a row block."""
    before = A.set_keep_supports(keep)
    try:
        for D, Nk in ((64, 25), (128, 32), (64, 1), (128, 64), (64, 33)):
            run_case(3, 8, 2, 700, Nk, D, F32, alpha=alpha, lq=[700, 0, 290], lk=[Nk, Nk, (Nk + 1) // 2])
            run_case(3, 8, 8, 690, Nk, D, F32, alpha=alpha, q_scale=0.05)
    finally:
        A.set_keep_supports(before)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("alpha", [1.25, 1.5, 2.0])
def test_many_row_blocks_over_few_keys_in_16_bits(dtype, alpha):
    for D, Nk in ((64, 25), (128, 32), (64, 1), (128, 128), (64, 97)):
        run_case(3, 8, 2, 700, Nk, D, dtype, alpha=alpha, lq=[700, 0, 290], lk=[Nk, Nk, (Nk + 1) // 2])
    run_case(3, 8, 8, 690, 70, 128, dtype, alpha=alpha, q_scale=0.05)


def test_supports_of_more_query_rows_than_16_bits_name():
    run_case(1, 8, 1, 9000, 600, 128, BF16, lq=[1100])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_more_keys_than_16_bits_name(dtype, D):
    run_case(1, 2, 1, 40, 66000, D, dtype, train=D == 64)
    run_case(1, 1, 1, 1, 66000, D, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_alpha_close_to_one(dtype):
    for alpha in (1.01, 1.001):
        run_case(1, 2, 1, 40, 200, 64, dtype, alpha=alpha)
        run_case(1, 2, 1, 2, 2500, 128, dtype, alpha=alpha)


@pytest.mark.parametrize("shape", [(2, 4, 2, 3, 700, 64, F32), (2, 4, 2, 100, 700, 64, F32), (2, 4, 2, 100, 700, 64, BF16), (2, 4, 2, 100, 700, 32, F16), (2, 4, 2, 40, 2500, 128, F16), (*SUPPORTS, BF16)])
def test_scratch_may_hold_anything(shape):
    q, k, v, do = (t.to(DEV) for t in inputs(*shape, q_scale=2.0))
    lens = {"varlen_q": torch.tensor([1, 77] * (shape[0] // 2), device=DEV), "varlen_k": torch.tensor([500, 0] * (shape[0] // 2), device=DEV)}

    def step(args):
        ts = [t.clone().requires_grad_(True) for t in (q, k, v)]
        out = A.cross_attention(*ts, **args)
        with torch.no_grad():
            return out.detach(), A.cross_attention(q, k, v, **args), *torch.autograd.grad(out, ts, do)

    for args in ({}, lens):
        results = []
        for fill in (0, 255, 1, 127):
            torch.cuda.synchronize()
            torch.cuda.empty_cache()
            soil = torch.full((2 << 30,), fill, dtype=torch.uint8, device=DEV)  # (what the allocator hands out next)
            soil_small = [torch.full((1 << 19,), fill, dtype=torch.uint8, device=DEV) for _ in range(64)]
            del soil, soil_small
            results.append(step(args))
        for other in results[1:]:
            for a, b in zip(results[0], other):
                assert torch.equal(a, b)


def test_few_queries_of_a_batch_in_more_than_one_launch():
    """64 rows of 131072 keys: 64 MiB of workspace an item."""
    B, Nk, D = 20, 131072, 32
    g = torch.Generator(device=DEV).manual_seed(0)
    q = torch.randn(B, 64, 1, D, generator=g, device=DEV).to(BF16)
    k = torch.randn(1, 1, Nk, D, generator=g, device=DEV).to(BF16).repeat(B, 1, 1, 1)
    lens = torch.tensor([1000 + b for b in range(B)], device=DEV)
    out = A.cross_attention(q, k, k, varlen_k=lens)
    for b in (0, 15, 16, 19):
        want, tol = ref.attend(q[b, :, 0].cpu(), k[b, 0, :1000 + b].cpu(), k[b, 0, :1000 + b].cpu(), 1.5, roundings=2)
        ref.check(out[b, :, 0], want, tol, f"item {b}")


@pytest.mark.parametrize("q_scale", [0.02, 0.2])
def test_supports_of_flat_scores(q_scale):
    run_case(*SUPPORTS, BF16, q_scale=q_scale, **SUPPORTS_LENGTHS)


@pytest.mark.parametrize("keep", ["never", "always"])
def test_supports_of_some_rows_and_heads_only(keep):
    """Rows of equal scores among sharp ones (their row blocks overflow the lists), a flat head, an item without keys."""
    B, Hq, Hkv, Nq, Nk, D = 3, 4, 2, 1030, 2600, 128
    q, k, v, do = inputs(B, Hq, Hkv, Nq, Nk, D, BF16, seed=3, q_scale=2.0)
    q[0, 1, 100:110] = 0
    q[0, 2:] *= 0.01
    q[2, :, -1] = 0
    lq, lk = [1030, 900, 1030], [2600, 0, 2048]
    want = reference(q, k, v, do, 1.5, lq, lk, True)
    ts = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    lens = {"varlen_q": torch.tensor(lq, device=DEV), "varlen_k": torch.tensor(lk, device=DEV)}
    before = A.set_keep_supports(keep)
    try:
        out = A.cross_attention(*ts, **lens)
        grads = torch.autograd.grad(out, ts, do.to(DEV))
    finally:
        A.set_keep_supports(before)
    for name, got, pair in zip(("out", "dq", "dk", "dv"), (out, *grads), want):
        ref.check(got, *pair, f"{name}, supports kept {keep}")


@pytest.mark.parametrize("keep", ["never", "always"])
@pytest.mark.parametrize("D, alpha", [(64, 1.5), (128, 1.5), (64, 1.25), (128, 2.0), (64, 1.75)])
def test_lists_kept_in_single_precision(keep, D, alpha):
    """Sharp rows, a row block of equal scores, whose lists overflow, a row of one member, items without queries or keys."""
    B, Hq, Hkv, Nq, Nk = 4, 4, 2, 170, 1100
    q, k, v, do = inputs(B, Hq, Hkv, Nq, Nk, D, F32, seed=5, q_scale=2.0)
    q[0, 1, 70] = 0
    q[1, 0, :40] *= 40
    v[1] += 30
    lq, lk = [170, 129, 0, 33], [1100, 901, 500, 0]
    want = reference(q, k, v, do, alpha, lq, lk, True)
    ts = [t.to(DEV).requires_grad_(True) for t in (spoil(q, lq), spoil(k, lk), spoil(v, lk))]
    lens = {"varlen_q": torch.tensor(lq, device=DEV), "varlen_k": torch.tensor(lk, device=DEV)}
    before = A.set_keep_supports(keep)
    try:
        out = A.cross_attention(*ts, alpha=alpha, **lens)
        grads = torch.autograd.grad(out, ts, spoil(do, lq).to(DEV))
    finally:
        A.set_keep_supports(before)
    for name, got, pair in zip(("out", "dq", "dk", "dv"), (out, *grads), want):
        ref.check(got, *pair, f"{name}, lists kept {keep}, D={D} alpha={alpha}")


@pytest.mark.parametrize("keep", ["never", "always"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D, alpha", [(64, 1.5), (128, 1.5), (64, 1.25), (128, 2.0)])
def test_lists_kept_in_16_bits(keep, dtype, D, alpha):
    """As above, with more keys than a workgroup's registers hold."""
    B, Hq, Hkv, Nq, Nk = 4, 4, 2, 170, 2300
    q, k, v, do = inputs(B, Hq, Hkv, Nq, Nk, D, dtype, seed=5, q_scale=2.0)
    q[0, 1, 70] = 0
    q[1, 0, :40] *= 40
    lq, lk = [170, 129, 0, 33], [2300, 901, 500, 0]
    want = reference(q, k, v, do, alpha, lq, lk, True)
    ts = [t.to(DEV).requires_grad_(True) for t in (spoil(q, lq), spoil(k, lk), spoil(v, lk))]
    lens = {"varlen_q": torch.tensor(lq, device=DEV), "varlen_k": torch.tensor(lk, device=DEV)}
    before = A.set_keep_supports(keep)
    try:
        out = A.cross_attention(*ts, alpha=alpha, **lens)
        grads = torch.autograd.grad(out, ts, spoil(do, lq).to(DEV))
    finally:
        A.set_keep_supports(before)
    for name, got, pair in zip(("out", "dq", "dk", "dv"), (out, *grads), want):
        ref.check(got, *pair, f"{name}, lists kept {keep}, D={D} alpha={alpha}")


def test_a_captured_training_step_on_the_supports():
    q, k, v, do = (t.to(DEV) for t in inputs(*SUPPORTS, BF16, q_scale=2.0))
    lens = torch.tensor(SUPPORTS_LENGTHS["lk"], device=DEV)

    def step(*ts):
        out = A.cross_attention(*ts, varlen_k=lens)
        return out, *torch.autograd.grad(out, ts, do)

    ts = [t.detach().requires_grad_(True) for t in (q, k, v)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(*ts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step(*ts)
    for i in range(4):
        q.copy_(torch.randn(q.shape).to(BF16))
        lens[1] = 700 * i
        graph.replay()
        torch.cuda.synchronize()
        # (other leaves of the same numbers: what the graph captured belongs to its own)
        for a, b in zip(results, step(*(t.detach().clone().requires_grad_(True) for t in (q, k, v)))):
            assert torch.equal(a, b)


def test_lengths_beyond_the_tensor_and_below_zero():
    q, k, v, do = (t.to(DEV) for t in inputs(2, 2, 2, 10, 20, 64, BF16))
    full = A.cross_attention(q, k, v)
    for n in (1, 10):
        a, b = q[:, :, :n].contiguous(), A.cross_attention(q, k, v, varlen_q=torch.tensor([99, -5], device=DEV), varlen_k=torch.tensor([10 ** 12, 20], device=DEV))
        assert torch.equal(b[0], full[0]) and (b[1] == 0).all()
        c = A.cross_attention(a, k, v, varlen_k=torch.tensor([2 ** 40, -1], device=DEV))
        assert torch.isfinite(c).all() and (c[1] == 0).all() and (c[0] != 0).any()


@pytest.mark.parametrize("shape", [(2, 4, 2, 3, 700, 64, F32), (2, 4, 2, 100, 700, 64, F32), (2, 4, 2, 100, 700, 64, BF16)])
def test_lengths_changed_between_forward_and_backward(shape):
    q, k, v, do = (t.to(DEV) for t in inputs(*shape))
    for name in ("varlen_q", "varlen_k"):
        ts = [t.clone().requires_grad_(True) for t in (q, k, v)]
        lens = torch.tensor([2, 1], device=DEV)
        out = A.cross_attention(*ts, **{name: lens})
        lens.fill_(3)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out, ts, do)


def test_nothing_to_do():
    q, k, v, do = (t.to(DEV) for t in inputs(2, 2, 2, 10, 20, 64, BF16))
    for t in (q, k, v):
        t.requires_grad_(True)
    assert A.cross_attention(q[:, :, :0].contiguous(), k, v).shape == (2, 2, 0, 64)
    out = A.cross_attention(q, k[:, :, :0].contiguous(), v[:, :, :0].contiguous())
    assert (out == 0).all()
    dq, dk = torch.autograd.grad(out, (q, k), do)
    assert (dq == 0).all() and (dk == 0).all()
    empty = A.cross_attention(q[:0], k[:0], v[:0])
    assert empty.shape == (0, 2, 10, 64)


def test_only_some_inputs_want_a_gradient():
    q, k, v, do = (t.to(DEV) for t in inputs(1, 4, 2, 20, 30, 64, F32))
    wants = [t.clone().requires_grad_(True) for t in (q, k, v)]
    all3 = torch.autograd.grad(A.cross_attention(*wants), wants, do)
    for i in range(3):
        args = [w if j == i else t for j, (w, t) in enumerate(zip(wants, (q, k, v)))]
        got, = torch.autograd.grad(A.cross_attention(*args), (wants[i],), do)
        assert torch.equal(got, all3[i])
    # an upstream gradient of another layout
    odd = do.transpose(1, 2).contiguous().transpose(1, 2)
    for a, b in zip(torch.autograd.grad(A.cross_attention(*wants), wants, odd), all3):
        assert torch.equal(a, b)


def test_the_gradient_is_the_difference():
    """fp32 outputs of the kernel itself, 0.02 apart along a direction; alpha = 1.333 has two continuous derivatives."""
    q, k, v, do = (t.to(DEV) for t in inputs(1, 2, 1, 40, 100, 64, F32))
    for i in range(3):
        ts = [t.clone().requires_grad_(True) for t in (q, k, v)]
        out = A.cross_attention(*ts, alpha=1.333)
        got, = torch.autograd.grad(out, (ts[i],), do)
        way = torch.randn(got.shape, generator=torch.Generator().manual_seed(i)).to(DEV)
        h = 0.01
        with torch.no_grad():
            ends = []
            for sign in (1, -1):
                moved = [q, k, v]
                moved[i] = moved[i] + sign * h * way
                ends.append((A.cross_attention(*moved, alpha=1.333).double() * do.double()).sum())
        slope = ((ends[0] - ends[1]) / (2 * h)).item()
        # central differences of a step h are off by h^2 / 6 times a third derivative of the loss's size (some thousand terms of order one add up to some
        # fifty), and by fp32's roundings of the outputs over 2 h
        assert abs(slope - (got.double() * way.double()).sum().item()) < 0.02 * abs(slope) + 0.2


def test_same_lengths_agree_with_the_block_mask_variant():
    q, k, v, do = (t.to(DEV) for t in inputs(2, 4, 4, 256, 256, 64, F32))
    a, b = A.cross_attention(q, k, v), A.adasplash_v1(q, k, v)
    assert torch.equal(a, b)  # (the same kernel on the same numbers)


def test_offsets_beyond_32_bits():
    """K and V of more than 2^31 elements; only the last item's head is looked at."""
    B, Nk, D = 2100, 8192, 128
    k = torch.zeros(B, 1, Nk, D, dtype=F16, device=DEV)
    k[-1] = torch.randn(1, Nk, D, device=DEV)
    q = torch.randn(B, 1, 3, D, device=DEV).to(F16)
    want, tol = ref.attend(q[-1, 0].cpu(), k[-1, 0].cpu(), k[-1, 0].cpu(), 1.5, roundings=2)
    ref.check(A.cross_attention(q, k, k)[-1, 0], want, tol, "split over the keys")
    q = q.expand(B, 1, 3, D).repeat(1, 1, 7, 1)
    out = A.cross_attention(q, k, k)
    ref.check(out[-1, 0, :3], want, tol, "rows")


def test_two_streams_at_once():
    cases = [[t.to(DEV) for t in inputs(2, 4, 2, n, 700, 64, BF16, seed=n)] for n in (1, 1, 40, 130, 1, 40)]
    want = [A.cross_attention(q, k, v) for q, k, v, _ in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, (q, k, v, _) in enumerate(cases):
        with torch.cuda.stream(streams[i % 2]):
            got.append(A.cross_attention(q, k, v))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_a_captured_forward():
    lens = torch.tensor([700, 3], device=DEV)
    for n in (1, 40):
        q, k, v, _ = (t.to(DEV) for t in inputs(2, 4, 2, n, 700, 64, BF16))
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            A.cross_attention(q, k, v, varlen_k=lens)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = A.cross_attention(q, k, v, varlen_k=lens)
        for i in range(4):
            q.copy_(torch.randn(q.shape).to(BF16))
            lens[1] = 100 * i
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, A.cross_attention(q, k, v, varlen_k=lens))


def test_a_decoder_layer_generates_what_it_was_trained_on():
    """Two layers' worth of a decoder: self attention over a paged cache and attention to an encoder's states, token by token, against the whole sequence at
    once (causal self attention in 64 bits)."""
    from adasplash_amd.paged import PagedCache
    from oracle import exact

    g = torch.Generator().manual_seed(9)
    B, Hq, Hkv, D, T, S = 2, 4, 2, 64, 12, 50
    q, xq = (torch.randn(B, Hq, T, D, generator=g).to(DEV) for _ in range(2))
    k, v = (torch.randn(B, Hkv, T, D, generator=g).to(DEV) for _ in range(2))
    ek, ev = (torch.randn(B, Hkv, S, D, generator=g).to(DEV) for _ in range(2))
    lens = torch.tensor([50, 31], device=DEV)
    whole_self = exact.dense_entmax_attention(*(t.cpu() for t in (q, k, v)), 1.5, True)
    whole_cross = A.cross_attention(xq, ek, ev, varlen_k=lens)
    cache = PagedCache(10, 4, B, Hkv, D, T, dtype=F32)
    for t in range(T):
        cache.append(k[:, :, t:t + 1], v[:, :, t:t + 1])
        step = cache.attend(q[:, :, t:t + 1])
        assert (step.double().cpu() - whole_self[:, :, t:t + 1]).abs().max() < 1e-4
        step = A.cross_attention(xq[:, :, t:t + 1].contiguous(), ek, ev, varlen_k=lens)
        # (two fp32 results of the same sums in another order: both within the tolerance of fp32 parity, 1e-4)
        assert (step - whole_cross[:, :, t:t + 1]).abs().max() < 1e-4
