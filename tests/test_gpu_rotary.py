"""Heads normed and turned by positions on the GPU: types, head dims, layouts, views, gradients, and the way into a cache's pages."""

import pytest
import torch

import adasplash_amd as A
from tests import positions_reference as pos
from tests.op_reference import check

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def weights_of(D, dtype, g):
    return [(1 + 0.3 * torch.randn(D, generator=g)).to(dtype) for _ in range(2)]


def run(q, k, positions, rot, layout, weights=(None, None), eps=1e-6, factor=1.0, train=True, what="", base=10000.0):
    """q, k on the CPU, as the call takes them; forward and gradients against the reference."""
    print(what, tuple(q.shape), None if k is None else tuple(k.shape), q.dtype, "rot", rot, layout, flush=True)
    f = pos.frequencies_of(rot, base)
    g = torch.Generator().manual_seed(11)
    leaves = [t.to(DEV).requires_grad_(train) if t is not None else None for t in (q, k, *weights)]
    qd, kd, qw, kw = leaves
    outs = A.rotary(qd, kd, positions.to(DEV), f.to(DEV), layout=layout, q_weight=qw, k_weight=kw, eps=eps, factor=factor)
    assert (outs[1] is None) == (k is None)
    douts, tokens = [], (lambda t: positions if t.dim() == 4 and positions.dim() == 1 else (positions[:, None] if t.dim() == 4 else positions[:, None]))
    for name, x, w, out in (("q", q, weights[0], outs[0]), ("k", k, weights[1], outs[1])):
        if x is None:
            continue
        assert out.shape == x.shape and out.dtype == x.dtype and out.is_contiguous()
        want, tol = pos.forward_tolerance(x, tokens(x), f, layout, w, eps, factor)
        check(out, want, tol, f"{what} {name}")
        douts.append(torch.randn(x.shape, generator=g).to(x.dtype))
    if not train:
        return outs
    wanted = [t for t in leaves if t is not None]
    grads = torch.autograd.grad([o for o in outs if o is not None], wanted, [d.to(DEV) for d in douts])
    grads = dict(zip([id(t) for t in wanted], grads))
    for name, x, w, xd, wd, dy in (("q", q, weights[0], qd, qw, douts[0]), ("k", k, weights[1], kd, kw, douts[-1])):
        if x is None:
            continue
        (dx, dx_tol), more = pos.backward(x, dy, tokens(x), f, layout, w, eps, factor)
        check(grads[id(xd)], dx, dx_tol, f"{what} d{name}")
        assert grads[id(xd)].dtype == x.dtype
        if w is not None:
            check(grads[id(wd)], more[0], more[1], f"{what} d{name}_weight")
            assert grads[id(wd)].dtype == w.dtype
    return outs


def heads(B, H, N, D, dtype, seed=0, scale=1.5):
    return (torch.randn(B, H, N, D, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_types_and_head_dims(dtype, D, layout):
    q, k = heads(2, 6, 37, D, dtype, 1), heads(2, 3, 37, D, dtype, 2)
    g = torch.Generator().manual_seed(3)
    for norm in (False, True):
        for rot in sorted({D, D // 2 // 8 * 8, 8}):
            run(q, k, torch.arange(37) * 5, rot, layout, weights_of(D, dtype, g) if norm else (None, None), what=f"norm={norm}")


@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 255, 1000, 4099])
def test_lengths(N):
    g = torch.Generator().manual_seed(3)
    run(heads(1, 4, N, 128, BF16, 1), heads(1, 1, N, 128, BF16, 2), torch.arange(N), 128, "half", weights_of(128, BF16, g), what="length")
    run(heads(3, 2, N, 64, F32, 1), heads(3, 2, N, 64, F32, 2), torch.arange(N), 32, "interleaved", weights_of(64, F32, g), what="length")


@pytest.mark.parametrize("Hq, Hkv", [(1, 1), (7, 7), (9, 3), (33, 11), (64, 8)])
def test_heads(Hq, Hkv):
    run(heads(2, Hq, 21, 64, BF16, 1), heads(2, Hkv, 21, 64, BF16, 2), torch.arange(21), 64, "half", weights_of(64, BF16, torch.Generator().manual_seed(3)), what="heads")


def test_positions():
    q, k = heads(3, 4, 19, 64, F32, 1), heads(3, 2, 19, 64, F32, 2)
    g = torch.Generator().manual_seed(4)
    each = torch.randint(0, 5000, (3, 19), generator=g)
    run(q, k, each, 64, "half", what="of each item")
    run(q, k, each.int(), 64, "half", what="of each item, 32 bits")
    run(q, k, each.t().contiguous().t(), 64, "half", what="of each item, other strides")
    run(q, k, torch.arange(40)[::2][:19], 64, "interleaved", what="every second")
    run(q, k, -torch.arange(19), 64, "half", what="negative")
    run(q, k, torch.full((19,), 7), 64, "half", what="all the same")
    run(q, k, 1000000 + 7919 * torch.arange(19), 64, "half", what="far")
    run(q, k, (1 << 31) - 5 + 1000003 * torch.arange(19), 64, "half", what="beyond 32 bits")
    run(q, k, torch.arange(19), 64, "half", base=1.0, what="all frequencies 1")


def test_weights():
    q, k = heads(2, 4, 33, 128, BF16, 1), heads(2, 2, 33, 128, BF16, 2)
    g = torch.Generator().manual_seed(5)
    w16, w32 = weights_of(128, BF16, g), weights_of(128, F32, g)
    at = torch.arange(33)
    run(q, k, at, 128, "half", (w16[0], None), what="of q")
    run(q, k, at, 128, "half", (None, w16[1]), what="of k")
    run(q, k, at, 128, "half", w32, what="in 32 bits")
    run(q, k, at, 128, "half", (w32[0], w16[1]), what="of two types")
    run(q, None, at, 64, "interleaved", (w32[0], None), what="q alone")
    run(q, k, at, 0, "half", w16, what="norms alone")
    run(q, k, at, 128, "half", w16, eps=0.5, factor=1.3, what="eps and factor")
    big, small = heads(1, 2, 9, 64, F32, 6, 1e15), heads(1, 2, 9, 64, F32, 7, 1e-6)
    run(big, small, torch.arange(9), 64, "half", weights_of(64, F32, g), eps=1e-12, what="large and small heads")


def test_zeros_stay_zeros():
    q = torch.zeros(1, 2, 5, 64)
    out, _ = A.rotary(q.to(DEV), None, torch.arange(5, device=DEV), pos.frequencies_of(64).to(DEV), q_weight=torch.ones(64, device=DEV))
    assert torch.equal(out.cpu(), q)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views(dtype):
    """What a projection leaves: token behind token, q, k and v in one tensor; gradients come back in the projection's order."""
    B, N, Hq, Hkv, D = 2, 45, 6, 2, 64
    g = torch.Generator().manual_seed(6)
    f = pos.frequencies_of(64).to(DEV)
    at = torch.arange(N, device=DEV)
    packed = torch.randn(B, N, (Hq + 2 * Hkv) * D, generator=g).to(dtype)
    leaf = packed.to(DEV).requires_grad_(True)
    q, k, _ = (t.view(B, N, -1, D).transpose(1, 2) for t in leaf.split([Hq * D, Hkv * D, Hkv * D], -1))
    outs = A.rotary(q, k, at, f)
    dy = [torch.randn(o.shape, generator=g).to(dtype).to(DEV) for o in outs]
    grad = torch.autograd.grad(outs, leaf, dy)[0]
    for i, (x, out) in enumerate(((q, outs[0]), (k, outs[1]))):
        want, tol = pos.forward_tolerance(x.detach().cpu(), torch.arange(N), f.cpu())
        check(out, want, tol, f"packed {i}")
    (dq, tol), _ = pos.backward(q.detach().cpu(), dy[0].cpu(), torch.arange(N), f.cpu())
    check(grad[..., : Hq * D].reshape(B, N, Hq, D).transpose(1, 2), dq, tol, "packed dq")
    assert (grad[..., (Hq + Hkv) * D:] == 0).all()
    x = torch.randn(B, N, Hq, D, generator=g).to(dtype).to(DEV).requires_grad_(True)
    out, _ = A.rotary(x.transpose(1, 2), None, at, f)
    assert torch.autograd.grad(out, x, dy[0])[0].is_contiguous()
    # rows that do not lie on 16 bytes, an inner stride, one row for all, an upstream gradient of another order
    odd = torch.randn(B * Hq * N * D + 1, generator=g).to(dtype)
    for what, x in (("off", odd.to(DEV)[1:].view(B, Hq, N, D)), ("odd rows", torch.randn(B, Hq, N, D + 1, generator=g).to(dtype).to(DEV)[..., 1:]),
                    ("inner", torch.randn(B, Hq, D, N, generator=g).to(dtype).to(DEV).transpose(2, 3)), ("one", odd.to(DEV)[:D].expand(B, Hq, N, D)),
                    ("every second token", torch.randn(B, Hq, 2 * N, D, generator=g).to(dtype).to(DEV)[:, :, ::2])):
        x = x.detach().requires_grad_(True)
        out, _ = A.rotary(x, None, at, f)
        want, tol = pos.forward_tolerance(x.detach().cpu(), torch.arange(N), f.cpu())
        check(out, want, tol, what)
        up = dy[0].transpose(1, 2).contiguous().transpose(1, 2)
        (dx, tol), _ = pos.backward(x.detach().cpu(), up.cpu(), torch.arange(N), f.cpu())
        check(torch.autograd.grad(out, x, up)[0], dx, tol, what + " gradient")


def test_tokens_of_three_dimensions():
    g = torch.Generator().manual_seed(7)
    for T in (1, 50):
        run(torch.randn(T, 6, 64, generator=g).to(BF16), torch.randn(T, 2, 64, generator=g).to(BF16), torch.randint(0, 900, (T,), generator=g), 64, "half",
            weights_of(64, BF16, g), what="tokens")


def test_nothing_to_turn():
    f = pos.frequencies_of(64).to(DEV)
    w = torch.ones(64, device=DEV, requires_grad=True)
    for shape in ((0, 4, 6, 64), (2, 4, 0, 64), (2, 0, 6, 64)):
        q = torch.zeros(shape, device=DEV, requires_grad=True)
        out, k = A.rotary(q, None, torch.arange(shape[2], device=DEV), f, q_weight=w)
        assert out.shape == shape and k is None
        dq, dw = torch.autograd.grad(out, (q, w), torch.zeros_like(out))
        assert dq.shape == shape and (dw == 0).all()


def test_what_is_not_used_has_no_gradient():
    f = pos.frequencies_of(64).to(DEV)
    q, k = heads(1, 2, 9, 64, F32, 1), heads(1, 1, 9, 64, F32, 2)
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, torch.ones(64), torch.ones(64))]
    a, b = A.rotary(leaves[0], leaves[1], torch.arange(9, device=DEV), f, q_weight=leaves[2], k_weight=leaves[3])
    for out, mine, other in ((a, (0, 2), (1, 3)), (b, (1, 3), (0, 2))):
        grads = torch.autograd.grad(out, leaves, torch.ones_like(out), retain_graph=True, allow_unused=True)
        for i in mine:
            assert grads[i] is not None and torch.isfinite(grads[i]).all()
        for i in other:
            assert grads[i] is None or (grads[i] == 0).all()
    # only some of the inputs want one
    out, _ = A.rotary(leaves[0].detach(), leaves[1].detach(), torch.arange(9, device=DEV), f, q_weight=leaves[2])
    out.sum().backward()
    assert torch.isfinite(leaves[2].grad).all()
    with torch.no_grad():
        assert not A.rotary(leaves[0], None, torch.arange(9, device=DEV), f)[0].requires_grad


def test_values_that_are_not_finite_stay_in_their_rows():
    q = heads(1, 3, 20, 64, BF16, 1)
    for i, bad in enumerate((float("nan"), float("inf"), -float("inf"))):
        q[0, i, 5 + i, 7] = bad
    f, at, w = pos.frequencies_of(64), torch.arange(20), torch.ones(64, dtype=BF16)
    clean = torch.where(torch.isfinite(q.float()), q, torch.zeros_like(q))
    got, _ = A.rotary(q.to(DEV), None, at.to(DEV), f.to(DEV), q_weight=w.to(DEV))
    want, _ = A.rotary(clean.to(DEV), None, at.to(DEV), f.to(DEV), q_weight=w.to(DEV))
    rows = torch.ones(1, 3, 20, dtype=torch.bool)
    for i in range(3):
        rows[0, i, 5 + i] = False
    assert torch.equal(got.cpu()[rows], want.cpu()[rows])


def test_calls_return_the_same_bits_and_can_be_captured():
    g = torch.Generator().manual_seed(8)
    q, k = (t.to(DEV).requires_grad_(True) for t in (heads(2, 8, 700, 128, BF16, 1), heads(2, 2, 700, 128, BF16, 2)))
    ws = [w.to(DEV).requires_grad_(True) for w in weights_of(128, BF16, g)]
    f, at = pos.frequencies_of(128).to(DEV), torch.arange(700, device=DEV)
    dy = [torch.randn(t.shape, generator=g).to(BF16).to(DEV) for t in (q, k)]

    def step():
        outs = A.rotary(q, k, at, f, q_weight=ws[0], k_weight=ws[1])
        return [*outs, *torch.autograd.grad(outs, (q, k, *ws), dy)]

    first = [t.clone() for t in step()]
    for a, b in zip(first, step()):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a, b in zip(first, step()):
            assert torch.equal(a, b)
    torch.cuda.synchronize()
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = A.rotary(q, k, at, f, q_weight=ws[0], k_weight=ws[1])
        for i in range(3):
            at.copy_(torch.arange(700, device=DEV) + 100 * i)
            for o in outs:
                o.zero_()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, A.rotary(q, k, at, f, q_weight=ws[0], k_weight=ws[1])):
                assert torch.equal(a, b)


def test_a_captured_training_step():
    """Forward and gradients in one graph, with leaves of its own beside eager steps, replayed on other rows and positions."""
    g = torch.Generator().manual_seed(18)
    leaves = [t.to(DEV) for t in (heads(2, 8, 300, 128, BF16, 3), heads(2, 2, 300, 128, BF16, 4), *weights_of(128, BF16, g))]
    f, at = pos.frequencies_of(128).to(DEV), torch.arange(300, device=DEV)
    dy = [torch.randn(t.shape, generator=g).to(BF16).to(DEV) for t in leaves[:2]]

    def step(q, k, wq, wk):
        outs = A.rotary(q, k, at, f, q_weight=wq, k_weight=wk)
        return [*outs, *torch.autograd.grad(outs, (q, k, wq, wk), dy)]

    ts = [t.detach().requires_grad_(True) for t in leaves]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*ts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step(*ts)
    for i in range(4):
        leaves[0].copy_(torch.randn(leaves[0].shape, generator=g).to(BF16))
        at.copy_(torch.arange(300, device=DEV) + 1000 * i)
        for r in results:
            r.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(results, step(*(t.detach().clone().requires_grad_(True) for t in leaves))):
            assert torch.equal(a, b)


def test_no_second_derivatives():
    q = heads(1, 2, 5, 32, F32, 1).to(DEV).requires_grad_(True)
    out, _ = A.rotary(q, None, torch.arange(5, device=DEV), pos.frequencies_of(32).to(DEV))
    with pytest.raises(RuntimeError, match="first derivatives only"):
        torch.autograd.grad(out.square().sum(), q, create_graph=True)
    out, _ = A.rotary(q, None, torch.arange(5, device=DEV), pos.frequencies_of(32).to(DEV))
    assert torch.autograd.grad(out.square().sum(), q)[0].shape == q.shape


@pytest.mark.parametrize("dtype, D, page, layout, norm", [(BF16, 128, 16, "half", True), (F16, 64, 7, "interleaved", False), (F32, 32, 1, "half", True), (F32, 256, 100, "interleaved", True),
                                                          (BF16, 16, 8, "half", False)])
def test_keys_on_the_way_to_their_slots(dtype, D, page, layout, norm):
    g = torch.Generator().manual_seed(9)
    H, pages = 3, 40 if page > 1 else 300
    for T in (1, 9, 211):
        k, v = (torch.randn(T, H, D, generator=g).to(dtype) for _ in range(2))
        at = torch.randint(0, 100000, (T,), generator=g)
        slots = torch.randperm(pages * page, generator=g)[:T]
        slots[::5] = -1
        if T > 9:
            slots[1], slots[2] = pages * page, 1 << 40
        w = weights_of(D, dtype, g)[0] if norm else None
        f = pos.frequencies_of(D)
        for slots_first in (False, True):
            shape = (pages, page, H, D) if slots_first else (pages, H, page, D)
            kp, vp = (torch.full(shape, 7.0, dtype=dtype, device=DEV) for _ in range(2))
            if slots_first:
                kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
            A.write_pages(k.to(DEV), v.to(DEV), slots.to(DEV), kp, vp, positions=at.to(DEV),
                          rotary=A.Rotary(f.to(DEV), layout, k_weight=w.to(DEV) if norm else None, factor=1.25))
            want, tol = pos.forward_tolerance(k, at[:, None], f, layout, w, 1e-6, 1.25)
            there = (slots >= 0) & (slots < pages * page)
            rows = [x.transpose(1, 2).reshape(-1, H, D).cpu() for x in (kp, vp)]
            check(rows[0][slots[there]], want[there], tol[there], f"T={T} keys")
            assert torch.equal(rows[1][slots[there]], v[there])
            left = torch.ones(pages * page, dtype=torch.bool)
            left[slots[there]] = False
            assert all((r[left] == 7.0).all() for r in rows)
    # views of a projection
    kv = torch.randn(20, 2, H, D, generator=g).to(dtype).to(DEV)
    slots = torch.arange(20, device=DEV)
    outs = []
    for k, v in ((kv[:, 0], kv[:, 1]), (kv[:, 0].contiguous(), kv[:, 1].contiguous())):
        kp, vp = (torch.zeros(pages, H, page, D, dtype=dtype, device=DEV) for _ in range(2))
        A.write_pages(k, v, slots, kp, vp, positions=slots, rotary=A.Rotary(f.to(DEV), layout))
        outs.append((kp, vp))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def test_rows_beyond_32_bits():
    """q of more than 2^31 elements: its last tokens, forward and gradient."""
    H, N, D = 4, 1 << 21 | 7, 256
    f = pos.frequencies_of(64).to(DEV)
    q = torch.empty(1, H, N, D, dtype=BF16, device=DEV)
    last = heads(1, H, 40, D, BF16, 1)
    q.zero_()
    q[:, :, -40:] = last.to(DEV)
    q.requires_grad_(True)
    w = weights_of(D, BF16, torch.Generator().manual_seed(3))[0]
    out, _ = A.rotary(q, None, torch.arange(N, device=DEV), f, q_weight=w.to(DEV))
    at = torch.arange(N - 40, N)
    want, tol = pos.forward_tolerance(last, at, f.cpu(), "half", w)
    check(out[:, :, -40:], want, tol, "last tokens")
    dy = torch.zeros_like(out)
    dy[:, :, -40:] = 1.0
    (dx, tol), _ = pos.backward(last, torch.ones_like(last), at, f.cpu(), "half", w)
    got = torch.autograd.grad(out, q, dy)[0]
    check(got[:, :, -40:], dx, tol, "last gradients")
    assert (got[:, :, :64] == 0).all()
