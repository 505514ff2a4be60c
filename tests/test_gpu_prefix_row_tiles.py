"""Attention behind a common prefix with several sixteens of rows to a workgroup, parts of every size and both kernels: each case names the parts and rows that it is there for, so that other rules of sharing out show here."""

import ctypes

import pytest
import torch

import adasplash_amd as A
from adasplash_amd import _lib
from tests import op_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
PAGE = 16
CODE = {F32: 0, BF16: 1, F16: 2}

# requests, heads, K/V heads, head_dim, type, pages of the prefix -> keys of a part, sixteens of rows (0: the kernel of up to sixteen rows)
CASES = [
    (64, 32, 8, 128, BF16, 512, 512, 4),
    (16, 176, 16, 64, F16, 400, 512, 4),   # 176 rows: the last workgroup's are not all there
    (8, 512, 32, 64, BF16, 256, 512, 4),
    (3, 15 * 64, 64, 64, BF16, 256, 512, 3),  # 45 rows
    (3, 30 * 24, 24, 64, BF16, 256, 512, 2),  # 90 rows
    (8, 128, 16, 32, F32, 512, 512, 2),
    (4, 33 * 16, 16, 64, F16, 256, 256, 4),
    (4, 33 * 8, 8, 128, BF16, 256, 256, 2),
    (4, 64 * 8, 8, 64, BF16, 128, 128, 4),
    (3, 64 * 8, 8, 64, F32, 128, 128, 2),
    (8, 512, 32, 128, F32, 128, 256, 4),   # rows of 512 bytes
    (8, 17 * 32, 32, 256, BF16, 128, 256, 4),
    (4, 60 * 16, 16, 256, F16, 64, 256, 2),
    (3, 128, 2, 256, BF16, 64, 64, 1),
    (8, 512, 32, 256, F32, 64, 128, 2),    # of 1024
    (3, 40 * 16, 16, 256, F32, 64, 128, 2),
    (3, 128, 2, 256, F32, 64, 64, 1),
    (2, 256, 64, 64, BF16, 64, 128, 0),
    (2, 512, 64, 64, F16, 128, 256, 0),
    (3, 320, 64, 64, BF16, 256, 512, 0),
    (2, 256, 64, 64, BF16, 512, 1024, 0),
    (4, 32, 32, 128, F32, 1024, 1024, 0),
]


def shared_out(B, Hq, Hkv, D, dtype, most, front):
    part, tiles = ctypes.c_int(-1), ctypes.c_int(-1)
    _lib.load().adsp_attn_paged_shared_parts(B, Hq, Hkv, D, CODE[dtype], most, PAGE, front, ctypes.addressof(part), ctypes.addressof(tiles))
    return part.value, tiles.value


def reference(q, k, v, alpha):
    with torch.device(DEV):
        return ref.attend(q, k, v, alpha)


class Batch:
    """Requests behind the first pages of one another, in a shuffled cache on the GPU."""

    def __init__(self, B, Hq, Hkv, D, dtype, front, seed):
        self.g = torch.Generator(DEV).manual_seed(seed)
        self.B, self.Hq, self.Hkv, self.D, self.dtype, self.front = B, Hq, Hkv, D, dtype, front
        own = 4
        self.width = front + own
        pages = front + B * own + 5
        self.k, self.v = (self.randn(pages, Hkv, PAGE, D) for _ in range(2))
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(DEV)
        self.prefix = order[:front].int()
        self.spare = order[-5:].int()
        self.tables = torch.cat([self.prefix.expand(B, front), order[front:front + B * own].view(B, own).int()], 1).contiguous()
        self.n = front * PAGE
        self.lengths = torch.tensor([self.n + 1 + (11 * b) % (own * PAGE) for b in range(B)], device=DEV)
        self.q = self.randn(B, Hq, 1, D)

    def randn(self, *shape):
        return torch.randn(shape, generator=self.g, device=DEV).to(self.dtype)

    def check(self, what, alpha=1.5, without=()):
        """Every request, up to eight of its heads; without: (head, key) that have no weight, {head: None} rows of zeros."""
        print(what, flush=True)
        out = A.paged_attention(self.q, self.k, self.v, self.tables, self.lengths, alpha=alpha, prefix_table=self.prefix)
        assert torch.isfinite(out).all(), what
        G, none = self.Hq // self.Hkv, {h: key for h, key in without}
        heads = sorted({h * max(self.Hkv - 1, 0) // 7 for h in range(8)})
        for b, n in enumerate(self.lengths.tolist()):
            pages = self.tables[b].long()
            there = ((pages >= 0) & (pages < self.k.shape[0])).repeat_interleave(PAGE)[:n]
            at = pages.clamp(0, self.k.shape[0] - 1)
            rows = [t[at].transpose(1, 2).reshape(-1, self.Hkv, self.D)[:n] for t in (self.k, self.v)]
            for h in heads:
                got = out[b, h * G:(h + 1) * G, 0]
                keep = there.clone()
                if h in none:
                    keep[none[h]] = False
                want, tol = reference(self.q[b, h * G:(h + 1) * G, 0], rows[0][keep, h], rows[1][keep, h], alpha)
                ref.check(got, want.cpu(), tol.cpu(), f"{what}: request {b} head {h}")
        return out


@pytest.mark.parametrize("B, Hq, Hkv, D, dtype, front, part, tiles", CASES)
def test_every_way_of_sharing_out(B, Hq, Hkv, D, dtype, front, part, tiles):
    x = Batch(B, Hq, Hkv, D, dtype, front, seed=B + D)
    assert shared_out(B, Hq, Hkv, D, dtype, x.width * PAGE, front) == (part, tiles)
    out = x.check("all of it")
    assert torch.equal(out, A.paged_attention(x.q, x.k, x.v, x.tables, x.lengths, prefix_table=x.prefix))
    lengths, tables, prefix, q = x.lengths.clone(), x.tables.clone(), x.prefix.clone(), x.q
    # requests that end inside the prefix, around the ends of parts, and empty ones
    ends = [0, 1, part - 1, part, part + 1, x.n // 2, x.n - 1, x.n]
    for b in range(0, B, 2):
        x.lengths[b] = ends[b // 2 % len(ends)] if b > 0 else ends[B % len(ends)]
    x.check("ends inside")
    x.lengths = lengths.clone()
    # tables that differ from the prefix in one entry: first, last, at a part's border, somewhere
    for i, b in enumerate(range(B - 1, -1, -3)):
        x.tables[b, (0, front - 1, part // PAGE, part // PAGE - 1, front // 3)[i % 5]] = x.spare[i % 5]
    x.check("other pages")
    x.tables = tables.clone()
    # pages that are none, for all of the requests and of one
    for at in (0, part // PAGE, part // PAGE + 3, front - 1):
        x.tables[:, at], x.prefix[at] = -1, -1
    x.tables[B // 2, 1] = x.k.shape[0]
    x.check("holes", alpha=1.25)
    x.q = (q.float() * 0.03).to(dtype)
    x.check("holes and flat scores", alpha=2.0)
    x.tables, x.prefix = tables.clone(), prefix.clone()
    # flat scores: steps on all of them
    x.check("flat scores")
    x.q = (q.float() * 0.4).to(dtype)
    x.check("scores between", alpha=1.75)
    x.q = (q.float() * 5).to(dtype)
    x.check("few keys with weight")
    # keys of the prefix that are not finite
    x.q = q.clone()
    x.q[..., 0] = q[..., 0].abs() + 0.125
    places = {0: (part - 1, float("nan")), (Hkv - 1) // 7: (part, -float("inf")), Hkv - 1: (x.n - 2, float("nan"))}
    for h, (key, value) in places.items():
        x.k[x.prefix[key // PAGE].long(), h, key % PAGE, 0] = value
    x.check("keys that are not finite", without=[(h, key) for h, (key, _) in places.items()])
    key = part // 2
    x.k[x.prefix[key // PAGE].long(), 2 * (Hkv - 1) // 7, key % PAGE, 0] = float("inf")
    out = A.paged_attention(x.q, x.k, x.v, x.tables, x.lengths, prefix_table=x.prefix).view(B, Hkv, -1, D)
    h = 2 * (Hkv - 1) // 7
    assert (out[:, h] == 0).all() and (out[:, Hkv - 1] != 0).any() and torch.isfinite(out).all()
