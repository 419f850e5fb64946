"""The arithmetic of the paged attention, bit by bit: every part of q counts,
long sums do not drift, every row counts once.  Inputs and tolerances are those
of paged_precision.py, where mistakes are planted on the CPU."""
from __future__ import annotations

import numpy as np
import pytest

import paged_precision as pp

pytestmark = pytest.mark.gpu

# (heads, KV heads, head_dim), type, page, queries, shared rows (0: the plain
# call): every kernel and every form of a shared prefix.
ROUTES = [
    pytest.param((14, 2, 64), "bf16", 16, 5, 0, id="plain-64"),
    pytest.param((8, 8, 32), "bf16", 8, 3, 0, id="plain-32"),
    pytest.param((32, 8, 128), "bf16", 32, 3, 0, id="plain-128"),
    pytest.param((22, 2, 64), "bf16", 64, 2, 0, id="plain-11-heads"),
    pytest.param((14, 2, 64), "f32", 16, 3, 0, id="plain-f32-64"),
    pytest.param((8, 8, 32), "f32", 16, 3, 0, id="plain-f32-32"),
    pytest.param((16, 1, 128), "f32", 16, 3, 0, id="plain-f32-128"),
    pytest.param((4, 4, 6), "f32", 16, 3, 0, id="plain-cores"),
    pytest.param((4, 4, 6), "bf16", 16, 3, 0, id="plain-cores-bf16"),
    pytest.param((14, 2, 64), "bf16", 16, 40, 9000, id="prefix"),
    pytest.param((14, 2, 64), "bf16", 32, 9, 65000, id="prefix-one-tile"),
    pytest.param((12, 4, 64), "bf16", 8, 10, 40003, id="prefix-30-rows"),
    pytest.param((12, 4, 64), "bf16", 256, 70, 4200, id="prefix-two-tiles"),
    pytest.param((8, 8, 32), "bf16", 16, 37, 4100, id="packed-32"),
    pytest.param((12, 4, 64), "f32", 16, 19, 9000, id="packed-f32"),
    pytest.param((32, 8, 128), "bf16", 16, 40, 3000, id="packed-128"),
]


def tokens(shared, n):
    """Rows of n queries, behind a shared part."""
    return [shared + 17 + 61 * i % 400 for i in range(n)]


class Rows:
    """A pool filled by make(positions) -> (k, v) of shape [len, KV heads, hd],
    per owner (the shared part or a sequence), pages in random order."""

    def __init__(self, tg, backend, shape, dtype, page, n, shared, make, lens=None, seed=0):
        import torch
        H, G, D = shape
        rng = np.random.default_rng(seed)
        dt = torch.bfloat16 if dtype == "bf16" else torch.float32
        self.sh = shared // page * page
        self.lens = tokens(self.sh, n) if lens is None else lens
        owners = [self.sh] + [x - self.sh for x in self.lens]
        need = [-(-x // page) for x in owners]
        order = torch.from_numpy(rng.permutation(sum(need) + 1).astype(np.int32))
        at = np.cumsum([0] + need)
        cols = need[0] + max(need[1:])
        table = torch.full((n, cols), int(order[-1]), dtype=torch.int32)
        pools = [torch.full((sum(need) + 1, G, page, D), float("nan"), dtype=dt, device="cuda")
                 for _ in range(2)]
        self.own = []
        for o, m in enumerate(owners):
            pages = order[at[o]:at[o + 1]]
            if o:
                table[o - 1, :need[0]] = order[:need[0]]
                table[o - 1, need[0]:need[0] + need[o]] = pages
            kv = make(o, m)
            self.own.append(kv)
            for pool, x in zip(pools, kv):
                full = torch.zeros(need[o] * page, G, D, dtype=dt, device="cuda")
                full[:m] = x.to(dt)
                pool[pages.long().cuda()] = full.view(need[o], page, G, D).permute(0, 2, 1, 3)
        self.table = table.cuda()
        self.past = torch.tensor([x - 1 for x in self.lens], dtype=torch.int32).cuda()
        self.cache = tg.PagedKVCache(backend, 1, sum(need) + 1, page, H, G, D,
                                     tg.DTYPE_BF16 if dtype == "bf16" else tg.DTYPE_F32,
                                     max_pos=64, k=pools[0][None].contiguous(),
                                     v=pools[1][None].contiguous())
        self.shared, self.backend = shared, backend

    def attend(self, q):
        import torch
        out = torch.full_like(q, 7.0)
        before = self.backend.launch_count()
        if self.shared:
            self.cache.attention_shared(0, q, self.past, self.table, self.shared, out)
        else:
            self.cache.attention(0, q, self.past, self.table, out)
        # A prefix that is attended for all takes two launches more.
        assert self.backend.launch_count() - before == (3 if self.shared else 1)
        self.backend.synchronize()
        return out


@pytest.mark.parametrize("shape,dtype,page,n,shared", ROUTES)
def test_every_part_of_q_counts(tg, backend, shape, dtype, page, n, shared):
    import torch
    H, G, D = shape
    rng = np.random.default_rng(D + n)
    q = pp.coherent_queries(rng, n * H, D)
    k = torch.from_numpy(pp.key(D)).cuda()
    plus = {}

    def make(owner, m):
        sign = torch.from_numpy(np.where(rng.random(m) < 0.5, 1.0, -1.0).astype(np.float32)).cuda()
        plus[owner] = int((sign > 0).sum())
        one = torch.ones(m, G, D, device="cuda") * sign[:, None, None]
        return one * k, one

    p = Rows(tg, backend, shape, dtype, page, n, shared, make)
    out = p.attend(torch.from_numpy(q.reshape(n, H * D)).cuda()).cpu().numpy().reshape(n, H, D)
    tol = pp.two_key_tolerance(D, dtype)
    for s in range(n):
        a = plus[0] + plus[s + 1]
        want = pp.two_key_result(q.reshape(n, H, D)[s], a, p.lens[s] - a)
        err = np.abs(out[s] - want[:, None]).max()
        assert err <= tol, (s, err, tol)


@pytest.mark.parametrize("shape,dtype,page,n,shared", ROUTES + [
    pytest.param((14, 2, 64), "bf16", 16, 1, 100_003, id="one-long"),
    pytest.param((12, 4, 64), "f32", 64, 2, 50_021, id="two-long-f32")])
def test_every_row_counts_once(tg, backend, shape, dtype, page, n, shared):
    """With q = 0 every weight is 1, and over values of random bits every sum
    is a whole number: the result is a count over a count, off by the rounding
    of a reciprocal and a product."""
    import torch
    H, G, D = shape
    gen = torch.Generator(device="cuda").manual_seed(n)
    counts = []

    def make(owner, m):
        v = torch.randint(0, 2, (m, G, D), generator=gen, device="cuda").float()
        counts.append(v.double().sum(0))
        return torch.randn(m, G, D, generator=gen, device="cuda"), v

    plain = "long" if n <= 2 else ""
    p = Rows(tg, backend, shape, dtype, page, n, 0 if plain else shared, make,
             lens=[shared + 31 * i for i in range(n)] if plain and shared else None)
    out = p.attend(torch.zeros(n, H * D, device="cuda")).double().view(n, G, H // G, D)
    for s in range(n):
        want = ((counts[0] + counts[s + 1]) / p.lens[s])[:, None]
        assert ((out[s] - want).abs() <= 2.0 ** -22 * want).all(), s


@pytest.mark.parametrize("dtype,n,rows,chunks", [("bf16", 37, 1 << 19, 1024), ("f32", 37, 1 << 17, 512)])
def test_long_sums_do_not_drift(tg, backend, dtype, n, rows, chunks):
    """With v = 1 the result is sum p / sum p: 1, whatever the scores, unless
    one of the sums loses more than the other over the chunks of a warp (two
    CTAs of eight warps share a stream).  Tables name few pages many times."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(5)
    pool, P = 64, 256
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    k = torch.randn(1, pool, 2, P, 64, generator=g, device="cuda").to(dt)
    c = tg.PagedKVCache(backend, 1, pool, P, max_pos=64,
                        dtype=tg.DTYPE_BF16 if dtype == "bf16" else tg.DTYPE_F32, k=k,
                        v=torch.ones_like(k))
    q = torch.randn(n, 896, generator=g, device="cuda")
    table = torch.randint(0, pool, (n, rows // P), generator=g, device="cuda", dtype=torch.int32)
    past = torch.full((n,), rows - 1, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(q)
    c.attention(0, q, past, table, out)
    backend.synchronize()
    err = (out.double() - 1).abs().max().item()
    assert err <= pp.chain_tolerance(chunks), err
    c.destroy()


def test_long_sums_of_a_prefix_do_not_drift(tg, backend):
    """The same behind a shared prefix of 400 steps a CTA; an accumulator
    gathers 16 steps of 8 products."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(6)
    pool, P, n, shared = 64, 256, 128, 64 * 18 * 400
    k = torch.randn(1, pool, 2, P, 64, generator=g, device="cuda").to(torch.bfloat16)
    c = tg.PagedKVCache(backend, 1, pool, P, max_pos=64, k=k, v=torch.ones_like(k))
    q = torch.randn(n, 896, generator=g, device="cuda")
    row = torch.randint(0, pool, (shared // P + 1,), generator=g, device="cuda", dtype=torch.int32)
    table = row.repeat(n, 1).contiguous()
    past = shared - 1 + torch.arange(n, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(q)
    c.attention_shared(0, q, past, table, shared, out)
    backend.synchronize()
    err = (out.double() - 1).abs().max().item()
    assert err <= pp.chain_tolerance(400, steps=128), err
    c.destroy()


@pytest.mark.parametrize("scale", [1.0, 8.0, 16.0])
@pytest.mark.parametrize("shape,dtype,page,n,shared", [
    r for r in ROUTES if r.id in ("plain-64", "plain-f32-64", "plain-128", "prefix",
                                  "prefix-one-tile", "packed-f32", "packed-128")])
def test_peaked_scores(tg, backend, shape, dtype, page, n, shared, scale):
    """Scores of up to 16 times the usual size, whose errors grow with them: on
    no route more than those of binary32 products, hd * 2^-24 of a key's sum
    of |q k| (and 3 * 2^-22 where fp32 rows are two tf32), plus 2^-16 of the
    weighted values for weights and sums."""
    import torch
    H, G, D = shape
    gen = torch.Generator(device="cuda").manual_seed(int(scale) + n)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32

    def make(owner, m):
        return [torch.randn(m, G, D, generator=gen, device="cuda").to(dt).float() for _ in range(2)]

    p = Rows(tg, backend, shape, dtype, page, n, shared, make)
    q = torch.randn(n, H * D, generator=gen, device="cuda") * scale
    out = p.attend(q).double().view(n, G, H // G, D)
    rel = D * 2.0 ** -24 + (0.0 if dtype == "bf16" else 3 * 2.0 ** -22)
    for s in range(0, n, max(1, n // 8)):
        k, v = (torch.cat([p.own[0][i], p.own[s + 1][i]]).double().transpose(0, 1) for i in range(2))
        x = q[s].double().view(G, H // G, D)
        w = torch.softmax(x @ k.transpose(1, 2) / D ** 0.5, -1)
        want = w @ v
        off = w * (rel * (x.abs() @ k.abs().transpose(1, 2)) / D ** 0.5)     # of a weight
        tol = off @ v.abs() + off.sum(-1, keepdim=True) * want.abs() + 2.0 ** -16 * (w @ v.abs())
        err = (out[s] - want).abs()
        assert (err <= tol).all(), (s, (err / tol).max().item())
