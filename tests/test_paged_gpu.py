"""The paged KV cache on the GPU against plain 64-bit forms: append with
rotation, decode attention through block tables, shared prefixes, page
selection, attention over listed pages.

Tolerances of the attention: with S the largest sum_d |q_d k_d| / sqrt(hd) of
a query, scores are off by at most S * 2^-16 (q and k split into two 16-bit
terms: 2^-17 relative; binary32 sums of up to 128 terms: 128 * 2^-24 = 2^-17),
which moves a weight by a factor within e^(+-2 S 2^-16); weights split the
same way and the binary32 sums add 2^-15 of the largest |v|."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

SHAPES = [(14, 2, 64), (8, 8, 32), (16, 1, 128), (12, 4, 64), (4, 4, 6), (22, 2, 64), (3, 1, 128)]


def f64(x):
    return np.asarray(x.float().cpu() if hasattr(x, "cpu") else x, np.float64)


class Pool:
    """A pool of NaN, a table over it in random page order, and rows for
    every sequence; the reference reads the same stored values."""

    def __init__(self, tg, backend, lens, shape=(14, 2, 64), dtype="bf16", page=16, seed=0,
                 shared=0, extra_cols=1, layers=1, layer=0, scale=1.0):
        import torch
        H, G, D = shape
        self.H, self.G, self.D, self.P = H, G, D, page
        rng = np.random.default_rng(seed)
        self.lens = list(lens)                       # rows per sequence, shared ones included
        n = len(self.lens)
        nsh = shared // page
        need = [max(0, -(-x // page) - nsh) for x in self.lens]
        cols = max([-(-x // page) for x in self.lens] + [nsh, 1]) + extra_cols
        total = nsh + sum(need) + 3
        order = rng.permutation(total)
        table = np.full((n, cols), order[-1], np.int32)    # unused entries: a page of NaN
        table[:, :nsh] = order[:nsh]
        at = nsh
        for s in range(n):
            table[s, nsh:nsh + need[s]] = order[at:at + need[s]]
            at += need[s]
        self.table_np = table
        dt = torch.bfloat16 if dtype == "bf16" else torch.float32
        size = (layers, total, G, page, D)
        kp = torch.full(size, float("nan"))
        vp = torch.full(size, float("inf"))
        for s in range(n):
            for j in range(-(-self.lens[s] // page)):
                r = min(page, self.lens[s] - j * page)
                if j < nsh and s != int(np.argmax(self.lens)):
                    continue                           # the longest sequence fills the shared pages
                if j < nsh:
                    r = page if self.lens[s] >= (j + 1) * page else r
                kp[layer, table[s, j], :, :r] = torch.from_numpy(
                    rng.standard_normal((G, r, D)).astype(np.float32) * scale)
                vp[layer, table[s, j], :, :r] = torch.from_numpy(
                    rng.standard_normal((G, r, D)).astype(np.float32))
        self.kp, self.vp = kp.to(dt).cuda(), vp.to(dt).cuda()
        lo, hi = self.kp.float().nan_to_num(nan=float("inf")).amin(3), \
            self.kp.float().nan_to_num(nan=float("-inf")).amax(3)
        self.bounds = torch.stack([lo, hi], 3).to(dt).contiguous()
        self.q = torch.from_numpy(rng.standard_normal((n, H * D)).astype(np.float32)).cuda()
        self.past = torch.tensor([x - 1 for x in self.lens], dtype=torch.int32).cuda()
        self.table = torch.from_numpy(table).cuda()
        self.out = torch.full((n, H * D), 7.0).cuda()
        self.layer = layer
        self.cache = tg.PagedKVCache(backend, layers, total, page, H, G, D,
                                     tg.DTYPE_BF16 if dtype == "bf16" else tg.DTYPE_F32,
                                     max_pos=4096, k=self.kp, v=self.vp, bounds=self.bounds)
        self._k, self._v = f64(self.kp[layer]), f64(self.vp[layer])

    def rows(self, s, g, entries=None):
        """K and V rows of sequence s, in 64 bits."""
        P, n = self.P, self.lens[s]
        entries = range(-(-n // P)) if entries is None else entries
        ks, vs = [], []
        for j in entries:
            r = min(P, n - j * P)
            if j < 0 or r <= 0:
                continue
            page = self.table_np[s, j]
            ks.append(self._k[page, g, :r])
            vs.append(self._v[page, g, :r])
        if not ks:
            return np.zeros((0, self.D)), np.zeros((0, self.D))
        return np.concatenate(ks), np.concatenate(vs)

    def check(self, out, pages=None, seqs=None):
        out, q = f64(out), f64(self.q)
        per = self.H // self.G
        for s in (range(len(self.lens)) if seqs is None else seqs):
            for g in range(self.G):
                k, v = self.rows(s, g, None if pages is None else pages[s][g])
                for h in range(g * per, (g + 1) * per):
                    sl = slice(h * self.D, (h + 1) * self.D)
                    if not len(k):
                        assert not out[s, sl].any(), (s, h)
                        continue
                    x = k @ q[s, sl] / np.sqrt(self.D)
                    w = np.exp(x - x.max())
                    ref = (w / w.sum()) @ v
                    S = (np.abs(k) @ np.abs(q[s, sl])).max() / np.sqrt(self.D)
                    tol = np.abs(v).max() * (2 * S * 2.0 ** -16 + 2.0 ** -15)
                    err = np.abs(out[s, sl] - ref).max()
                    assert err <= tol, (s, h, self.lens[s], err, tol)


# ------------------------------------------------------------------- append

def _append_case(rng, n, max_new, max_ctx, page, empty=True):
    new = rng.integers(0 if empty else 1, max_new + 1, n)
    pos0 = rng.integers(0, max_ctx + 1, n)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    cols = int((pos0 + new).max() + page - 1) // page + 1
    need = -(-(pos0 + new) // page)
    order = rng.permutation(int(need.sum()) + 2).astype(np.int32)
    table = np.full((n, cols), -1, np.int32)           # never read where nothing lies
    at = 0
    for s in range(n):
        table[s, :need[s]] = order[at:at + need[s]]
        at += need[s]
    return new, pos0.astype(np.int32), cu, table, len(order)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page,max_new", [(8, 1), (16, 45), (256, 3)])
def test_append(tg, backend, O, shape, dtype, page, max_new):
    import torch
    H, G, D = shape
    rng = np.random.default_rng(H * 1000 + page)
    n, pad, layers, layer = 7, 5, 2, 1
    new, pos0, cu, table, pages = _append_case(rng, n, max_new, 40, page)
    T = int(cu[-1]) + pad
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    k, v = (rng.standard_normal((T, G * D)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((T, H * D)).astype(np.float32)
    kp0 = torch.randn(layers, pages, G, page, D).to(dt).cuda()
    vp0 = torch.randn(layers, pages, G, page, D).to(dt).cuda()
    b0 = torch.randn(layers, pages, G, 2, D).to(dt).cuda()
    kp, vp, bd = kp0.clone(), vp0.clone(), b0.clone()
    cache = tg.PagedKVCache(backend, layers, pages, page, H, G, D,
                            tg.DTYPE_BF16 if dtype == "bf16" else tg.DTYPE_F32, max_pos=4096,
                            k=kp, v=vp, bounds=bd)
    q_out = torch.full((T, H * D), 3.0).cuda()
    cache.append(layer, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(),
                 torch.from_numpy(pos0).cuda(), torch.from_numpy(table).cuda(),
                 q=torch.from_numpy(q).cuda(), q_out=q_out, cu_tokens=torch.from_numpy(cu).cuda())
    backend.synchronize()
    want_k, want_v, want_b = kp0.clone().cpu(), vp0.clone().cpu(), b0.clone().cpu()
    want_q = np.full((T, H * D), 3.0, np.float32)      # padding tokens stay as they were
    for s in range(n):
        for i in range(new[s]):
            t, pos = cu[s] + i, int(pos0[s]) + i
            want_q[t] = O.rope_heads(q[t], H, D, pos)
            kr = torch.from_numpy(O.rope_heads(k[t], G, D, pos)).view(G, D).to(dt)
            pg, slot = table[s, pos // page], pos % page
            want_k[layer, pg, :, slot] = kr
            want_v[layer, pg, :, slot] = torch.from_numpy(v[t]).view(G, D).to(dt)
        if new[s]:
            end = int(pos0[s]) + int(new[s])
            for j in range(int(pos0[s]) // page, (end - 1) // page + 1):
                rows = want_k[layer, table[s, j], :, :min(page, end - j * page)].float()
                want_b[layer, table[s, j]] = torch.stack([rows.amin(1), rows.amax(1)], 1).to(dt)
    assert np.array_equal(q_out.cpu().numpy().view(np.uint32), want_q.view(np.uint32))
    assert torch.equal(kp.cpu(), want_k)
    assert torch.equal(vp.cpu(), want_v)
    assert torch.equal(bd.cpu(), want_b)
    cache.destroy()


def test_append_in_pieces_and_in_place(tg, backend):
    """Chunks and single tokens leave the pool and bounds that one call does;
    q rotated in place; rewritten rows (a rejected draft) renew the bounds."""
    import torch
    rng = np.random.default_rng(5)
    T, P = 77, 16
    k, v, q = (torch.from_numpy(rng.standard_normal((T, w)).astype(np.float32)).cuda()
               for w in (128, 128, 896))
    table = torch.arange(5, dtype=torch.int32).flip(0).view(1, 5).contiguous().cuda()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    caches = [tg.PagedKVCache(backend, 1, 5, P, max_pos=128, k=torch.zeros(5, 2, P, 64, dtype=torch.bfloat16).cuda(),
                              v=torch.zeros(5, 2, P, 64, dtype=torch.bfloat16).cuda(),
                              bounds=torch.zeros(5, 2, 2, 64, dtype=torch.bfloat16).cuda())
              for _ in range(2)]
    qa = torch.zeros_like(q)
    caches[0].append(0, k, v, i32(0), table, q=q, q_out=qa, cu_tokens=i32(0, T))
    qb = q.clone()
    draft = torch.full((9, 128), 1e4).cuda()
    caches[1].append(0, k[:30], v[:30], i32(0), table, q=qb[:30], cu_tokens=i32(0, 30))
    caches[1].append(0, draft, draft, i32(30), table, cu_tokens=i32(0, 9))
    for t in range(30, 41):
        caches[1].append(0, k[t:t + 1], v[t:t + 1], i32(t), table, q=qb[t:t + 1])
    caches[1].append(0, k[41:], v[41:], i32(41), table, q=qb[41:], cu_tokens=i32(0, T - 41))
    backend.synchronize()
    assert torch.equal(qa, qb)
    for a, b in zip(caches[0]._keep, caches[1]._keep):
        assert torch.equal(a, b)


# ---------------------------------------------------------------- attention

EDGES = [0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 255, 256, 257]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page", [8, 16, 64, 256])
def test_attention_lengths(tg, backend, shape, dtype, page):
    """Every length around tile and page ends, among them none; everything
    behind a sequence's rows is NaN and infinity."""
    p = Pool(tg, backend, EDGES, shape, dtype, page, seed=page, layers=2, layer=1)
    p.cache.attention(1, p.q, p.past, p.table, p.out)
    backend.synchronize()
    p.check(p.out)
    p.cache.destroy()


@pytest.mark.parametrize("dtype,page", [("bf16", 16), ("bf16", 128), ("f32", 32)])
def test_attention_split_streams(tg, backend, dtype, page):
    """Long and short sequences together: streams split over many CTAs; the
    same call again gives the same bits (arrival counters are back at 0)."""
    p = Pool(tg, backend, [30001, 5, 0, 4097, 12345], (14, 2, 64), dtype, page, seed=3, scale=1.5)
    p.cache.attention(0, p.q, p.past, p.table, p.out)
    again = p.out.clone()
    p.cache.attention(0, p.q, p.past, p.table, again)
    backend.synchronize()
    p.check(p.out)
    assert (p.out == again).all()


@pytest.mark.parametrize("shape", [(12, 1, 32), (6, 3, 32), (9, 9, 32)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page", [8, 32, 256])
def test_attention_narrow_heads(tg, backend, shape, dtype, page):
    """Rows of 64 and 128 bytes, groups of 1, 2 and 12 (two blocks of heads)."""
    p = Pool(tg, backend, [1, 0, 700, 31, 2049, 257], shape, dtype, page, seed=page + 1)
    p.cache.attention(0, p.q, p.past, p.table, p.out)
    backend.synchronize()
    p.check(p.out)
    p.cache.destroy()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_many_ragged_in_place(tg, backend, dtype):
    """Several streams of a CTA one after the other, empty ones between them,
    and the result written over the queries."""
    rng = np.random.default_rng(9)
    lens = rng.integers(1, 700, 333)
    lens[rng.integers(0, 333, 120)] = 0
    p = Pool(tg, backend, [int(x) for x in lens], (14, 2, 64), dtype, 16, seed=10)
    out = p.q.clone()
    p.cache.attention(0, p.q, p.past, p.table, p.out)
    p.cache.attention(0, out, p.past, p.table, out)
    backend.synchronize()
    assert (out == p.out).all()
    p.check(p.out, seqs=range(0, 333, 4))
    p.cache.destroy()


def test_attention_single_long_sequence(tg, backend):
    p = Pool(tg, backend, [100003], (14, 2, 64), "bf16", 64, seed=4)
    p.cache.attention(0, p.q, p.past, p.table, p.out)
    backend.synchronize()
    p.check(p.out)


def test_attention_peaked_scores(tg, backend):
    """Large scores: one key takes nearly all the weight, far keys underflow."""
    for dtype in ("bf16", "f32"):
        p = Pool(tg, backend, [500, 33], (14, 2, 64), dtype, 16, seed=6, scale=8.0)
        p.cache.attention(0, p.q, p.past, p.table, p.out)
        backend.synchronize()
        p.check(p.out)


def test_attention_more_queries_than_one_launch(tg, backend):
    import torch
    p = Pool(tg, backend, [3, 40, 0, 17], (14, 2, 64), "bf16", 16, seed=8)
    reps = 1100                                         # 4400 queries
    q, past, table = (x.repeat(reps, 1) if x.dim() > 1 else x.repeat(reps)
                      for x in (p.q, p.past, p.table))
    out = torch.full_like(q, 9.0)
    p.cache.attention(0, q, past, table, out)
    backend.synchronize()
    # Not the same bits for every copy of a query: where a launch's CTAs cut a
    # stream, its sums join in another order, which moves each result within
    # the binary32 share of the tolerance.  Every copy meets the tolerance.
    for i in range(0, reps, 11):
        p.check(out[4 * i:4 * i + 4])
    p.check(out[-4:])
    assert (out.view(reps, 4, -1)[:, 2] == 0).all()


def test_offsets_past_32_bits(tg, backend):
    """Pages whose elements lie behind 2^31: attention and append there."""
    import torch
    pages, P = 1_060_000, 16
    kp = torch.zeros(pages, 2, P, 64, dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros_like(kp)
    assert kp.numel() > 2 ** 31
    cache = tg.PagedKVCache(backend, 1, pages, P, max_pos=64, k=kp, v=vp)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(20, 128, generator=g, device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32).cuda()
    cu, zero = (torch.tensor(x, dtype=torch.int32).cuda() for x in ([0, 20], [0]))
    cache.append(0, k, v, zero, table, cu_tokens=cu)
    q = torch.randn(1, 896, generator=g, device="cuda")
    out = torch.zeros_like(q)
    cache.attention(0, q, torch.tensor([19], dtype=torch.int32).cuda(), table, out)
    backend.synchronize()
    rows = torch.cat([kp[-1], kp[-2, :, :4]], 1).double(), torch.cat([vp[-1], vp[-2, :, :4]], 1).double()
    assert torch.equal(rows[1].transpose(0, 1).reshape(20, 128).float(), v.bfloat16().float())
    w = torch.softmax(q.view(2, 7, 64).double() @ rows[0].transpose(1, 2) / 8, -1) @ rows[1]
    # |q.k| / 8 stays below 16 for 64 normal values; |v| below 6 (see above).
    assert (out.view(2, 7, 64).double() - w).abs().max() <= 6 * (32 * 2.0 ** -16 + 2.0 ** -15)
    assert not kp[:-2].view(torch.int16).any()
    cache.destroy()


# ------------------------------------------------------------ shared prefix

@pytest.mark.parametrize("shape", [(14, 2, 64), (12, 4, 64), (16, 1, 128), (8, 8, 32), (22, 2, 64)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page,shared", [(16, 0), (16, 200), (64, 700), (8, 1031)])
def test_attention_shared(tg, backend, shape, dtype, page, shared):
    """Suffixes of every kind, queries that end inside the shared part, an
    empty query; shared_len need not be a whole number of pages."""
    sh = shared // page * page
    lens = [sh, sh + 1, sh + 15, sh + 16, sh + 130, 0, sh // 2, min(1, sh), sh + 33, sh + 257]
    p = Pool(tg, backend, lens, shape, dtype, page, seed=shared, shared=shared)
    p.cache.attention_shared(0, p.q, p.past, p.table, shared, p.out)
    backend.synchronize()
    p.check(p.out)
    p.cache.destroy()


@pytest.mark.parametrize("n,shared,page,shape", [
    (1, 3000, 16, (14, 2, 64)), (19, 5000, 32, (14, 2, 64)), (37, 2049, 16, (14, 2, 64)),
    # From here on the prefix goes to the tensor cores: one tile of rows (the
    # keys shared out between both slots), two tiles, an odd number of them,
    # groups of 1 to 11, pages smaller and larger than a step.
    (10, 30011, 16, (14, 2, 64)), (19, 16000, 32, (14, 2, 64)), (37, 8001, 8, (14, 2, 64)),
    (150, 2111, 128, (14, 2, 64)), (64, 20000, 64, (14, 2, 64)), (70, 2000, 16, (4, 4, 64)),
    (40, 4444, 256, (12, 4, 64)), (30, 9000, 16, (22, 2, 64)), (131, 4100, 16, (3, 1, 64))])
def test_attention_shared_batches(tg, backend, n, shared, page, shape):
    """Suffixes of 0 to 300 rows, a query inside the shared part, an empty one."""
    rng = np.random.default_rng(n)
    sh = shared // page * page
    lens = [sh + int(x) for x in rng.integers(0, 300, n)]
    lens[n // 2] = 0 if n > 1 else lens[0]
    lens[n // 3] = sh - 5 if n > 3 else lens[n // 3]
    p = Pool(tg, backend, lens, shape, "bf16", page, seed=n, shared=shared, scale=1.5)
    p.cache.attention_shared(0, p.q, p.past, p.table, shared, p.out)
    again = p.out.clone()
    p.cache.attention_shared(0, p.q, p.past, p.table, shared, again)
    backend.synchronize()
    p.check(p.out, seqs=sorted(set(rng.choice(n, min(n, 8), replace=False)) | {n // 2, n // 3}))
    assert (p.out == again).all()


@pytest.mark.parametrize("n,shared,page,shape,dtype", [
    (37, 4100, 16, (8, 8, 32), "bf16"), (19, 9000, 8, (12, 4, 64), "f32"),
    (10, 30011, 64, (4, 1, 128), "bf16"), (100, 2000, 16, (6, 3, 32), "f32"),
    (3, 40000, 256, (3, 3, 64), "f32"), (1100, 210, 16, (8, 8, 32), "bf16"),
    (1100, 1100, 16, (8, 8, 32), "bf16")])
def test_attention_shared_small_groups(tg, backend, n, shared, page, shape, dtype):
    """Rows of several queries over the prefix together: whole and ragged
    blocks of eight, one block, more queries than one launch takes."""
    rng = np.random.default_rng(n + 1)
    sh = shared // page * page
    lens = [sh + int(x) for x in rng.integers(0, 90, n)]
    lens[n // 2] = 0
    lens[n // 3] = sh - 5 if n > 3 else lens[n // 3]
    p = Pool(tg, backend, lens, shape, dtype, page, seed=n, shared=shared, scale=1.5)
    p.cache.attention_shared(0, p.q, p.past, p.table, shared, p.out)
    again = p.out.clone()
    p.cache.attention_shared(0, p.q, p.past, p.table, shared, again)
    backend.synchronize()
    p.check(p.out, seqs=sorted(set(rng.choice(n, min(n, 12), replace=False)) | {n // 2, n // 3, n - 1}))
    assert (p.out == again).all()


@pytest.mark.parametrize("shape", [(14, 2, 64), (8, 8, 32)])
def test_shared_position_outside_the_table(tg, backend, shape):
    """Counts as empty, also where the prefix is attended by itself."""
    rng = np.random.default_rng(4)
    p = Pool(tg, backend, [6000 + int(x) for x in rng.integers(0, 40, 50)], shape, "bf16", 16,
             seed=6, shared=6000)
    past = p.past.clone()
    past[7] = 10 ** 6
    p.cache.attention_shared(0, p.q, past, p.table, 6000, p.out)
    with pytest.raises(tg.TGError) as e:
        backend.synchronize()
    assert e.value.status == tg.TG_ERR_DEVICE and "0x103" in e.value.message
    assert not p.out[7].any()
    p.check(p.out, seqs=[0, 6, 8, 49])


def test_shared_equals_plain(tg, backend):
    import torch
    p = Pool(tg, backend, [2100, 2048, 3000, 2047], (14, 2, 64), "bf16", 16, seed=2, shared=2048)
    plain = torch.zeros_like(p.out)
    p.cache.attention_shared(0, p.q, p.past, p.table, 2048, p.out)
    p.cache.attention(0, p.q, p.past, p.table, plain)
    backend.synchronize()
    p.check(p.out)
    p.check(plain)


# ---------------------------------------------------------------- selection

def _select_ref(p, n_sel, keep_first, keep_last):
    b, q = f64(p.bounds[p.layer]), f64(p.q)
    per = p.H // p.G
    out = np.full((len(p.lens), p.G, n_sel), -1, np.int32)
    for s, rows in enumerate(p.lens):
        nb = -(-rows // p.P)
        for g in range(p.G):
            score = np.full(nb, -np.inf)
            for j in range(nb):
                lo, hi = b[p.table_np[s, j], g]
                for h in range(g * per, (g + 1) * per):
                    x = q[s, h * p.D:(h + 1) * p.D]
                    score[j] = max(score[j], np.maximum(x * lo, x * hi).sum())
            score[:keep_first] = np.inf
            score[max(0, nb - keep_last):] = np.inf
            order = sorted(range(nb), key=lambda j: (-score[j], j))
            got = sorted(order[:n_sel])
            out[s, g, :len(got)] = got
    return out


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page,n_sel", [(8, 1), (16, 5), (16, 40), (32, 300)])
def test_select(tg, backend, shape, dtype, page, n_sel):
    import torch
    lens = [0, 1, page, page + 1, 5 * page, 5 * page + 1, 700, 40 * page, 1500]
    p = Pool(tg, backend, lens, shape, dtype, page, seed=n_sel)
    for first, last in ((1, 1), (0, 0), (3, 2)):
        pages = torch.full((len(lens), p.G, n_sel), 99, dtype=torch.int32).cuda()
        p.cache.select_pages(0, p.q, p.past, p.table, pages, first, last)
        backend.synchronize()
        assert np.array_equal(pages.cpu().numpy(), _select_ref(p, n_sel, first, last))


def test_select_ties_and_long(tg, backend):
    """Equal scores (pages named twice, zero queries) go to the lower index,
    over more pages than one pass of the block holds."""
    import torch
    page, lens = 16, [16 * 5000 + 3, 16 * 700]
    p = Pool(tg, backend, lens, (14, 2, 64), "bf16", page, seed=1)
    p.table_np[0, 100:5000:2] = p.table_np[0, 50]
    p.table_np[1, 1:650] = p.table_np[1, 0]
    p.table = torch.from_numpy(p.table_np).cuda()
    for zero in (False, True):
        if zero:
            p.q.zero_()
            p.q[:, ::2] = -0.0
        for n_sel in (1, 37, 256, 2600):
            pages = torch.zeros(2, 2, n_sel, dtype=torch.int32).cuda()
            p.cache.select_pages(0, p.q, p.past, p.table, pages, 1, 1)
            backend.synchronize()
            assert np.array_equal(pages.cpu().numpy(), _select_ref(p, n_sel, 1, 1))


def test_select_nan_ranks_last(tg, backend):
    import torch
    p = Pool(tg, backend, [640], (14, 2, 64), "f32", 16, seed=1)
    p.bounds[0, int(p.table_np[0, 7])] = float("nan")
    p.bounds[0, int(p.table_np[0, 9]), :, 1] = float("inf")
    p.bounds[0, int(p.table_np[0, 9]), :, 0] = float("-inf")
    pages = torch.zeros(1, 2, 39, dtype=torch.int32).cuda()
    p.cache.select_pages(0, p.q, p.past, p.table, pages, 0, 0)
    one = torch.zeros(1, 2, 1, dtype=torch.int32).cuda()
    p.cache.select_pages(0, p.q, p.past, p.table, one, 0, 0)
    backend.synchronize()
    for g in range(2):
        assert pages[0, g].tolist() == [j for j in range(40) if j != 7]
    assert one.flatten().tolist() == [9, 9]


# ------------------------------------------------------------ listed pages

@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page,n_sel", [(8, 3), (16, 10), (64, 5)])
def test_attention_sparse(tg, backend, shape, dtype, page, n_sel):
    import torch
    rng = np.random.default_rng(page)
    lens = [0, 1, page + 1, 9 * page, 20 * page - 3, 37 * page + 5]
    p = Pool(tg, backend, lens, shape, dtype, page, seed=page)
    sel = np.full((len(lens), p.G, n_sel), -1, np.int32)
    for s, rows in enumerate(lens):
        nb = -(-rows // page)
        for g in range(p.G):
            m = min(nb, n_sel)
            pick = rng.permutation(nb)[:m]
            if s % 2:
                pick.sort()
            sel[s, g, :m] = pick
    sel[-1, 0, 0] = nb - 1                             # the partial page, not in order
    sel[-1, 0, 1:] = [j for j in range(nb - 1)][:n_sel - 1]
    sel[-2, p.G - 1, 1] = -1                            # a hole
    sel[-2, 0, 0] = 10 ** 6 if p.G > 1 else sel[-2, 0, 0]   # holds no position of the sequence
    p.cache.attention_sparse(0, p.q, p.past, p.table, torch.from_numpy(sel).cuda(), p.out)
    backend.synchronize()
    ref = [[[j for j in sel[s, g] if 0 <= j < -(-lens[s] // page)] for g in range(p.G)]
           for s in range(len(lens))]
    p.check(p.out, ref)


def test_sparse_twice_and_none(tg, backend):
    """An entry listed twice counts twice; a list of nothing gives zeros;
    long lists split over CTAs."""
    import torch
    p = Pool(tg, backend, [400, 400, 60000], (14, 2, 64), "bf16", 16, seed=9)
    sel = np.full((3, 2, 1500), -1, np.int32)
    sel[0, :, :3] = [4, 4, 2]
    sel[2, :] = np.sort(np.random.default_rng(0).permutation(3750)[:1500])
    p.cache.attention_sparse(0, p.q, p.past, p.table, torch.from_numpy(sel).cuda(), p.out)
    backend.synchronize()
    p.check(p.out, [[[4, 4, 2]] * 2, [[]] * 2, list(sel[2])])


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_loop(tg, backend, dtype):
    """As a server runs it: a common prompt once, every sequence's own tokens
    behind it, then single-token steps with all three readers, every step one
    graph replay; checked against 64-bit attention over what was appended."""
    import torch
    H, G, D, P, n, sh, steps = 14, 2, 64, 16, 5, 96, 20
    g = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    dt, code = (torch.bfloat16, tg.DTYPE_BF16) if dtype == "bf16" else (torch.float32, tg.DTYPE_F32)
    cols, pages = 12, 6 + 5 * 6
    kp = torch.zeros(pages, G, P, D, dtype=dt, device="cuda")
    vp = torch.zeros_like(kp)
    c = tg.PagedKVCache(backend, 1, pages, P, H, G, D, code, max_pos=256, k=kp, v=vp)
    table = torch.zeros(n, cols, dtype=torch.int32)
    table[:, :6] = torch.arange(6)
    table[:, 6:] = 6 + torch.arange(30).view(5, 6)
    table = table.cuda()
    backend.set_stream(torch.cuda.current_stream().cuda_stream)
    c.append(0, rnd(sh, 128), rnd(sh, 128), i32([0]), table[:1].contiguous(), cu_tokens=i32([0, sh]))
    new = [1, 7, 0, 16, 33]
    cu = i32([0] + list(np.cumsum(new)))
    c.append(0, rnd(sum(new), 128), rnd(sum(new), 128), i32([sh] * n), table, cu_tokens=cu)
    pos = i32([sh + x for x in new])
    k, v, q, qr = rnd(n, 128), rnd(n, 128), rnd(n, 896), rnd(n, 896)
    outs = [torch.zeros(n, 896, device="cuda") for _ in range(3)]
    sel = torch.zeros(n, G, 6, dtype=torch.int32, device="cuda")

    def step():
        c.append(0, k, v, pos, table, q=q, q_out=qr)
        c.attention(0, qr, pos, table, outs[0])
        c.attention_shared(0, qr, pos, table, sh, outs[1])
        c.select_pages(0, qr, pos, table, sel)
        c.attention_sparse(0, qr, pos, table, sel, outs[2])

    step()
    torch.cuda.synchronize()
    own = torch.cuda.Stream()
    backend.set_stream(own.cuda_stream)                # a stream that can be captured
    backend.graph_begin()
    step()
    graph = backend.graph_end()
    for _ in range(steps):
        pos += 1
        for x in (k, v, q):
            x.copy_(rnd(*x.shape))
        torch.cuda.synchronize()
        graph.launch()
        backend.synchronize()
        for s in range(n):
            rows = int(pos[s]) + 1
            for h in range(H):
                kk = kp[table[s].long(), h // 7].reshape(-1, D)[:rows].double()
                vv = vp[table[s].long(), h // 7].reshape(-1, D)[:rows].double()
                x = kk @ qr[s, h * D:(h + 1) * D].double() / 8
                tol = 6 * (2 * 24 * 2.0 ** -16 + 2.0 ** -15)   # |v| < 6, sum |q k| / 8 < 24
                ref = torch.softmax(x, 0) @ vv
                for o in outs[:2]:
                    assert (o[s, h * D:(h + 1) * D].double() - ref).abs().max() <= tol
                keep = torch.cat([torch.arange(j * P, min(rows, (j + 1) * P))
                                  for j in sel[s, h // 7].tolist() if j >= 0]).cuda()
                ref = torch.softmax(x[keep], 0) @ vv[keep]
                assert (outs[2][s, h * D:(h + 1) * D].double() - ref).abs().max() <= tol
    graph.destroy()
    torch.cuda.synchronize()
    backend.set_stream(torch.cuda.current_stream().cuda_stream)


def test_graphs_survive_larger_calls(tg):
    """A captured graph keeps its scratch when later calls need more, and two
    graphs replayed in turn do not disturb each other."""
    import torch
    be = tg.CudaBackend(0)
    small = Pool(tg, be, [900, 40], (14, 2, 64), "bf16", 16, seed=1)
    big = Pool(tg, be, [5000] * 40, (14, 2, 64), "bf16", 16, seed=2)
    pages = torch.zeros(2, 2, 8, dtype=torch.int32).cuda()
    torch.cuda.synchronize()

    def call(p):
        p.cache.attention(0, p.q, p.past, p.table, p.out)

    graphs = []
    for p in (small, big):
        call(p)
        if p is small:
            p.cache.select_pages(0, p.q, p.past, p.table, pages)
        be.synchronize()
        be.graph_begin()
        call(p)
        if p is small:
            p.cache.select_pages(0, p.q, p.past, p.table, pages)
        graphs.append(be.graph_end())
    want = [p.out.clone() for p in (small, big)]
    want_pages = pages.clone()
    for _ in range(3):
        for p in (small, big):
            p.out.zero_()
        pages.zero_()
        torch.cuda.synchronize()
        graphs[0].launch()
        graphs[1].launch()
        be.synchronize()
        assert torch.equal(small.out, want[0]) and torch.equal(big.out, want[1])
        assert torch.equal(pages, want_pages)
    small.check(small.out)
    for g in graphs:
        g.destroy()
    be.shutdown()


def test_host_arrays_and_batches(tg, backend):
    """numpy arguments (staged) inside and outside a batch."""
    p = Pool(tg, backend, [5, 0, 300], (14, 2, 64), "bf16", 16, seed=12)
    q, past, table = (x.cpu().numpy() for x in (p.q, p.past, p.table))
    out = np.full(q.shape, 5.0, np.float32)
    p.cache.attention(0, q, past, table, out)
    p.check(out)
    sel = np.zeros((3, 2, 4), np.int32)
    out2, out3 = np.zeros_like(out), np.zeros_like(out)
    backend.metal_batch_begin()
    p.cache.attention_shared(0, q, past, table, 0, out2)
    p.cache.select_pages(0, q, past, table, sel)
    backend.metal_batch_end()
    p.check(out2)
    assert np.array_equal(sel, _select_ref(p, 4, 1, 1))
    p.cache.attention_sparse(0, q, past, table, sel, out3)
    p.check(out3, [[[j for j in sel[s, g] if j >= 0] for g in range(2)] for s in range(3)])
    k = np.ones((1, 128), np.float32)
    q_out = np.full((2, 896), 4.0, np.float32)
    p.cache.append(0, np.repeat(k, 2, 0), np.repeat(k, 2, 0), past[:1], table[:1],
                   q=q[:2].copy(), q_out=q_out, cu_tokens=np.array([0, 1], np.int32))
    assert (q_out[1] == 4.0).all() and not (q_out[0] == 4.0).all()   # row 1 is padding


# ------------------------------------------------------------------ refusals

def test_refusals(tg, backend):
    import torch
    bad = [dict(page_size=12), dict(page_size=4), dict(page_size=512), dict(n_pages=0),
           dict(n_layers=0), dict(max_pos=0), dict(rope_base=0.0), dict(dtype=3),
           dict(head_dim=63), dict(n_head=15), dict(n_pages=1 << 27)]
    base = dict(n_layers=1, n_pages=4, page_size=16)
    for b in bad:
        with pytest.raises(tg.TGError) as e:
            tg.PagedKVCache(backend, **{**base, **b})
        assert e.value.status == tg.TG_ERR_INVALID_ARG, b
    pool = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16).cuda()
    with pytest.raises(tg.TGError):
        tg.PagedKVCache(backend, 1, 4, 16, k=pool)            # k without v
    with pytest.raises(ValueError):
        tg.PagedKVCache(backend, 1, 5, 16, k=pool, v=pool)    # sizes
    with pytest.raises(ValueError):
        tg.PagedKVCache(backend, 1, 4, 16, k=pool.float(), v=pool.float())
    host = np.zeros((4, 2, 16, 64), np.uint16)
    with pytest.raises(tg.TGError):
        tg.PagedKVCache(backend, 1, 4, 16, k=host, v=host)
    p = Pool(tg, backend, [20, 3], (14, 2, 64), "bf16", 16)
    c, i32 = p.cache, lambda *x: np.array(x, np.int32)
    pages = torch.zeros(2, 2, 4, dtype=torch.int32).cuda()
    q, past, table = (x.cpu().numpy() for x in (p.q, p.past, p.table))
    out = np.zeros_like(q)
    for call in (lambda: c.attention(1, p.q, p.past, p.table, p.out),
                 lambda: c.attention(-1, p.q, p.past, p.table, p.out),
                 lambda: c.attention_shared(0, p.q, p.past, p.table, -1, p.out),
                 lambda: c.attention_shared(0, p.q, p.past, p.table, 10 ** 6, p.out),
                 lambda: c.select_pages(0, p.q, p.past, p.table, pages, -1, 0),
                 lambda: c.attention(0, q, i32(-2, 3), table, out),
                 lambda: c.attention(0, q, i32(5000, 3), table, out),
                 lambda: c.attention(0, q, past, table * 0 - 1, out),
                 lambda: c.append(0, q[:, :128].copy(), q[:, :128].copy(), i32(0), table[:1]),
                 lambda: c.append(0, q[:, :128].copy(), q[:, :128].copy(), i32(-1, 0), table),
                 lambda: c.append(0, q[:, :128].copy(), q[:, :128].copy(), i32(5000, 0), table),
                 lambda: c.append(0, q[:, :128].copy(), q[:, :128].copy(), i32(0, 0), table,
                                  cu_tokens=i32(0, 3, 2)),
                 lambda: c.append(0, q[:, :128].copy(), q[:, :128].copy(), i32(0, 0), table,
                                  cu_tokens=i32(0, 1, 3)),
                 lambda: c.append(0, q[:, :128].copy(), q[:, :128].copy(), i32(0, 0), table + 999)):
        with pytest.raises(tg.TGError) as e:
            call()
        assert e.value.status == tg.TG_ERR_INVALID_ARG
    for call in (lambda: c.attention(0, p.q[:1], p.past, p.table, p.out),
                 lambda: c.attention(0, p.q.double(), p.past, p.table, p.out),
                 lambda: c.attention(0, p.q, p.past.long(), p.table, p.out),
                 lambda: c.attention(0, p.q, p.past, p.table[0], p.out),
                 lambda: c.attention(0, p.q, p.past[:1], p.table, p.out),
                 lambda: c.attention(0, p.q, p.past, p.table.t(), p.out),
                 lambda: c.select_pages(0, p.q, p.past, p.table, pages[:1]),
                 lambda: c.append(0, p.q[:, :128].contiguous(), p.q[:1, :128].contiguous(), p.past, p.table),
                 lambda: c.append(0, p.q[:, :128].contiguous(), p.q[:, :128].contiguous(), p.past, p.table,
                                  q_out=p.q)):
        with pytest.raises(ValueError):
            call()
    none = tg.PagedKVCache(backend, 1, 4, 16, with_bounds=False)
    assert none.layer_ptrs(0)[2] is None
    with pytest.raises(tg.TGError) as e:
        none.select_pages(0, p.q, p.past, p.table, pages)
    assert e.value.status == tg.TG_ERR_UNSUPPORTED
    other = tg.CudaBackend(0)
    L = tg.lib()
    assert L.tg_paged_attention(other.handle, c.handle, 0, 0, None, None, None, 1, None) == \
        tg.TG_ERR_INVALID_ARG                                # a cache of another context
    other.shutdown()
    c.attention(0, p.q, p.past, p.table, p.out)               # and all is well after them
    backend.synchronize()
    p.check(p.out)


def test_device_errors_are_reported(tg, backend):
    """Positions and pages out of range in device arrays: the rows concerned
    are left out, the others are right, and the error surfaces at the sync."""
    import torch
    p = Pool(tg, backend, [20, 300, 33], (14, 2, 64), "bf16", 16)
    past = p.past.clone()
    past[0] = 10 ** 6
    p.cache.attention(0, p.q, past, p.table, p.out)
    with pytest.raises(tg.TGError) as e:
        backend.synchronize()
    assert e.value.status == tg.TG_ERR_DEVICE and "0x103" in e.value.message
    assert not p.out[0].any()
    p.check(p.out, seqs=[1, 2])
    table = p.table.clone()
    table[0, 1] = 10 ** 6
    table[2, 0] = -5
    pages = torch.zeros(3, 2, 2, dtype=torch.int32).cuda()
    for call in (lambda: p.cache.attention(0, p.q, p.past, table, p.out),
                 lambda: p.cache.attention_shared(0, p.q, p.past, table, 0, p.out),
                 lambda: p.cache.select_pages(0, p.q, p.past, table, pages),
                 lambda: p.cache.append(0, p.q[:, :128].contiguous(), p.q[:, :128].contiguous(),
                                        p.past, table)):
        call()
        with pytest.raises(tg.TGError) as e:
            backend.synchronize()
        assert e.value.status == tg.TG_ERR_DEVICE and "0x106" in e.value.message
    p.cache.attention(0, p.q, p.past, p.table, p.out)
    backend.synchronize()
