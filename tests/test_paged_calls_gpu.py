"""Calls of the paged cache that its header allows and that are easily left
out: rows of one sequence in one append, keys that are NaN, tiny queries,
tables with dropped pages, contexts in two threads."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def i32(x):
    import torch
    return torch.tensor(np.asarray(x), dtype=torch.int32).cuda()


# ------------------------------------------- rows of one sequence in one append

def _rows_of_sequences(rng, lens, tokens, page, chunk, order):
    """Table rows (sequence, first position, tokens) of a call that appends
    tokens[s] tokens behind lens[s] rows of sequence s, `chunk` at a time."""
    rows = []
    for s, (n, m) in enumerate(zip(lens, tokens)):
        at = 0
        while at < m:
            step = min(chunk or int(rng.integers(1, 2 * page)), m - at)
            rows.append((s, n + at, step))
            at += step
    if order == "down":
        rows.reverse()
    elif order == "mixed":
        rows = [rows[i] for i in rng.permutation(len(rows))]
    return rows


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape,page", [((14, 2, 64), 16), ((8, 8, 32), 8), ((4, 4, 6), 256),
                                        ((16, 1, 128), 64)])
@pytest.mark.parametrize("chunk,order", [(1, "up"), (1, "down"), (1, "mixed"), (2, "mixed"),
                                         (0, "up"), (0, "mixed")])
def test_append_rows_of_one_sequence(tg, backend, O, dtype, shape, page, chunk, order):
    """Several rows with the same entries (a draft as a row per token, a prompt
    in chunks): one pair of bounds per page, over the tokens of all rows."""
    import torch
    H, G, D = shape
    rng = np.random.default_rng(page + chunk)
    lens = [0, 5, page - 1, page, 2 * page + 3, 7, 3 * page - 2]
    tokens = [3, 1, 2, 5, 2 * page + 1, 0, 4]
    cols = 6
    order_np = rng.permutation(len(lens) * cols).astype(np.int32)
    own = order_np.reshape(len(lens), cols)             # pages of the sequences
    rows = _rows_of_sequences(rng, lens, tokens, page, chunk, order)
    table = own[[s for s, _, _ in rows]]
    pos0 = np.array([p for _, p, _ in rows], np.int32)
    cu = np.concatenate([[0], np.cumsum([m for _, _, m in rows])]).astype(np.int32)
    T = int(cu[-1])
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    k, v = (rng.standard_normal((T, G * D)).astype(np.float32) for _ in range(2))
    k[rng.random(T) < 0.3] *= 20.0                      # a missed key shows in the bounds
    size = (1, order_np.size, G, page, D)
    kp0, vp0 = torch.randn(size).to(dt), torch.randn(size).to(dt)
    b0 = torch.full((1, order_np.size, G, 2, D), 9.0).to(dt)
    kp, vp, bd = kp0.cuda(), vp0.cuda(), b0.cuda()
    cache = tg.PagedKVCache(backend, 1, order_np.size, page, H, G, D,
                            tg.DTYPE_BF16 if dtype == "bf16" else tg.DTYPE_F32, max_pos=4096,
                            k=kp, v=vp, bounds=bd)
    cache.append(0, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), i32(pos0), i32(table),
                 cu_tokens=None if chunk == 1 else i32(cu))
    backend.synchronize()
    want_k, want_v, want_b = kp0.clone(), vp0.clone(), b0.clone()
    for i, (s, p0, m) in enumerate(rows):
        for x in range(m):
            t, pos = cu[i] + x, p0 + x
            pg, slot = own[s, pos // page], pos % page
            want_k[0, pg, :, slot] = torch.from_numpy(O.rope_heads(k[t], G, D, pos)).view(G, D).to(dt)
            want_v[0, pg, :, slot] = torch.from_numpy(v[t]).view(G, D).to(dt)
    for s, (n, m) in enumerate(zip(lens, tokens)):
        for j in range(n // page, (n + m - 1) // page + 1) if m else ():
            x = want_k[0, own[s, j], :, :min(page, n + m - j * page)].float()
            want_b[0, own[s, j]] = torch.stack([x.amin(1), x.amax(1)], 1).to(dt)
    assert torch.equal(kp.cpu(), want_k)
    assert torch.equal(vp.cpu(), want_v)
    assert torch.equal(bd.cpu(), want_b)
    cache.destroy()


@pytest.mark.parametrize("where", ["device", "host"])
def test_append_to_a_padded_batch(tg, backend, O, where):
    """Rows without tokens are padding, whatever their position and entries."""
    import torch
    rng = np.random.default_rng(3)
    P, n = 16, 70
    live = np.flatnonzero(rng.random(n) < 0.5)
    pos0, table = np.full(n, -1, np.int32), np.full((n, 3), -1, np.int32)
    pos0[live] = rng.integers(0, 3 * P, len(live))
    for i, s in enumerate(live):
        table[s, pos0[s] // P] = i
    cu = np.concatenate([[0], np.cumsum(np.isin(np.arange(n), live))]).astype(np.int32)
    T = n                                                # tokens of the live rows, then padding
    k, q = (rng.standard_normal((T, w)).astype(np.float32) for w in (128, 896))
    kp, vp = (torch.zeros(1, len(live), 2, P, 64).cuda() for _ in range(2))
    bd = torch.full((1, len(live), 2, 2, 64), 5.0).cuda()
    c = tg.PagedKVCache(backend, 1, len(live), P, dtype=tg.DTYPE_F32, max_pos=64, k=kp, v=vp, bounds=bd)
    put = (lambda x: torch.from_numpy(x).cuda()) if where == "device" else (lambda x: x.copy())
    out = put(np.full_like(q, 3.0))
    c.append(0, put(k), put(k), put(pos0), put(table), q=put(q), q_out=out, cu_tokens=put(cu))
    backend.synchronize()
    out = out.cpu().numpy() if where == "device" else out
    for i, s in enumerate(live):
        want = O.rope_heads(k[i], 2, 64, int(pos0[s])).reshape(2, 64)
        assert np.array_equal(kp[0, i, :, pos0[s] % P].cpu().numpy(), want)
        assert np.array_equal(out[i], O.rope_heads(q[i], 14, 64, int(pos0[s])))
        if pos0[s] % P == 0:
            assert np.array_equal(bd[0, i].cpu().numpy(), np.stack([want, want], 1))
    assert (out[len(live):] == 3.0).all()
    c.destroy()


# ------------------------------------------------------------------- NaN keys

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 3])
def test_append_nan_key_reaches_the_bounds(tg, backend, dtype, rows):
    """A page with a NaN key has NaN bounds in its dimension pair (the rotation
    mixes two), whether the row is new or was there, and is selected last."""
    import torch
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    P, T = 16, 80
    rng = np.random.default_rng(rows)
    k, v = (rng.standard_normal((T, 128)).astype(np.float32) for _ in range(2))
    k[5, 10] = k[37, 64 + 3] = np.nan                    # pages 0 and 2, KV heads 0 and 1
    kp, vp = (torch.zeros(1, 5, 2, P, 64, dtype=dt).cuda() for _ in range(2))
    bd = torch.zeros(1, 5, 2, 2, 64, dtype=dt).cuda()
    c = tg.PagedKVCache(backend, 1, 5, P, dtype=tg.DTYPE_BF16 if dtype == "bf16" else tg.DTYPE_F32,
                        max_pos=128, k=kp, v=vp, bounds=bd)
    kd, vd = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()
    table = i32(np.arange(5)[None].repeat(rows, 0))
    cut = [0, 7, 40, T] if rows == 3 else [0, T]         # three rows of one sequence, or one
    c.append(0, kd[:T], vd[:T], i32(cut[:-1]), table, cu_tokens=i32(cut))
    c.append(0, kd[6:7], vd[6:7], i32([6]), table[:1].contiguous())    # page 0 again: the row was there
    q = torch.from_numpy(rng.standard_normal((1, 896)).astype(np.float32)).cuda()
    pages = torch.zeros(1, 2, 4, dtype=torch.int32).cuda()
    c.select_pages(0, q, i32([T - 1]), table[:1].contiguous(), pages, 0, 0)
    backend.synchronize()
    nan = torch.isnan(bd.float().cpu())[0]
    want = torch.zeros(5, 2, 2, 64, dtype=torch.bool)
    want[0, 0, :, 10:12] = True
    want[2, 1, :, 2:4] = True
    assert torch.equal(nan, want)
    rest = ~want
    rows_k = kp.float().cpu()[0]
    rows_k[0, :, 7:] = rows_k[0, :, :1]                  # the last append renewed 7 rows
    ref = torch.stack([rows_k.amin(2), rows_k.amax(2)], 2)
    assert torch.equal(bd.float().cpu()[0][rest], ref[rest])
    assert pages[0, 0].tolist() == [1, 2, 3, 4] and pages[0, 1].tolist() == [0, 1, 3, 4]
    c.destroy()


# ------------------------------------------------- selection at the range's ends

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape", [(14, 2, 64), (16, 1, 128), (8, 8, 32), (4, 4, 6)])
@pytest.mark.parametrize("q_exp,b_exp", [(0, 0), (-120, 0), (-128, 0), (-136, 0), (-144, 0),
                                         (-70, -70), (0, -130), (60, 60)])
def test_select_small_and_large_values(tg, backend, dtype, shape, q_exp, b_exp):
    """The order is that of the binary64 scores where binary32 is subnormal or
    overflows too."""
    import torch
    H, G, D = shape
    rng = np.random.default_rng(D)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    nb, P, n = 300, 8, 3
    lo = rng.standard_normal((nb, G, D)) - 1.0
    hi = lo + np.abs(rng.standard_normal((nb, G, D)))
    bounds = torch.from_numpy((np.stack([lo, hi], 2) * 2.0 ** b_exp)).to(dt)[None].contiguous()
    q = torch.from_numpy((rng.standard_normal((n, H * D)) * 2.0 ** q_exp).astype(np.float32))
    pool = [torch.zeros(1, nb, G, P, D, dtype=dt).cuda() for _ in range(2)]
    c = tg.PagedKVCache(backend, 1, nb, P, H, G, D,
                        tg.DTYPE_BF16 if dtype == "bf16" else tg.DTYPE_F32, max_pos=64, k=pool[0],
                        v=pool[1], bounds=bounds.cuda())
    table = np.stack([rng.permutation(nb) for _ in range(n)])
    n_sel = 40
    pages = torch.zeros(n, G, n_sel, dtype=torch.int32).cuda()
    c.select_pages(0, q.cuda(), i32([nb * P - 1] * n), i32(table), pages, 0, 0)
    backend.synchronize()
    b = bounds[0].double().numpy()
    x = q.double().numpy().reshape(n, G, H // G, D)
    for s in range(n):
        for g in range(G):
            bl, bh = b[table[s], g, 0], b[table[s], g, 1]
            score = np.maximum(x[s, g][:, None] * bl, x[s, g][:, None] * bh).sum(-1).max(0)
            order = sorted(range(nb), key=lambda j: (-score[j], j))
            assert pages[s, g].tolist() == sorted(order[:n_sel]), (s, g)
    c.destroy()


@pytest.mark.parametrize("fill", [float("nan"), 1e30])
def test_select_ignores_pages_of_nobody(tg, backend, fill):
    """Bounds of a page that no table names change neither the result nor the
    work (they once widened the set of pages to be scored again to all of
    them: 36 times the time)."""
    import torch
    nb, n, n_sel = 8187, 4, 256                          # the last pass of a row is not full
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(1, nb + 1, 2, 64, generator=g, device="cuda")
    bounds = torch.stack([x - 0.5, x + 0.5], 3).to(torch.bfloat16).contiguous()
    pool = torch.zeros(1, nb + 1, 2, 8, 64, dtype=torch.bfloat16, device="cuda")
    c = tg.PagedKVCache(backend, 1, nb + 1, 8, max_pos=64, k=pool, v=pool, bounds=bounds)
    table = (torch.arange(nb, dtype=torch.int32, device="cuda") + 1).repeat(n, 1).contiguous()
    q = torch.randn(n, 896, generator=g, device="cuda")
    past = i32([nb * 8 - 1] * n)
    backend.set_stream(torch.cuda.current_stream().cuda_stream)
    results, times = [], []
    for value in (0.0, fill):
        bounds[:, 0] = value
        pages = torch.zeros(n, 2, n_sel, dtype=torch.int32, device="cuda")
        best = float("inf")
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(10):
                c.select_pages(0, q, past, table, pages, 0, 0)
            b.record()
            backend.synchronize()
            best = min(best, a.elapsed_time(b))
        results.append(pages)
        times.append(best)
    assert torch.equal(results[0], results[1])
    assert times[1] < 4 * times[0], times
    c.destroy()


@pytest.mark.parametrize("times", [50.0, 5000.0])
@pytest.mark.parametrize("shape,dtype", [((14, 2, 64), "bf16"), ((32, 8, 128), "bf16"),
                                         ((12, 4, 64), "f32"), ((4, 4, 6), "f32")])
def test_select_outlier_dimension(tg, backend, shape, dtype, times):
    """A key dimension that is far larger than the others widens the set of
    pages that are scored again (past the 256 that one CTA ranks by itself);
    the result is the exact one."""
    import torch
    H, G, D = shape
    rng = np.random.default_rng(D)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    nb, P, n, n_sel = 3000, 8, 2, 500
    lo = rng.standard_normal((nb, G, D)) * 0.01 - 0.5
    hi = lo + np.abs(rng.standard_normal((nb, G, D))) * 0.01
    lo[..., 3] *= times
    hi[..., 3] = lo[..., 3] + np.abs(rng.standard_normal((nb, G)))
    bounds = torch.from_numpy(np.stack([lo, hi], 2)).to(dt)[None].contiguous()
    q = torch.from_numpy(rng.standard_normal((n, H * D)).astype(np.float32))
    pool = torch.zeros(1, nb, G, P, D, dtype=dt).cuda()
    c = tg.PagedKVCache(backend, 1, nb, P, H, G, D,
                        tg.DTYPE_BF16 if dtype == "bf16" else tg.DTYPE_F32, max_pos=64, k=pool,
                        v=pool, bounds=bounds.cuda())
    table = np.stack([rng.permutation(nb) for _ in range(n)])
    pages = torch.zeros(n, G, n_sel, dtype=torch.int32).cuda()
    c.select_pages(0, q.cuda(), i32([nb * P - 1] * n), i32(table), pages)
    backend.synchronize()
    b = bounds[0].double().numpy()
    x = q.double().numpy().reshape(n, G, H // G, D)
    for s in range(n):
        for g in range(G):
            bl, bh = b[table[s], g, 0], b[table[s], g, 1]
            score = np.maximum(x[s, g][:, None] * bl, x[s, g][:, None] * bh).sum(-1).max(0)
            score[0] = score[-1] = np.inf
            order = sorted(range(nb), key=lambda j: (-score[j], j))
            assert pages[s, g].tolist() == sorted(order[:n_sel]), (s, g)
    c.destroy()


# ------------------------------------------------------------ dropped pages

def test_sparse_reads_listed_entries_only(tg, backend):
    """A table whose unlisted entries are no pages (dropped ones), on the host
    and on the device; a listed one that is none is refused or reported."""
    import torch
    from test_paged_gpu import Pool
    p = Pool(tg, backend, [20 * 16 - 3, 40, 9], (14, 2, 64), "bf16", 16, seed=2)
    sel = np.full((3, 2, 4), -1, np.int32)
    sel[0, 0], sel[0, 1] = [0, 3, 7, 19], [2, 3, 19, 10 ** 6]
    sel[1, :, :2] = [0, 2]
    sel[1, 1, 3] = 1                       # behind the first min(n_sel, 3) entries: not read
    sel[2, :, 0] = 0
    table = np.full_like(p.table_np, -1)
    for s in range(3):
        for j in set(sel[s, :, :min(4, -(-p.lens[s] // 16))].flatten()) & set(range(table.shape[1])):
            table[s, j] = p.table_np[s, j]
    ref = [[[j for j in sel[s, g, :min(4, -(-p.lens[s] // 16))] if 0 <= j < -(-p.lens[s] // 16)]
            for g in range(2)] for s in range(3)]
    p.cache.attention_sparse(0, p.q, p.past, i32(table), torch.from_numpy(sel).cuda(), p.out)
    backend.synchronize()
    p.check(p.out, ref)
    q, past = p.q.cpu().numpy(), p.past.cpu().numpy()
    out = np.zeros_like(q)
    p.cache.attention_sparse(0, q, past, table, sel, out)
    p.check(out, ref)
    out[:] = 0
    p.cache.attention_sparse(0, q, past, table, torch.from_numpy(sel).cuda(), out)   # a device list
    p.check(out, ref)
    bad = table.copy()
    bad[0, 7] = -1
    with pytest.raises(tg.TGError) as e:
        p.cache.attention_sparse(0, q, past, bad, sel, out)
    assert e.value.status == tg.TG_ERR_INVALID_ARG and "[0][7]" in e.value.message
    with pytest.raises(tg.TGError) as e:
        p.cache.attention_sparse(0, q, past, bad, torch.from_numpy(sel).cuda(), out)
    assert e.value.status == tg.TG_ERR_DEVICE and "0x106" in e.value.message
    with pytest.raises(tg.TGError) as e:                       # the dense call reads them all
        p.cache.attention(0, q, past, table, out)
    assert e.value.status == tg.TG_ERR_INVALID_ARG
    p.cache.destroy()


# ------------------------------------------------------------ rotation tables

@pytest.mark.parametrize("max_pos", [0, -1, 2 ** 24 + 1, 2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1])
def test_max_pos_is_bounded(tg, backend, max_pos):
    with pytest.raises(tg.TGError) as e:
        tg.PagedKVCache(backend, 1, 4, 16, max_pos=max_pos)
    assert e.value.status == tg.TG_ERR_INVALID_ARG and "max_pos" in e.value.message


def test_rotation_table_that_does_not_fit(tg):
    """A status and a context that goes on, not an exception or the host's
    memory: 2^31 positions of 128 dimensions are 1 TB."""
    import torch
    be = tg.CudaBackend(0)
    x = torch.ones(1, 128, device="cuda")
    L = tg.lib()
    assert L.tg_rope_op(be.handle, x.data_ptr(), 1, 128, 2 ** 30, 1e6) == tg.TG_ERR_OUT_OF_MEMORY
    assert L.tg_rope_op(be.handle, x.data_ptr(), 1, 128, 2 ** 31 - 1, 1e6) == tg.TG_ERR_INVALID_ARG
    assert L.tg_rope_op(be.handle, x.data_ptr(), 1, 128, 0, 1e6) == tg.TG_OK
    be.synchronize()
    assert (x == 1).all()
    be.shutdown()


def test_positions_across_the_pieces_of_a_table(tg, backend, O):
    """Bit for bit the rotation of the oracle, wherever the table was cut."""
    import torch
    pos = [0, 1, 32767, 32768, 65535, 65536, 65537, 131071, 131072, 200_000, 262_142]
    n, P = len(pos), 256
    rng = np.random.default_rng(0)
    k = rng.standard_normal((n, 128)).astype(np.float32)
    kp, vp = (torch.zeros(1, n, 2, P, 64, device="cuda") for _ in range(2))
    c = tg.PagedKVCache(backend, 1, n, P, dtype=tg.DTYPE_F32, max_pos=262_143, k=kp, v=vp)
    table = np.full((n, 1024), -1)
    for s in range(n):
        table[s, pos[s] // P] = s
    kd = torch.from_numpy(k).cuda()
    c.append(0, kd, kd, i32(pos), i32(table))
    backend.synchronize()
    for s in range(n):
        want = O.rope_heads(k[s], 2, 64, pos[s]).reshape(2, 64)
        got = kp[0, s, :, pos[s] % P].cpu().numpy()
        assert np.array_equal(got.view(np.uint32), want.view(np.uint32)), pos[s]
    c.destroy()


# ------------------------------------------------------- contexts of threads

def test_contexts_in_threads(tg):
    """A context, cache and stream per thread, calling at once: every thread
    has the results that it has alone."""
    import threading

    from test_paged_gpu import Pool
    n, shared = 40, 8200
    made = []
    for i in range(4):
        be = tg.CudaBackend(0)
        p = Pool(tg, be, [shared // 16 * 16 + 7 * i + j for j in range(n)], (14, 2, 64), "bf16",
                 16, seed=i, shared=shared)
        made.append((be, p))
    import torch
    torch.cuda.synchronize()
    failed = []

    def work(be, p):
        try:
            for _ in range(20):
                p.cache.attention_shared(0, p.q, p.past, p.table, shared, p.out)
                p.cache.attention(0, p.q, p.past, p.table, p.out)
            p.out.zero_()
            torch.cuda.synchronize()
            p.cache.attention_shared(0, p.q, p.past, p.table, shared, p.out)
            be.synchronize()
        except Exception as e:  # noqa: BLE001 - handed to the test's own thread
            failed.append(e)

    threads = [threading.Thread(target=work, args=x) for x in made]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for be, p in made:
        p.check(p.out, seqs=[0, n // 2, n - 1])
        be.shutdown()


# ------------------------------------------------------- forms of a shared call

@pytest.mark.parametrize("shape,dtype,n,shared,launches", [
    ((8, 8, 64), "bf16", 1, 65536, 1), ((14, 2, 64), "bf16", 1, 131072, 1),   # nothing is shared
    ((8, 1, 64), "bf16", 1, 131072, 1), ((4, 1, 128), "f32", 1, 131072, 1),
    ((14, 2, 64), "bf16", 2, 65536, 1), ((14, 2, 64), "bf16", 32, 2048, 1),
    ((8, 8, 32), "bf16", 1000, 200, 1), ((32, 8, 128), "bf16", 256, 300, 1),
    ((8, 8, 64), "bf16", 8, 65536, 3), ((14, 2, 64), "bf16", 64, 8192, 3),    # much is
    ((8, 8, 32), "bf16", 1000, 900, 3), ((12, 4, 64), "f32", 1000, 900, 3),
    ((4, 4, 6), "bf16", 64, 65536, 1)])                                       # CUDA cores
def test_shared_form_by_what_it_saves(tg, backend, shape, dtype, n, shared, launches):
    """A prefix is attended for all queries where that is worth two launches
    more: never for one query (which took a form of 2.3 times the time over
    65536 rows of 8 KV heads), also for short ones of many queries."""
    import torch
    H, G, D = shape
    g = torch.Generator(device="cuda").manual_seed(n)
    P, pool = 256, 8
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    k, v = (torch.randn(1, pool, G, P, D, generator=g, device="cuda").to(dt) for _ in range(2))
    c = tg.PagedKVCache(backend, 1, pool, P, H, G, D,
                        tg.DTYPE_BF16 if dtype == "bf16" else tg.DTYPE_F32, max_pos=64, k=k, v=v)
    row = torch.randint(0, pool, (shared // P + 2,), generator=g, device="cuda", dtype=torch.int32)
    table = row.repeat(n, 1).contiguous()
    past = shared + torch.arange(n, dtype=torch.int32, device="cuda") % 200
    q = torch.randn(n, H * D, generator=g, device="cuda")
    outs = [torch.zeros_like(q) for _ in range(2)]
    before = backend.launch_count()
    c.attention_shared(0, q, past, table, shared, outs[0])
    assert backend.launch_count() - before == launches
    c.attention(0, q, past, table, outs[1])
    backend.synchronize()
    # Two ways to the same sums (|v| < 6): 2^-15 of it, and scores below 40 in
    # binary32 products.
    assert (outs[0] - outs[1]).abs().max() <= 6 * (2.0 ** -15 + 2 * 40 * D * 2.0 ** -24)
    c.destroy()


# ----------------------------------------------------- caches and captures

def test_destroy_inside_a_capture_is_refused(tg):
    """The capture goes on and its graph runs; the cache is destroyed after it,
    or by the shutdown when Python dropped it in between."""
    import torch

    from test_paged_gpu import Pool
    be = tg.CudaBackend(0)
    p = Pool(tg, be, [300, 7], (14, 2, 64), "bf16", 16, seed=3)
    other, dropped = (tg.PagedKVCache(be, 1, 4, 16) for _ in range(2))
    torch.cuda.synchronize()
    p.cache.attention(0, p.q, p.past, p.table, p.out)
    be.synchronize()
    be.graph_begin()
    p.cache.attention(0, p.q, p.past, p.table, p.out)
    with pytest.raises(tg.TGError) as e:
        other.destroy()
    assert e.value.status == tg.TG_ERR_STATE
    del dropped
    graph = be.graph_end()
    p.out.zero_()
    torch.cuda.synchronize()
    graph.launch()
    be.synchronize()
    p.check(p.out)
    other.destroy()
    graph.destroy()
    be.shutdown()
