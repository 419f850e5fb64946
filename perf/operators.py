"""Measured cases of the paged-cache operators: appending rotated keys and
values to a paged KV cache, decode attention over it, decode attention of a
batch that shares a long prefix, selection of pages by a bound on their
scores, and attention over the selected pages.

``run`` computes each operator in its plain form (elementary torch
operations) or, with ``own``, through the package's public calls.
"""
from __future__ import annotations

import importlib.util
import math
import os
import sys

import torch

own = False

DEV = "cuda"
ROPE_BASE = 1000000.0
MAX_POS = 131072          # positions of the rotation table
NEG = float("-inf")
DT = {"bf16": torch.bfloat16, "f32": torch.float32}

# Qwen2-0.5B's attention shape (14 query heads, 2 KV heads, 64), the other
# shapes are those of this repository's tests.
QWEN = {"n_head": 14, "n_kv": 2, "hd": 64}


# --------------------------------------------------------------------- cases

def listed():
    return [
        # One decode step of a served batch: a new token for each of 64 sequences.
        dict(QWEN, name="append decode", op="append", dtype="bf16", page=16, n=64,
             ctx_lo=1, ctx_hi=4096, new_lo=1, new_hi=1, pad=0),
        # Prompts of a served batch entering the cache, ragged, some of them
        # behind an earlier chunk, with padding tokens behind the last one.
        dict(QWEN, name="append prompts", op="append", dtype="bf16", page=16, n=16,
             ctx_lo=0, ctx_hi=1500, new_lo=3, new_hi=2048, pad=37),
        # The reference's own case: one sequence at the end of its 256 positions, fp32.
        dict(QWEN, name="attend one fp32", op="attend", dtype="f32", page=16, n=1,
             len_lo=256, len_hi=256),
        # A ragged fp32 batch of short sequences.
        dict(QWEN, name="attend ragged fp32", op="attend", dtype="f32", page=32, n=64,
             len_lo=0, len_hi=256),
        # Bandwidth-bound batched decode.
        dict(QWEN, name="attend batch", op="attend", dtype="bf16", page=16, n=256,
             len_lo=4096, len_hi=4096),
        # A few very long sequences: the work is split along them.
        dict(QWEN, name="attend long", op="attend", dtype="bf16", page=64, n=4,
             len_lo=131072, len_hi=131072),
        # A batch of chats behind one system prompt, each with its own short tail.
        dict(QWEN, name="shared prompt", op="shared", dtype="bf16", page=16, n=32,
             shared=2053, len_lo=1, len_hi=256),
        # Many questions about one long document.
        dict(QWEN, name="shared document", op="shared", dtype="bf16", page=32, n=128,
             shared=32768, len_lo=1, len_hi=1024),
        # Page selection of a served batch, and of a few very long sequences.
        dict(QWEN, name="select batch", op="select", dtype="bf16", page=16, n=64,
             len_lo=1000, len_hi=8192, n_sel=64),
        dict(QWEN, name="select long", op="select", dtype="bf16", page=16, n=4,
             len_lo=131072, len_hi=131072, n_sel=256),
        # Attention over the pages selected in those two.
        dict(QWEN, name="sparse batch", op="sparse", dtype="bf16", page=16, n=64,
             len_lo=1000, len_hi=8192, n_sel=64),
        dict(QWEN, name="sparse long", op="sparse", dtype="bf16", page=16, n=4,
             len_lo=131072, len_hi=131072, n_sel=256),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "shared", "select", "sparse"])
    n_head, n_kv, hd = rng.choice([(14, 2, 64)] * 3 + [(12, 4, 64), (8, 8, 32), (16, 1, 128)])
    c = {"op": op, "n_head": n_head, "n_kv": n_kv, "hd": hd,
         "dtype": rng.choice(["bf16", "bf16", "f32"]), "page": rng.choice([8, 16, 32, 64, 128])}
    row = 2 * n_kv * hd * DT[c["dtype"]].itemsize   # bytes of K and V per position
    if op == "append":
        c["n"] = _log_int(rng, 1, 256)
        c["new_hi"] = rng.choice([1, _log_int(rng, 2, max(2, 16384 // c["n"]))])
        c["new_lo"] = 1 if c["new_hi"] == 1 else rng.randint(0, c["new_hi"])
        c["ctx_lo"] = 0
        c["ctx_hi"] = _log_int(rng, 1, 4096)
        c["pad"] = rng.choice([0, rng.randint(1, 50)])
    elif op == "shared":
        c["n"] = _log_int(rng, 1, 128)
        c["shared"] = _log_int(rng, 100, min(65536, 128 * 32768 * 896 // (c["n"] * n_head * hd)))
        c["len_lo"], c["len_hi"] = 1, _log_int(rng, 1, 1024)
    else:
        # Rows of all sequences together: at most 400 MB of keys and values.
        c["n"] = _log_int(rng, 1, 256)
        # A selection leaves something out: the longest sequence has 8 pages or more.
        c["len_hi"] = _log_int(rng, 8 * c["page"] if op == "select" else 1,
                               min(131072, 400_000_000 // (row * c["n"])))
        c["len_lo"] = rng.choice([c["len_hi"], rng.randint(0, c["len_hi"])])
        if op == "select":
            c["n_sel"] = _log_int(rng, 3, min(512, c["len_hi"] // c["page"] // 2))
        elif op == "sparse":
            c["n_sel"] = _log_int(rng, 2, 512)
    return c


# ------------------------------------------------------------------- inputs

def _spread(lo, hi, n):
    """n whole numbers evenly over [lo, hi], both ends among them."""
    if n == 1:
        return [hi]
    return [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lens(case):
    """Rows that each sequence attends (its own ones behind a shared prefix)."""
    return _spread(case["len_lo"], case["len_hi"], case["n"])


def _shared_rows(case):
    return case["shared"] // case["page"] * case["page"]


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _shuffled(gen, values):
    t = torch.tensor(values, dtype=torch.int32, device=DEV)
    return t[torch.randperm(len(values), generator=gen, device=DEV)]


def _table(gen, need, cols):
    """A block table of need[s] pages for sequence s, pages in random order
    over the pool; page 0 is the empty page that unused entries name."""
    n = need.numel()
    total = int(need.sum())
    perm = torch.randperm(total, generator=gen, device=DEV).to(torch.int32) + 1
    table = torch.zeros(n, cols, dtype=torch.int32, device=DEV)
    use = torch.arange(cols, device=DEV)[None, :] < need[:, None]
    table[use] = perm
    return table, total + 1


def _rows(gen, dtype, n_pages, n_kv, page, hd):
    """Keys (or values): neighbours are alike, as those of a text are, so a
    page has a direction of its own."""
    x = _normal(gen, n_pages, n_kv, 1, hd) * 0.6
    return (_normal(gen, n_pages, n_kv, page, hd) * 0.8 + x).to(DT[dtype])


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    n, P = case["n"], case["page"]
    H, G, D = case["n_head"], case["n_kv"], case["hd"]
    st = dict(case)
    if case["op"] == "append":
        ctx, new = _spread(case["ctx_lo"], case["ctx_hi"], n), _spread(case["new_lo"], case["new_hi"], n)
        order = torch.randperm(n, generator=gen, device=DEV)
        # Short and long prompts over short and long contexts, in any order.
        pos0, new = (torch.tensor(x, dtype=torch.int32, device=DEV)[order]
                     for x in (ctx, new[n // 3:] + new[:n // 3]))
        cu = torch.zeros(n + 1, dtype=torch.int32, device=DEV)
        cu[1:] = torch.cumsum(new, 0)
        toks = sum(_spread(case["new_lo"], case["new_hi"], n)) + case["pad"]
        cols = (case["ctx_hi"] + case["new_hi"] + P - 1) // P
        table, pages = _table(gen, (pos0 + new + P - 1) // P, cols)
        st.update(k=_normal(gen, toks, G * D), v=_normal(gen, toks, G * D),
                  q=_normal(gen, toks, H * D), pos0=pos0, cu=cu, toks=toks, table=table,
                  q_out=torch.zeros(toks, H * D, device=DEV),
                  # One decode step needs no offsets: token s is sequence s's.
                  single=case["new_lo"] == case["new_hi"] == 1 and case["pad"] == 0)
    else:
        lens = _shuffled(gen, _lens(case))
        sh = _shared_rows(case) if case["op"] == "shared" else 0
        cols = (sh + case["len_hi"] + P - 1) // P
        table, pages = _table(gen, (lens + P - 1) // P, max(cols - sh // P, 1))
        if sh:
            prefix = torch.arange(pages, pages + sh // P, device=DEV, dtype=torch.int32)
            prefix = prefix[torch.randperm(sh // P, generator=gen, device=DEV)]
            table = torch.cat([prefix[None].expand(n, -1), table], 1).contiguous()
            pages += sh // P
        st.update(q=_normal(gen, n, H * D) * 1.5, past=lens + (sh - 1), table=table,
                  out=torch.zeros(n, H * D, device=DEV))
        if case["op"] in ("select", "sparse"):
            st["pages_out"] = torch.zeros(n, G, case["n_sel"], dtype=torch.int32, device=DEV)
        if case["op"] == "sparse":
            nb = (lens + P - 1) // P
            cols = table.shape[1]
            j = torch.arange(cols, device=DEV)
            score = torch.rand(n, G, cols, generator=gen, device=DEV)
            score = torch.where(j == (nb - 1)[:, None, None], 2.0, score)   # the newest page
            score = torch.where(j < nb[:, None, None], score, -1.0)
            m = min(case["n_sel"], cols)
            top, idx = torch.topk(score, m, dim=2)
            idx = torch.where(top >= 0, idx, cols).sort(dim=2).values
            st["sel"] = torch.full((n, G, case["n_sel"]), -1, dtype=torch.int32, device=DEV)
            st["sel"][:, :, :m] = torch.where(idx < cols, idx, -1).to(torch.int32)
    rows = (pages, G, P, D)
    st["kp"] = _rows(gen, case["dtype"], *rows)
    st["vp"] = _rows(gen, case["dtype"], *rows)
    st["bounds"] = torch.stack([st["kp"].amin(2), st["kp"].amax(2)], 2).contiguous()
    st["bounds"][0] = 0
    if own:   # the handle that a program keeps for its pool
        st["cache"] = _package().PagedKVCache(
            _backend(), 1, pages, P, n_head=H, n_kv_head=G, head_dim=D,
            dtype=_package().DTYPE_BF16 if case["dtype"] == "bf16" else _package().DTYPE_F32,
            max_pos=MAX_POS, rope_base=ROPE_BASE, k=st["kp"], v=st["vp"], bounds=st["bounds"])
    torch.cuda.synchronize()
    return st


# ---------------------------------------------------------- the own calls

_kept = {}


def _package():
    """The package (its folder's name has a dot: loaded by its path)."""
    name = "tmac_gguf_cpp_b200"
    if name not in sys.modules:
        root = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "tmac_gguf.cpp_b200")
        spec = importlib.util.spec_from_file_location(
            name, os.path.join(root, "__init__.py"), submodule_search_locations=[root])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


def _backend():
    """The device's backend, on the current stream: what made the inputs is
    ordered before the calls."""
    if "be" not in _kept:
        _kept["be"] = _package().CudaBackend(torch.cuda.current_device())
    stream = torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())
    if _kept.get("stream") != stream:
        _kept["be"].set_stream(stream)
        _kept["stream"] = stream
    return _kept["be"]


def _run_own(st):
    _backend()
    c = st["cache"]
    if st["op"] == "append":
        c.append(0, st["k"], st["v"], st["pos0"], st["table"], q=st["q"], q_out=st["q_out"],
                 cu_tokens=None if st["single"] else st["cu"])
        return {"q": st["q_out"], "k": st["kp"], "v": st["vp"], "bounds": st["bounds"]}
    if st["op"] == "attend":
        c.attention(0, st["q"], st["past"], st["table"], st["out"])
    elif st["op"] == "shared":
        c.attention_shared(0, st["q"], st["past"], st["table"], st["shared"], st["out"])
    elif st["op"] == "select":
        c.select_pages(0, st["q"], st["past"], st["table"], st["pages_out"], keep_first=1,
                       keep_last=1)
        return st["pages_out"]
    else:
        c.attention_sparse(0, st["q"], st["past"], st["table"], st["sel"], st["out"])
    return st["out"]


# -------------------------------------------------------------- plain forms

def _angles(pos, D):
    """cos and sin of the rotation angles: base and product rounded to 32
    bits as the rotation's definition has them, cos and sin in 64."""
    e = torch.arange(0, D, 2, device=DEV, dtype=torch.float32) / D
    theta = 1.0 / torch.pow(torch.tensor(ROPE_BASE, dtype=torch.float64, device=DEV),
                            e.double()).float()
    a = (pos.float()[:, None] * theta).double()
    return a.cos().float(), a.sin().float()


def _rotate(x, cos, sin):
    """x [tokens, heads, D], adjacent pairs."""
    a, b = x[..., 0::2], x[..., 1::2]
    c, s = cos[:, None], sin[:, None]
    return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)


def _plain_append(st):
    n, P, H, G, D, T = st["n"], st["page"], st["n_head"], st["n_kv"], st["hd"], st["toks"]
    kp, vp, bd, table, pos0, cu = (st[x] for x in ("kp", "vp", "bounds", "table", "pos0", "cu"))
    t = torch.arange(T, device=DEV)
    s = torch.searchsorted(cu, t.to(cu.dtype), right=True) - 1
    live = s < n                       # the others are padding
    s = s.clamp(max=n - 1)
    pos = torch.where(live, pos0[s] + t - cu[s], 0)
    cos, sin = _angles(pos, D)
    q = _rotate(st["q"].view(T, H, D), cos, sin).view(T, H * D)
    st["q_out"].copy_(torch.where(live[:, None], q, st["q_out"]))
    page = torch.where(live, table[s, pos // P], 0).long()
    slot = torch.where(live, pos % P, 0).long()
    keep = live[:, None, None]
    for pool, x in ((kp, _rotate(st["k"].view(T, G, D), cos, sin)), (vp, st["v"].view(T, G, D))):
        pool[page, :, slot] = torch.where(keep, x.to(pool.dtype), pool[page, :, slot])
    # The bounds of every page that a sequence wrote to, over its rows so far.
    new = cu[1:] - cu[:-1]
    end = pos0 + new
    first = pos0 // P
    j = first[:, None] + torch.arange(st["new_hi"] // P + 2, device=DEV)
    wrote = (new[:, None] > 0) & (j * P < end[:, None])
    pg = torch.where(wrote, table.gather(1, j.clamp(max=table.shape[1] - 1).long()), 0).long()
    rows = kp[pg]                                            # [n, pages, G, P, D]
    seen = (j[:, :, None] * P + torch.arange(P, device=DEV) < end[:, None, None])[:, :, None, :, None]
    lo = torch.where(seen, rows, float("inf")).amin(3)
    hi = torch.where(seen, rows, NEG).amax(3)
    bd[pg] = torch.where(wrote[:, :, None, None, None], torch.stack([lo, hi], 3), 0).to(bd.dtype)
    return {"q": st["q_out"], "k": kp, "v": vp, "bounds": bd}


def _softmax_sum(scores, values):
    """sum of softmax(scores) * values; zeros where every score is -inf."""
    m = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(m > NEG, m, 0.0))
    total = p.sum(-1, keepdim=True)
    return (p @ values) / torch.where(total > 0, total, 1.0)


def _pages_rows(pool, pages):
    """Rows of pages [n, b] of a pool as [n, G, b * P, D] in 32 bits."""
    x = pool[pages.long()].permute(0, 2, 1, 3, 4)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1]).float()


def _plain_attend(st):
    n, H, G, D = st["n"], st["n_head"], st["n_kv"], st["hd"]
    q = st["q"].view(n, G, H // G, D)
    k, v = _pages_rows(st["kp"], st["table"]), _pages_rows(st["vp"], st["table"])
    s = (q @ k.transpose(2, 3)) / math.sqrt(D)
    at = torch.arange(k.shape[2], device=DEV)
    s = torch.where(at <= st["past"][:, None, None, None], s, NEG)
    return _softmax_sum(s, v).reshape(n, H * D)


def _plain_shared(st):
    n, H, G, D, P = st["n"], st["n_head"], st["n_kv"], st["hd"], st["page"]
    q = st["q"].view(n, G, H // G, D)
    nsh = st["shared"] // P
    k0, v0 = (_pages_rows(st[x], st["table"][:1, :nsh])[0] for x in ("kp", "vp"))
    k1, v1 = (_pages_rows(st[x], st["table"][:, nsh:]) for x in ("kp", "vp"))
    qg = q.transpose(0, 1).reshape(G, -1, D)
    s0 = (qg @ k0.transpose(1, 2)).view(G, n, H // G, -1).transpose(0, 1) / math.sqrt(D)
    s1 = (q @ k1.transpose(2, 3)) / math.sqrt(D)
    past = st["past"][:, None, None, None]
    s0 = torch.where(torch.arange(nsh * P, device=DEV) <= past, s0, NEG)
    s1 = torch.where(torch.arange(s1.shape[3], device=DEV) + nsh * P <= past, s1, NEG)
    m = torch.maximum(s0.amax(-1, keepdim=True) if nsh else torch.full_like(s1[..., :1], NEG),
                      s1.amax(-1, keepdim=True))
    m = torch.where(m > NEG, m, 0.0)
    p0, p1 = torch.exp(s0 - m), torch.exp(s1 - m)
    total = p0.sum(-1, keepdim=True) + p1.sum(-1, keepdim=True)
    o0 = (p0.transpose(0, 1).reshape(G, n * (H // G), -1) @ v0).view(G, n, H // G, D).transpose(0, 1)
    return ((o0 + p1 @ v1) / torch.where(total > 0, total, 1.0)).reshape(n, H * D)


def _plain_select(st):
    n, H, G, D, P = st["n"], st["n_head"], st["n_kv"], st["hd"], st["page"]
    # The choice between two pages next to the border goes by 64-bit sums.
    q = st["q"].view(n, G, H // G, D).double()
    b = st["bounds"][st["table"].long()].double()            # [n, pages, G, 2, D]
    lo, hi = b[:, :, :, 0].permute(0, 2, 3, 1), b[:, :, :, 1].permute(0, 2, 3, 1)
    score = (q.clamp(min=0) @ hi + q.clamp(max=0) @ lo).amax(2)   # [n, G, pages]
    nb = ((st["past"] + P) // P)[:, None, None]
    j = torch.arange(score.shape[2], device=DEV)
    score = torch.where((j < 1) | (j >= nb - 1), float("inf"), score)
    score = torch.where(j < nb, score, NEG)
    m = min(st["n_sel"], score.shape[2])
    top, idx = torch.sort(score, dim=2, descending=True, stable=True)
    none = score.shape[2]
    idx = torch.where(idx[:, :, :m] < nb, idx[:, :, :m], none).sort(dim=2).values
    out = torch.full_like(st["pages_out"], -1)
    out[:, :, :m] = torch.where(idx < none, idx, -1).to(torch.int32)
    return out


def _plain_sparse(st):
    n, H, G, D, P = st["n"], st["n_head"], st["n_kv"], st["hd"], st["page"]
    q, sel = st["q"].view(n, G, H // G, D), st["sel"].long()
    page = st["table"].long()[:, None].expand(-1, G, -1).gather(2, sel.clamp(min=0))
    g = torch.arange(G, device=DEV)[None, :, None]
    k, v = (st[x][page, g].reshape(n, G, -1, D).float() for x in ("kp", "vp"))
    at = sel[..., None] * P + torch.arange(P, device=DEV)
    seen = ((sel[..., None] >= 0) & (at <= st["past"][:, None, None, None])).view(n, G, 1, -1)
    s = torch.where(seen, (q @ k.transpose(2, 3)) / math.sqrt(D), NEG)
    return _softmax_sum(s, v).reshape(n, H * D)


_PLAIN = {"append": _plain_append, "attend": _plain_attend, "shared": _plain_shared,
          "select": _plain_select, "sparse": _plain_sparse}


def run(state):
    return _run_own(state) if own else _PLAIN[state["op"]](state)


# ------------------------------------------------------------- the least work

def work(case):
    H, G, D, P, n = (case[x] for x in ("n_head", "n_kv", "hd", "page", "n"))
    e = DT[case["dtype"]].itemsize
    io = 2 * n * H * D * 4                                   # q in, output out
    if case["op"] == "append":
        toks = sum(_spread(case["new_lo"], case["new_hi"], n))
        pages = max(n if case["new_hi"] else 0, toks // P)
        return {"bytes": toks * (2 * H * D * 4 + 2 * G * D * 4 + 2 * G * D * e)
                + pages * 2 * G * D * e, "flops": 3 * toks * (H + G) * D}
    lens = _lens(case)
    if case["op"] == "shared":
        sh = _shared_rows(case)
        return {"bytes": (sh + sum(lens)) * 2 * G * D * e + io,
                "flops": 4 * H * D * (n * sh + sum(lens))}
    if case["op"] == "select":
        pages = sum(-(-x // P) for x in lens)
        return {"bytes": pages * 2 * G * D * e + io // 2 + n * G * case["n_sel"] * 4,
                "flops": 2 * H * D * pages}
    if case["op"] == "sparse":
        lens = [min(x, case["n_sel"] * P) for x in lens]
    return {"bytes": sum(lens) * 2 * G * D * e + io, "flops": 4 * H * D * sum(lens)}


# ------------------------------------------------------- the values in 64 bits

def _exact_append(st):
    n, P, H, G, D = st["n"], st["page"], st["n_head"], st["n_kv"], st["hd"]
    k, v, bd, q = (st[x].double() for x in ("kp", "vp", "bounds", "q_out"))
    table, pos0, cu = (st[x].tolist() for x in ("table", "pos0", "cu"))
    dims = torch.arange(D // 2, device=DEV)
    power = torch.tensor(ROPE_BASE, device=DEV, dtype=torch.float64) ** (
        (2 * dims).float() / torch.tensor(float(D), device=DEV)).double()
    inv = (1.0 / power.float()).float()
    for s in range(n):
        a, b = cu[s], cu[s + 1]
        if a == b:
            continue
        pos = torch.arange(pos0[s], pos0[s] + b - a, device=DEV)
        angle = (pos.float()[:, None] * inv[None]).double()
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]     # e^(i angle)
        for x, to, heads in ((st["q"], "q", H), (st["k"], "k", G)):
            z = torch.view_as_complex(x[a:b].double().view(b - a, heads, D // 2, 2).contiguous())
            r = torch.view_as_real(z * turn).reshape(b - a, heads, D)
            if to == "q":
                q[a:b] = r.view(b - a, H * D)
            else:
                kr = r
        page = st["table"][s].long()[pos // P]
        k[page, :, pos % P] = kr
        v[page, :, pos % P] = st["v"][a:b].double().view(b - a, G, D)
        for j in range(pos0[s] // P, (pos0[s] + b - a - 1) // P + 1):
            rows = k[table[s][j], :, :min(P, pos0[s] + b - a - j * P)]
            bd[table[s][j], :, 0], bd[table[s][j], :, 1] = rows.amin(1), rows.amax(1)
    return {"q": q, "k": k, "v": v, "bounds": bd}


def _exact_rows(st, s, g, pages, valid):
    k = st["kp"][pages, g].double().reshape(-1, st["hd"])[valid]
    v = st["vp"][pages, g].double().reshape(-1, st["hd"])[valid]
    per = st["n_head"] // st["n_kv"]
    q = st["q"][s].double().view(st["n_head"], st["hd"])[g * per:(g + 1) * per]
    return torch.softmax(q @ k.T * st["hd"] ** -0.5, -1) @ v


def _exact_attend(st, sparse=False):
    n, P, H, G, D = st["n"], st["page"], st["n_head"], st["n_kv"], st["hd"]
    out = torch.zeros(n, G, H // G, D, dtype=torch.float64, device=DEV)
    slots = torch.arange(P, device=DEV)
    for s, past in enumerate(st["past"].tolist()):
        if past < 0:
            continue
        for g in range(G):
            j = torch.arange(past // P + 1, device=DEV)
            if sparse:
                j = st["sel"][s, g].long()
                j = j[j >= 0]
            valid = (j[:, None] * P + slots <= past).view(-1)
            out[s, g] = _exact_rows(st, s, g, st["table"][s].long()[j], valid)
    return out.view(n, H * D)


def _exact_select(st):
    n, P, H, G, D = st["n"], st["page"], st["n_head"], st["n_kv"], st["hd"]
    out = torch.full((n, G, st["n_sel"]), -1, dtype=torch.int32)
    for s, past in enumerate(st["past"].tolist()):
        nb = (past + P) // P
        for g in range(G if nb else 0):
            b = st["bounds"][st["table"][s, :nb].long(), g].double()
            best = torch.full((nb,), NEG, dtype=torch.float64, device=DEV)
            for h in range(g * (H // G), (g + 1) * (H // G)):
                q = st["q"][s, h * D:(h + 1) * D].double()
                best = torch.maximum(best, torch.maximum(b[:, 0] * q, b[:, 1] * q).sum(1))
            best[0] = best[nb - 1] = float("inf")
            order = sorted(range(nb), key=lambda i, v=best.tolist(): (-v[i], i))
            got = sorted(order[:st["n_sel"]])
            out[s, g, :len(got)] = torch.tensor(got, dtype=torch.int32)
    return out


def exact(case, seed):
    if case["op"] != "append" and case["n"] * case["n_kv"] > 4096:
        return None
    st = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(st)
    if case["op"] == "select":
        return _exact_select(st)
    return _exact_attend(st, sparse=case["op"] == "sparse")
