"""The operators around decoding with drafted tokens, as measurable cases.

Five families, each one call (or the short run of calls) that a serving or training program makes of them: attention of a tree
of drafted tokens over a KV cache, rotary positions with several axes, forking sequences whose cache pages are shared, moving
the accepted rows of a draft behind their prefix, and reserving and freeing pages.  `run` computes each in plain torch
operations, or, where `own` is true, through the framework's entry points.  A case is a dict of plain values; lengths and
trees come from the case's own `shape_seed`, so that the work of a case does not depend on the seed of its inputs.
"""
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _fa():
    pkg = os.path.join(os.getcwd(), "flash-attention-npu_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import flash_attn_npu_3
    return flash_attn_npu_3


def listed():
    return [
        # One user's decoding step with a small draft tree: everything in it is latency.
        {"name": "tree_single", "family": "tree", "dtype": "bf16", "b": 1, "t": 8, "lo": 1500, "hi": 1500, "hq": 32, "hkv": 8,
         "d": 128, "page": 64, "left": -1, "softcap": 0.0, "rotary": "half", "axes": 1, "ragged": False, "shape_seed": 1},
        # A serving batch of mixed lengths, 26 drafted tokens a sequence, some sequences with fewer.
        {"name": "tree_batch", "family": "tree", "dtype": "bf16", "b": 16, "t": 26, "lo": 1024, "hi": 8192, "hq": 32, "hkv": 8,
         "d": 128, "page": 256, "left": -1, "softcap": 0.0, "rotary": "half", "axes": 1, "ragged": True, "shape_seed": 2},
        # Long contexts and large trees: 64 drafted tokens, 256 stacked query rows a KV head.
        {"name": "tree_long", "family": "tree", "dtype": "fp16", "b": 8, "t": 64, "lo": 4096, "hi": 32768, "hq": 32, "hkv": 8,
         "d": 128, "page": 128, "left": -1, "softcap": 0.0, "rotary": "none", "axes": 1, "ragged": False, "shape_seed": 3},
        # A layer with a sliding window and capped scores, an odd tree, a query group of 7, a dense cache, image positions.
        {"name": "tree_window_softcap", "family": "tree", "dtype": "bf16", "b": 5, "t": 13, "lo": 700, "hi": 4000, "hq": 14,
         "hkv": 2, "d": 64, "page": 0, "left": 1024, "softcap": 30.0, "rotary": "interleaved", "axes": 3, "ragged": False,
         "shape_seed": 4},
        # One new token for each of 33 sequences, three position axes: the smallest rotary call.
        {"name": "rotary_step", "family": "rotary", "dtype": "bf16", "b": 33, "s": 1, "hq": 32, "hkv": 8, "d": 128, "rd": 128,
         "axes": 3, "cyclic": False, "interleaved": False, "table": "fp32", "packed": False, "grad": False},
        # A training step's rotary embedding over image and text tokens, forward and backward.
        {"name": "rotary_train", "family": "rotary", "dtype": "bf16", "b": 4, "s": 4096, "hq": 32, "hkv": 8, "d": 128, "rd": 128,
         "axes": 3, "cyclic": True, "interleaved": False, "table": "fp32", "packed": True, "grad": True},
        # Beam search over two prompts: four beams each, forked, reordered and freed again.
        {"name": "fork_beams", "family": "fork", "caches": 4, "pages": 256, "page": 64, "h": 8, "d": 128, "b": 2, "n": 8,
         "lo": 700, "hi": 2500, "reorder": True, "shape_seed": 5},
        # Many samples of each of 16 prompts in all layers' caches.
        {"name": "fork_samples", "family": "fork", "caches": 16, "pages": 768, "page": 64, "h": 4, "d": 128, "b": 16, "n": 128,
         "lo": 500, "hi": 2300, "reorder": False, "shape_seed": 6},
        # The accepted tokens of one sequence's draft, in a few layers.
        {"name": "accept_single", "family": "compact", "caches": 4, "pages": 64, "page": 64, "h": 8, "d": 128, "b": 1, "t": 8,
         "lo": 1500, "hi": 1500, "shape_seed": 7},
        # The accepted tokens of a serving batch, in all layers' caches.
        {"name": "accept_batch", "family": "compact", "caches": 16, "pages": 448, "page": 64, "h": 8, "d": 128, "b": 48, "t": 64,
         "lo": 100, "hi": 500, "shape_seed": 8},
        # Pages for the drafts of a small batch, handed out and returned.
        {"name": "turnover_small", "family": "turnover", "pages": 1000, "page": 16, "b": 7, "width": 128, "lo": 100, "hi": 1900,
         "extra": 33, "shape_seed": 9},
        # The same for a large server: many sequences, long tables, a large pool.
        {"name": "turnover_large", "family": "turnover", "pages": 290000, "page": 16, "b": 512, "width": 2048, "lo": 100,
         "hi": 16000, "extra": 64, "shape_seed": 10},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    family = rng.choice(["tree", "tree", "tree", "rotary", "rotary", "fork", "compact", "turnover"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    shape_seed = rng.randrange(1 << 20)
    if family == "tree":
        hkv = rng.choice([1, 2, 4, 8, 8])
        g = rng.choice([1, 2, 3, 4, 4, 7, 8])
        g = g if hkv * g <= 32 else 4
        b, t, d = _log(rng, 1, 16), _log(rng, 1, 100), rng.choice([64, 128, 128, 128, 256])
        hi = min(_log(rng, 100, 16000), 8 * 64 * 32768 * 32 * 128 // (b * t * hkv * g * d))
        return {"family": family, "dtype": dtype, "b": b, "t": t, "lo": max(1, hi // 8), "hi": hi,
                "hq": hkv * g, "hkv": hkv, "d": d, "page": rng.choice([0, 16, 64, 64, 128, 256]),
                "left": _log(rng, 16, 2048) if rng.random() < 0.2 else -1, "softcap": 30.0 if rng.random() < 0.2 else 0.0,
                "rotary": rng.choice(["none", "half", "half", "interleaved"]), "axes": rng.choice([1, 1, 3]),
                "ragged": rng.random() < 0.5, "shape_seed": shape_seed}
    if family == "rotary":
        hkv = rng.choice([1, 2, 4, 8, 8, 16])
        hq = hkv * rng.choice([1, 2, 4])
        d = rng.choice([64, 96, 128, 128, 256])
        rd = rng.choice([d, d, d // 2, d // 4 + 8])
        b = _log(rng, 1, 64)
        s = _log(rng, 1, max(1, min(8192, 16384 * 40 * 128 // (b * (hq + hkv) * d))))
        return {"family": family, "dtype": dtype, "b": b, "s": s, "hq": hq, "hkv": hkv, "d": d, "rd": rd,
                "axes": rng.choice([1, 2, 3, 3, 4]), "cyclic": rng.random() < 0.4, "interleaved": rng.random() < 0.4,
                "table": rng.choice(["fp32", "same"]), "packed": rng.random() < 0.4, "grad": rng.random() < 0.5}
    if family == "fork":
        page = rng.choice([16, 32, 64, 64, 128])
        b, h, d = _log(rng, 1, 16), rng.choice([2, 4, 8]), rng.choice([64, 128])
        n = _log(rng, 1, 128)
        hi = _log(rng, page, 2000)
        need = b * (hi // page + 1) + 2 * n
        caches = max(1, min(_log(rng, 1, 16), (1 << 29) // (need * page * h * d * 2)))
        return {"family": family, "caches": caches, "pages": need + rng.randrange(40), "page": page, "h": h, "d": d, "b": b, "n": n,
                "lo": max(1, hi // 6), "hi": hi, "reorder": rng.random() < 0.5, "shape_seed": shape_seed}
    if family == "compact":
        page, t = rng.choice([16, 32, 64, 64, 128]), _log(rng, 2, 100)
        b, h, d = _log(rng, 1, 48), rng.choice([2, 4, 8]), rng.choice([64, 128])
        hi = _log(rng, 20, 1200)
        need = b * ((hi + t) // page + 1)
        caches = max(1, min(_log(rng, 1, 32), (1 << 30) // (need * page * h * d * 2)))
        return {"family": family, "caches": caches, "pages": need + rng.randrange(40), "page": page, "h": h, "d": d, "b": b, "t": t,
                "lo": max(1, hi // 6), "hi": hi, "shape_seed": shape_seed}
    page = rng.choice([16, 16, 32, 64])
    b, hi = _log(rng, 1, 512), _log(rng, 40, 16000)
    extra = _log(rng, 1, 300)
    hi = max(1, min(hi, (300000 // b - 3) * page - extra))
    width = (hi + extra) // page + 1 + rng.randrange(50)
    return {"family": family, "pages": b * ((hi + extra) // page + 2) + rng.randrange(100), "page": page, "b": b,
            "width": width, "lo": max(1, hi // 100), "hi": hi, "extra": extra, "shape_seed": shape_seed}


# ---- shapes of a case: lengths, trees, page tables (the same for every seed of its inputs) -----------------------------
def _lens(case, rng):
    return [rng.randint(case["lo"], case["hi"]) for _ in range(case["b"])]


def _tables(lens, page, width, pages, rng):
    """Every sequence's pages, in an order as a running server has it; -1 behind them.  What is not handed out is free."""
    order = list(range(pages))
    rng.shuffle(order)
    rows, at = [], 0
    for n in lens:
        k = -(-n // page)
        rows.append(order[at:at + k] + [-1] * (width - k))
        at += k
    assert at <= pages
    return rows


def _trees(case, rng):
    """Parents of every drafted token: the first token of a level extends the likeliest branch, others branch off anywhere
    up to 12 tokens deep.  A ragged case has sequences with fewer tokens (-2: no token here)."""
    b, t = case["b"], case["t"]
    out = []
    for _ in range(b):
        n = rng.randint((t + 1) // 2, t) if case["ragged"] else t
        parents, depth = [], []
        for i in range(n):
            p = i - 1 if i and rng.random() < 0.3 else rng.randint(-1, i - 1)
            while p >= 0 and depth[p] >= 12:
                p = parents[p]
            parents.append(p)
            depth.append(0 if p < 0 else depth[p] + 1)
        out.append(parents + [-2] * (t - n))
    return out


def _depths(parents):
    out = []
    for p in parents:
        out.append(-1 if p < -1 else 0 if p < 0 else out[p] + 1)
    return out


def _sections(case):
    """Pairs of each axis: half of them for the first, the rest shared evenly, as with time, height and width."""
    pairs, n = case.get("rd", case.get("d")) // 2, case["axes"]
    if n == 1:
        return None
    rest = [pairs // 2 // (n - 1)] * (n - 1)
    return [pairs - sum(rest)] + rest


def _kept(case, rng):
    """The accepted tokens of each sequence: the likeliest tokens in order as far as they hold, then a later branch."""
    t = case["t"]
    rows, counts = [], []
    for _ in range(case["b"]):
        count = rng.randint(0, min(t, 9))
        lead = rng.randint(0, count)
        if t - count < count - lead:
            lead = count
        rows.append(list(range(lead)) + sorted(rng.sample(range(count, t), count - lead)) + [-1] * (t - count))
        counts.append(count)
    return rows, counts


def _fork_parents(case, rng):
    return [rng.randrange(case["b"]) for _ in range(case["n"])]


def _tree_shape(case):
    rng = random.Random(case["shape_seed"])
    lens = _lens(case, rng)
    trees = _trees(case, rng)
    page, t = case["page"], case["t"]
    table, pages = None, 0
    if page:
        width = -(-(case["hi"] + t) // page)
        pages = sum(-(-(n + t) // page) for n in lens) + 3
        table = _tables([n + t for n in lens], page, width, pages, rng)
        table = [[max(x, 0) for x in row] for row in table]     # entries that no length reaches may hold anything
    return lens, trees, table, pages


def _cos_sin(rows, pairs, device, dtype):
    ang = torch.arange(rows, dtype=torch.float64, device=device)[:, None] \
        * 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device=device) / pairs)
    return ang.cos().to(dtype), ang.sin().to(dtype)


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    family = case["family"]

    def randn(*shape, dtype):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dtype)

    def i32(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    st = {"case": case}
    if family == "tree":
        lens, trees, table, pages = _tree_shape(case)
        dt, b, t, hq, hkv, d = _DTYPES[case["dtype"]], case["b"], case["t"], case["hq"], case["hkv"], case["d"]
        shape = (pages, case["page"], hkv, d) if case["page"] else (b, case["hi"] + t, hkv, d)
        st.update(q=randn(b, t, hq, d, dtype=dt), k=randn(b, t, hkv, d, dtype=dt), v=randn(b, t, hkv, d, dtype=dt),
                  k_cache=randn(*shape, dtype=dt), v_cache=randn(*shape, dtype=dt), parents=i32(trees), lens=i32(lens),
                  table=None if table is None else i32(table), cos=None, sin=None, positions=None, sections=None)
        if case["rotary"] != "none":
            st["cos"], st["sin"] = _cos_sin(case["hi"] + t + 16, d // 2, dev, dt)
            if case["axes"] > 1:
                # text advances all axes together; image tokens of a draft differ in height and width
                base = i32(lens)[None, :, None] // 2
                st["positions"] = (base + torch.randint(0, 16, (case["axes"], b, t), generator=gen, device=dev)).int()
                st["sections"] = _sections(case)
        return st
    if family == "rotary":
        dt = _DTYPES[case["dtype"]]
        b, s, hq, hkv, d = case["b"], case["s"], case["hq"], case["hkv"], case["d"]
        lead = (b * s,) if case["packed"] else (b, s)
        # q and k are slices of one projection, as they come out of it
        qkv = randn(*lead, hq + 2 * hkv, d, dtype=dt)
        st.update(q=qkv[..., :hq, :], k=qkv[..., hq:hq + hkv, :], sections=_sections(case))
        rows = 2 * s + 64
        st["cos"], st["sin"] = _cos_sin(rows, case["rd"] // 2, dev, torch.float32 if case["table"] == "fp32" else dt)
        # the first axis runs with the tokens from where each sequence stands, the others over the patches of images
        steps = (torch.arange(s, device=dev) + torch.randint(0, s + 1, (b, 1), generator=gen, device=dev)).reshape(lead)
        patch = torch.randint(0, 64, (case["axes"] - 1,) + lead, generator=gen, device=dev)
        st["positions"] = torch.cat((steps[None], patch)).int()
        if case["axes"] == 1:
            st["positions"] = st["positions"][0]
        if case["grad"]:
            st["q"], st["k"] = st["q"].detach().requires_grad_(True), st["k"].detach().requires_grad_(True)
            st["dq"], st["dk"] = randn(*lead, hq, d, dtype=dt), randn(*lead, hkv, d, dtype=dt)
        return st
    rng = random.Random(case["shape_seed"])
    lens = _lens(case, rng)
    page, b = case["page"], case["b"]
    order = random.Random(seed)                                 # which pages a sequence got depends on what ran before
    if family == "turnover":
        table = _tables(lens, page, case["width"], case["pages"], order)
    elif family == "fork":
        table = _tables(lens, page, -(-case["hi"] // page) + 1, case["pages"], order)
    else:
        table = _tables([n + case["t"] for n in lens], page, -(-(case["hi"] + case["t"]) // page), case["pages"], order)
    st.update(lens=i32(lens), table=i32(table))
    st["refs"] = (torch.bincount(st["table"].flatten().long() + 1, minlength=case["pages"] + 1)[1:]).int()
    if family != "turnover":
        st["caches"] = randn(case["caches"], case["pages"], page, case["h"], case["d"], dtype=torch.bfloat16)
    if family == "fork":
        st["parents"] = i32(_fork_parents(case, rng))
        st["order"] = i32([rng.randrange(case["n"]) for _ in range(case["n"])])
    if family == "compact":
        kept, counts = _kept(case, rng)
        st.update(kept=i32(kept), counts=i32(counts))
    return st


# ---- the framework's calls --------------------------------------------------------------------------------------------
def _run_own(st):
    fa, case = _fa(), st["case"]
    family = case["family"]
    if family == "tree":
        out, lse = fa.flash_attn_tree_with_kvcache(
            st["q"], st["k_cache"], st["v_cache"], st["k"], st["v"], st["parents"], cache_seqlens=st["lens"],
            page_table=st["table"], rotary_cos=st["cos"], rotary_sin=st["sin"], rotary_positions=st["positions"],
            rotary_sections=st["sections"], rotary_interleaved=case["rotary"] == "interleaved",
            window_size=(case["left"], -1), softcap=case["softcap"], return_softmax_lse=True)
        return {"out": out, "lse": lse, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    if family == "rotary":
        q, k = fa.rotary_axes_func(st["q"], st["k"], st["cos"], st["sin"], st["positions"], sections=st["sections"],
                                   sections_cyclic=case["cyclic"], interleaved=case["interleaved"])
        if not case["grad"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    if family == "fork":
        table, lens, missing = fa.kvcache_fork(st["caches"], st["refs"], st["table"], st["lens"], st["parents"], keep_parents=True)
        got = {"lens": lens, "missing": missing}
        if case["reorder"]:
            got["table"] = table
            table, lens, again = fa.kvcache_fork(st["caches"], st["refs"], table, lens, st["order"])
            got.update(lens2=lens, missing2=again)
        got.update(held=st["refs"].clone(), last=table.clone())
        fa.kvcache_free(st["refs"], table, page_size=case["page"])
        got.update(refs=st["refs"], caches=st["caches"].view(torch.int16), freed=table)
        return got
    if family == "compact":
        lens = fa.kvcache_compact(st["caches"], st["lens"], st["kept"], st["counts"], page_table=st["table"])
        return {"lens": lens, "caches": st["caches"].view(torch.int16)}
    missing = fa.kvcache_reserve(st["refs"], st["table"], st["lens"], page_size=case["page"], extra=case["extra"])
    held, table = st["refs"].clone(), st["table"].clone()
    fa.kvcache_free(st["refs"], st["table"], st["lens"], page_size=case["page"])
    return {"missing": missing, "held": held, "table_held": table, "refs": st["refs"], "table": st["table"]}


# ---- the plain form ---------------------------------------------------------------------------------------------------
def _axis_of_pair(pairs, sections, cyclic, device):
    """Which position axis turns pair i."""
    i = torch.arange(pairs, device=device)
    if sections is None:
        return torch.zeros_like(i)
    sec = torch.tensor(sections, device=device)
    if cyclic:
        axis = i % len(sections)
        return torch.where(i < len(sections) * sec[axis], axis, torch.zeros_like(i))
    return (i[:, None] >= sec.cumsum(0)[None, :]).sum(1)


def _rotate(x, cos, sin, interleaved):
    """x (..., heads, d) with cos, sin (..., 1, pairs), in 32 bits; the columns behind the pairs stay."""
    pairs = cos.shape[-1]
    xf = x.float()
    turned, rest = xf[..., :2 * pairs], xf[..., 2 * pairs:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = turned[..., :pairs], turned[..., pairs:]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((y, rest), -1).to(x.dtype)


def _angles(cos, sin, positions, axis):
    """cos and sin (tokens.., 1, pairs) of positions (axes, tokens..)."""
    i = torch.arange(axis.numel(), device=axis.device)
    pos = positions.long().clamp(0, cos.shape[0] - 1)[axis].movedim(0, -1)
    return cos.float()[pos, i][..., None, :], sin.float()[pos, i][..., None, :]


def _plain_tree(st):
    case = st["case"]
    b, t, hq, hkv, d = case["b"], case["t"], case["hq"], case["hkv"], case["d"]
    dev = st["q"].device
    lens, parents = st["lens"].long(), st["parents"].long()
    idx = torch.arange(t, device=dev)
    # ancestors with the token itself: the sum of all powers of the parent matrix
    real = (parents >= 0) & (parents < idx)
    up = torch.zeros(b, t, t, device=dev).scatter_(2, parents.clamp(0, t - 1)[..., None], real.float()[..., None])
    eye = torch.eye(t, device=dev)
    reach = torch.linalg.solve_triangular(eye - up, eye.expand(b, t, t), upper=False, unitriangular=True) > 0.5
    alive = (reach & (parents == -1)[:, None, :]).any(2)
    depth = reach.sum(2) - 1
    q, k, v = st["q"], st["k"], st["v"]
    if st["cos"] is not None:
        pos = (lens[:, None] + depth)[None] if st["positions"] is None else st["positions"]
        cos, sin = _angles(st["cos"], st["sin"], pos, _axis_of_pair(d // 2, st["sections"], False, dev))
        q, k = _rotate(q, cos, sin, case["rotary"] == "interleaved"), _rotate(k, cos, sin, case["rotary"] == "interleaved")
    rows = lens[:, None] + idx
    bi = torch.arange(b, device=dev)[:, None].expand(b, t)[alive]
    if st["table"] is not None:
        table, page = st["table"].long(), case["page"]
        outer, inner = table.gather(1, rows // page)[alive], (rows % page)[alive]
        st["k_cache"][outer, inner], st["v_cache"][outer, inner] = k[alive], v[alive]
        kk, vv = (c[table].reshape(b, -1, hkv, d) for c in (st["k_cache"], st["v_cache"]))
    else:
        st["k_cache"][bi, rows[alive]], st["v_cache"][bi, rows[alive]] = k[alive], v[alive]
        kk, vv = st["k_cache"], st["v_cache"]
    n = kk.shape[1]
    col = torch.arange(n, device=dev)
    see = alive[:, :, None] & (col < lens[:, None, None])
    rel = (col[None] - lens[:, None])
    in_tree = (rel >= 0) & (rel < t)
    see = see | (reach.gather(2, rel.clamp(0, t - 1)[:, None, :].expand(b, t, n)) & in_tree[:, None, :] & alive[:, :, None])
    if case["left"] >= 0:
        where = torch.where(in_tree, lens[:, None] + depth.gather(1, rel.clamp(0, t - 1)), col[None].expand(b, n))
        see = see & (where[:, None, :] >= (lens[:, None] + depth)[:, :, None] - case["left"])
    g = hq // hkv
    qg = q.float().reshape(b, t, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * t, d)
    s = (qg @ kk.permute(0, 2, 3, 1).float()).reshape(b, hkv, g, t, n) * d ** -0.5
    if case["softcap"] > 0:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    s = s.masked_fill(~see[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True).clamp_min(-3e38)
    e = torch.exp(s - m)
    z = e.sum(-1, keepdim=True)
    used = (torch.arange(n, device=dev) < (lens + t)[:, None])[:, :, None, None]
    vv = torch.where(used, vv, torch.zeros_like(vv)).permute(0, 2, 1, 3).float()
    o = (e / z.clamp_min(1e-38)).reshape(b, hkv, g * t, n) @ vv
    out = o.reshape(b, hkv, g, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, hq, d).to(st["q"].dtype)
    lse = torch.where(z > 0, m + torch.log(z), torch.full_like(z, float("inf")))[..., 0].reshape(b, hq, t)
    return {"out": out, "lse": lse, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _lowest_free(refs, wanted):
    """A page for every true entry of `wanted` in order, the lowest free ones; -1 where none is left."""
    order = torch.argsort((refs != 0).int(), stable=True)
    rank = wanted.int().flatten().cumsum(0) - 1
    have = wanted.flatten() & (rank < (refs == 0).sum())
    page = torch.where(have, order[rank.clamp(0, refs.numel() - 1)], torch.full_like(order[:1], -1))
    return page.reshape(wanted.shape), (wanted.flatten() & ~have).sum().int().reshape(1)


def _count(refs, table, add):
    """Adds `add` to the count of every page that the table names."""
    spare = torch.zeros(refs.numel() + 1, dtype=torch.int32, device=refs.device)
    spare.index_add_(0, table.flatten().long() + 1, torch.ones_like(table.flatten(), dtype=torch.int32))
    refs += add * spare[1:]


def _plain_fork(caches, refs, table, lens, parents, keep, page):
    width = table.shape[1]
    col = torch.arange(width, device=table.device)
    new_lens = lens[parents.long()]
    new = torch.where(col < ((new_lens + page - 1) // page)[:, None], table[parents.long()], torch.full_like(table[:1], -1))
    _count(refs, new, 1)
    if not keep:
        _count(refs, table, -1)
    # the partly filled last page: a holder keeps it only if it is the last one left
    fill = new_lens % page
    last = torch.where(fill > 0, new.gather(1, (new_lens // page).long().clamp(max=width - 1)[:, None])[:, 0], torch.full_like(fill, -1))
    before = ((last[:, None] == last[None, :]) & torch.ones(len(last), len(last), device=last.device).tril(-1).bool()).sum(1)
    copies = (last >= 0) & (refs[last.clamp_min(0).long()] - before > 1)
    dst, missing = _lowest_free(refs, copies)
    src = last[copies].long()
    refs -= torch.bincount(src, minlength=refs.numel()).int()
    to = dst[copies]
    ok = to >= 0
    refs[to[ok]] = 1
    at = (new_lens // page)[copies].long()
    new[copies.nonzero()[:, 0], at] = to.int()
    new_lens = new_lens.clone()
    new_lens[copies] = torch.where(ok, new_lens[copies], (at * page).int())
    rows = torch.arange(page, device=table.device) < fill[copies][ok][:, None]
    moved = torch.where(rows[None, :, :, None, None], caches[:, src[ok]], caches[:, to[ok]])
    caches[:, to[ok]] = moved
    return new, new_lens, missing


def _plain_free(refs, table, lens, page):
    col = torch.arange(table.shape[1], device=table.device)
    keep = torch.zeros_like(table[:, :1]) if lens is None else ((lens + page - 1) // page)[:, None]
    gone = torch.where(col >= keep, table, torch.full_like(table, -1))
    _count(refs, gone, -1)
    table.masked_fill_(col >= keep, -1)


def _run_plain(st):
    case = st["case"]
    family = case["family"]
    if family == "tree":
        return _plain_tree(st)
    if family == "rotary":
        axis = _axis_of_pair(case["rd"] // 2, st["sections"], case["cyclic"], st["q"].device)
        positions = st["positions"] if case["axes"] > 1 else st["positions"][None]
        cos, sin = _angles(st["cos"], st["sin"], positions, axis)
        q, k = _rotate(st["q"], cos, sin, case["interleaved"]), _rotate(st["k"], cos, sin, case["interleaved"])
        if not case["grad"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    if family == "fork":
        table, lens, missing = _plain_fork(st["caches"], st["refs"], st["table"], st["lens"], st["parents"], True, case["page"])
        got = {"lens": lens, "missing": missing}
        if case["reorder"]:
            got["table"] = table
            table, lens, again = _plain_fork(st["caches"], st["refs"], table, lens, st["order"], False, case["page"])
            got.update(lens2=lens, missing2=again)
        got.update(held=st["refs"].clone(), last=table.clone())
        _plain_free(st["refs"], table, None, case["page"])
        got.update(refs=st["refs"], caches=st["caches"].view(torch.int16), freed=table)
        return got
    if family == "compact":
        page = case["page"]
        i = torch.arange(case["t"], device=st["lens"].device)
        take = i < st["counts"][:, None]
        lens = st["lens"].long()[:, None]
        src, dst = (lens + st["kept"])[take], (lens + i)[take]
        seq = torch.arange(case["b"], device=take.device)[:, None].expand_as(take)[take]
        table = st["table"].long()
        rows = st["caches"][:, table[seq, src // page], src % page]
        st["caches"][:, table[seq, dst // page], dst % page] = rows
        return {"lens": st["lens"] + st["counts"], "caches": st["caches"].view(torch.int16)}
    page, table = case["page"], st["table"]
    col = torch.arange(case["width"], device=table.device)
    wanted = (col < ((st["lens"] + case["extra"] + page - 1) // page)[:, None]) & (table < 0)
    pages, missing = _lowest_free(st["refs"], wanted)
    table.copy_(torch.where(wanted, pages.int(), table))
    _count(st["refs"], torch.where(wanted, table, torch.full_like(table, -1)), 1)
    held, snapshot = st["refs"].clone(), table.clone()
    _plain_free(st["refs"], table, st["lens"], page)
    return {"missing": missing, "held": held, "table_held": snapshot, "refs": st["refs"], "table": table}


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    family = case["family"]
    if family == "tree":
        lens, trees, _, _ = _tree_shape(case)
        b, t, hq, hkv, d = case["b"], case["t"], case["hq"], case["hkv"], case["d"]
        pairs = rows = 0
        for n, parents in zip(lens, trees):
            seen = n if case["left"] < 0 else min(n, case["left"])
            depth = [x for x in _depths(parents) if x >= 0]
            rows += seen
            pairs += sum(seen + x + 1 for x in depth)
        return {"bytes": 4 * rows * hkv * d + 4 * b * t * hq * d + 8 * b * t * hkv * d + 4 * b * t * hq, "flops": 4 * d * hq * pairs}
    if family == "rotary":
        tokens, heads = case["b"] * case["s"], case["hq"] + case["hkv"]
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (4 * tokens * heads * case["d"] + 4 * tokens * case["axes"]),
                "flops": passes * 3 * tokens * heads * case["rd"]}
    rng = random.Random(case["shape_seed"])
    lens = _lens(case, rng)
    page = case["page"]
    if family == "turnover":
        return {"bytes": 2 * 4 * (case["b"] * case["width"] + case["pages"]), "flops": 2 * (case["b"] * case["width"] + case["pages"])}
    row = case["caches"] * case["h"] * case["d"] * 2
    if family == "compact":
        kept, counts = _kept(case, rng)
        moved = sum(x != i for r, c in zip(kept, counts) for i, x in enumerate(r[:c]))
        return {"bytes": 2 * moved * row + 4 * sum(counts), "flops": 0}
    parents = _fork_parents(case, rng)
    copied = sum(lens[p] % page for p in parents)
    if case["reorder"]:
        order = [rng.randrange(case["n"]) for _ in range(case["n"])]
        copied += sum((order.count(p) - 1) * (lens[parents[p]] % page) for p in set(order))
    width = -(-case["hi"] // page) + 1
    return {"bytes": 2 * copied * row + 8 * case["n"] * width, "flops": 0}


# ---- in 64 bits, from the definition ----------------------------------------------------------------------------------
def _exact_turn(x, cos, sin, positions, sections, cyclic, interleaved, back=False):
    """Each pair of x as a complex number times e^{i angle}; positions (axes, tokens..)."""
    pairs = cos.shape[1]
    axes = positions.shape[0]
    owner = []
    for i in range(pairs):
        if sections is None:
            owner.append(0)
        elif cyclic:
            owner.append(i % axes if i < axes * sections[i % axes] else 0)
        else:
            owner.append(next(a for a in range(axes) if i < sum(sections[:a + 1])))
    x = x.double()
    turn = torch.stack([torch.complex(cos.double()[positions[a].long(), i], sin.double()[positions[a].long(), i])
                        for i, a in enumerate(owner)], -1)[..., None, :]
    turn = turn.conj() if back else turn
    at = [2 * i for i in range(pairs)] if interleaved else list(range(pairs))
    to = [a + 1 for a in at] if interleaved else [a + pairs for a in at]
    z = torch.complex(x[..., at], x[..., to]) * turn
    y = x.clone()
    y[..., at], y[..., to] = z.real, z.imag
    return y


def _exact_tree(case, st):
    lens, trees, table, _ = _tree_shape(case)
    hq, hkv, d, t = case["hq"], case["hkv"], case["d"], case["t"]
    q, k = st["q"].double(), st["k"].double()
    dt = st["q"].dtype
    depths = [_depths(p) for p in trees]
    if st["cos"] is not None:
        pos = st["positions"]
        if pos is None:
            pos = torch.tensor([[n + max(x, 0) for x in ds] for n, ds in zip(lens, depths)], device=q.device)[None]
        # what stands in the cache, and what is multiplied with it, is rounded to the inputs' type by the operator's definition
        q, k = (_exact_turn(x, st["cos"], st["sin"], pos, st["sections"], False, case["rotary"] == "interleaved").to(dt).double() for x in (q, k))
    kc, vc = st["k_cache"].double(), st["v_cache"].double()
    out = torch.zeros(case["b"], t, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((case["b"], hq, t), float("inf"), dtype=torch.float64, device=q.device)
    for b in range(case["b"]):
        n, ds = lens[b], depths[b]
        for i in range(t):
            if ds[i] >= 0:
                at = (table[b][(n + i) // case["page"]], (n + i) % case["page"]) if table else (b, n + i)
                kc[at], vc[at] = k[b, i], st["v"][b, i].double()
        if table:
            pg = torch.tensor(table[b], device=q.device)
            kb, vb = kc[pg].flatten(0, 1)[:n + t], vc[pg].flatten(0, 1)[:n + t]
        else:
            kb, vb = kc[b, :n + t], vc[b, :n + t]
        where = torch.cat((torch.arange(n), n + torch.tensor(ds))).to(q.device)
        for i in range(t):
            if ds[i] < 0:
                continue
            see = torch.zeros(n + t, dtype=torch.bool, device=q.device)
            see[:n] = True
            a, mine = i, []
            while a >= 0:
                mine.append(n + a)
                a = trees[b][a]
            see[torch.tensor(mine, device=q.device)] = True
            if case["left"] >= 0:
                see &= where >= n + ds[i] - case["left"]
            s = torch.einsum("hgd,nhd->hgn", q[b, i].reshape(hkv, hq // hkv, d), kb).reshape(hq, -1) / math.sqrt(d)
            if case["softcap"] > 0:
                s = case["softcap"] * torch.tanh(s / case["softcap"])
            s[:, ~see] = float("-inf")
            lse[b, :, i] = torch.logsumexp(s, 1)
            w = torch.exp(s - lse[b, :, i, None]).reshape(hkv, hq // hkv, -1)
            vv = torch.where(see[:, None, None], vb, torch.zeros_like(vb))
            out[b, i] = torch.einsum("hgn,nhd->hgd", w, vv).reshape(hq, d)
    return {"out": out, "lse": lse, "k_cache": kc, "v_cache": vc}


def exact(case, seed):
    if case["family"] not in ("tree", "rotary"):
        return None                                             # rows are moved and whole numbers counted: nothing is rounded
    st = prepare(case, seed)
    if case["family"] == "tree":
        return _exact_tree(case, st)
    positions = st["positions"] if case["axes"] > 1 else st["positions"][None]
    args = (st["cos"], st["sin"], positions, st["sections"], case["cyclic"], case["interleaved"])
    got = {"q": _exact_turn(st["q"].detach(), *args), "k": _exact_turn(st["k"].detach(), *args)}
    if case["grad"]:
        got.update(dq=_exact_turn(st["dq"], *args, back=True), dk=_exact_turn(st["dk"], *args, back=True))
    return got
